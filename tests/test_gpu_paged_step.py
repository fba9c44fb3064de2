"""The decode step of a batch as a server runs it: prompts into pages, then steps of grow,
4-bit QKV projection, RoPE + append, paged attention and 4-bit output projection over
several layers, with forks, dropped candidates and compaction in between; eager and as one
captured graph; against the contiguous path of one sequence and against 64 bits."""
import numpy as np
import pytest
import torch

import oracle
import paged_reference as ref
from attn_mi355x import hipgraph

pytestmark = pytest.mark.gpu

LAYERS, HIDDEN, HQ, HKV, D, GROUP, MOST = 3, 256, 8, 2, 64, 64, 512
QD, KVD = HQ * D, HKV * D
TOTAL = QD + 2 * KVD
rotates = lambda layer: layer % 4 != 1  # noqa: E731  (one layer without rotation)


class Server:
    def __init__(self, attn, gpu, page, pages, seqs, columns, seed):
        self.attn, self.gpu, self.seqs = attn, gpu, seqs
        rng = np.random.default_rng(seed)
        f16 = lambda *s, scale=1.0: (scale * rng.standard_normal(s)).astype(np.float16)  # noqa: E731
        self.dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(gpu)  # noqa: E731
        self.w = []
        for _ in range(LAYERS):
            qkv, out = f16(TOTAL, HIDDEN, scale=HIDDEN**-0.5), f16(HIDDEN, QD, scale=QD**-0.5)
            self.w.append((ref.w4_quantize(qkv, GROUP), ref.w4_quantize(out, GROUP),
                           attn.w4_pack(self.dev(qkv), TOTAL, HIDDEN, GROUP),
                           attn.w4_pack(self.dev(out), HIDDEN, QD, GROUP)))
        cos, sin = oracle.rope_tables(MOST, D, 5.0e6)
        self.host_tables = [t.view(np.float16).reshape(MOST, D // 2) for t in (cos, sin)]
        self.cos, self.sin = (self.dev(t) for t in self.host_tables)
        self.cache = attn.PagedKVCache(LAYERS, pages, page, HKV, D, seqs, columns, gpu)
        self.cache.pool.fill_(float("nan"))  # rows that nobody wrote
        buf = lambda *s: torch.zeros(*s, dtype=torch.float16, device=gpu)  # noqa: E731
        self.x, self.qkv, self.q, self.o = buf(seqs, HIDDEN), buf(seqs, TOTAL), buf(seqs, QD), buf(seqs, QD)
        self.grow = torch.zeros(seqs, dtype=torch.int32, device=gpu)
        self.positions = torch.zeros(seqs, dtype=torch.int32, device=gpu)

    def step(self, stream=None):
        """One token more for each sequence with grow = 1, x in place."""
        a, c, B = self.attn, self.cache, self.seqs
        c.grow(self.grow, stream)
        for layer in range(LAYERS):
            _, _, qkv, out = self.w[layer]
            a.w4_matvec(self.x, self.qkv, *qkv, B, HIDDEN, TOTAL, GROUP, stream=stream)
            at = self.qkv.data_ptr()
            c.append(layer, at, at + 2 * QD, at + 2 * (QD + KVD), self.cos, self.sin,
                     self.positions, B, HQ, MOST, TOTAL, TOTAL, rotates(layer), q_out=self.q,
                     stream=stream)
            c.decode(layer, self.q, self.o, HQ, stream=stream)
            a.w4_matvec(self.o, self.x, *out, B, QD, HIDDEN, GROUP, residual=self.x,
                        stream=stream)

    def set_inputs(self, x, live):
        """New hidden states; sequences not in `live` are padding of the batch."""
        lens = self.cache.seq_lens.tolist()
        self.x.copy_(self.dev(x))
        self.grow.copy_(torch.tensor([int(b in live) for b in range(self.seqs)], dtype=torch.int32))
        self.positions.copy_(torch.tensor([lens[b] if b in live else -1 for b in range(self.seqs)],
                                          dtype=torch.int32))


def rotate(x, cos, sin):
    a, b = x[..., :D // 2], x[..., D // 2:]
    return np.concatenate([a * cos - b * sin, b * cos + a * sin], -1)


class Model64:
    """The same step of one sequence in 64 bits, rounded to fp16 where the server holds
    fp16: projections, rotated keys and queries, attention, hidden states."""

    def __init__(self, server):
        self.s = server
        self.k = [[] for _ in range(LAYERS)]
        self.v = [[] for _ in range(LAYERS)]

    def copy(self):
        m = Model64(self.s)
        m.k, m.v = [list(x) for x in self.k], [list(x) for x in self.v]
        return m

    def step(self, x):
        r = lambda a: np.asarray(a).astype(np.float16).astype(np.float64)  # noqa: E731
        pos = len(self.k[0])
        cos, sin = (t[pos].astype(np.float64) for t in self.s.host_tables)
        for layer in range(LAYERS):
            qkv, out = self.s.w[layer][:2]
            y = r(ref.w4_product(*qkv, GROUP, x[None])[0][0])
            q, k = y[:QD].reshape(HQ, D), y[QD:QD + KVD].reshape(HKV, D)
            if rotates(layer):
                q, k = r(rotate(q, cos, sin)), r(rotate(k, cos, sin))
            self.k[layer].append(k)
            self.v[layer].append(y[QD + KVD:].reshape(HKV, D))
            K, V = np.array(self.k[layer]), np.array(self.v[layer])
            o = [ref.decode(q[g * 4:g * 4 + 4], K[:, g], V[:, g], D**-0.5)[0] for g in range(HKV)]
            x = r(ref.w4_product(*out, GROUP, r(np.concatenate(o).reshape(1, -1)), x[None])[0][0])
        return x


def hidden(rng, n):
    return rng.standard_normal((n, HIDDEN)).astype(np.float16)


def check(got, exp):
    """Each of the step's six roundings to fp16 per layer (two projections, rotation,
    weights and output of the attention, hidden state) is off by half a step, 2^-11 of values
    whose size is that of the hidden states (unit variance, up to about 4); an error of one
    layer's output passes the next layers' residual stream and is added to, and through their
    attention at most doubled: 6 * 2^-11 * 4 * (1 + 2 + 4) below 0.09 at worst; a page or a
    position mixed up changes the values by their own size."""
    assert np.abs(got.astype(np.float64) - exp).max() < 0.09


@pytest.mark.parametrize("page", [16, 5])
def test_steps_with_forks_and_compaction(attn, gpu, page):
    print(f"[case] page={page}", flush=True)
    B = 6
    s = Server(attn, gpu, page, 60, B, 80 // page, 1)
    rng = np.random.default_rng(2)
    models = {0: Model64(s), 1: Model64(s), 3: Model64(s)}

    def run(steps):
        for _ in range(steps):
            x = hidden(rng, B)
            s.set_inputs(x, models)
            s.step()
            torch.cuda.synchronize()
            assert s.cache.status.tolist() == [0, 0]
            got = s.x.cpu().numpy()
            for b, m in models.items():
                check(got[b], m.step(x[b]))

    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    run(18)
    # two candidates of sequence 0, one of 3; their last pages are shared until they grow
    s.cache.fork(ints([-1, -1, 0, -1, 0, 3]))
    models.update({2: models[0].copy(), 4: models[0].copy(), 5: models[3].copy()})
    run(7)
    # sequence 0 ends, 2 and 5 lose their last tokens, the pool is compacted
    keep = [0, -1, 20, -1, -1, 3]
    s.cache.free(ints(keep))
    del models[0]
    for b, n in ((2, 20), (5, 3)):
        for layer in range(LAYERS):
            del models[b].k[layer][n:], models[b].v[layer][n:]
    s.cache.compact()
    run(5)
    used = int((s.cache.ref_counts > 0).sum())
    assert used <= 60 and sum(s.cache.ref_counts.tolist()) == sum(
        ref.pages_for(n, page) for n in s.cache.seq_lens.tolist())


def test_prompt_then_steps_as_the_contiguous_path(attn, gpu):
    """A prompt through the framework's own projection, RoPE and prefill, its keys and values
    put into pages; then steps whose attention equals that of the contiguous cache."""
    N, page, Hq, Hkv, Dh = 254, 16, 16, 4, 128
    qd, kvd = Hq * Dh, Hkv * Dh
    rng = np.random.default_rng(5)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(gpu)  # noqa: E731
    most = 300
    cos, sin = (dev(t.view(np.float16)) for t in oracle.rope_tables(most, Dh, 5.0e6))
    flat = attn.KVCache(1, most, Hkv, Dh, gpu)
    cache = attn.PagedKVCache(1, 40, page, Hkv, Dh, 2, 20, gpu)
    grow = torch.tensor([0, N], dtype=torch.int32, device=gpu)
    cache.grow(grow)
    qkv = dev(rng.standard_normal((N, qd + 2 * kvd)).astype(np.float16))
    at, stride = qkv.data_ptr(), qd + 2 * kvd
    seq = torch.ones(N, dtype=torch.int32, device=gpu)
    pos = torch.arange(N, dtype=torch.int32, device=gpu)
    q_out = torch.empty(N, qd, dtype=torch.float16, device=gpu)
    cache.append(0, at, at + 2 * qd, at + 2 * (qd + kvd), cos, sin, pos, N, Hq, most, stride,
                 stride, q_out=q_out, seq_ids=seq)
    attn.rope_store_kv(at, at + 2 * qd, at + 2 * (qd + kvd), flat.k(0), flat.v(0), cos, sin, N,
                       Hq, Hkv, Dh, stride, stride, 0, True)
    out = torch.empty(N, qd, dtype=torch.float16, device=gpu)
    attn.prefill(at, flat.k(0), flat.v(0), out, N, Hq, Hkv, Dh, stride, kvd)
    torch.cuda.synchronize()
    assert torch.equal(q_out, qkv[:, :qd])
    rows = cache.page_table[1, pos.long() // page].long() * page + pos % page
    assert torch.equal(cache.k(0).view(-1, kvd)[rows], flat.k(0)[:N])
    assert torch.equal(cache.v(0).view(-1, kvd)[rows], flat.v(0)[:N])
    grow = torch.tensor([0, 1], dtype=torch.int32, device=gpu)
    ws = attn.decode_workspace(Hq, most, Dh, gpu)
    for step in range(20):
        n = N + step + 1
        x = dev(rng.standard_normal((2, qd + 2 * kvd)).astype(np.float16))
        cache.grow(grow)
        pos = torch.tensor([-1, n - 1], dtype=torch.int32, device=gpu)
        q = torch.zeros(2, qd, dtype=torch.float16, device=gpu)
        at = x.data_ptr()
        cache.append(0, at, at + 2 * qd, at + 2 * (qd + kvd), cos, sin, pos, 2, Hq, most, stride,
                     stride, q_out=q)
        o = torch.full((2, qd), 9.0, dtype=torch.float16, device=gpu)
        cache.decode(0, q, o, Hq)
        one = at + 2 * stride
        attn.rope_store_kv(one, one + 2 * qd, one + 2 * (qd + kvd), flat.k(0), flat.v(0), cos, sin,
                           1, Hq, Hkv, Dh, stride, stride, n - 1, True)
        exp = torch.empty(qd, dtype=torch.float16, device=gpu)
        attn.decode(one, flat.k(0), flat.v(0), exp, *ws, 1, n, n - 1, Hq, Hkv, Dh)
        torch.cuda.synchronize()
        assert (o[0] == 9).all() and torch.equal(q[1], x[1, :qd])
        k, v = (t(0)[:n].cpu().numpy().reshape(n, Hkv, Dh) for t in (flat.k, flat.v))
        for g in range(Hkv):
            mine = slice(g * 4 * Dh, (g + 1) * 4 * Dh)
            e64, bound = ref.decode(q[1, mine].cpu().numpy().reshape(4, Dh), k[:, g], v[:, g],
                                    Dh**-0.5)
            for got in (o[1, mine], exp[mine]):
                err = np.abs(got.cpu().numpy().reshape(4, Dh).astype(np.float64) - e64)
                # the contiguous path's weights are fp16 without the scale and its states
                # fp16: two more half steps of the weighted magnitudes
                assert (err <= 2 * bound + 2.0**-24).all()


def test_captured_steps(attn, gpu):
    """The whole step as one graph: lengths, positions, padding and tables change between
    replays on the device alone; every replay equals the eager step bit for bit."""
    B, page = 5, 16
    eager, graph = (Server(attn, gpu, page, 40, B, 6, 3) for _ in range(2))
    rng = np.random.default_rng(4)
    stream = torch.cuda.Stream()
    sp = stream.cuda_stream
    graph.set_inputs(hidden(rng, B), {0, 2})
    graph.step()  # workspaces exist before the capture
    graph.cache.free()
    graph.cache.pool.fill_(float("nan"))
    torch.cuda.synchronize()
    hipgraph.begin_capture(sp)
    graph.step(sp)
    g, exe = hipgraph.end_capture(sp)
    parents = torch.tensor([-1, 0, -1, -1, 2], dtype=torch.int32, device=gpu)
    live = {0, 2}
    for turn in range(24):
        if turn == 17:
            for s in (eager, graph):
                s.cache.fork(parents)
            live = {0, 1, 2, 4}
        if turn == 20:
            live = {0, 4}
        x = hidden(rng, B)
        for s in (eager, graph):
            s.set_inputs(x, live)
        eager.step()
        torch.cuda.synchronize()
        hipgraph.launch(exe, sp)
        hipgraph.synchronize(sp)
        rows = sorted(live)
        assert torch.equal(eager.x[rows], graph.x[rows]), turn
        assert torch.equal(eager.cache.page_table, graph.cache.page_table)
        assert torch.equal(eager.cache.seq_lens, graph.cache.seq_lens)
        assert torch.equal(eager.cache.ref_counts, graph.cache.ref_counts)
    hipgraph.destroy(g, exe)


def test_two_caches_on_two_streams(attn, gpu):
    """Two servers that run at the same time, each on its own stream with its own state."""
    servers = [Server(attn, gpu, 8, 60, 4, 12, 7 + i) for i in range(2)]
    alone = [Server(attn, gpu, 8, 60, 4, 12, 7 + i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in servers]
    rng = np.random.default_rng(9)
    for _ in range(12):
        x = [hidden(rng, 4) for _ in servers]
        for s, xx in zip(servers + alone, x + x):
            s.set_inputs(xx, {0, 1, 3})
        torch.cuda.synchronize()
        for s, st in zip(servers, streams):
            s.step(st)
        torch.cuda.synchronize()
        for s in alone:
            s.step()
            torch.cuda.synchronize()
        for a, b in zip(servers, alone):
            assert torch.equal(a.x[[0, 1, 3]], b.x[[0, 1, 3]])
