"""Decode attention over pages against 64 bits: lengths from nothing to long, page sizes
that end inside every tile, head layouts, strides, NaN in cache rows nobody should read,
page numbers out of range, captured calls whose lengths change between replays."""
import numpy as np
import pytest
import torch

import paged_reference as ref
from attn_mi355x import hipgraph

pytestmark = pytest.mark.gpu
OUT = 77.0  # what outputs hold before a call


class Case:
    def __init__(self, attn, gpu, lens, page, Hq, Hkv, D, seed=0, pad=0, kfill=np.nan,
                 columns=None, spare=2):
        print(f"[case] lens={lens if len(lens) < 9 else len(lens)} page={page} heads={Hq}/{Hkv} "
              f"D={D} pad={pad}", flush=True)
        self.attn, self.gpu = attn, gpu
        self.Hq, self.Hkv, self.D, self.page = Hq, Hkv, D, page
        self.lay = lay = ref.Layout(lens, page, seed, columns=columns, spare=spare)
        rng = np.random.default_rng(seed + 1)
        # rows that belong to no sequence hold NaN
        self.k, self.v = (np.full((lay.pages * page, Hkv, D), kfill, np.float16) for _ in "kv")
        for b in range(len(lens)):
            r = lay.rows(b)
            for x in (self.k, self.v):
                x[r] = rng.standard_normal((len(r), Hkv, D))
        self.stride = Hq * D + pad
        self.q = (2 * rng.standard_normal((len(lens), self.stride))).astype(np.float16)
        self.upload()

    def upload(self):
        dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(self.gpu)  # noqa: E731
        self.dq, self.dk, self.dv = dev(self.q), dev(self.k), dev(self.v)
        self.table = dev(self.lay.table)
        self.lens = dev(np.array(self.lay.lens, dtype=np.int32))
        B = len(self.lay.lens)
        # 64 guard values behind the outputs and behind the workspace
        self.out = torch.full((B * self.Hq * self.D + 64,), OUT, dtype=torch.float16,
                              device=self.gpu)
        n = int(self.attn.lib().attn_paged_decode_workspace_bytes(B, self.Hq, self.Hkv, self.D))
        self.ws = torch.full((n + 64,), 0xFF, dtype=torch.uint8, device=self.gpu)

    def call(self, stream=None):
        lay = self.lay
        self.attn.paged_decode(self.dq, self.dk, self.dv, self.out, self.table, self.lens,
                               len(lay.lens), lay.columns, lay.pages, self.page, self.Hq,
                               self.Hkv, self.D, self.ws, self.stride, stream)

    def got(self):
        torch.cuda.synchronize()
        assert (self.ws[-64:] == 0xFF).all() and (self.out[-64:] == OUT).all()
        return self.out[:-64].cpu().numpy().reshape(len(self.lay.lens), self.Hq, self.D)

    def check(self, got, lens=None, skip=()):
        G, D = self.Hq // self.Hkv, self.D
        for b, n in enumerate(self.lay.lens if lens is None else lens):
            if b in skip:
                continue
            if n <= 0:
                assert (got[b] == OUT).all(), b
                continue
            rows = self.lay.rows(b, n)
            for g in range(self.Hkv):
                q = self.q[b, g * G * D:(g + 1) * G * D].reshape(G, D)
                exp, bound = ref.decode(q, self.k[rows, g], self.v[rows, g], D**-0.5)
                err = np.abs(got[b, g * G:(g + 1) * G].astype(np.float64) - exp)
                assert (err <= bound).all(), (b, n, g, err.max(), (err / bound).max())


# how a call is split: table rows of a few hundred keys take one kernel, wide ones two; the
# generic kernel is the one of other head dims and unaligned tensors
@pytest.fixture(params=["one kernel", "two kernels", "generic"])
def form(request, attn):
    attn.set_option("decode_force_generic", int(request.param == "generic"))
    yield request.param
    attn.set_option("decode_force_generic", 0)


def columns_of(form, page, high):
    return -(-5000 // page) if form == "two kernels" else -(-high // page) + 1


# lengths around 8, 16, 32, 64 and the page's end
LENS = [1, 0, 7, 8, 9, 31, 32, 33, 63, 64, 65, 100, 127, 129, 254, 300]


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 32, 64, 100, 128])
@pytest.mark.parametrize("Hq,Hkv,D", [(16, 4, 128), (16, 4, 64)])
def test_pages_and_lengths(attn, gpu, form, page, Hq, Hkv, D):
    c = Case(attn, gpu, LENS, page, Hq, Hkv, D, seed=page,
             columns=columns_of(form, page, max(LENS)))
    c.call()
    c.check(c.got())


@pytest.mark.parametrize("Hq,Hkv,D,pad", [
    (16, 16, 128, 0), (16, 8, 128, 0), (8, 2, 128, 8), (8, 8, 64, 0), (32, 8, 64, 0),
    (1, 1, 128, 0), (6, 2, 64, 16), (17, 1, 128, 0), (40, 2, 64, 0), (16, 1, 128, 0),
    (4, 2, 128, 3),             # rows of q that are not 16-byte aligned
    (4, 2, 32, 0), (4, 2, 96, 0), (2, 1, 256, 0), (3, 3, 5, 1)])
def test_head_layouts(attn, gpu, Hq, Hkv, D, pad):
    c = Case(attn, gpu, [300, 1, 40, 0, 700], 16, Hq, Hkv, D, seed=Hq + D, pad=pad)
    c.call()
    c.check(c.got())


@pytest.mark.parametrize("Hq,Hkv,D,page,lens", [
    (16, 4, 128, 64, [32768]), (16, 4, 128, 16, [5000, 17, 1, 0, 9001, 2000]),
    (16, 4, 64, 32, [12345, 3]), (8, 8, 64, 16, [4097, 4096, 4095]),
    (16, 4, 128, 7, [3000, 200])])
def test_long_sequences(attn, gpu, Hq, Hkv, D, page, lens):
    c = Case(attn, gpu, lens, page, Hq, Hkv, D, seed=len(lens))
    c.call()
    c.check(c.got())


@pytest.mark.parametrize("columns", [None, 100])
@pytest.mark.parametrize("B,high", [(200, 60), (70, 900), (1100, 9), (64, 40), (65, 40)])
def test_many_sequences(attn, gpu, B, high, columns):
    rng = np.random.default_rng(B)
    lens = rng.integers(0, high + 1, B).tolist()
    c = Case(attn, gpu, lens, 16, 8, 2, 128, seed=B, columns=columns)
    c.call()
    c.check(c.got())


@pytest.mark.parametrize("D", [128, 64])
def test_rising_scores(attn, gpu, D):
    """Maxima that move all the way along the keys, and weights that span hundreds of
    powers of two."""
    c = Case(attn, gpu, [1500, 40], 16, 16, 4, D, seed=5)
    for b in range(2):
        rows = c.lay.rows(b)
        c.k[rows] *= np.linspace(0.1, 12.0, len(rows))[:, None, None].astype(np.float16)
    c.upload()
    c.call()
    c.check(c.got())


@pytest.mark.parametrize("size", [300.0, 3000.0, 30000.0])
@pytest.mark.parametrize("D", [128, 64])
def test_scores_far_past_the_steps_of_fp32(attn, gpu, form, D, size):
    """Scores of 10^6 to 10^11, whose neighbours in fp32 are up to 8192 apart: the one key
    that points along the query has all the weight, the others point away."""
    c = Case(attn, gpu, [200], 16, 8, 2, D, seed=17, columns=columns_of(form, 16, 200))
    rng = np.random.default_rng(18)
    sign = rng.choice([-1.0, 1.0], (c.Hkv, D))
    c.q[0] = np.repeat(size * sign, c.Hq // c.Hkv, axis=0).ravel()
    rows = c.lay.rows(0)
    # sums of odd values, so that products with the scale are not exact in fp32
    c.k[rows] = -sign * (size * rng.uniform(0.5, 1.0, (len(rows), c.Hkv, D)))
    c.k[rows[77]] = sign * (size * rng.uniform(0.5, 1.0, (c.Hkv, D)))
    c.upload()
    c.call()
    got = c.got()[0]
    exp = np.repeat(c.v[rows[77]], c.Hq // c.Hkv, axis=0)
    assert np.array_equal(got.view(np.uint16), exp.view(np.uint16))


@pytest.mark.parametrize("D", [128, 64])
def test_many_small_weights_keep_their_sum(attn, gpu, D):
    """One key whose weight is 2^17 times the others': alone they would vanish in fp16,
    together they carry a fifth of the output."""
    n = 30000
    c = Case(attn, gpu, [n], 16, 4, 1, D, seed=6)
    rows = c.lay.rows(0)
    c.q[:] = 0
    c.q[:, ::D] = 1.0
    c.k[rows] = 0
    c.k[rows[1234], :, 0] = np.float16(17 * np.log(2) * D**0.5)
    c.v[rows] = 1.0
    c.v[rows[1234]] = -1.0
    c.upload()
    c.call()
    c.check(c.got())


def test_infinities_and_nan_stay_where_they_are(attn, gpu, form):
    """A NaN in V reaches its dim of its KV head's queries of its sequence, a NaN in K
    that head's queries, an infinite V its dim; other sequences are as they would be."""
    c = Case(attn, gpu, [200, 200, 200, 200], 16, 8, 2, 128, seed=8,
             columns=columns_of(form, 16, 200))
    c.v[c.lay.rows(0)[150], 1, 7] = np.nan
    c.k[c.lay.rows(1)[3], 0, 9] = np.nan
    c.v[c.lay.rows(2)[199], 0, 100] = np.inf
    c.upload()
    c.call()
    got = c.got()
    c.check(got, skip=(0, 1, 2))
    exp = np.zeros((4, 8, 128), dtype=bool)
    exp[0, 4:, 7] = True
    exp[1, :4] = True
    assert np.array_equal(np.isnan(got), exp)
    assert (got[2, :4, 100] == np.inf).all() and np.isinf(got).sum() == 4


@pytest.mark.parametrize("bad", [-1, 2**30, -2**31])
@pytest.mark.parametrize("at", [0, 5, 18])
def test_page_out_of_range(attn, gpu, form, bad, at):
    """Its sequence is NaN, the others are not touched by it; entries past a sequence's
    end are never used (the layout fills them with numbers out of range)."""
    c = Case(attn, gpu, [300, 300, 33], 16, 16, 4, 128, seed=9, columns=columns_of(form, 16, 300))
    c.table[1, at] = bad
    c.call()
    got = c.got()
    assert np.isnan(got[1]).all()
    c.check(got, skip=(1,))


@pytest.mark.parametrize("keys", [64, 1600])
def test_lengths_past_the_table_are_cut(attn, gpu, keys):
    c = Case(attn, gpu, [keys, 32], 16, 16, 4, 128, seed=10, columns=keys // 16)
    c.lens[0] = 2**31 - 1
    c.lens[1] = -5
    c.call()
    c.check(c.got(), lens=[keys, 0])


def test_captured_call_with_changing_lengths(attn, gpu):
    """One captured call; lengths, tables and queries change in place between replays,
    with eager calls in between; another captured call shares the workspace."""
    lens = [3000, 10, 700, 64]
    c = Case(attn, gpu, lens, 16, 16, 4, 128, seed=11)
    stream = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        hipgraph.begin_capture(stream.cuda_stream)
        c.call(stream.cuda_stream)
        graphs.append(hipgraph.end_capture(stream.cuda_stream))
    rng = np.random.default_rng(12)
    for turn in range(5):
        now = [int(rng.integers(0, n + 1)) for n in lens] if turn else lens
        c.lens.copy_(torch.tensor(now, dtype=torch.int32))
        c.out.fill_(OUT)
        torch.cuda.synchronize()
        hipgraph.launch(graphs[0][1], stream.cuda_stream)
        hipgraph.launch(graphs[1][1], stream.cuda_stream)
        hipgraph.synchronize(stream.cuda_stream)
        replayed = c.got()
        c.check(replayed, lens=now)
        c.out.fill_(OUT)
        c.call()
        assert np.array_equal(c.got(), replayed)
    for g in graphs:
        hipgraph.destroy(*g)


def test_batch_without_keys(attn, gpu, form):
    c = Case(attn, gpu, [0] * 70, 16, 8, 2, 128, seed=15, columns=columns_of(form, 16, 400))
    c.call()
    assert (c.got() == OUT).all()


def test_same_bits_every_time(attn, gpu):
    c = Case(attn, gpu, [5000, 123, 1], 16, 16, 4, 128, seed=13)
    c.call()
    first = c.got().copy()
    for _ in range(3):
        c.out.fill_(OUT)
        c.ws.fill_(0xFF)
        c.call()
        assert np.array_equal(c.got(), first)


@pytest.mark.parametrize("columns", [8, 100])
def test_pool_past_four_gigabytes(attn, gpu, columns):
    """Pages whose byte offset passes 32 bits: 2^21 rows of 4 KiB in each of K and V,
    sequences on the pool's last pages and its first."""
    Hq, Hkv, D, page, pages = 16, 16, 128, 16, 2**17
    free, _ = torch.cuda.mem_get_info()
    assert free > 40 * 2**30
    rows = pages * page
    k = torch.empty(rows, Hkv, D, dtype=torch.float16, device=gpu)
    v = torch.empty_like(k)
    lens = [100, 33]
    table = np.full((2, columns), -1, dtype=np.int32)
    table[0, :7] = [pages - 1, 0, pages - 2, 2**16, 3, pages - 9, 2**16 - 1]
    table[1, :3] = [2**16 + 1, 5, pages - 5]
    rng = np.random.default_rng(14)
    q = (2 * rng.standard_normal((2, Hq, D))).astype(np.float16)
    held = []
    for b, n in enumerate(lens):
        t = np.arange(n)
        r = table[b, t // page].astype(np.int64) * page + t % page
        kb, vb = (rng.standard_normal((n, Hkv, D)).astype(np.float16) for _ in "kv")
        k[torch.from_numpy(r).to(gpu)] = torch.from_numpy(kb).to(gpu)
        v[torch.from_numpy(r).to(gpu)] = torch.from_numpy(vb).to(gpu)
        held.append((kb, vb))
    out = torch.empty(2, Hq, D, dtype=torch.float16, device=gpu)
    ws = attn.paged_decode_workspace(2, Hq, Hkv, D, gpu)
    attn.paged_decode(torch.from_numpy(q).to(gpu), k, v, out, torch.from_numpy(table).to(gpu),
                      torch.tensor(lens, dtype=torch.int32, device=gpu), 2, columns, pages, page, Hq,
                      Hkv, D, ws)
    torch.cuda.synchronize()
    got = out.cpu().numpy().astype(np.float64)
    for b in range(2):
        for g in range(Hkv):
            exp, bound = ref.decode(q[b, g:g + 1], held[b][0][:, g], held[b][1][:, g], D**-0.5)
            assert (np.abs(got[b, g] - exp[0]) <= bound[0]).all()


@pytest.mark.parametrize("Hq,Hkv,D,page", [(16, 4, 128, 16), (16, 4, 64, 7)])
@pytest.mark.parametrize("columns", [40, 1000])
def test_pool_that_no_cache_keeps(attn, gpu, Hq, Hkv, D, page, columns):
    """K and V of more than 100 MiB, which are read with another hint."""
    spare = 110 * 2**20 // (4 * Hkv * D * page)
    c = Case(attn, gpu, [260, 3, 0, 100], page, Hq, Hkv, D, seed=16, columns=columns, spare=spare)
    c.call()
    c.check(c.got())
