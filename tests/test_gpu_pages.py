"""Page management against bookkeeping in Python, page by page: random runs of grow, fork,
free and compact, pools that run short, copies of shared pages, sizes that fit no vector."""
import numpy as np
import pytest
import torch

import paged_reference as ref
from attn_mi355x import hipgraph

pytestmark = pytest.mark.gpu


class Both:
    """A PagedKVCache and its bookkeeping in Python."""

    def __init__(self, attn, gpu, layers, pages, page, Hkv, D, seqs, columns, seed):
        self.cache = c = attn.PagedKVCache(layers, pages, page, Hkv, D, seqs, columns, gpu)
        self.rng = np.random.default_rng(seed)
        data = self.rng.integers(-2**15, 2**15, c.pool.shape, dtype=np.int16)
        c.pool.view(torch.int16).copy_(torch.from_numpy(data))
        self.model = ref.Pool(pages, page, columns, seqs, data)
        self.gpu = gpu

    def ints(self, x):
        return torch.tensor([int(v) for v in x], dtype=torch.int32, device=self.gpu)

    def check(self, what):
        torch.cuda.synchronize()
        c, m = self.cache, self.model
        assert c.seq_lens.tolist() == m.lens, what
        assert c.ref_counts.tolist() == m.refs, what
        assert c.page_table.tolist() == m.table, what
        assert np.array_equal(c.pool.view(torch.int16).cpu().numpy(), m.contents), what

    def grow(self, amounts):
        self.cache.status.fill_(-7)
        self.cache.grow(self.ints(amounts))
        exp = self.model.grow([int(a) for a in amounts])
        self.check("grow")
        assert tuple(self.cache.status.tolist()) == exp
        return exp

    def free(self, keep=None):
        self.cache.free(None if keep is None else self.ints(keep))
        self.model.free(None if keep is None else [int(k) for k in keep])
        self.check("free")

    def fork(self, parents):
        self.cache.fork(self.ints(parents))
        self.model.fork([int(p) for p in parents])
        self.check("fork")

    def compact(self):
        self.cache.compact()
        used = self.model.compact()
        self.check("compact")
        assert self.cache.num_used.tolist() == [used]


@pytest.mark.parametrize("layers,pages,page,Hkv,D,seqs,columns", [
    (1, 40, 4, 1, 8, 6, 8), (3, 300, 16, 2, 16, 20, 12), (1, 9000, 1, 1, 3, 70, 200),
    (2, 64, 5, 1, 2, 9, 30), (1, 5000, 2, 1, 8, 1100, 9)])
def test_random_runs(attn, gpu, layers, pages, page, Hkv, D, seqs, columns):
    print(f"[case] pages={pages} page={page} seqs={seqs}", flush=True)
    x = Both(attn, gpu, layers, pages, page, Hkv, D, seqs, columns, seqs)
    rng = x.rng
    most = columns * page
    met = set()
    for step in range(30):
        what = rng.choice(["grow", "grow", "grow", "fork", "free", "compact"])
        if what == "grow":
            room = np.array([most - n for n in x.model.lens])
            # mostly what fits a row, now and then what does not; rows that stay as they are
            amounts = np.minimum(rng.integers(-1, 2 + pages * page // (2 * seqs), seqs),
                                 room if rng.random() < 0.9 else 2 * most)
            met.add(("grow", x.grow(amounts) == (0, 0)))
        elif what == "fork":
            x.fork(np.where(rng.random(seqs) < 0.4, rng.integers(-1, seqs + 1, seqs), -1))
        elif what == "free":
            keep = rng.integers(0, most, seqs)
            x.free(np.where(rng.random(seqs) < 0.5, -1, np.where(rng.random(seqs) < 0.6, 0, keep)))
        else:
            x.compact()
        met.add(what)
    assert {"grow", "fork", "free", "compact", ("grow", True)} <= met
    x.free()
    assert not any(x.model.refs)


def test_short_pool_changes_nothing(attn, gpu):
    x = Both(attn, gpu, 1, 10, 4, 1, 8, 3, 8, 1)
    assert x.grow([12, 8, 4]) == (0, 0)         # six pages
    assert x.grow([1, 16, 4]) == (2, 0)         # six more of four
    assert x.grow([1, 2, 29]) == (0, 1)         # a row of eight pages
    assert x.grow([2**31 - 1, 0, 0]) == (0, 1)
    assert x.grow([4, 8, 4]) == (0, 0)
    assert x.grow([0, 0, 1]) == (1, 0)
    assert x.grow([-2**31, 0, 0]) == (0, 0)


@pytest.mark.parametrize("pages", [20479, 20480, 20481, 40000, 70001, 174080])
@pytest.mark.parametrize("where", ["last", "few", "one a round", "far apart", "none"])
def test_free_pages_far_up_a_large_pool(attn, gpu, pages, where):
    """The lowest free pages lie behind thousands that are in use."""
    print(f"[case] {pages} pages, {where}", flush=True)
    rng = np.random.default_rng(pages)
    free = {"last": [pages - 1], "none": [], "few": sorted(rng.choice(pages, 5, replace=False)),
            "one a round": list(range(4095, pages, 4096)),
            "far apart": [p for p in (3, 4095, 4096, 20479, 20480, 36863, 36864, 53247, 69999,
                                      150000, pages - 2) if p < pages]}[where]
    free = sorted({int(p) for p in free})
    seqs, columns = 7, 16
    cache = attn.PagedKVCache(1, pages, 1, 1, 8, seqs, columns, gpu)
    pool = cache.pool.view(torch.int16).clone()
    for need in sorted({min(len(free), 1), min(len(free), 4), min(len(free), 60), len(free) + 1}):
        refs = torch.ones(pages, dtype=torch.int32)
        refs[free] = 0
        cache.ref_counts.copy_(refs)
        cache.seq_lens.zero_()
        cache.page_table.fill_(-1)
        grow = [min(columns, max(0, need - columns * b)) for b in range(seqs)]
        cache.grow(torch.tensor(grow, dtype=torch.int32, device=gpu))
        torch.cuda.synchronize()
        if need > len(free):
            assert cache.status.tolist() == [1, 0]
            assert cache.seq_lens.tolist() == [0] * seqs
        else:
            assert cache.status.tolist() == [0, 0]
            assert cache.seq_lens.tolist() == grow
            table = cache.page_table.cpu().reshape(seqs, columns)
            taken = [int(table[b, j]) for b in range(seqs) for j in range(grow[b])]
            assert taken == free[:need]
            refs[taken] = 1
        assert torch.equal(cache.ref_counts.cpu(), refs)
    assert torch.equal(cache.pool.view(torch.int16), pool)


def test_forks_copy_their_last_page_when_they_grow(attn, gpu):
    x = Both(attn, gpu, 2, 30, 4, 1, 8, 6, 6, 2)
    x.grow([6, 8, 0, 0, 0, 0])                  # row 0 ends inside a page, row 1 at its end
    x.fork([-1, -1, 0, 0, 1, 1])
    x.grow([0, 0, 1, 0, 1, 0])                  # one copy (row 2), one plain new page (row 4)
    x.grow([1, 1, 0, 1, 0, 0])                  # rows 0 and 3 still share: both copy
    x.grow([1, 0, 1, 1, 1, 1])                  # no page is shared any more but full ones
    x.free([0, 0, -1, -1, -1, -1])
    x.compact()
    x.free()
    x.compact()                                 # nothing in use


def test_fork_rules(attn, gpu):
    x = Both(attn, gpu, 1, 20, 4, 1, 8, 5, 4, 3)
    x.grow([5, 0, 0, 0, 0])
    x.fork([-1, 0, 1, 99, 0])    # row 2's parent has a parent itself; row 3's does not exist
    assert x.model.lens == [5, 5, 0, 0, 5]
    x.fork([1, 0, 2, 3, -5])     # rows that hold a sequence, rows that name themselves
    assert x.model.lens == [5, 5, 0, 0, 5]


def test_fork_between_two_tables(attn, gpu):
    """The whole of a beam step: children in a second table, then the old rows are freed."""
    pages, page, columns = 24, 4, 5
    lens, table = [9, 4, 0], np.full((3, columns), -1, dtype=np.int32)
    table[0, :3], table[1, :1] = [3, 1, 7], [0]
    refs = np.zeros(pages, dtype=np.int32)
    refs[[3, 1, 7, 0]] = 1
    dev = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device=gpu)  # noqa: E731
    a, la, r = dev(table), dev(lens), dev(refs)
    b, lb = dev(np.full((4, columns), -1)), dev([0] * 4)
    attn.pages_fork(a, la, b, lb, dev([0, 0, 1, 2]), r, 3, 4, columns, pages, page)
    attn.pages_free(a, la, r, 3, columns, pages, page)
    torch.cuda.synchronize()
    assert lb.tolist() == [9, 9, 4, 0] and la.tolist() == [0, 0, 0]
    assert b.tolist() == [[3, 1, 7, -1, -1]] * 2 + [[0, -1, -1, -1, -1], [-1] * columns]
    exp = np.zeros(pages, dtype=int)
    exp[[3, 1, 7]], exp[0] = 2, 1
    assert r.tolist() == exp.tolist()


def test_numbers_out_of_range_name_nothing(attn, gpu):
    pages, page, columns = 6, 4, 3
    dev = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device=gpu)  # noqa: E731
    table, lens = dev([[-1, 2, 6], [2**30, 1, 5]]), dev([12, 2**31 - 1])
    refs = dev([1] * pages)
    attn.pages_free(table, lens, refs, 2, columns, pages, page)
    torch.cuda.synchronize()
    assert refs.tolist() == [1, 0, 0, 1, 1, 0] and lens.tolist() == [0, 0]
    pool = torch.arange(2 * pages * 8, dtype=torch.int16, device=gpu).view(2, pages, 8)
    before = pool.clone()
    attn.pages_copy(pool, 2, 8, dev([-1, 3, 6, 2]), dev([0, 6, 1, 5]), 4, pages)
    torch.cuda.synchronize()
    before[:, 5] = before[:, 2]
    assert torch.equal(pool, before)


@pytest.mark.parametrize("elements,planes,stride,offset", [
    (8, 1, 0, 0), (8192, 3, 0, 0), (8200, 2, 0, 0), (40000, 2, 0, 0), (7, 3, 0, 0),
    (16384, 2, 16384 * 20 + 8, 0), (100, 2, 2003, 0), (64, 2, 0, 1)])
def test_copy_sizes(attn, gpu, elements, planes, stride, offset):
    print(f"[case] {elements} x {planes}, stride {stride}, offset {offset}", flush=True)
    pages = 20
    size = (stride or pages * elements) * planes
    data = np.random.default_rng(elements).integers(-2**15, 2**15, size + offset, dtype=np.int16)
    pool = torch.from_numpy(data).to(gpu)
    rng = np.random.default_rng(1)
    order = rng.permutation(pages)
    src, dst = order[:9].astype(np.int32), order[9:18].astype(np.int32)
    dst[4] = src[4]  # onto itself
    attn.pages_copy(pool[offset:], planes, elements, torch.from_numpy(src).to(gpu),
                    torch.from_numpy(dst).to(gpu), 9, pages, plane_stride=stride)
    torch.cuda.synchronize()
    exp = data.copy()
    for p in range(planes):
        plane = exp[offset + p * (stride or pages * elements):][:pages * elements]
        plane = plane.reshape(pages, elements)
        plane[dst] = plane[src]
    assert np.array_equal(pool.cpu().numpy(), exp)


def test_captured_steps(attn, gpu):
    """fork, grow, free and compact as one captured graph, replayed; the state between
    replays is changed by eager calls."""
    x = Both(attn, gpu, 2, 60, 4, 1, 8, 8, 6, 4)
    c, m = x.cache, x.model
    x.grow([7, 3, 10, 0, 0, 0, 0, 0])
    parents, amounts, keep = [-1, -1, -1, 0, 0, 1, 2, -1], [1, 0, 2, 1, 5, 1, 0, 3], [-1] * 3 + [0] * 5
    d = [x.ints(v) for v in (parents, amounts, keep)]
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    sp = stream.cuda_stream
    hipgraph.begin_capture(sp)
    c.fork(d[0], sp)
    c.grow(d[1], sp)
    c.free(d[2], sp)
    c.compact(sp)
    graph, exe = hipgraph.end_capture(sp)
    for turn in range(4):
        hipgraph.launch(exe, sp)
        hipgraph.synchronize(sp)
        m.fork(parents)
        m.grow(amounts)
        m.free(keep)
        m.compact()
        x.check(f"replay {turn}")
        x.free([4, 1, -1, -1, -1, -1, -1, -1])
        x.grow([0, 2, 0, 0, 0, 0, 0, 0])
    hipgraph.destroy(graph, exe)
