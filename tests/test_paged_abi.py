"""Paged-cache and 4-bit entry points without a GPU: what they refuse, what is a no-op,
the sizes they ask for, and the references' own consistency.  CPU only."""
import numpy as np
import pytest

import paged_reference as ref

INVALID = 1  # hipErrorInvalidValue
P = 4096     # a non-null, aligned address that no accepted call of this file reads


def append(lib, **change):
    a = dict(q=P, k=P, v=P, q_out=None, kp=P, vp=P, cos=P, sin=P, table=P, seq=P, pos=P, tokens=4,
             seqs=4, columns=8, pages=16, page=16, most=100, hq=16, hkv=4, d=128, qs=0, ks=0,
             apply=1, stream=None)
    assert set(change) <= set(a)
    a.update(change)
    return lib.attn_paged_rope_store_kv(*a.values())


def decode(lib, **change):
    a = dict(q=P, kp=P, vp=P, out=P, table=P, lens=P, seqs=4, columns=8, pages=16, page=16, hq=16,
             hkv=4, d=128, qs=0, ws=P, stream=None)
    assert set(change) <= set(a)
    a.update(change)
    return lib.attn_paged_decode(*a.values())


def test_append_refusals(attn):
    lib = attn.lib()
    assert append(lib, tokens=0, q=None, table=None) == 0
    assert append(lib, hq=0, hkv=0) == 0
    for name in ("q", "k", "v", "kp", "vp", "cos", "sin", "table", "pos"):
        assert append(lib, **{name: None}) == INVALID, name
    assert append(lib, seq=None, tokens=5) == INVALID  # more tokens than sequences
    for change in (dict(d=127), dict(d=0), dict(page=0), dict(pages=2**31), dict(columns=2**31),
                   dict(page=2**20, pages=2**11), dict(page=2**20, columns=2**11),
                   dict(tokens=2**31), dict(most=2**31), dict(d=2**16), dict(hq=2**16),
                   dict(seqs=2**31)):
        assert append(lib, **change) == INVALID, change


def test_decode_refusals(attn):
    lib = attn.lib()
    assert decode(lib, seqs=0, q=None) == 0
    assert decode(lib, columns=0) == 0 and decode(lib, hq=0) == 0
    for name in ("q", "kp", "vp", "out", "table", "lens", "ws"):
        assert decode(lib, **{name: None}) == INVALID, name
    for change in (dict(hkv=0), dict(hkv=3), dict(d=0), dict(d=257), dict(page=0),
                   dict(pages=2**31), dict(page=2**20, pages=2**11), dict(seqs=2**16),
                   dict(page=2**20, columns=2**11), dict(hq=2**16, hkv=2**16)):
        assert decode(lib, **change) == INVALID, change


def test_page_management_refusals(attn):
    lib = attn.lib()
    # copy(pool, planes, stride, elements, src, dst, n, pages)
    copy = lambda *a: lib.attn_pages_copy(*a, None)  # noqa: E731
    assert copy(None, 2, 0, 64, None, None, 0, 8) == 0
    assert copy(None, 0, 0, 64, None, None, 3, 8) == 0
    assert copy(P, 2, 0, 0, P, P, 3, 8) == INVALID
    assert copy(P, 2, 511, 64, P, P, 3, 8) == INVALID  # planes overlap
    assert copy(None, 2, 0, 64, P, P, 3, 8) == INVALID
    assert copy(P, 2, 0, 64, None, P, 3, 8) == INVALID
    assert copy(P, 2, 0, 64, P, None, 3, 8) == INVALID
    assert copy(P, 2, 0, 64, P, P, 2**31, 8) == INVALID
    assert copy(P, 2**31, 0, 64, P, P, 1, 8) == INVALID
    assert copy(P, 2**30, 0, 2**40, P, P, 1, 2**30) == INVALID
    # free(table, lens, keep, refs, seqs, columns, pages, page)
    free = lambda *a: lib.attn_pages_free(*a, None)  # noqa: E731
    assert free(None, None, None, None, 0, 8, 8, 16) == 0
    for a in ((None, P, P, P), (P, None, P, P), (P, P, P, None)):
        assert free(*a, 2, 8, 8, 16) == INVALID
    assert free(P, P, None, P, 2, 8, 8, 0) == INVALID
    # fork(src table, src lens, dst table, dst lens, parents, refs, n src, n dst, ...)
    fork = lambda *a: lib.attn_pages_fork(*a, None)  # noqa: E731
    assert fork(None, None, None, None, None, None, 2, 0, 8, 8, 16) == 0
    for i in range(6):
        a = [P, P, 2 * P, 2 * P, P, P]
        a[i] = None
        assert fork(*a, 2, 2, 8, 8, 16) == INVALID, i
    assert fork(P, P, P, 2 * P, P, P, 2, 2, 8, 8, 16) == INVALID   # one table, two lengths
    assert fork(P, P, 2 * P, P, P, P, 2, 2, 8, 8, 16) == INVALID   # two tables, one length
    assert fork(P, P, P, P, P, P, 2, 3, 8, 8, 16) == INVALID       # one table, two sizes
    # grow(pool, planes, stride, elements, table, lens, grow, refs, status, seqs, ..., ws)
    grow = lambda *a: lib.attn_pages_grow(*a, None)  # noqa: E731
    assert grow(None, 2, 0, 64, None, None, None, None, None, 0, 8, 8, 16, None) == 0
    for i in (0, 4, 5, 6, 7, 8):
        a = [P, 2, 0, 64, P, P, P, P, P]
        a[i] = None
        assert grow(*a, 2, 8, 8, 16, P) == INVALID, i
    assert grow(P, 2, 0, 64, P, P, P, P, P, 2, 8, 8, 16, None) == INVALID
    assert grow(P, 2, 0, 64, P, P, P, P, P, 2, 8, 8, 16, P + 2) == INVALID
    assert grow(P, 0, 0, 64, P, P, P, P, P, 2, 8, 8, 16, P) == INVALID
    # compact(pool, planes, stride, elements, table, lens, refs, table out, refs out, used, ...)
    compact = lambda *a: lib.attn_pages_compact(*a, None)  # noqa: E731
    assert compact(None, 2, 0, 64, None, None, None, None, None, None, 2, 8, 0, 16, None) == 0
    for i in (0, 4, 5, 6, 7, 8, 9):
        a = [P, 2, 0, 64, P, P, P, P, P, P]
        a[i] = None
        assert compact(*a, 2, 8, 8, 16, P) == INVALID, i
    assert compact(P, 2, 0, 64, P, P, P, P, P, P, 2, 8, 8, 16, None) == INVALID
    assert attn.lib().attn_pages_workspace_bytes(3, 100) >= 4 * (4 * 3 + 3 * 100)


def test_w4_refusals(attn):
    lib = attn.lib()
    pack = lambda *a: lib.attn_w4_pack(*a, None)  # noqa: E731
    assert pack(None, None, None, 0, 64, 32) == 0 and pack(None, None, None, 64, 0, 32) == 0
    for a in ((None, P, P), (P, None, P), (P, P, None), (P, P + 8, P)):
        assert pack(*a, 64, 64, 32) == INVALID
    for group in (0, 16, 33, 2**32):
        assert pack(P, P, P, 64, 64, group) == INVALID
    assert pack(P, P, P, 2**31, 64, 32) == INVALID
    # (x, y, packed, scales, residual, tokens, in, out, group, x stride, y stride)
    mv = lambda *a: lib.attn_w4_matvec(*a, None)  # noqa: E731
    assert mv(None, None, None, None, None, 0, 64, 64, 32, 0, 0) == 0
    assert mv(None, None, None, None, None, 1, 64, 0, 32, 0, 0) == 0
    for i in range(4):
        a = [P, P, P, P, None]
        a[i] = None
        assert mv(*a, 1, 64, 64, 32, 0, 0) == INVALID, i
    assert mv(P, P, P + 8, P, None, 1, 64, 64, 32, 0, 0) == INVALID
    for group in (0, 16, 40):
        assert mv(P, P, P, P, None, 1, 64, 64, group, 0, 0) == INVALID
    assert mv(P, P, P, P, None, 2**16, 64, 64, 32, 0, 0) == INVALID
    assert lib.attn_w4_weight_bytes(17, 129) == 4 * 1024
    assert lib.attn_w4_weight_bytes(16, 128) == 1024
    assert lib.attn_w4_scale_count(17, 129, 64) == 32 * 3
    assert lib.attn_w4_scale_count(17, 129, 0) == 0


def test_w4_rows_of_y_that_overlap_are_refused(attn):
    mv = lambda *a: attn.lib().attn_w4_matvec(*a, None)  # noqa: E731
    assert mv(P, P, P, P, None, 2, 64, 64, 32, 0, 63) == INVALID
    assert mv(P, P, P, P, P, 64, 0, 64, 32, 0, 8) == INVALID


def test_cache_refuses_lists_that_are_too_short(attn):
    import torch
    cache = attn.PagedKVCache(1, 8, 4, 1, 8, 3, 2, device="cpu")
    short = torch.zeros(2, dtype=torch.int32)
    for call in (cache.grow, cache.free, cache.fork):
        with pytest.raises(attn.AttnError, match="2 entries, needs 3"):
            call(short)
    for lists in ((short, None), (torch.zeros(3, dtype=torch.int32), short)):
        with pytest.raises(attn.AttnError, match="2 entries, needs 3"):
            cache.append(0, P, P, P, P, P, lists[0], 3, 1, 8, seq_ids=lists[1])


def test_wrappers_refuse_other_integers(attn):
    """Page numbers and lengths in 64 bits, or in another order, never reach the library."""
    import torch
    good = torch.zeros(4, 4, dtype=torch.int32)
    for bad in (good.long(), good.float(), good.t()[1:], good[:, ::2]):
        with pytest.raises(attn.AttnError, match="kv_lens must be a contiguous int32"):
            attn.paged_decode(P, P, P, P, good, bad, 4, 4, 8, 16, 4, 2, 64, P)
        with pytest.raises(attn.AttnError, match="page_table must be"):
            attn.pages_free(bad, good, good, 4, 4, 8, 16)
        with pytest.raises(attn.AttnError, match="positions must be"):
            attn.paged_rope_store_kv(P, P, P, P, P, P, P, good, bad, 4, 4, 4, 8, 16, 9, 4, 2, 64)
    for w in (torch.zeros(4, 64), torch.zeros(64, 4, dtype=torch.float16).t(),
              torch.zeros(4, 63, dtype=torch.float16)):
        with pytest.raises(attn.AttnError, match="4 x 64 contiguous fp16"):
            attn.w4_pack(w, 4, 64, 32)


@pytest.mark.parametrize("N,K", [(1, 1), (16, 128), (35, 300)])
def test_reference_words_hold_every_code(N, K):
    codes = np.random.default_rng(N).integers(0, 16, (N, K))
    words = ref.w4_words(codes)
    for n in range(N):
        for k in range(K):
            j, s, a, e = k // 128, k % 128 // 32, k % 32 // 8, k % 8
            w = int(words[n // 16, j].reshape(-1)[4 * (16 * a + n % 16) + s])
            assert w >> (4 * (e // 2) + 16 * (e % 2)) & 15 == codes[n, k]
