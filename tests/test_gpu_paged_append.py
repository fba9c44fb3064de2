"""RoPE + append into pages: every value equals rope_store_kv's for the same position, bit
for bit; tokens that name no cache row leave everything alone."""
import numpy as np
import pytest
import torch

import oracle

pytestmark = pytest.mark.gpu
FILL = np.uint16(0x5A5A)


def setup(T, B, page, Hq, Hkv, D, seed, columns, most, pad=0, one_each=False):
    rng = np.random.default_rng(seed)
    stride = (Hq + 2 * Hkv) * D + pad
    qkv = rng.standard_normal((T, stride)).astype(np.float16).view(np.uint16)
    seq = np.arange(T) if one_each else rng.integers(0, B, T)
    pos = np.zeros(T, dtype=np.int32)
    for b in range(B):  # distinct positions within a sequence
        mine = np.flatnonzero(seq == b)
        pos[mine] = rng.choice(min(most, columns * page), len(mine), replace=False)
    pages = B * columns + 1
    table = rng.permutation(pages)[:B * columns].reshape(B, columns).astype(np.int32)
    cos, sin = oracle.rope_tables(most, D, 5.0e6)
    return stride, qkv, seq.astype(np.int32), pos, pages, table, cos, sin


def expected(qkv, seq, pos, table, pages, page, Hq, Hkv, D, stride, cos, sin, apply, live):
    q = qkv.copy()
    kp, vp = (np.full((pages * page, Hkv * D), FILL, np.uint16) for _ in "kv")
    qd, kvd = Hq * D, Hkv * D
    for t in np.flatnonzero(live):
        row = int(table[seq[t], pos[t] // page]) * page + pos[t] % page
        one = q[t].copy()
        cache = np.zeros(2 * kvd, np.uint16)
        p = int(pos[t]) if apply else 0
        # one token at "position 0" of tables that start at its row
        oracle.rope_store_kv(one, one[qd:], one[qd + kvd:], cache, cache[kvd:],
                             cos.reshape(-1, D // 2)[p:p + 1], sin.reshape(-1, D // 2)[p:p + 1],
                             1, Hq, Hkv, D, stride, stride, 0, apply)
        q[t, :qd] = one[:qd]
        kp[row], vp[row] = cache[:kvd], cache[kvd:]
    return q, kp, vp


def dev(a, gpu):
    return torch.from_numpy(np.ascontiguousarray(a).view(np.int16 if a.dtype == np.uint16
                                                         else a.dtype)).to(gpu)


def bits(t):
    return t.cpu().numpy().view(np.uint16)


@pytest.mark.parametrize("apply", [True, False])
@pytest.mark.parametrize("T,B,page,Hq,Hkv,D,pad,one", [
    (1, 1, 16, 16, 4, 128, 0, True), (64, 64, 16, 16, 4, 128, 0, True),
    (200, 3, 16, 16, 4, 128, 0, False), (77, 5, 7, 8, 8, 64, 8, False),
    (50, 4, 1, 32, 8, 64, 0, False), (33, 2, 24, 4, 2, 32, 3, False),
    (20, 2, 5, 3, 1, 6, 1, False), (40, 40, 128, 16, 8, 128, 0, True)])
def test_append_bitexact(attn, gpu, T, B, page, Hq, Hkv, D, pad, one, apply):
    print(f"[case] T={T} B={B} page={page} {Hq}/{Hkv}x{D} pad={pad} apply={apply}", flush=True)
    columns, most = max(3, -(-T * 2 // page)), 2 * T + 40
    stride, qkv, seq, pos, pages, table, cos, sin = setup(T, B, page, Hq, Hkv, D, T, columns,
                                                          most, pad, one)
    live = np.ones(T, dtype=bool)
    if T > 10:  # tokens of a padded batch, and every kind that is out of range
        for t, p in ((2, -1), (5, most), (6, -2**31)):
            pos[t], live[t] = p, False
        if not one:
            seq[8], live[8] = B, False
            seq[9], live[9] = -3, False
        table[seq[3], pos[3] // page] = pages
        for t in range(T):
            if live[t] and table[seq[t], pos[t] // page] == pages:
                live[t] = False
    q_e, kp_e, vp_e = expected(qkv, seq, pos, table, pages, page, Hq, Hkv, D, stride, cos, sin,
                               apply, live)
    qd, kvd = Hq * D, Hkv * D
    for out_of_place in (True, False):
        x = dev(qkv, gpu)
        kp, vp = (torch.full((pages * page, kvd), int(FILL), dtype=torch.int16, device=gpu)
                  for _ in "kv")
        q_out = torch.full((T + 1, qd), int(FILL), dtype=torch.int16, device=gpu)
        at = x.data_ptr()
        attn.paged_rope_store_kv(
            at, at + 2 * qd, at + 2 * (qd + kvd), kp, vp, dev(cos, gpu), dev(sin, gpu),
            dev(table, gpu), dev(pos, gpu), T, B, columns, pages, page, most, Hq, Hkv, D, stride,
            stride, apply, q_out=q_out if out_of_place else None,
            seq_ids=None if one else dev(seq, gpu))
        torch.cuda.synchronize()
        assert np.array_equal(bits(kp), kp_e) and np.array_equal(bits(vp), vp_e)
        if out_of_place:
            assert np.array_equal(bits(x), qkv)
            exp = np.full((T + 1, qd), FILL)
            exp[:T][live] = q_e[live, :qd]
            assert np.array_equal(bits(q_out), exp)
        else:
            assert np.array_equal(bits(x), q_e)
            assert (bits(q_out) == FILL).all()


def test_positions_past_the_tables_row(attn, gpu):
    """A position beyond max_pages pages, with rotation tables that reach further."""
    T = B = 2
    stride, qkv, seq, pos, pages, table, cos, sin = setup(T, B, 4, 4, 2, 64, 1, 2, 100, 0, True)
    pos[:] = [8, 7]  # two pages of four rows hold positions 0..7
    kp, vp = (torch.full((pages * 4, 128), int(FILL), dtype=torch.int16, device=gpu) for _ in "kv")
    x = dev(qkv, gpu)
    at = x.data_ptr()
    attn.paged_rope_store_kv(at, at + 512, at + 768, kp, vp, dev(cos, gpu), dev(sin, gpu),
                             dev(table, gpu), dev(pos, gpu), T, B, 2, pages, 4, 100, 4, 2, 64,
                             stride, stride)
    torch.cuda.synchronize()
    q_e, kp_e, vp_e = expected(qkv, seq, pos, table, pages, 4, 4, 2, 64, stride, cos, sin, True,
                               np.array([False, True]))
    assert np.array_equal(bits(kp), kp_e) and np.array_equal(bits(vp), vp_e)
    assert np.array_equal(bits(x), q_e)


def test_unaligned_tensors(attn, gpu):
    """The pool two bytes off a 16-byte boundary: the element-wise kernel, same bits."""
    T, B, page, Hq, Hkv, D = 9, 2, 16, 4, 2, 64
    stride, qkv, seq, pos, pages, table, cos, sin = setup(T, B, page, Hq, Hkv, D, 3, 4, 64)
    kvd, qd = Hkv * D, Hq * D
    _, kp_e, vp_e = expected(qkv, seq, pos, table, pages, page, Hq, Hkv, D, stride, cos, sin,
                             True, np.ones(T, dtype=bool))
    kp, vp = (torch.full((pages * page * kvd + 1,), int(FILL), dtype=torch.int16, device=gpu)
              for _ in "kv")
    x = dev(qkv, gpu)
    at = x.data_ptr()
    attn.paged_rope_store_kv(at, at + 2 * qd, at + 2 * (qd + kvd), kp[1:], vp[1:], dev(cos, gpu),
                             dev(sin, gpu), dev(table, gpu), dev(pos, gpu), T, B, 4, pages, page,
                             64, Hq, Hkv, D, stride, stride, seq_ids=dev(seq, gpu))
    torch.cuda.synchronize()
    assert np.array_equal(bits(kp)[1:], kp_e.ravel()) and bits(kp)[0] == FILL
    assert np.array_equal(bits(vp)[1:], vp_e.ravel())
