"""4-bit weights: the packer against numpy bit for bit, the products against 64 bits."""
import numpy as np
import pytest
import torch

import paged_reference as ref
from attn_mi355x import hipgraph

pytestmark = pytest.mark.gpu


def dev(a, gpu):
    return torch.from_numpy(np.ascontiguousarray(a)).to(gpu)


def weights(N, K, group, seed):
    """Codes over the whole range and scales of different rows and groups far apart."""
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 16, (N, K))
    scales = np.zeros((-(-K // group), -(-N // 16) * 16), dtype=np.float16)
    scales[:, :N] = np.exp(rng.uniform(-6, -2, (scales.shape[0], N)))
    return codes, scales


@pytest.mark.parametrize("N,K,group", [(16, 128, 32), (1, 1, 32), (17, 129, 64), (100, 1000, 128),
                                       (2048, 2048, 128), (33, 257, 32), (5, 4096, 4096),
                                       (48, 96, 96)])
def test_pack_bitexact(attn, gpu, N, K, group):
    rng = np.random.default_rng(N + K)
    w = rng.standard_normal((N, K)).astype(np.float16)
    w[0] = 0                                    # a scale of zero
    if N > 4:
        w[1] *= np.float16(6e-8)                # values and scales below the normal range
        w[2] *= np.float16(10000)
        w[3, :K // 2] = 7.0 * 2.0**-3           # ties and the range's ends
        w[3, K // 2:] = np.resize(np.array([7, -7, 0.5, 1.5, -2.5], dtype=np.float16), K - K // 2)
    packed, scales = attn.w4_pack(dev(w, gpu), N, K, group)
    torch.cuda.synchronize()
    codes, exp = ref.w4_quantize(w, group)
    full = np.zeros((exp.shape[0], -(-N // 16) * 16), dtype=np.float16)
    full[:, :N] = exp
    assert np.array_equal(scales.cpu().numpy().reshape(full.shape).view(np.uint16),
                          full.view(np.uint16))
    assert np.array_equal(packed.cpu().numpy().view(np.uint32), ref.w4_words(codes).ravel())


def test_pack_of_no_numbers(attn, gpu):
    """An infinity or a NaN in a group: products with its row are no number."""
    w = np.ones((3, 64), dtype=np.float16)
    w[0, 5], w[1, 40] = np.inf, np.nan
    packed, scales = attn.w4_pack(dev(w, gpu), 3, 64, 32)
    y = torch.zeros(3, dtype=torch.float16, device=gpu)
    attn.w4_matvec(torch.ones(64, dtype=torch.float16, device=gpu), y, packed, scales, 1, 64, 3, 32)
    torch.cuda.synchronize()
    y = y.cpu().numpy()
    assert np.isnan(y[:2]).all() and abs(y[2] - 64) <= 64 * 2.0**-10


def product(attn, gpu, T, N, K, group, seed, x_pad=0, y_pad=0, residual=None, x_off=0):
    """residual: None, "apart" or "in place"."""
    rng = np.random.default_rng(seed + 1)
    codes, scales = weights(N, K, group, seed)
    xs, ys = K + x_pad, N + y_pad
    x = np.full(T * xs + x_off + 8, np.nan, dtype=np.float16)  # NaN between and behind the rows
    rows = x[x_off:x_off + T * xs].reshape(T, xs)
    rows[:, :K] = rng.standard_normal((T, K))
    y = np.full((T, ys), 55.0, dtype=np.float16)
    r = None
    if residual:
        r = np.full((T, ys), np.nan, dtype=np.float16)
        r[:, :N] = rng.standard_normal((T, N)) * 3
        if residual == "in place":
            y[:, :N] = r[:, :N]
    dy = dev(np.concatenate([y.ravel(), np.full(16, 55.0, np.float16)]), gpu)
    dr = dy if residual == "in place" else dev(r, gpu) if residual else None
    args = (dev(x, gpu)[x_off:], dy, dev(ref.w4_words(codes).view(np.int32), gpu),
            dev(scales, gpu), T, K, N, group)
    attn.w4_matvec(*args, residual=dr, x_stride=xs, y_stride=ys)
    torch.cuda.synchronize()
    got = dy.cpu().numpy()
    assert (got[-16:] == 55).all()
    got = got[:-16].reshape(T, ys)
    assert (got[:, N:] == 55).all()
    exp, bound = ref.w4_product(codes, scales[:, :N], group, rows[:, :K],
                                r[:, :N] if residual else None)
    err = np.abs(got[:, :N].astype(np.float64) - exp)
    assert (err <= bound).all(), (T, N, K, group, err.max(), (err / bound).max())


@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("T,N,K", [
    (1, 1, 1), (1, 16, 128), (1, 2048, 2048), (2, 100, 257), (3, 17, 31), (5, 48, 33),
    (1, 33, 5000), (16, 64, 512), (17, 130, 640), (33, 96, 1111), (64, 40, 384), (65, 16, 256),
    (130, 24, 160), (1, 5000, 96)])
def test_products(attn, gpu, T, N, K, group):
    print(f"[case] T={T} N={N} K={K} group={group}", flush=True)
    product(attn, gpu, T, N, K, group, T + N + K)


@pytest.mark.parametrize("residual", [None, "apart", "in place"])
@pytest.mark.parametrize("T,N,K,x_pad,y_pad,x_off", [
    (1, 2048, 2048, 0, 0, 0), (4, 50, 256, 8, 8, 0), (4, 50, 256, 3, 5, 0), (7, 33, 300, 0, 1, 1),
    (20, 64, 136, 8, 0, 0), (40, 80, 1000, 0, 16, 8)])
def test_strides_and_residuals(attn, gpu, T, N, K, x_pad, y_pad, x_off, residual):
    print(f"[case] T={T} N={N} K={K} pads {x_pad} {y_pad} offset {x_off} {residual}", flush=True)
    product(attn, gpu, T, N, K, 64, T + N, x_pad, y_pad, residual, x_off)


def test_the_layers_of_a_model(attn, gpu):
    """The widths of a layer, one token and a batch."""
    for T in (1, 33):
        for N, K, group in ((2048, 2048, 128), (2048, 11008, 32), (11008, 2048, 64)):
            print(f"[case] T={T} N={N} K={K}", flush=True)
            product(attn, gpu, T, N, K, group, T, residual="apart")


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T,N,K", [
    (64, 8200, 160), (50, 8208, 200), (100, 6000, 96), (64, 16400, 104), (17, 16390, 72),
    (64, 32784, 40), (48, 32770, 264), (33, 32768, 48), (16, 32784, 88), (5, 32800, 136),
    (16, 6150, 1000), (130, 4100, 392), (33, 2060, 640), (64, 2050, 4240),
    (64, 8200, 164), (20, 32768, 36),   # columns that take element loads
    (16, 4100, 300), (40, 1500, 256)])
def test_many_rows(attn, gpu, T, N, K, group):
    """The tiles of more rows and tokens a wave, rows and tokens that end inside them."""
    print(f"[case] T={T} N={N} K={K} group={group}", flush=True)
    product(attn, gpu, T, N, K, group, T, residual="apart")


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T,N,K", [
    (1, 40, 1027), (4, 100, 2050), (12, 60, 1281), (16, 4100, 447), (16, 6150, 1001), (33, 2060, 641),
    (64, 8200, 161), (40, 16400, 199), (100, 6000, 97), (48, 32770, 261), (5, 32800, 135),
    (64, 2050, 4241), (65, 16400, 5), (20, 300, 127), (20, 300, 129)])
def test_odd_columns(attn, gpu, T, N, K, group):
    """Rows of x at every element: no 16-byte boundary, the tile with the row's end."""
    print(f"[case] T={T} N={N} K={K} group={group}", flush=True)
    product(attn, gpu, T, N, K, group, T, x_off=T % 3)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T,N,K", [
    (16, 65600, 72), (7, 65540, 135), (60, 28700, 133), (64, 28720, 264), (33, 11008, 176),
    (48, 10930, 171), (32, 12288, 168), (25, 12270, 143), (80, 11000, 104), (16, 12300, 392)])
def test_workgroups_that_share_x(attn, gpu, T, N, K, group):
    """Either side of the sizes from which workgroups take more rows or tokens."""
    print(f"[case] T={T} N={N} K={K} group={group}", flush=True)
    product(attn, gpu, T, N, K, group, T, residual="in place")


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T,N,K", [(16, 40, 8200), (7, 33, 8192), (8, 300, 8064), (5, 17, 8072),
                                   (33, 2050, 8328), (64, 2040, 8208), (64, 2050, 8208)])
def test_many_columns(attn, gpu, T, N, K, group):
    """Few rows of many columns, split between more waves."""
    print(f"[case] T={T} N={N} K={K} group={group}", flush=True)
    product(attn, gpu, T, N, K, group, T, x_pad=8, residual="apart")


def test_infinity_in_one_token_stays_there(attn, gpu):
    N, K = 40, 200
    codes, scales = weights(N, K, 32, 1)
    x = np.random.default_rng(2).standard_normal((5, K)).astype(np.float16)
    clean = x.copy()
    x[1, 0], x[3, K - 1] = np.inf, np.nan
    y = torch.empty(5, N, dtype=torch.float16, device=gpu)
    attn.w4_matvec(dev(x, gpu), y, dev(ref.w4_words(codes).view(np.int32), gpu),
                   dev(scales, gpu), 5, K, N, 32)
    torch.cuda.synchronize()
    got = y.cpu().numpy()
    exp, bound = ref.w4_product(codes, scales[:, :N], 32, clean)
    for t in (0, 2, 4):
        assert (np.abs(got[t].astype(np.float64) - exp[t]) <= bound[t]).all()
    assert not np.isfinite(got[1]).any() and np.isnan(got[3]).all()


def test_no_columns(attn, gpu):
    y = torch.full((2, 20), 9.0, dtype=torch.float16, device=gpu)
    r = torch.arange(40, dtype=torch.float16, device=gpu).view(2, 20)
    attn.w4_matvec(None, y, None, None, 2, 0, 20, 32, residual=r)
    torch.cuda.synchronize()
    assert torch.equal(y, r)
    attn.w4_matvec(None, y, None, None, 2, 0, 20, 32)
    torch.cuda.synchronize()
    assert (y == 0).all()


def test_captured_product(attn, gpu):
    """Replays with new inputs and a residual added in place, eager work in between."""
    N, K, T = 300, 700, 3
    codes, scales = weights(N, K, 64, 5)
    w, s = dev(ref.w4_words(codes).view(np.int32), gpu), dev(scales, gpu)
    x = torch.empty(T, K, dtype=torch.float16, device=gpu)
    y, z = (torch.empty(T, N, dtype=torch.float16, device=gpu) for _ in "yz")
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    hipgraph.begin_capture(stream.cuda_stream)
    attn.w4_matvec(x, y, w, s, T, K, N, 64, residual=y, stream=stream.cuda_stream)
    graph, exe = hipgraph.end_capture(stream.cuda_stream)
    for turn in range(4):
        g = torch.Generator().manual_seed(turn)
        x.copy_(torch.randn(T, K, generator=g))
        y.copy_(torch.randn(T, N, generator=g))
        z.copy_(y)
        attn.w4_matvec(x, z, w, s, T, K, N, 64, residual=z)
        torch.cuda.synchronize()
        hipgraph.launch(exe, stream.cuda_stream)
        hipgraph.synchronize(stream.cuda_stream)
        assert torch.equal(y, z)
    hipgraph.destroy(graph, exe)
