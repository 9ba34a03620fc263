"""The layer operators on the GPU against plain 64-bit forms."""
import math

import numpy as np
import pytest
import torch

import layer_reference as ref
from liteform_ae_b200 import _cabi, hyb, layer

pytestmark = pytest.mark.gpu

F32, BF16, F16, E4M3 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn
U32 = ref.U[F32]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rows_of(shape, dtype, g, dev, pitch=None, shift=0):
    """Random rows with a row stride of `pitch` elements, `shift` elements into their buffer."""
    M, N = shape
    v = torch.randn(shape, generator=g).to(dtype)
    pitch = N if pitch is None else pitch
    buf = torch.zeros(M * pitch + shift + 32, dtype=dtype, device=dev)
    t = torch.as_strided(buf, (M, N), (pitch, 1), shift)
    t.copy_(v)
    return t, v.double()


# ---- norm -------------------------------------------------------------------------------------------
def check_norm(x, r, w, eps, n, xv, rv, wv):
    """n: what rms_norm returned; ...v: the 64-bit values of its inputs."""
    dt = x.dtype
    hv = xv
    if r is not None:
        hv = (xv.float() + rv.float()).to(dt).double()     # one addition in 32 bits, one rounding
        assert torch.equal(n.h.cpu().double(), hv)
    N = xv.shape[1]
    ms = hv.square().sum(1) / N
    rstd = (ms + eps) ** -0.5
    # a sum of N squares is off by N + 1 roundings at most (all terms positive), the quotient and eps by 2, the
    # root halves that; rsqrtf by 2 units in the last place
    off = ((N + 3) / 2 + 4) * U32 * 1.01
    ref.close(n.rstd, rstd, off * rstd, "rstd")
    y = hv * rstd[:, None] * wv
    yoff = (off + 2 * U32) * y.abs()
    if n.y.dtype != E4M3:
        ref.close(n.y, y, ref.rounded(y, yoff, n.y.dtype), "y")
        return
    amax = y.abs().amax(1)
    ref.close(n.scale, amax / 448, (off + 5 * U32) * amax / 448, "scale")
    back = n.y.cpu().double() * n.scale.cpu().double()[:, None]
    # the stored value is within half a step of y / scale (2^-4 relative, 2^-10 below the normal numbers), the scale
    # as it is stored; y / scale itself is off as y is, plus the reciprocal and two products
    s = n.scale.cpu().double()[:, None]
    t = yoff + 4 * U32 * y.abs()
    ref.close(back, y, t + 2.0 ** -4 * (y.abs() + t) + 2.0 ** -10 * s, "8-bit rows")
    q = n.y.cpu().double().abs().amax(1)
    assert bool(((q == 448) | (amax < 1e-30)).all()), "the largest value of a row is stored as 448"


@pytest.mark.parametrize("M,N", [(1, 1), (1, 4096), (3, 7), (5, 8), (33, 47), (130, 128), (17, 300), (9, 512), (4, 1000), (70, 64),
                                 (3, 2048), (2, 8192), (2, 5001), (2, 20000), (1, 70001), (600, 16), (129, 33)])
@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, E4M3), (F32, E4M3), (F16, E4M3), (BF16, F32)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(cuda_device, M, N, dtype, out, residual):
    g = gen(M * 7 + N)
    x, xv = rows_of((M, N), dtype, g, cuda_device)
    r, rv = rows_of((M, N), dtype, g, cuda_device) if residual else (None, None)
    w = (1 + 0.1 * torch.randn(N, generator=g)).to(dtype).to(cuda_device)
    n = layer.rms_norm(x, w, residual=r, eps=1e-5, out_dtype=out)
    assert n.y.dtype == out and n.y.shape == (M, N)
    check_norm(x, r, w, 1e-5, n, xv, rv, w.cpu().double())


@pytest.mark.parametrize("N,pitch,shift", [(47, 50, 1), (64, 72, 0), (64, 72, 8), (128, 129, 3), (96, 104, 2), (1024, 1031, 5), (24, 24, 1)])
@pytest.mark.parametrize("dtype,out", [(BF16, E4M3), (F32, F32), (F16, BF16)])
def test_norm_strides(cuda_device, N, pitch, shift, dtype, out):
    g, M = gen(N), 37
    x, xv = rows_of((M, N), dtype, g, cuda_device, pitch, shift)
    r, rv = rows_of((M, N), dtype, g, cuda_device, pitch + 8, 0)
    w = (1 + 0.1 * torch.randn(N, generator=g)).to(cuda_device)       # a float32 weight beside 16-bit rows
    buf = torch.zeros(M * pitch + shift + 8, device=cuda_device).to(out)
    y = torch.as_strided(buf, (M, N), (pitch, 1), shift)
    hbuf = torch.full((M * pitch + shift + 8,), 7.0, dtype=dtype, device=cuda_device)
    h = torch.as_strided(hbuf, (M, N), (pitch, 1), shift)
    n = layer.rms_norm(x, w, residual=r, eps=1e-6, out=y, sum_out=h)
    check_norm(x, r, w, 1e-6, n, xv, rv, w.cpu().double())
    inside = torch.zeros_like(hbuf, dtype=torch.bool)
    torch.as_strided(inside, (M, N), (pitch, 1), shift).fill_(True)
    assert bool((hbuf[~inside] == 7).all()) and bool((buf[~inside].float() == 0).all()), "what lies between the rows stays"


def test_norm_in_place(cuda_device):
    g = gen(4)
    for N in (64, 61, 6000):
        x, xv = rows_of((21, N), BF16, g, cuda_device)
        r, rv = rows_of((21, N), BF16, g, cuda_device)
        w = torch.ones(N, dtype=BF16, device=cuda_device)
        n = layer.rms_norm(x, w, residual=r, sum_out=r)
        assert n.h is r
        check_norm(x, r, w, 1e-6, n, xv, rv, w.cpu().double())


@pytest.mark.parametrize("N", [8, 47, 128, 4096])
@pytest.mark.parametrize("out", [F32, E4M3])
def test_norm_special_rows(cuda_device, N, out):
    x = torch.randn(6, N, generator=gen(N))
    x[0] = 0
    x[1, N // 2] = float("nan")
    x[2, N - 1] = float("inf")
    x[3] = 1e-30
    x[4] *= 1e15
    w = torch.ones(N, device=cuda_device)
    n = layer.rms_norm(x.to(cuda_device), w, out_dtype=out, eps=1e-6)
    y = n.y.float().cpu()
    assert bool((y[0] == 0).all()) and bool(torch.isnan(y[1]).all())
    assert bool(torch.isnan(y[2, N - 1])) and float(n.rstd[2]) == 0     # infinity times 0
    ok = [0, 3, 4, 5]
    if out == E4M3:
        assert float(n.scale[0]) == 0 and bool(torch.isnan(n.scale[1:3]).all())
        ok = [4, 5]
        assert bool(torch.isfinite(n.y.float()[3]).all())
    sub = layer.NormOutput(n.y[ok], n.scale[ok] if out == E4M3 else None, n.h[ok], n.rstd[ok])
    check_norm(x[ok].to(cuda_device), None, w, 1e-6, sub, x[ok].double(), None, w.cpu().double())


def norm_grad64(dy, h, w, rstd, dh):
    N = h.shape[1]
    n = h * rstd[:, None]
    t = dy * w
    c = (t * n).sum(1, keepdim=True) / N
    dx = rstd[:, None] * (t - n * c) + (0 if dh is None else dh)
    # roundings: t and n one each, the sum N + 3 of its size, then three products and two additions
    size = rstd[:, None] * (t.abs() + n.abs() * (t * n).abs().sum(1, keepdim=True) / N * (N + 4)) + (0 if dh is None else dh.abs())
    return dx, 6 * U32 * size, (dy * n).sum(0), ((dy * n).abs().sum(0)) * (h.shape[0] + 3) * U32


@pytest.mark.parametrize("M,N", [(1, 1), (1, 4096), (3, 7), (33, 47), (700, 128), (2000, 64), (17, 300), (1300, 512), (5, 1000), (3, 8192),
                                 (2, 5001), (3, 20001), (1500, 33)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("with_dh", [False, True])
def test_norm_backward(cuda_device, M, N, dtype, with_dh):
    g = gen(M + N)
    dy, dyv = rows_of((M, N), dtype, g, cuda_device)
    h, hv = rows_of((M, N), dtype, g, cuda_device)
    dh, dhv = rows_of((M, N), dtype, g, cuda_device) if with_dh else (None, None)
    w = (1 + 0.1 * torch.randn(N, generator=g)).to(dtype).to(cuda_device)
    rstd = (hv.square().mean(1) + 1e-6).rsqrt().float().to(cuda_device)
    dx, dw = layer.rms_norm_backward(dy, h, w, rstd, dh=dh)
    want, off, dwv, dwoff = norm_grad64(dyv, hv, w.cpu().double(), rstd.cpu().double(), dhv)
    ref.close(dx, want, ref.rounded(want, off, dtype), "dx")
    ref.close(dw, dwv, dwoff + ref.TINY[F32], "dw")
    again = layer.rms_norm_backward(dy, h, w, rstd, dh=dh)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


@pytest.mark.parametrize("N,pitch,shift", [(47, 50, 1), (64, 72, 8), (128, 129, 3), (96, 104, 0)])
def test_norm_backward_strides_and_in_place(cuda_device, N, pitch, shift):
    g, M = gen(N), 45
    dy, dyv = rows_of((M, N), BF16, g, cuda_device, pitch, shift)
    h, hv = rows_of((M, N), BF16, g, cuda_device, pitch + 1, 0)
    dh, dhv = rows_of((M, N), BF16, g, cuda_device, pitch, 0)
    w = torch.randn(N, generator=g).to(cuda_device)
    rstd = torch.rand(M, generator=g).to(cuda_device)
    want, off, dwv, dwoff = norm_grad64(dyv, hv, w.cpu().double(), rstd.cpu().double(), dhv)
    dx, dw = layer.rms_norm_backward(dy, h, w, rstd, dh=dh, dx=dh)
    assert dx is dh
    ref.close(dx, want, ref.rounded(want, off, BF16), "dx")
    ref.close(dw, dwv, dwoff, "dw")


def test_norm_gradient_by_differences(cuda_device):
    """Along a random direction, against central differences of the 64-bit norm."""
    g = gen(9)
    M, N, eps = 12, 40, 1e-5
    x, w, dy = (torch.randn(s, generator=g, dtype=torch.float64).float().double() for s in ((M, N), (N,), (M, N)))
    f = lambda x, w: float((dy * (x * (x.square().mean(1, keepdim=True) + eps).rsqrt() * w)).sum())
    ux, uw = torch.randn(M, N, generator=g, dtype=torch.float64), torch.randn(N, generator=g, dtype=torch.float64)
    d = 1e-5
    dev = lambda t: t.float().to(cuda_device)
    n = layer.rms_norm(dev(x), dev(w), eps=eps)
    dx, dw = layer.rms_norm_backward(dev(dy), n.h, dev(w), n.rstd)
    for got, diff in ((float((dx.cpu().double() * ux).sum()), (f(x + d * ux, w) - f(x - d * ux, w)) / (2 * d)),
                      (float((dw.cpu().double() * uw).sum()), (f(x, w + d * uw) - f(x, w - d * uw)) / (2 * d))):
        # 480 terms of size about 1, each known to about N roundings; differences of third order: d^2 ~ 1e-10
        assert abs(got - diff) < 480 * N * U32 + 1e-6


def test_norm_refusals(cuda_device):
    x = torch.randn(4, 16, device=cuda_device)
    w = torch.ones(16, device=cuda_device)
    for call in (lambda: layer.rms_norm(x, w[:8]), lambda: layer.rms_norm(x[0], w), lambda: layer.rms_norm(x.t(), torch.ones(4, device=cuda_device)),
                 lambda: layer.rms_norm(x.double(), w), lambda: layer.rms_norm(x, w, residual=x.bfloat16()),
                 lambda: layer.rms_norm(x, w, residual=x[:3]), lambda: layer.rms_norm(x, w, sum_out=x),
                 lambda: layer.rms_norm(x, w, scale=w[:4]), lambda: layer.rms_norm(x, w.cpu()),
                 lambda: layer.rms_norm(x, w, out=torch.empty(4, 15, device=cuda_device)),
                 lambda: layer.rms_norm(x, w, out=x.bfloat16(), out_dtype=F32), lambda: layer.rms_norm(x[:1].expand(4, 16), w),
                 lambda: layer.rms_norm_backward(x, x.bfloat16(), w, w[:4]), lambda: layer.rms_norm_backward(x, x, w, w),
                 lambda: layer.rms_norm_backward(x, x, w, w[:4], dh=x[:2])):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(_cabi.LiteformError):
        layer.rms_norm(x, w, eps=-1.0)
    assert layer.rms_norm(x[:0], w).y.shape == (0, 16)
    dx, dw = layer.rms_norm_backward(x[:0], x[:0], w, w[:0])
    assert dx.shape == (0, 16) and float(dw.abs().sum()) == 0


# ---- product ----------------------------------------------------------------------------------------
def pattern(M, K, seed, mean=6.0, longest=0, empty=0.2):
    """CSR arrays (CPU): some rows empty, row `M // 2` of `longest` entries."""
    rng = np.random.default_rng(seed)
    lens = np.minimum(rng.poisson(mean, M), K)
    lens[rng.random(M) < empty] = 0
    if longest and M:
        lens[M // 2] = min(longest, K)
    cols = [np.sort(rng.choice(K, n, replace=False)) for n in lens]
    indptr = np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)
    indices = (np.concatenate(cols) if len(cols) else np.zeros(0)).astype(np.int32)
    vals = rng.uniform(-1, 1, len(indices)).astype(np.float32)
    return torch.from_numpy(indptr), torch.from_numpy(indices), torch.from_numpy(vals)


def csr_on(dev, p, shape, with_values=True):
    return hyb.DeviceCsr(p[0].to(dev), p[1].to(dev), p[2].to(dev) if with_values else None, shape)


def features(K, N, dtype, g, dev, pitch=None, shift=0):
    """(B, scale, 64-bit rows)"""
    if dtype != E4M3:
        B, v = rows_of((K, N), dtype, g, dev, pitch, shift)
        return B, None, v
    q, v = rows_of((K, N), E4M3, g, dev, pitch, shift)
    scale = torch.rand(K, generator=g) + 0.01
    return q, scale.to(dev), v * scale.double()[:, None]


TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (E4M3, BF16), (E4M3, F32), (BF16, F32), (F32, F16), (E4M3, F16)]


@pytest.mark.parametrize("M,K,N,mean,longest", [
    (1, 1, 1, 1, 0), (1, 50, 64, 20, 50), (40, 30, 8, 3, 0), (64, 64, 32, 6, 0), (100, 80, 47, 6, 0), (90, 600, 128, 10, 600),
    (50, 40, 300, 6, 0), (33, 3000, 16, 8, 3000), (70, 5000, 33, 30, 5000), (20, 2500, 520, 30, 2500), (300, 64, 1, 4, 0),
    (257, 100, 1024, 5, 0), (700, 500, 96, 14, 0), (5, 7, 2, 2, 0), (400, 9000, 7, 20, 9000)])
@pytest.mark.parametrize("dtype,out", TYPES)
def test_product(cuda_device, M, K, N, mean, longest, dtype, out):
    g = gen(M + K + N)
    p = pattern(M, K, M + N, mean, longest)
    A = csr_on(cuda_device, p, (M, K))
    B, scale, Bv = features(K, N, dtype, g, cuda_device)
    bias = torch.randn(N, generator=g).to(out)
    R, Rv = rows_of((M, N), out, g, cuda_device)
    name = ref.ACTS[(M + N) % 5]
    z, y, zoff, yoff = ref.product(ref.dense(*p, (M, K)), Bv, bias, name, Rv, out)
    pre = torch.empty((M, N), dtype=out, device=cuda_device)
    kw = dict(scale=scale, bias=bias.to(cuda_device), activation=name, residual=R, preact=pre, out_dtype=out)
    got = layer.spmm_csr_act(A, B, **kw)
    assert got.dtype == out
    ref.close(pre, z, zoff, "z")
    ref.close(got, y, yoff, "y")
    assert torch.equal(layer.spmm_csr_act(A, B, **kw), got), "the same call gives the same bits"


@pytest.mark.parametrize("name", ref.ACTS)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("N", [48, 21])
def test_product_epilogues(cuda_device, name, residual, bias, N):
    g = gen(N)
    M, K = 80, 60
    p = pattern(M, K, 5)
    A = csr_on(cuda_device, p, (M, K), with_values=False)       # all ones
    B, _, Bv = features(K, N, F32, g, cuda_device)
    R, Rv = rows_of((M, N), BF16, g, cuda_device) if residual else (None, None)    # another type than the result's
    b = torch.randn(N, generator=g).half() if bias else None
    got = layer.spmm_csr_act(A, B, bias=None if b is None else b.to(cuda_device), activation=name, residual=R)
    z, y, _, off = ref.product(ref.dense(p[0], p[1], None, (M, K)), Bv, b, name, Rv, F32)
    ref.close(got, y, off, name)


@pytest.mark.parametrize("dtype", [F32, BF16, F16, E4M3])
@pytest.mark.parametrize("N,pitch,shift", [(64, 64, 1), (64, 80, 0), (64, 80, 16), (31, 32, 0), (31, 33, 2), (128, 131, 7), (200, 208, 0),
                                           (17, 48, 0), (260, 261, 1)])
def test_product_strides(cuda_device, dtype, N, pitch, shift):
    g = gen(N + shift)
    M, K = 150, 90
    out = BF16 if dtype == E4M3 else dtype
    p = pattern(M, K, 8, 9.0, 90)
    A = csr_on(cuda_device, p, (M, K))
    B, scale, Bv = features(K, N, dtype, g, cuda_device, pitch, shift)
    R, Rv = rows_of((M, N), out, g, cuda_device, pitch + 3, shift)
    z, y, _, off = ref.product(ref.dense(*p, (M, K)), Bv, None, "gelu", Rv, out)
    buf = torch.full((M * pitch + shift + 16,), 5.0, dtype=out, device=cuda_device)
    C = torch.as_strided(buf, (M, N), (pitch, 1), shift)
    got = layer.spmm_csr_act(A, B, scale=scale, activation="gelu", residual=R, out=C)
    assert got is C
    ref.close(C, y, off)
    inside = torch.zeros_like(buf, dtype=torch.bool)
    torch.as_strided(inside, (M, N), (pitch, 1), shift).fill_(True)
    assert bool((buf[~inside] == 5).all()), "what lies between the rows stays"


def test_product_adds_to_its_own_output(cuda_device):
    g = gen(1)
    M, K, N = 120, 70, 64
    p = pattern(M, K, 2, 8.0, 70)
    A = csr_on(cuda_device, p, (M, K))
    B, _, Bv = features(K, N, BF16, g, cuda_device)
    C, Cv = rows_of((M, N), BF16, g, cuda_device)
    layer.spmm_csr_act(A, B, activation="silu", residual=C, out=C)
    _, y, _, off = ref.product(ref.dense(*p, (M, K)), Bv, None, "silu", Cv, BF16)
    ref.close(C, y, off)


@pytest.mark.parametrize("dtype", [F32, BF16, F16, E4M3])
@pytest.mark.parametrize("N", [64, 50])
def test_entries_of_value_zero_pass_nothing_on(cuda_device, dtype, N):
    """Rows of B that only entries of value 0 point at may hold anything."""
    g = gen(3)
    M, K = 60, 40
    indptr, indices, vals = pattern(M, K, 4, 6.0, 40)
    bad = (indices % 5) == 2
    vals[bad] = 0.0
    A = csr_on(cuda_device, (indptr, indices, vals), (M, K))
    B, scale, Bv = features(K, N, dtype, g, cuda_device)
    B.view(torch.uint8 if dtype == E4M3 else B.dtype)[2::5] = 0x7f if dtype == E4M3 else float("nan")
    if scale is not None:
        scale[2::5] = float("inf")
    Bv[2::5] = 0
    got = layer.spmm_csr_act(A, B, scale=scale, out_dtype=F32)
    _, y, _, off = ref.product(ref.dense(indptr, indices, vals, (M, K)), Bv, None, "none", None, F32)
    ref.close(got, y, off)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_infinities_and_nan_stay_in_their_rows(cuda_device, dtype):
    M, K, N = 64, 64, 40
    indptr = torch.arange(M + 1, dtype=torch.int64) * 2
    indices = torch.stack([torch.arange(M) // 2, 32 + torch.arange(M) // 2], 1).reshape(-1).int()
    A = hyb.DeviceCsr(indptr.to(cuda_device), indices.to(cuda_device), torch.ones(2 * M, device=cuda_device), (M, K))
    B = torch.ones(K, N, dtype=dtype)
    B[3, 5], B[7, 6], B[9, 7], B[41, 7] = float("inf"), float("nan"), float("inf"), float("-inf")
    y = layer.spmm_csr_act(A, B.to(cuda_device), activation="relu").float().cpu()
    want = torch.full((M, N), 2.0)
    want[6:8, 5], want[14:16, 6], want[18:20, 7] = float("inf"), float("nan"), float("nan")
    assert torch.equal(torch.nan_to_num(y, nan=-1.0), torch.nan_to_num(want, nan=-1.0))


@pytest.mark.parametrize("name", ref.ACTS)
def test_matrix_without_entries(cuda_device, name):
    M, N = 77, 40
    z64 = torch.zeros(M + 1, dtype=torch.int64, device=cuda_device)
    A = hyb.DeviceCsr(z64, torch.empty(0, dtype=torch.int32, device=cuda_device), None, (M, 9))
    g = gen(0)
    bias = torch.randn(N, generator=g)
    R, Rv = rows_of((M, N), F32, g, cuda_device)
    B = torch.full((9, N), float("nan"), device=cuda_device)
    got = layer.spmm_csr_act(A, B, bias=bias.to(cuda_device), activation=name, residual=R)
    _, y, _, off = ref.product(torch.zeros(M, 9, dtype=torch.float64), torch.zeros(9, N, dtype=torch.float64), bias, name, Rv, F32)
    ref.close(got, y, off)


def test_row_range_and_slices(cuda_device):
    g = gen(2)
    M, K, N = 200, 90, 64
    p = pattern(M, K, 3, 12.0, 90)
    A = csr_on(cuda_device, p, (M, K))
    B, _, Bv = features(K, N, BF16, g, cuda_device)
    full = ref.product(ref.dense(*p, (M, K)), Bv, None, "silu", None, BF16)
    for r0, r1 in ((0, 200), (0, 1), (99, 101), (150, 200), (30, 30), (199, 200)):
        got = layer.spmm_csr_act(A, B, activation="silu", row_range=(r0, r1))
        ref.close(got, full[1][r0:r1], full[3][r0:r1], f"rows {r0} to {r1}")
        e0, e1 = int(p[0][r0]), int(p[0][r1])
        part = hyb.DeviceCsr(A.indptr[r0:r1 + 1].clone() - e0, A.indices[e0:e1].clone(), A.data[e0:e1].clone(), (r1 - r0, K))
        ref.close(layer.spmm_csr_act(part, B, activation="silu"), full[1][r0:r1], full[3][r0:r1])


def test_far_rows_of_b(cuda_device):
    """Offsets beyond 32 bits, in elements and in bytes."""
    K, N = (1 << 22) + 5, 1040
    B = torch.empty((K, N), dtype=E4M3, device=cuda_device)
    scale = torch.ones(K, device=cuda_device)
    cols = torch.tensor([0, 1, (1 << 21) + 3, K - 2, K - 1])
    g = gen(5)
    v = torch.randn(5, N, generator=g).to(E4M3)
    B.view(torch.uint8)[cols.to(cuda_device)] = v.view(torch.uint8).to(cuda_device)
    A = hyb.DeviceCsr(torch.tensor([0, 5, 5, 6], device=cuda_device), torch.cat([cols, cols[4:]]).int().to(cuda_device),
                      torch.ones(6, device=cuda_device), (3, K))
    got = layer.spmm_csr_act(A, B, scale=scale, out_dtype=F32)
    want = torch.stack([v.double().sum(0), torch.zeros(N, dtype=torch.float64), v[4].double()])
    ref.close(got, want, 8 * U32 * torch.stack([v.double().abs().sum(0)] * 3))


@pytest.mark.parametrize("shape,N,seed", [((60, 31), 40, 1), ((31, 900), 33, 2), ((900, 31), 64, 3), ((1, 400), 16, 4), ((400, 1), 17, 5)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("ones", [False, True])
def test_product_with_the_transposed_pattern(cuda_device, shape, N, seed, dtype, ones):
    g = gen(seed)
    p = pattern(*shape, seed, 8.0, 700)
    A = csr_on(cuda_device, p, shape)
    T = layer.CsrTranspose.of(A)
    B, _, Bv = features(shape[0], N, dtype, g, cuda_device)
    got = layer.spmm_csr_act(T, B, values=None if ones else A.data, out_dtype=F32)
    a = ref.dense(p[0], p[1], None if ones else p[2], shape).t().contiguous()
    _, y, _, off = ref.product(a, Bv, None, "none", None, F32)
    ref.close(got, y, off)


def test_product_refusals(cuda_device):
    p = pattern(20, 30, 1)
    A = csr_on(cuda_device, p, (20, 30))
    B = torch.randn(30, 16, device=cuda_device)
    q = B.to(E4M3)
    one = torch.ones(30, device=cuda_device)
    bad_values = hyb.DeviceCsr(A.indptr, A.indices, A.data[:-1], (20, 30))
    half = hyb.DeviceCsr(A.indptr, A.indices, A.data.half(), (20, 30))
    call = layer.spmm_csr_act
    for f in (lambda: call(A, B[:29]), lambda: call(A, q), lambda: call(A, q, scale=one[:29]), lambda: call(A, B, activation="tanh"),
              lambda: call(A, B, bias=one[:15]), lambda: call(A, B, bias=one[:16].double()), lambda: call(A, B, residual=B),
              lambda: call(A, B, out=torch.empty(20, 15, device=cuda_device)), lambda: call(A, B, out_dtype=E4M3),
              lambda: call(A, B, preact=torch.empty(20, 16, dtype=BF16, device=cuda_device)), lambda: call(A, B.t()),
              lambda: call(A, B.cpu()), lambda: call(A, B, bias=one[:16].cpu()), lambda: call(A, B, row_range=(3, 21)),
              lambda: call(A, B, values=A.data), lambda: call(bad_values, B), lambda: call(half, B), lambda: call(A, B.double()),
              lambda: call(A, B[:1].expand(30, 16)), lambda: layer.spmm_csr_act_backward(A, None, B, B[:20]),
              lambda: layer.spmm_csr_act_backward(A, None, B, B[:20], need=("dX",)),
              lambda: layer.spmm_csr_act_backward(A, None, q, B[:20], need=("dvalues",)),
              lambda: layer.spmm_csr_grad_values(A, B, B[:19]), lambda: layer.spmm_csr_grad_values(A, B, B[:20], activation="relu"),
              lambda: layer.act_backward(B, activation="relu"), lambda: layer.act_backward(B, B.half(), "relu"),
              lambda: layer.act_backward(B, need_dz=False, need_dbias=False)):
        with pytest.raises(ValueError):
            f()


# ---- gradients --------------------------------------------------------------------------------------
def gradients64(A, Bv, dyv, zv, name, dz_dtype):
    """dB, dvalues (dense), dbias and bounds; dz is rounded to `dz_dtype` for dB."""
    s = ref.slope(zv, name) if name != "none" else torch.ones_like(zv)
    dz = dyv * s
    soff = ref.SLOPE_ERROR * (1 + zv.abs()) if name not in ("none", "relu") else torch.zeros_like(zv)
    dzoff = dyv.abs() * soff + 2 * U32 * dz.abs()
    if name == "none":
        rz = dzoff * 0                                      # dy itself
    else:
        rz = ref.rounded(dz, dzoff, dz_dtype)
    M = A.shape[0]
    n = (A != 0).sum(0).double()[:, None]
    dB = A.t() @ dz
    dBoff = A.abs().t() @ rz + (n + 3) * U32 * (A.abs().t() @ (dz.abs() + rz))
    dv, N = dz @ Bv.t(), Bv.shape[1]
    dvoff = dzoff @ Bv.abs().t() + (N + 3) * U32 * ((dz.abs() + dzoff) @ Bv.abs().t())
    db = dz.sum(0)
    return dz, rz, dB, dBoff, dv, dvoff, db, dzoff.sum(0) + (M + 2) * U32 * (dz.abs() + dzoff).sum(0)


@pytest.mark.parametrize("M,K,N,mean,longest", [(1, 1, 1, 1, 0), (1, 60, 64, 20, 60), (40, 30, 8, 3, 0), (100, 80, 47, 6, 0),
                                                (90, 600, 128, 10, 600), (50, 40, 300, 6, 0), (600, 30, 32, 8, 0), (33, 2000, 256, 9, 2000),
                                                (130, 90, 1030, 5, 0), (2000, 40, 16, 5, 0)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_gradients(cuda_device, M, K, N, mean, longest, dtype):
    g = gen(M * 3 + N)
    p = pattern(M, K, M + K, mean, longest)
    A = csr_on(cuda_device, p, (M, K))
    T = layer.CsrTranspose.of(A)
    B, _, Bv = features(K, N, dtype, g, cuda_device)
    dy, dyv = rows_of((M, N), dtype, g, cuda_device)
    z, zv = rows_of((M, N), dtype, g, cuda_device)
    a = ref.dense(*p, (M, K))
    for name in ref.ACTS:
        got = layer.spmm_csr_act_backward(A, T, B, dy, preact=z, activation=name)
        dz, rz, dB, dBoff, dv, dvoff, db, dboff = gradients64(a, Bv, dyv, zv, name, dtype)
        ref.close(got.dB, dB, ref.rounded(dB, dBoff, dtype), name + " dB")
        rows = torch.repeat_interleave(torch.arange(M), torch.diff(p[0]))
        ref.close(got.dvalues, dv[rows, p[1].long()], dvoff[rows, p[1].long()] + ref.TINY[F32], name + " dvalues")
        ref.close(got.dbias, db, dboff + ref.TINY[F32], name + " dbias")
        own, _ = layer.act_backward(dy, z, name, need_dbias=False)
        ref.close(own, dz, ref.rounded(dz, rz, dtype), name + " dz")
        again = layer.spmm_csr_act_backward(A, T, B, dy, preact=z, activation=name)
        assert all(torch.equal(x, y) for x, y in zip(got, again)), "the same call gives the same bits"


@pytest.mark.parametrize("N,pitch,shift", [(64, 64, 1), (64, 72, 8), (31, 33, 2), (128, 131, 7), (17, 48, 0), (260, 264, 0)])
@pytest.mark.parametrize("dtype,dyt", [(F32, F32), (BF16, BF16), (F16, F32), (F32, BF16)])
def test_gradient_strides_and_mixed_types(cuda_device, N, pitch, shift, dtype, dyt):
    g = gen(N)
    M, K = 120, 80
    p = pattern(M, K, 8, 9.0, 80)
    A = csr_on(cuda_device, p, (M, K))
    B, _, Bv = features(K, N, dtype, g, cuda_device, pitch, shift)
    dy, dyv = rows_of((M, N), dyt, g, cuda_device, pitch + 1, shift)
    z, zv = rows_of((M, N), dyt, g, cuda_device, pitch, 0)
    got = layer.spmm_csr_act_backward(A, layer.CsrTranspose.of(A), B, dy, preact=z, activation="silu")
    _, _, dB, dBoff, dv, dvoff, db, dboff = gradients64(ref.dense(*p, (M, K)), Bv, dyv, zv, "silu", dyt)
    rows = torch.repeat_interleave(torch.arange(M), torch.diff(p[0]))
    assert got.dB.dtype == dtype
    ref.close(got.dB, dB, ref.rounded(dB, dBoff, dtype), "dB")
    ref.close(got.dvalues, dv[rows, p[1].long()], dvoff[rows, p[1].long()] + ref.TINY[F32], "dvalues")
    ref.close(got.dbias, db, dboff + ref.TINY[F32], "dbias")


def test_slopes_far_out(cuda_device):
    """No NaN where the slope is plainly 0 or 1."""
    z = torch.tensor([[-float("inf"), -1e38, -1e20, -200.0, 200.0, 1e20, 1e38, float("inf")]], device=cuda_device)
    one = torch.ones_like(z)
    want = torch.tensor([[0.0, 0, 0, 0, 1, 1, 1, 1]])
    for name in ref.ACTS[1:]:
        assert torch.equal(layer.act_backward(one, z, name, need_dbias=False)[0].cpu() + 0.0, want), name
    nan = torch.full((1, 8), float("nan"), device=cuda_device)
    for name in ("silu", "gelu", "gelu_tanh"):
        assert bool(torch.isnan(layer.act_backward(one, nan, name, need_dbias=False)[0]).all())


def test_gradient_by_differences(cuda_device):
    """Of the whole layer, norm included, along random directions, against central differences in 64 bits."""
    g = gen(11)
    M, K, N, eps = 30, 25, 24, 1e-5
    indptr, indices, vals = pattern(M, K, 7)
    r64 = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).float().double()
    x, w, b, dy, v = r64(K, N), r64(N), r64(N), r64(M, N), vals.double()

    def f(x, w, b, v):
        n = x * (x.square().mean(1, keepdim=True) + eps).rsqrt() * w
        return float((dy * ref.act(ref.dense(indptr, indices, v, (M, K)) @ n + b, "gelu")).sum())

    A = csr_on(cuda_device, (indptr, indices, vals), (M, K))
    dev = lambda t: t.float().to(cuda_device)
    n = layer.rms_norm(dev(x), dev(w), eps=eps)
    z = torch.empty(M, N, device=cuda_device)
    layer.spmm_csr_act(A, n.y, bias=dev(b), activation="gelu", preact=z)
    got = layer.spmm_csr_act_backward(A, layer.CsrTranspose.of(A), n.y, dev(dy), preact=z, activation="gelu")
    dx, dw = layer.rms_norm_backward(got.dB, n.h, dev(w), n.rstd)
    d = 1e-5
    args = [x, w, b, v]
    for i, grad in enumerate((dx, dw, got.dbias, got.dvalues)):
        u = torch.randn(args[i].shape, generator=g, dtype=torch.float64)
        hi, lo = ([a + s * d * u if j == i else a for j, a in enumerate(args)] for s in (1, -1))
        diff = (f(*hi) - f(*lo)) / (2 * d)
        # some thousand terms of size about 1, each known to about 100 roundings; differences of third order: d^2 ~ 1e-10
        assert abs(float((grad.cpu().double() * u).sum()) - diff) < 4000 * 100 * U32 + 1e-5, i


# ---- together, as they are used ---------------------------------------------------------------------
@pytest.mark.parametrize("N", [64, 40])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_two_layers_in_8_bits(cuda_device, N, dtype):
    """norm to 8 bits, product, activation, residual, twice; each step against the 64-bit step on its own inputs."""
    g = gen(N)
    M = 500
    p = pattern(M, M, 6, 9.0, 400)
    A, a = csr_on(cuda_device, p, (M, M)), ref.dense(*p, (M, M))
    x, _ = rows_of((M, N), dtype, g, cuda_device)
    r, _ = rows_of((M, N), dtype, g, cuda_device)
    for step in range(2):
        w = (1 + 0.1 * torch.randn(N, generator=g)).to(dtype).to(cuda_device)
        b = torch.randn(N, generator=g).to(dtype).to(cuda_device)
        n = layer.rms_norm(x, w, residual=r, out_dtype=E4M3)
        check_norm(x, r, w, 1e-6, n, x.cpu().double(), r.cpu().double(), w.cpu().double())
        y = layer.spmm_csr_act(A, n.y, scale=n.scale, bias=b, activation="silu", out_dtype=dtype)
        _, want, _, off = ref.product(a, n.y.cpu().double() * n.scale.cpu().double()[:, None], b.cpu(), "silu", None, dtype)
        ref.close(y, want, off)
        x, r = y, n.h


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_calls_on_two_streams_and_in_a_graph(cuda_device, dtype):
    g = gen(8)
    M, K, N = 300, 250, 96
    p = pattern(M, K, 9, 12.0, 250)
    A = csr_on(cuda_device, p, (M, K))
    T = layer.CsrTranspose.of(A)
    mats = [[rows_of(s, dtype, g, cuda_device)[0] for s in ((K, N), (M, N), (K, N))] for _ in range(2)]
    w = torch.ones(N, device=cuda_device)

    def step(x, dy, dh):
        n = layer.rms_norm(x, w)
        z = torch.empty_like(dy)
        y = layer.spmm_csr_act(A, n.y, activation="gelu", residual=dy, preact=z)
        gr = layer.spmm_csr_act_backward(A, T, n.y, dy, preact=z, activation="gelu")
        dx, dw = layer.rms_norm_backward(gr.dB, n.h, w, n.rstd, dh=dh)
        return y, gr.dvalues, gr.dbias, dx, dw

    want = [step(*m) for m in mats]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in mats]
    for _ in range(3):
        got = []
        for s, m in zip(streams, mats):
            with torch.cuda.stream(s):
                got.append(step(*m))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    graph = torch.cuda.CUDAGraph()
    held = [t.clone() for t in mats[0]]
    with torch.cuda.graph(graph):
        out = step(*held)
    for i in (1, 0, 1):
        for t, m in zip(held, mats[i]):
            t.copy_(m)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(want[i], out))


def test_workspace_is_reused(cuda_device):
    g = gen(8)
    M, K, N = 300, 2500, 96
    p = pattern(M, K, 9, 12.0, 2500)
    A = csr_on(cuda_device, p, (M, K))
    B = torch.randn(K, N, generator=g).to(cuda_device)
    ws = hyb.Workspace(cuda_device)
    want = layer.spmm_csr_act(A, B)
    for _ in range(2):
        assert torch.equal(layer.spmm_csr_act(A, B, workspace=ws), want)
        dz, db = layer.act_backward(want, want, "silu", workspace=ws)
        assert torch.equal(db, layer.act_backward(want, want, "silu")[1])


def test_workspace_of_another_device_or_too_small(cuda_device):
    class Small(hyb.Workspace):
        def get(self, nbytes, slot=0):
            return super().get(nbytes, slot)[:nbytes - 16]

    p = pattern(20, 30, 1)
    A = csr_on(cuda_device, p, (20, 30))
    B = torch.randn(30, 16, device=cuda_device)
    with pytest.raises(ValueError):
        layer.spmm_csr_act(A, B, workspace=hyb.Workspace("cpu"))
    with pytest.raises(_cabi.LiteformError):
        layer.spmm_csr_act(A, B, workspace=Small(cuda_device))
    with pytest.raises(_cabi.LiteformError):
        layer.act_backward(B, workspace=Small(cuda_device))


# ---- graphs large enough for every length of range, rows of many pieces, runs of empty rows ----------
def big_pattern(M, K, entries, hubs, hub_len, used, seed, dev):
    """CSR arrays on the device: `used` of the rows hold entries, `hubs` of them `hub_len`."""
    g = torch.Generator(device=dev).manual_seed(seed)
    where = torch.randperm(M, generator=g, device=dev)[:used]
    r = where[torch.randint(0, used, (entries,), generator=g, device=dev)]
    r = torch.cat([r] + [torch.full((hub_len,), int(h), device=dev) for h in where[:hubs]])
    c = torch.randint(0, K, (r.numel(),), generator=g, device=dev)
    keys = torch.unique(r * K + c)
    rows = torch.div(keys, K, rounding_mode="floor")
    indptr = torch.zeros(M + 1, dtype=torch.int64, device=dev)
    torch.cumsum(torch.bincount(rows, minlength=M), 0, out=indptr[1:])
    vals = torch.rand(keys.numel(), generator=g, device=dev) * 2 - 1
    return rows, hyb.DeviceCsr(indptr, (keys - rows * K).int(), vals, (M, K))


@pytest.mark.parametrize("M,K,entries,hubs,hub_len,used,N", [
    (1 << 18, 1 << 17, 6_000_000, 3, 60_000, 1 << 18, 24),        # ranges of 1024 entries
    (50_000, 90_000, 1_000_000, 20, 5000, 50_000, 40),            # 256
    (300_000, 2000, 100, 0, 0, 60, 16),                           # nearly all rows empty
    (3, 2_000_000, 10, 3, 900_000, 3, 8),                         # three rows of nearly a million entries
    (200_000, 64, 30_000, 2, 60, 5, 33)])
@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, BF16), (E4M3, F16)])
def test_large_graphs(cuda_device, M, K, entries, hubs, hub_len, used, N, dtype, out):
    rows, A = big_pattern(M, K, entries, hubs, hub_len, used, M, cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(N)
    B = torch.randn((K, N), generator=g, device=cuda_device).to(dtype)
    scale = torch.rand(K, generator=g, device=cuda_device) + 0.1 if dtype == E4M3 else None
    Bv = B.double() * (1 if scale is None else scale.double()[:, None])
    R = torch.randn((M, N), generator=g, device=cuda_device).to(out)
    got = layer.spmm_csr_act(A, B, scale=scale, activation="relu", residual=R)  if dtype != E4M3 else \
        layer.spmm_csr_act(A, B, scale=scale, activation="relu", residual=R, out_dtype=out)
    full = lambda v, X: torch.sparse_csr_tensor(A.indptr, A.indices.long(), v, size=(M, K)) @ X
    z, size = full(A.data.double(), Bv), full(A.data.double().abs(), Bv.abs())
    n = torch.diff(A.indptr).double()[:, None]
    y = z.clamp(min=0) + R.double()
    off = (n + 3) * U32 * 1.01 * size + U32 * y.abs()
    ref.close(got, y.cpu(), ref.rounded(y, off, out).cpu())
    if dtype == E4M3:
        return
    dy = torch.randn((M, N), generator=g, device=cuda_device).to(dtype)
    dv = layer.spmm_csr_grad_values(A, B, dy)
    at = torch.randint(0, A.nnz, (min(A.nnz, 200_000),), generator=g, device=cuda_device)
    prod = dy[rows[at]].double() * Bv[A.indices[at].long()]
    ref.close(dv[at], prod.sum(1).cpu(), ((N + 3) * U32 * prod.abs().sum(1)).cpu(), "dvalues")
    T = layer.CsrTranspose.of(A)
    dB = layer.spmm_csr_act(T, dy, values=A.data, out_dtype=F32)
    tr = lambda v, X: torch.sparse_csr_tensor(T.indptr, T.indices.long(), v[T.order.long()], size=(K, M)) @ X
    want, size = tr(A.data.double(), dy.double()), tr(A.data.double().abs(), dy.double().abs())
    n = torch.diff(T.indptr).double()[:, None]
    ref.close(dB, want.cpu(), ((n + 3) * U32 * 1.01 * size + ref.TINY[F32]).cpu(), "dB")


def test_values_of_other_numbers_than_the_matrix_has(cuda_device):
    """nnz bounds what is read: a matrix whose row pointers promise more entries than there are stays inside them."""
    indptr = torch.tensor([0, 4, 9, 40], device=cuda_device)
    A = hyb.DeviceCsr(indptr, torch.arange(12, dtype=torch.int32, device=cuda_device), torch.ones(12, device=cuda_device), (3, 64))
    B = torch.ones(64, 16, device=cuda_device)
    y = layer.spmm_csr_act(A, B)
    assert torch.equal(y[:, 0].cpu(), torch.tensor([4.0, 5.0, 3.0]))


def test_infer(cuda_device):
    """The pipeline's layers against the same steps, each from its own inputs, in 64 bits."""
    from liteform_ae_b200 import pipeline, synth
    from liteform_ae_b200.format_matrix_market import MTX
    c = synth.zipf_rows(M=2048, seed=5)
    m = MTX.from_csr(c.indptr, c.indices, c.data, c.shape, "t")
    g, N = gen(3), 48
    x = torch.randn(2048, N, generator=g).bfloat16().to(cuda_device)
    layers = [dict(norm=(1 + 0.1 * torch.randn(N, generator=g)).to(cuda_device), bias=torch.randn(N, generator=g).to(cuda_device),
                   activation="silu"), dict(norm=torch.ones(N, device=cuda_device), activation="gelu"),
              dict(norm=torch.ones(N, device=cuda_device))]
    A = m.csr_device(cuda_device)
    for bits in (True, False):
        got = pipeline.infer(m, x, layers, eight_bits=bits)
        h, y = x, None
        for i, p in enumerate(layers):
            n = layer.rms_norm(h if y is None else y, p["norm"], residual=None if y is None else h, out_dtype=E4M3 if bits else BF16)
            check_norm(h if y is None else y, None if y is None else h, None, 1e-6, n, (h if y is None else y).cpu().double(),
                       None if y is None else h.cpu().double(), p["norm"].cpu().double())
            f = n.y.cpu().double() * (n.scale.cpu().double()[:, None] if bits else 1)
            a = ref.dense(A.indptr.cpu(), A.indices.cpu(), A.data.cpu(), A.shape)
            h = n.h
            _, want, _, off = ref.product(a, f, None if p.get("bias") is None else p["bias"].cpu(), p.get("activation") or "none",
                                          h.cpu() if i == 2 else None, BF16)
            y = layer.spmm_csr_act(A, n.y, scale=n.scale, bias=p.get("bias"), activation=p.get("activation"),
                                   residual=h if i == 2 else None, out_dtype=BF16)
            ref.close(y, want, off)
        assert torch.equal(got, y)
    with pytest.raises(ValueError):
        pipeline.infer(m, x, [])


def test_pattern_types_are_checked(cuda_device):
    p = pattern(20, 30, 1)
    A = csr_on(cuda_device, p, (20, 30))
    T = layer.CsrTranspose.of(A)
    B, Bt = torch.randn(30, 16, device=cuda_device), torch.randn(20, 16, device=cuda_device)
    with_order = lambda order: layer.CsrTranspose(T.indptr, T.indices, order, T.shape)
    for f in (lambda: layer.spmm_csr_act(hyb.DeviceCsr(A.indptr.int(), A.indices, A.data, A.shape), B),
              lambda: layer.spmm_csr_act(hyb.DeviceCsr(A.indptr, A.indices.long(), A.data, A.shape), B),
              lambda: layer.spmm_csr_grad_values(hyb.DeviceCsr(A.indptr, A.indices.long(), A.data, A.shape), B, Bt),
              lambda: layer.spmm_csr_act(with_order(T.order.long()), Bt, values=A.data),
              lambda: layer.spmm_csr_act(with_order(T.order[:-1]), Bt, values=A.data),
              lambda: layer.spmm_csr_act(with_order(T.order.cpu()), Bt, values=A.data)):
        with pytest.raises(ValueError):
            f()


def test_value_gradient_of_a_slice(cuda_device):
    p = pattern(40, 30, 2)
    A = csr_on(cuda_device, p, (40, 30))
    B, dy = torch.randn(30, 16, device=cuda_device), torch.randn(40, 16, device=cuda_device)
    full = layer.spmm_csr_grad_values(A, B, dy)
    r0, r1 = 11, 29
    e0, e1 = int(A.indptr[r0]), int(A.indptr[r1])
    out = torch.full((A.nnz,), 7.0, device=cuda_device)
    layer.spmm_csr_grad_values(hyb.DeviceCsr(A.indptr[r0:r1 + 1], A.indices, A.data, (r1 - r0, 30)), B, dy[r0:r1], out=out)
    # the same products, perhaps added up in another order: 16 terms, each sum rounded
    off = 16 * 2.0 ** -24 * (dy.abs().amax() * B.abs().amax()) * 16
    assert (out[:e1 - e0] - full[e0:e1]).abs().max() <= off and (out[e1 - e0:] == 7.0).all()


@pytest.mark.parametrize("N", [16, 40, 47])
@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, BF16), (E4M3, BF16), (E4M3, F32)])
def test_mostly_empty_rows(cuda_device, N, dtype, out):
    M, K = 20000, 300
    g = gen(N)
    p = pattern(M, K, N, 0.003, 200, empty=0.0)
    assert 200 < len(p[1]) < 400
    A = csr_on(cuda_device, p, (M, K))
    B, scale, Bv = features(K, N, dtype, g, cuda_device)
    R, Rv = rows_of((M, N), out, g, cuda_device)
    _, y, _, yoff = ref.product(ref.dense(*p, (M, K)), Bv, None, "silu", Rv, out)
    ref.close(layer.spmm_csr_act(A, B, scale=scale, activation="silu", residual=R, out_dtype=out), y, yoff, "y")
    if dtype == E4M3:
        return
    dy, dyv = rows_of((M, N), out, g, cuda_device)
    rows = torch.repeat_interleave(torch.arange(M), torch.diff(p[0]))
    terms = dyv[rows] * Bv[p[1].long()]
    # N products, each rounded, and their sums: N units of the magnitudes' sum cover both
    off = (N + 1) * 2.0 ** -24 * terms.abs().sum(1)
    ref.close(layer.spmm_csr_grad_values(A, B, dy), terms.sum(1), off, "dvalues")


@pytest.mark.parametrize("M,N,pitch", [(8000, 128, 128), (3000, 47, 47), (700, 1000, 1000), (200, 300, 301), (60, 4096, 4096), (40, 9000, 9001)])
@pytest.mark.parametrize("residual", [False, True])
def test_eight_bit_rows_are_rounded_to_nearest(cuda_device, M, N, pitch, residual):
    """Stored is 448 h w / max|h w| to the nearest value, halves to the even one.  For bfloat16 h and w both products are
    exact in 64 bits; a quotient that is a half is one there too (it has five bits), and any other is at least 2^-22 of itself
    away from one: its two integers have 16 and 19 bits.  So the 64-bit quotient, through float32, rounds as the true one."""
    g = gen(N)
    x, xv = rows_of((M, N), BF16, g, cuda_device, pitch)
    r, rv = rows_of((M, N), BF16, g, cuda_device, pitch) if residual else (None, None)
    w = (1 + 0.1 * torch.randn(N, generator=g)).to(BF16).to(cuda_device)
    n = layer.rms_norm(x, w, residual=r, out_dtype=E4M3)
    p = n.h.cpu().double() * w.cpu().double()
    want = (448 * p / p.abs().amax(1, keepdim=True)).float().to(E4M3).float()
    got = n.y.cpu().float()
    assert int((got != want).sum()) == 0


def test_eight_bit_rows_of_tiny_numbers(cuda_device):
    """A reciprocal of max|h w| would overflow; y itself is an ordinary number, since eps is smaller still."""
    x = torch.randn(5, 64, generator=gen(1)) * torch.tensor([[1e-19], [1e-30], [1e-36], [1e-38], [0.0]])
    w = torch.full((64,), 1e-9)
    n = layer.rms_norm(x.to(cuda_device), w.to(cuda_device), eps=1e-37, out_dtype=E4M3)
    y = x.double() * (x.double().square().mean(1, keepdim=True) + 1e-37) ** -0.5 * w.double()
    y = torch.where(y.abs().amax(1, keepdim=True) < 448 * 2.0 ** -126, torch.zeros_like(y), y)
    s = n.scale.cpu().double()[:, None]
    back = n.y.cpu().double() * s
    # half a step of 2^-4, 2^-10 of the scale below the normal numbers; h w itself is a subnormal number in the later rows, known to
    # 2^-150 * rstd (below 2^-88 here); eps in 32 bits and the square's sum: 2^-20
    off = 2.0 ** -4 * y.abs() * 1.01 + 2.0 ** -10 * s + 2.0 ** -88 + 2.0 ** -20 * y.abs()
    assert bool(((back - y).abs() <= off).all()) and bool((back[4] == 0).all())


def test_outputs_in_the_memory_of_inputs_are_refused(cuda_device):
    M = N = 32
    p = pattern(M, M, 1)
    A = csr_on(cuda_device, p, (M, M))
    T = layer.CsrTranspose.of(A)
    wide = torch.randn(M + 8, 3 * N, device=cuda_device)
    B, side, w = wide[:M, :N], wide[:M, N:2 * N], torch.ones(N, device=cuda_device)
    v = torch.ones(M, device=cuda_device)
    for f in (lambda: layer.spmm_csr_act(A, B, out=wide[5:25, :N], row_range=(5, 25)),      # rows of B that other rows read
              lambda: layer.spmm_csr_act(A, B, out=wide[8:, :N]), lambda: layer.spmm_csr_act(A, B, preact=wide[:M, N - 1:2 * N - 1]),
              lambda: layer.spmm_csr_act(A, B, out=side, preact=side), lambda: layer.spmm_csr_act(A, B, out=side, preact=wide[1:M + 1, N:2 * N]),
              lambda: layer.spmm_csr_act(A, B, out=side, residual=wide[1:M + 1, N:2 * N]),
              lambda: layer.spmm_csr_act(A, B, preact=side, residual=wide[1:M + 1, N:2 * N]),
              lambda: layer.spmm_csr_act(T, B, values=A.data, out=B), lambda: layer.rms_norm(B, w, out=wide[1:M + 1, :N]),
              lambda: layer.rms_norm(B, w, residual=side, sum_out=side, out=side),
              lambda: layer.rms_norm(B, w, residual=side, sum_out=wide[2:M + 2, :N]), lambda: layer.rms_norm(B, v, rstd=v),
              lambda: layer.rms_norm(B, w, out_dtype=E4M3, scale=v, rstd=v), lambda: layer.rms_norm_backward(B, side, w, v, dx=wide[3:M + 3, :N]),
              lambda: layer.rms_norm_backward(B, side, w, v, dweight=v), lambda: layer.act_backward(B, side, "silu", dz=wide[1:M + 1, :N]),
              lambda: layer.act_backward(B, side, "silu", dbias=wide[0, :N]),
              lambda: layer.spmm_csr_grad_values(A, B, side, out=wide.view(-1)[:A.nnz])):
        with pytest.raises(ValueError, match="lies in the memory of"):
            f()


def test_outputs_beside_or_in_place_of_inputs(cuda_device):
    """Column slices of one buffer, and the inputs that an output may be, give what separate outputs give."""
    g = gen(3)
    for N in (32, 33):
        M = 70
        A = csr_on(cuda_device, pattern(M, M, 1, 8.0, 70), (M, M))
        for dtype in (F32, BF16):
            wide = torch.randn(M, 3 * N, generator=g).to(dtype).to(cuda_device)
            B, C, R = (wide[:, i * N:(i + 1) * N] for i in range(3))
            same = lambda x, y: torch.equal(x, y)
            want = layer.spmm_csr_act(A, B, activation="gelu", residual=R)
            assert same(layer.spmm_csr_act(A, B, activation="gelu", residual=R, out=C), want)
            pre = torch.empty(M, N, dtype=dtype, device=cuda_device)
            layer.spmm_csr_act(A, B, activation="gelu", preact=pre)
            res = R.clone()
            assert same(layer.spmm_csr_act(A, B, activation="gelu", residual=res, preact=res), want) and same(res, pre)
            w = torch.randn(N, generator=g).to(cuda_device)
            n = layer.rms_norm(B, w, residual=R)
            for i in range(2):
                x, r = B.clone(), R.clone()
                assert same(layer.rms_norm(x, w, residual=r, out=(x, r)[i]).y, n.y)
                x, r = B.clone(), R.clone()
                m = layer.rms_norm(x, w, residual=r, sum_out=(x, r)[i], out=(x, r)[1 - i])
                assert same(m.y, n.y) and same(m.h, n.h)
            want = layer.act_backward(B, R, "silu")
            for i in range(2):
                x, r = B.clone(), R.clone()
                assert all(same(*p) for p in zip(layer.act_backward(x, r, "silu", dz=(x, r)[i]), want))
            want = layer.rms_norm_backward(B, R, w, n.rstd, dh=C)
            for i in range(3):
                x, r, c = B.clone(), R.clone(), C.clone()
                assert all(same(*p) for p in zip(layer.rms_norm_backward(x, r, w, n.rstd, dh=c, dx=(x, r, c)[i]), want))


@pytest.mark.parametrize("name", ref.ACTS)
@pytest.mark.parametrize("N", [16, 21])
def test_gradient_of_float16_beyond_its_range(cuda_device, name, N):
    """dz beyond 65504, and below the smallest float16, where dB is an ordinary number: A's values bring it back."""
    g = gen(N)
    M, K = 64, 48
    indptr, indices, vals = pattern(M, K, 6, 8.0)
    dyv = torch.randn(M, N, generator=g)
    dyv[::2] = torch.sign(dyv[::2]) * 65000.0
    dyv[1::2] *= 2.0 ** -24
    vals *= torch.repeat_interleave(torch.tensor([2.0 ** -18, 2.0 ** 20]).repeat(M // 2), torch.diff(indptr))
    zv = (1.5 + torch.rand(M, N, generator=g)).half().double()      # where the slopes of silu and gelu are above 1
    zv[1::2] -= 5
    A = csr_on(cuda_device, (indptr, indices, vals), (M, K))
    B, _, Bv = features(K, N, F16, g, cuda_device)
    dy, z = dyv.half().to(cuda_device), zv.half().to(cuda_device)
    got = layer.spmm_csr_act_backward(A, layer.CsrTranspose.of(A), B, dy, preact=z, activation=name)
    dz_dtype = F16 if name in ("none", "relu") else F32
    _, _, dB, dBoff, _, _, db, dboff = gradients64(ref.dense(indptr, indices, vals, (M, K)), Bv, dyv.half().double(), zv, name, dz_dtype)
    assert float(dB.abs().max()) < 6e4
    ref.close(got.dB, dB, ref.rounded(dB, dBoff, F16), name)
    ref.close(got.dbias, db, dboff + ref.TINY[F32], name)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("N,pitch,shift", [(64, 64, 0), (64, 72, 4), (31, 33, 2), (300, 300, 0)])
def test_act_backward_into_float32(cuda_device, dtype, N, pitch, shift):
    g, M = gen(N), 90
    dy, dyv = rows_of((M, N), dtype, g, cuda_device, N + 1)
    z, zv = rows_of((M, N), dtype, g, cuda_device)
    for name in ref.ACTS:
        buf = torch.full((M * pitch + shift + 8,), 3.0, device=cuda_device)
        dz = torch.as_strided(buf, (M, N), (pitch, 1), shift)
        want = dyv * (ref.slope(zv, name) if name != "none" else 1)
        off = (0 if name in ("none", "relu") else ref.SLOPE_ERROR) * (1 + zv.abs()) * dyv.abs() + 2 * U32 * want.abs()
        got, db = layer.act_backward(dy, z, name, dz=dz)
        assert got is dz
        ref.close(dz, want, off, name)
        assert torch.equal(layer.act_backward(dy, z, name, dz_dtype=F32)[0], dz) and bool((buf[:shift] == 3).all())
        assert torch.equal(layer.act_backward(dy, z, name, need_dz=False)[1], db)
    for f in (lambda: layer.act_backward(dy, z, "silu", dz_dtype=F16 if dtype == BF16 else BF16), lambda: layer.act_backward(dy, z, "silu", dz=dz, dz_dtype=dtype),
              lambda: layer.act_backward(dz, dz.clone(), "silu", dz_dtype=dtype), lambda: layer.act_backward(dy, z, "silu", dz_dtype=E4M3)):
        with pytest.raises(ValueError):
            f()


# Relative bounds of the activations, in units of U = 2^-24.  silu: expf and the reciprocal are off by a unit in the last place (2 U)
# each, 1 + p, p r and the product with z by U: 7 U; in 16 bits 2^x by 4 U, its argument by a rounded constant and product, 1.5 |u| U.
# gelu_tanh: 4 roundings in u add 4 |u| U.  gelu: the series is off by 2.9e-7 (5 U), the reciprocal's other half unit counts
# 2.6-fold, 2^x is off by 4 U, three products by 3 U: 16 U; three roundings in the exponent z^2 / 2 add 1.5 z^2 U.  Slopes add two
# terms with 3 more roundings; in 16 bits s (1 - s) is off by U of s where s is near 1.
def activation_forms(z, name, dtype):
    """(value, slope's two terms, relative bound), all accurate in the lower tail."""
    if name == "gelu":
        phi, c = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), torch.special.erfc(-z * math.sqrt(0.5)) / 2
        return z * c, (c, z * phi), (16 + 1.5 * z * z) * U32
    k0, k1 = (1.0, 0.0) if name == "silu" else (2 * math.sqrt(2 / math.pi), 0.044715)
    u = k0 * z * (1 + k1 * z * z)
    s, d = torch.special.expit(u), torch.special.expit(u) * torch.special.expit(-u)
    off = 8 + (4 * u.abs() if name == "gelu_tanh" else 0) + (0 if dtype == F32 else 2 + 1.5 * u.abs())
    return z * s, (s, z * d * k0 * (1 + 3 * k1 * z * z)), off * U32


@pytest.mark.parametrize("name", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_tails_of_the_activations(cuda_device, name, dtype):
    """For z in [-9, 9], relative to the results themselves: a tail that is lost, or known to an absolute error, fails."""
    z = torch.linspace(-9, 9, 8192).to(dtype)
    N, dev = len(z), cuda_device
    A = hyb.DeviceCsr(torch.tensor([0, 1, 1], device=dev), torch.zeros(1, dtype=torch.int32, device=dev), None, (2, 1))
    want, (s, t), off = activation_forms(z.double(), name, dtype)
    B = z[None].to(dev)
    ref.close(layer.spmm_csr_act(A, B, activation=name)[0], want, ref.rounded(want, off * want.abs(), dtype), name)
    ref.close(layer.spmm_csr_act(A, B * 0, bias=B[0], activation=name)[1], want, ref.rounded(want, off * want.abs(), dtype), name + " of a bias")
    slope, off = s + t, (off + 3 * U32) * (s + t.abs()) + (0 if dtype == F32 else U32 * t.abs() / (1 - s).clamp(min=U32))
    one = torch.ones_like(B)
    ref.close(layer.act_backward(one, B, name, need_dbias=False)[0][0], slope, ref.rounded(slope, off, dtype), name + " slope")
    unit = torch.zeros_like(B)      # one column at a time, unrounded: the slope times 1
    for i in range(0, N, 1024):
        unit.zero_()[0, i] = 1
        dv = layer.spmm_csr_grad_values(A, B * 0 + 1, torch.cat([unit, unit]), torch.cat([B, B]), name)
        ref.close(dv, slope[i:i + 1], off[i:i + 1] + ref.TINY[F32], name + " value gradient")


# ---- more rows than a launch has places for: every thread takes several, the last turn is ragged -------
# (148 * 12 blocks of 256 threads or 148 * 6 of 512 forward, 148 * 3 or 148 blocks backward, 148 * 6 for dz)
@pytest.mark.parametrize("M,N,extra", [(2000, 4096, 0), (1000, 8192, 8), (20001, 512, 0), (120001, 32, 8), (60001, 47, 1), (30001, 96, 5),
                                       (1900, 1030, 0), (1001, 4097, 1), (2111, 264, 8)])
@pytest.mark.parametrize("dtype,out", [(BF16, E4M3), (F32, F32)])
@pytest.mark.parametrize("form", ["x", "x + r", "into x", "into r"])
def test_norm_of_many_rows(cuda_device, M, N, extra, dtype, out, form):
    g = gen(N)
    x, xv = rows_of((M, N), dtype, g, cuda_device, N + extra)
    r, rv = (None, None) if form == "x" else rows_of((M, N), dtype, g, cuda_device, N + extra)
    w = (1 + 0.1 * torch.randn(N, generator=g)).to(dtype).to(cuda_device)
    n = layer.rms_norm(x, w, residual=r, eps=1e-5, out_dtype=out, sum_out={"into x": x, "into r": r}.get(form))
    check_norm(x, r, w, 1e-5, n, xv, rv, w.cpu().double())


@pytest.mark.parametrize("M,N,extra", [(5000, 512, 0), (1000, 4096, 8), (1000, 20001, 0), (40001, 64, 8), (9000, 47, 1), (700, 8192, 0), (3001, 1030, 2),
                                       (2000, 264, 0), (500, 2056, 0)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("form", ["plain", "dh", "in place"])
def test_norm_backward_of_many_rows(cuda_device, M, N, extra, dtype, form):
    g = gen(M + N)
    dy, dyv = rows_of((M, N), dtype, g, cuda_device, N + extra)
    h, hv = rows_of((M, N), dtype, g, cuda_device, N + extra)
    dh, dhv = (None, None) if form == "plain" else rows_of((M, N), dtype, g, cuda_device, N + extra)
    w = (1 + 0.1 * torch.randn(N, generator=g)).to(dtype).to(cuda_device)
    rstd = (hv.square().mean(1) + 1e-6).rsqrt().float().to(cuda_device)
    dx, dw = layer.rms_norm_backward(dy, h, w, rstd, dh=dh, dx=dy if form == "in place" else None)
    want, off, dwv, dwoff = norm_grad64(dyv, hv, w.cpu().double(), rstd.cpu().double(), dhv)
    ref.close(dx, want, ref.rounded(want, off, dtype), "dx")
    ref.close(dw, dwv, dwoff + ref.TINY[F32], "dw")


@pytest.mark.parametrize("M,N,extra", [(3000, 1030, 0), (100_000, 16, 0), (100_001, 17, 2), (40_000, 64, 8), (1500, 5000, 0)])
@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("name", ["none", "silu", "gelu"])
def test_act_backward_of_many_rows(cuda_device, M, N, extra, dtype, out, name):
    g = gen(M)
    dy, dyv = rows_of((M, N), dtype, g, cuda_device, N + extra)
    z, zv = rows_of((M, N), dtype, g, cuda_device, N)
    s = ref.slope(zv, name) if name != "none" else torch.ones_like(zv)
    want = dyv * s
    off = (ref.SLOPE_ERROR * (1 + zv.abs()) * dyv.abs() if name != "none" else 0) + 2 * U32 * want.abs()
    dz, db = layer.act_backward(dy, z, name, dz_dtype=out)
    ref.close(dz, want, ref.rounded(want, off, out), "dz")
    ref.close(db, want.sum(0), off.sum(0) + (M + 2) * U32 * (want.abs() + off).sum(0) + ref.TINY[F32], "dbias")


def test_tensors_that_require_a_gradient_are_refused(cuda_device):
    M, N = 20, 16
    A = csr_on(cuda_device, pattern(M, M, 1), (M, M))
    T = layer.CsrTranspose.of(A)
    t, w, r = torch.randn(M, N, device=cuda_device), torch.ones(N, device=cuda_device), torch.ones(M, device=cuda_device)
    p, q, v = t.clone().requires_grad_(), w.clone().requires_grad_(), A.data.clone().requires_grad_()
    trained = hyb.DeviceCsr(A.indptr, A.indices, v, (M, M))
    calls = [lambda: layer.rms_norm(p, w), lambda: layer.rms_norm(t, q), lambda: layer.rms_norm(t, w, residual=p),
             lambda: layer.rms_norm_backward(p, t, w, r), lambda: layer.rms_norm_backward(t, t, q, r), lambda: layer.spmm_csr_act(A, p),
             lambda: layer.spmm_csr_act(A, t, bias=q), lambda: layer.spmm_csr_act(A, t, residual=p), lambda: layer.spmm_csr_act(trained, t),
             lambda: layer.spmm_csr_act(T, t, values=v), lambda: layer.act_backward(p), lambda: layer.act_backward(t, p, "silu"),
             lambda: layer.spmm_csr_grad_values(A, p, t), lambda: layer.spmm_csr_act_backward(trained, T, t, t)]
    for f in calls:
        with pytest.raises(ValueError, match="no_grad"):
            f()
        with torch.no_grad():
            f()


def test_transposed_patterns_are_validated(cuda_device):
    for M, K in ((40, 30), (1, 50), (30, 1), (5, 0), (0, 5)):
        A = csr_on(cuda_device, pattern(M, K, 3) if M and K else (torch.zeros(M + 1, dtype=torch.int64), torch.empty(0, dtype=torch.int32), torch.empty(0)), (M, K))
        T = layer.CsrTranspose.of(A)
        T.validate()
        T.validate(A)
    A = csr_on(cuda_device, pattern(40, 30, 3), (40, 30))
    T = layer.CsrTranspose.of(A)
    other = csr_on(cuda_device, pattern(40, 30, 3), (40, 30))
    other.indices = (29 - other.indices)      # as many entries, elsewhere
    swapped = T.order.clone()
    swapped[:2] = T.order[:2].flip(0)
    far = T.indices.clone()
    far[-1] = 40
    for t, a in ((T, other), (layer.CsrTranspose(T.indptr, T.indices, swapped, T.shape), A), (layer.CsrTranspose(T.indptr, far, T.order, T.shape), None),
                 (layer.CsrTranspose(T.indptr, T.indices, T.order, (30, 39)), A), (layer.CsrTranspose(T.indptr.flip(0), T.indices, T.order, T.shape), None)):
        with pytest.raises(ValueError):
            t.validate(a)


def test_captured_calls_leave_the_workspace_alone(cuda_device):
    """A workspace that has grown since the capture is no part of the replay."""
    g = gen(8)
    M, K, N = 300, 2500, 96
    A = csr_on(cuda_device, pattern(M, K, 9, 12.0, 2500), (M, K))
    B, dy = torch.randn(K, N, generator=g).to(cuda_device), torch.randn(M, N, generator=g).to(cuda_device)
    h, w, r = torch.randn(M, N, generator=g).to(cuda_device), torch.ones(N, device=cuda_device), torch.ones(M, device=cuda_device)
    ws = hyb.Workspace(cuda_device)
    step = lambda: (layer.spmm_csr_act(A, B, workspace=ws), *layer.act_backward(dy, dy, "silu", workspace=ws),
                    *layer.rms_norm_backward(dy, h, w, r, workspace=ws))
    want = [t.clone() for t in step()]
    held = ws._buf
    assert held is not None and held.numel() >= 1000
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    assert ws._buf is held
    held.fill_(0x5a)            # as if it were another tensor's by now
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(out, want)) and bool((held == 0x5a).all())


@pytest.mark.parametrize("dtype", [F32, BF16, E4M3])
@pytest.mark.parametrize("N", [64, 33])
def test_scales_of_any_type_and_ranges_of_a_transposed_pattern(cuda_device, dtype, N):
    g = gen(N)
    M, K = 150, 110
    p = pattern(M, K, 4, 9.0, 110)
    A = csr_on(cuda_device, p, (M, K))
    T = layer.CsrTranspose.of(A)
    a = ref.dense(*p, (M, K))
    for m, at, rows, ad in ((A, None, K, a), (T, A.data, M, a.t().contiguous())):
        B, _, Bv = features(rows, N, F32 if dtype == E4M3 else dtype, g, cuda_device)
        if dtype == E4M3:
            B, Bv = B.to(E4M3), B.to(E4M3).cpu().double()
        s = torch.rand(rows, generator=g) * 2 - 1
        n = ad.shape[0]
        R, Rv = rows_of((n, N), F32, g, cuda_device)
        z, y, zoff, yoff = ref.product(ad, Bv * s.double()[:, None], None, "silu", Rv, F32)
        kw = dict(scale=s.to(cuda_device), activation="silu", values=at, out_dtype=F32)
        ref.close(layer.spmm_csr_act(m, B, residual=R, **kw), y, yoff)
        for r0, r1 in ((0, 1), (37, 90), (n - 1, n), (50, 50)):
            pre = torch.empty(r1 - r0, N, device=cuda_device)
            ref.close(layer.spmm_csr_act(m, B, residual=R[r0:r1], preact=pre, row_range=(r0, r1), **kw), y[r0:r1], yoff[r0:r1], (r0, r1))
            ref.close(pre, z[r0:r1], zoff[r0:r1], (r0, r1))
