"""The block-scaled e4m3 operators, the root-mean-square norm and the cross attention on the GPU against their 64-bit forms (block_ref.py,
which derives each bound), at the sizes, strides and masks where they could go wrong."""
import math

import pytest
import torch

import block_ref as R
from uc2_amd import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(shape, seed, dtype=F32, std=1.0):
    return (torch.randn(*shape, generator=gen(seed), device=DEV) * std).to(dtype)


# ---- quantisation ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (3, 129), (7, 500), (5, 512), (130, 1000), (17, 1024), (4100, 777), (1, 4096)])
def test_quantize_rows_is_the_format(dtype, M, K):
    x = normal((M, K), M + K, dtype) * torch.exp(2 * normal((M, 1), 5)).to(dtype)
    a = ops.fp8_quantize_block(x)
    v, e = R.quant_rows(x)
    got, ge = R.rows_values(a)
    assert torch.equal(ge, e) and torch.equal(got, v)
    assert not a.data[:, K:].any()


def test_quantize_rows_borders_and_tiny_values():
    # maxima at 448 2^e exactly, one step over it, powers of two, and values that the block's scale makes subnormal
    x = torch.zeros(8, 256, device=DEV)
    for i, top in enumerate([448.0, 449.0, 448.0 * 2 ** -20, 448.0 * (1 + 2.0 ** -23), 1.0, 2.0 ** -100, 1e30, 3e38]):
        x[i, 3] = top
        x[i, 4:128] = -top * torch.linspace(0, 1, 124, device=DEV) ** 6
    x[1, 128:] = 2.0 ** -140                            # fp32 subnormals: the smallest exponent, 1, is kept
    a = ops.fp8_quantize_block(x)
    v, e = R.quant_rows(x)
    got, ge = R.rows_values(a)
    assert torch.equal(ge, e) and torch.equal(got, v)
    z = ops.fp8_quantize_block(torch.zeros(3, 130, device=DEV, dtype=BF16))
    assert not z.data.any()
    assert bool((R.rows_values(z)[1] == 1).all())


def test_quantize_keeps_nan_and_infinity_visible():
    x = normal((4, 300), 1, BF16)
    x[0, 5], x[1, 200], x[2, 299] = math.nan, math.inf, -math.inf
    v = ops.fp8_quantize_block(x).data.view(torch.float8_e4m3fn).float()
    assert torch.isnan(v[0, 5]) and torch.isnan(v[1, 200]) and torch.isnan(v[2, 299])
    assert torch.isfinite(v[3]).all() and torch.isfinite(v[0, 128:]).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N,K", [(1, 1), (128, 128), (129, 127), (300, 1000), (777, 260), (1024, 768)])
def test_quantize_weight_and_its_transposed_copy(dtype, N, K):
    w = normal((N, K), N + K, dtype)
    b, bt = ops.fp8_quantize_weight_block(w, transpose=True)
    v, e = R.quant_square(w)
    assert torch.equal(b.scale.long(), e) and torch.equal(R.weight_values(b, K), v)
    assert torch.equal(bt.scale.long(), e.t()) and torch.equal(R.weight_values(bt, N), v.t())
    assert not b.data[:, K:].any() and not bt.data[:, N:].any()
    one = ops.fp8_quantize_weight_block(w)
    assert torch.equal(one.data, b.data) and torch.equal(one.scale, b.scale)


def test_quantize_strided_rows():
    big = normal((9, 700), 3, BF16)
    for x in (big[:, 3:300], big[::2], big[:, :1], big.t()[:5]):
        a = ops.fp8_quantize_block(x)
        v, e = R.quant_rows(x)
        assert torch.equal(R.rows_values(a)[0], v)
    w = normal((200, 300), 4)
    assert torch.equal(R.weight_values(ops.fp8_quantize_weight_block(w[:, 1:260]), 259), R.quant_square(w[:, 1:260])[0])


# ---- product --------------------------------------------------------------------------------------------------------------------
GEMM_SIZES = [(1, 1, 1), (1, 1024, 4096), (8, 4096, 1024), (16, 17, 128), (17, 130, 256), (33, 1000, 300), (64, 255, 1024), (65, 129, 640),
              (128, 128, 128), (200, 777, 1000), (256, 256, 512), (512, 768, 768), (1030, 516, 384), (2048, 2304, 768), (1024, 1024, 1152),
              (4096, 2304, 768), (8300, 1100, 512), (33000, 256, 256), (4200, 2304, 1000), (4096, 2304, 1152),
              (4096, 2048, 4096), (4100, 2310, 3840)]                     # (scales of more than 28 blocks)


@pytest.mark.parametrize("M,N,K", GEMM_SIZES)
@pytest.mark.parametrize("bias", [False, True])
def test_gemm_block(M, N, K, bias):
    x = normal((M, K), 1, BF16) * torch.exp(normal((1, K), 2)).to(BF16)
    w = normal((N, K), 3, F32, K ** -0.5) * torch.exp(normal((N, 1), 4))
    b = normal((N,), 5) if bias else None
    a, q = ops.fp8_quantize_block(x), ops.fp8_quantize_weight_block(w)
    A, B = R.rows_values(a)[0], R.weight_values(q, K)
    got = ops.gemm_fp8_block(a, q, bias=b)
    R.assert_gemm(got, A, B, b, "%d x %d x %d" % (M, N, K))
    assert torch.equal(got, ops.gemm_fp8_block(a, q, bias=b))


@pytest.mark.parametrize("M,N,K", [(8460, 2310, 256), (8460, 2310, 1024), (8448, 2304, 3840), (8460, 2310, 4096), (16896, 1024, 7424)])
@pytest.mark.parametrize("bias", [False, True])
def test_gemm_block_more_tiles_than_compute_units(M, N, K, bias):
    """more than 256 whole 256 x 256 tiles: workgroups of the persistent kernel take a second one (2, 8, 30, 32 and 58 blocks of K: with one, two and three fills
    of the scales, and the next tile's first fill after a refill), nine columns of tiles, with and without remainders.  Each row and each
    128 columns have a scale of their own, so a tile that took another's scales would be off by a power of two"""
    g = gen(M + N + K)
    x = normal((M, K), 1, BF16) * torch.exp2(torch.randint(-6, 7, (M, 1), generator=g, device=DEV).float()).to(BF16)
    x *= torch.exp2(torch.randint(-3, 4, (1, K // 128, 1), generator=g, device=DEV).float()).expand(1, K // 128, 128).reshape(1, K).to(BF16)
    w = normal((N, K), 3, F32, K ** -0.5) * torch.exp2(torch.randint(-6, 7, ((N + 127) // 128, 1, K // 128, 1), generator=g, device=DEV).float()).expand(-1, 128, -1, 128).reshape(-1, K)[:N]
    b = normal((N,), 5) if bias else None
    a, q = ops.fp8_quantize_block(x), ops.fp8_quantize_weight_block(w)
    got = ops.gemm_fp8_block(a, q, bias=b)
    assert torch.equal(got, ops.gemm_fp8_block(a, q, bias=b))
    for r0 in range(0, M, 2112):                             # (the 64-bit product in parts)
        part = ops.BlockRows(a.data[r0:r0 + 2112], a.scale[:, r0:r0 + 2112], K)
        A, B = R.rows_values(part)[0], R.weight_values(q, K)
        R.assert_gemm(got[r0:r0 + 2112], A, B, b, "%d x %d x %d from row %d" % (M, N, K, r0))


def test_gemm_block_a_row_has_the_same_bits_among_others():
    """the operand bytes of a row do not depend on the rows beside it, nor do the product's bits where the same kernel runs: few rows, 64 x 64 tiles, 128 x 128
    tiles, whole 256 x 256 tiles, and with other values in the rows behind"""
    for N, K, sizes in ((640, 768, (3, 16)), (1024, 1024, (33, 50)), (2048, 512, (640, 700)), (4096, 384, (1280, 1400)), (2048, 512, (4096, 4352))):
        x, w = normal((sizes[1], K), 1, BF16), normal((N, K), 2)
        q = ops.fp8_quantize_weight_block(w)
        full, m = ops.fp8_quantize_block(x), sizes[0]
        some = ops.fp8_quantize_block(x[:m])
        assert torch.equal(some.data, full.data[:m]) and torch.equal(some.scale, full.scale[:, :m])
        want = ops.gemm_fp8_block(full, q)
        assert torch.equal(ops.gemm_fp8_block(some, q), want[:m]), (N, K, sizes)
        x[m:] = math.inf
        assert torch.equal(ops.gemm_fp8_block(ops.fp8_quantize_block(x), q)[:m], want[:m])


def test_gemm_block_rows_do_not_depend_on_the_others():
    """a row alone and among others: the same operand bytes; where both run the same kernel the same bits"""
    K, N = 768, 640
    x, w = normal((2048, K), 1, BF16), normal((N, K), 2)
    q = ops.fp8_quantize_weight_block(w)
    full = ops.gemm_fp8_block(ops.fp8_quantize_block(x), q)
    A, B = R.rows_values(ops.fp8_quantize_block(x[:3]))[0], R.weight_values(q, K)
    part = ops.gemm_fp8_block(ops.fp8_quantize_block(x[:3]), q)
    R.assert_gemm(part, A, B)
    R.assert_gemm(full[:3], A, B)


def test_gemm_block_scales_far_apart():
    """one block 2^60 above its neighbours, one 2^-60 below: the sums keep the large one's precision, nothing overflows"""
    x, w = normal((70, 512), 1, F32), normal((96, 512), 2)
    x[:, 128:256] *= 2.0 ** 60
    x[:, 256:384] *= 2.0 ** -60
    w[:, 384:] *= 2.0 ** -50
    a, q = ops.fp8_quantize_block(x), ops.fp8_quantize_weight_block(w)
    A, B = R.rows_values(a)[0], R.weight_values(q, 512)
    R.assert_gemm(ops.gemm_fp8_block(a, q), A, B)


def test_gemm_block_nan_reaches_its_row_only():
    x, w = normal((40, 256), 1, BF16), normal((48, 256), 2)
    x[7, 100] = math.nan
    y = ops.gemm_fp8_block(ops.fp8_quantize_block(x), ops.fp8_quantize_weight_block(w))
    assert torch.isnan(y[7]).all()
    assert torch.isfinite(y[:7]).all() and torch.isfinite(y[8:]).all()


def test_gemm_block_empty():
    q = ops.fp8_quantize_weight_block(normal((48, 256), 2))
    assert ops.gemm_fp8_block(ops.fp8_quantize_block(torch.empty(0, 256, device=DEV, dtype=BF16)), q).shape == (0, 48)


# ---- linear layer ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("M,N,K", [(1, 130, 64), (7, 96, 200), (100, 77, 129), (640, 512, 768), (1024, 768, 256), (2500, 333, 1000)])
@pytest.mark.parametrize("wtype", [F32, BF16])
def test_linear_block_forward_and_gradients(M, N, K, wtype):
    x, w, b, dy = normal((M, K), 1, BF16), normal((N, K), 2, wtype, K ** -0.5), normal((N,), 3), normal((M, N), 4, BF16)
    xg, wg, bg = (t.clone().requires_grad_() for t in (x, w, b))
    y = ops.linear_fp8_block(xg, wg, bg)
    dx, dw, db = torch.autograd.grad(y, [xg, wg, bg], dy)
    X, W, DY = R.quant_rows(x)[0], R.quant_square(w)[0], R.quant_rows(dy)[0]
    R.assert_gemm(y.detach(), X, W, b, "y")
    R.assert_gemm(dx, DY, W.t(), None, "dx")
    want, mag = R.mm(dy.double().t(), x.double()), R.mm(dy.double().abs().t(), x.double().abs())
    assert dw.dtype == wtype
    R.assert_within(dw, want, 2 * M * R.U[F32] * mag + R.U[wtype] * want.abs(), "dw")
    R.assert_within(db, dy.double().sum(0), M * R.U[F32] * dy.double().abs().sum(0) + 1e-30, "db")


def wgrad(M, N, K, dy, x, bias=True, lddw=None, off=0):
    """uc2_linear_wgrad on rows dy [M, N] and x [M, K] of any stride -> (dw [N, K], db)"""
    lddw = lddw or K
    dw = torch.full((N * lddw + off,), 7.0, device=DEV)[off:].view(N, lddw)
    db = torch.empty(N, device=DEV) if bias else None
    n = _lib.load().uc2_linear_wgrad_workspace(M, N, K)
    ws = torch.empty(n, dtype=torch.uint8, device=DEV)
    _lib.call("uc2_linear_wgrad", M, N, K, dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), dw.data_ptr(), lddw, _lib.ptr(db), ws.data_ptr(), n, _lib.stream())
    assert bool((dw[:, K:] == 7).all())
    return dw[:, :K], db


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 8, 8), (2, 7, 300), (65, 300, 3), (513, 1, 1000), (700, 9, 130), (4097, 257, 100), (5000, 5, 6), (1024, 256, 256), (1280, 512, 256),
                                   (1152, 256, 512), (40000, 64, 40)])
@pytest.mark.parametrize("odd", [False, True])
def test_linear_wgrad(M, N, K, odd):
    """odd: rows of an odd stride behind an odd offset, dw in wider rows.  Bound as above: M fp32 additions"""
    dy, x = normal((M, N + 3 * odd), 1, BF16)[:, odd:N + odd], normal((M, K + 5 * odd), 2, BF16)[:, 3 * odd:K + 3 * odd]
    dw, db = wgrad(M, N, K, dy, x, True, K + odd)
    want, mag = R.mm(dy.double().t(), x.double()), R.mm(dy.double().abs().t(), x.double().abs())
    R.assert_within(dw, want, 2 * M * R.U[F32] * mag + 1e-30, "dw")
    R.assert_within(db, dy.double().sum(0), M * R.U[F32] * dy.double().abs().sum(0) + 1e-30, "db")
    again, db2 = wgrad(M, N, K, dy, x)
    assert torch.equal(again, dw) and torch.equal(db2, db)
    assert torch.equal(wgrad(M, N, K, dy, x, False)[0], dw)


def test_linear_wgrad_into_a_result_of_any_alignment():
    M, N, K = 1280, 512, 256                                     # (whole tiles)
    dy, x = normal((M, N), 1, BF16), normal((M, K), 2, BF16)
    want, mag = R.mm(dy.double().t(), x.double()), R.mm(dy.double().abs().t(), x.double().abs())
    for off in (0, 1, 2):
        R.assert_within(wgrad(M, N, K, dy, x, off=off)[0], want, 2 * M * R.U[F32] * mag, "off by %d" % off)


@pytest.mark.parametrize("M,N", [(1, 1), (300, 5), (5000, 777), (9000, 2304)])
def test_linear_block_bias_gradient_alone(M, N):
    """a bias that is trained beside a weight that is not: in a fixed order too"""
    x, w, dy = normal((M, 64), 1, BF16), normal((N, 64), 2), normal((M, N), 3, BF16)
    b = torch.zeros(N, device=DEV, requires_grad=True)
    db, = torch.autograd.grad(ops.linear_fp8_block(x, w, b), [b], dy)
    R.assert_within(db, dy.double().sum(0), M * R.U[F32] * dy.double().abs().sum(0) + 1e-30, "db")
    for _ in range(3):
        assert torch.equal(torch.autograd.grad(ops.linear_fp8_block(x, w, b), [b], dy)[0], db)


def test_linear_wgrad_nan_stays_in_its_row_and_column():
    dy, x = normal((1500, 40), 1, BF16), normal((1500, 72), 2, BF16)
    dy[700, 3] = math.nan
    dw, db = wgrad(1500, 40, 72, dy, x)
    bad = torch.isnan(dw)
    assert bool(bad[3].all()) and int(bad.sum()) == 72 and bool(torch.isnan(db)[3]) and int(torch.isnan(db).sum()) == 1


def test_linear_block_leading_dimensions_and_partial_gradients():
    x, w = normal((3, 5, 256), 1, BF16), normal((130, 256), 2)
    y = ops.linear_fp8_block(x, w)
    assert y.shape == (3, 5, 130) and not y.requires_grad
    xg = x.clone().requires_grad_()
    dx, = torch.autograd.grad(ops.linear_fp8_block(xg, w).float().sum(), [xg])
    assert dx.shape == x.shape
    wg = w.clone().requires_grad_()
    dw, = torch.autograd.grad(ops.linear_fp8_block(x, wg).float().sum(), [wg])
    R.assert_within(dw, x.double().sum((0, 1)).expand(130, 256), 1e-5 * x.double().abs().sum((0, 1)).expand(130, 256))
    empty = torch.empty(0, 256, device=DEV, dtype=BF16).requires_grad_()
    out = ops.linear_fp8_block(empty, wg)
    dx, dw = torch.autograd.grad(out, [empty, wg], torch.empty(0, 130, device=DEV, dtype=BF16))
    assert dx.shape == (0, 256) and not dw.any()


# ---- root-mean-square norm ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,H", [(1, 1), (1, 8), (3, 7), (5, 512), (9, 513), (1000, 768), (37, 1000), (6, 1024), (5, 2048), (4, 2049), (3, 4100), (2, 8192),
                                 (2, 8193), (2, 16384)])
@pytest.mark.parametrize("with_res", [False, True])
def test_rms_norm_forward_and_gradients(dtype, M, H, with_res):
    x, w = normal((M, H), 1, dtype, 3.0), 1 + normal((H,), 2, F32, 0.2)
    res = normal((M, H), 3, dtype) if with_res else None
    dy, ds = normal((M, H), 4, dtype), normal((M, H), 5, dtype) if with_res else None
    eps, u, u32, r1 = 1e-5, R.U[dtype], R.U[F32], R.rms_rel(H)
    y64, s, r = R.rms(x, w, eps, res)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    if with_res:
        rg = res.clone().requires_grad_()
        y, sg = ops.rms_norm(xg, wg, eps, residual=rg)
        assert torch.equal(sg.detach(), s)
        dx, dres, dw = torch.autograd.grad([y, sg], [xg, rg, wg], [dy, ds])
        assert torch.equal(dx, dres)
    else:
        y = ops.rms_norm(xg, wg, eps)
        dx, dw = torch.autograd.grad(y, [xg, wg], dy)
    R.assert_within(y.detach(), y64, (r1 + 3 * u32 + u) * y64.abs(), "y")
    g, h = dy.double() * w.double(), s.double() * r
    c, cm = (g * h).mean(-1, keepdim=True), (g * h).abs().mean(-1, keepdim=True)
    want = r * (g - h * c) + (0 if ds is None else ds.double())
    mag = r * (g.abs() + h.abs() * cm)
    R.assert_within(dx, want, u * want.abs() + (2 * r1 + (H + 8) * u32) * mag + u32 * want.abs(), "dx")
    want, mag = (dy.double() * h).sum(0), (dy.double() * h).abs().sum(0)
    R.assert_within(dw, want, (M + 4) * u32 * mag + r1 * mag, "dw")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,H", [(2049, 768), (5003, 1000), (9000, 130), (1100, 2500), (700, 9000)])
def test_rms_norm_gradient_of_more_rows_than_workgroups(dtype, M, H):
    """more rows than the backward's 512 workgroups take at once: each goes over several, of every width of row"""
    x, w, res = normal((M, H), 1, dtype, 3.0), 1 + normal((H,), 2, F32, 0.2), normal((M, H), 3, dtype)
    dy, ds = normal((M, H), 4, dtype), normal((M, H), 5, dtype)
    eps, u, u32, r1 = 1e-5, R.U[dtype], R.U[F32], R.rms_rel(H)
    _, s, r = R.rms(x, w, eps, res)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    y, sg = ops.rms_norm(xg, wg, eps, residual=res)
    dx, dw = torch.autograd.grad([y, sg], [xg, wg], [dy, ds])
    g, h = dy.double() * w.double(), s.double() * r
    c, cm = (g * h).mean(-1, keepdim=True), (g * h).abs().mean(-1, keepdim=True)
    want, mag = r * (g - h * c) + ds.double(), r * (g.abs() + h.abs() * cm)
    R.assert_within(dx, want, u * want.abs() + (2 * r1 + (H + 8) * u32) * mag + u32 * want.abs(), "dx")
    want, mag = (dy.double() * h).sum(0), (dy.double() * h).abs().sum(0)
    R.assert_within(dw, want, (M + 4) * u32 * mag + r1 * mag, "dw")


def test_rms_norm_gradient_against_differences():
    M, H, eps = 5, 200, 1e-5
    x, w, dy = normal((M, H), 1), 1 + normal((H,), 2, F32, 0.2), normal((M, H), 3)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(ops.rms_norm(xg, wg, eps), [xg, wg], dy)
    f = lambda a, b: (R.rms(a, b, eps)[0] * dy.double()).sum()  # noqa: E731
    for seed in range(3):
        a, b, t = normal((M, H), 10 + seed).double(), normal((H,), 20 + seed).double(), 1e-4
        num = (f(x.double() + t * a, w.double() + t * b) - f(x.double() - t * a, w.double() - t * b)) / (2 * t)
        ana = (dx.double() * a).sum() + (dw.double() * b).sum()
        # differences: t^2 times a third derivative of order 1 per element; the gradients: 1e-5 of each product
        tol = 1e-5 * ((dx.double() * a).abs().sum() + (dw.double() * b).abs().sum()) + t * t * M * H
        assert abs(num - ana) < tol


def test_rms_norm_uses_of_the_stream():
    x, r, w = normal((6, 96), 1).requires_grad_(), normal((6, 96), 2).requires_grad_(), torch.ones(96, device=DEV, requires_grad=True)
    y, s = ops.rms_norm(x, w, 1e-6, residual=r)
    g = torch.autograd.grad(s.sum(), [x, r, w], retain_graph=True)            # the stream alone
    assert torch.equal(g[0], torch.ones_like(x)) and torch.equal(g[1], g[0]) and not g[2].any()
    y2 = ops.rms_norm(s, w, 1e-6)
    a = torch.autograd.grad(y.sum() + (2 * s).sum() + y2.sum(), [x])[0]
    X, Rr = x.detach().double().requires_grad_(), r.detach().double()
    S = X + Rr
    Y = S / torch.sqrt(S.pow(2).mean(-1, keepdim=True) + 1e-6)
    b = torch.autograd.grad(Y.sum() + (2 * S).sum() + Y.sum(), [X])[0]
    R.assert_within(a, b, 1e-5 * (b.abs() + 2))
    xs = normal((8, 300), 4, BF16)[:, 5:200]                                     # strided, unaligned rows
    y64, _, _ = R.rms(xs, torch.ones(195, device=DEV), 1e-6)
    R.assert_within(ops.rms_norm(xs, torch.ones(195, device=DEV)), y64, (R.U[BF16] + 1e-5) * y64.abs())
    assert ops.rms_norm(torch.empty(0, 96, device=DEV), torch.ones(96, device=DEV)).shape == (0, 96)
    e = torch.empty(0, 96, device=DEV).requires_grad_()
    dw, = torch.autograd.grad(ops.rms_norm(e, w), [w], torch.empty(0, 96, device=DEV))
    assert not dw.any()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,H", [(1, 1024), (8, 768), (5, 130), (33, 2100), (3, 9000), (700, 1000)])
def test_rms_norm_fp8_is_the_norm_quantised(dtype, M, H):
    x, res, w = normal((M, H), 1, dtype, 2.0), normal((M, H), 2, dtype), 1 + normal((H,), 3, F32, 0.2)
    a, s = ops.rms_norm_fp8(x, w, 1e-6, residual=res)
    y, s64, _ = R.rms(x, w, 1e-6, res)
    assert torch.equal(s, s64)
    got, e = R.rows_values(a)
    assert not a.data[:, H:].any()
    p = torch.nn.functional.pad(y, (0, -H % 128)).reshape(M, -1, 128).abs().amax(-1)
    rel = R.rms_rel(H) + 3 * R.U[F32]
    lo, hi = R.block_exponents(p * (1 - rel)), R.block_exponents(p * (1 + rel))
    assert bool(((e >= lo) & (e <= hi)).all())
    step = torch.exp2((e - 127).double()).repeat_interleave(128, 1)[:, :H]
    R.assert_within(got, y, torch.maximum(R.U["e4m3"] * y.abs(), 2.0 ** -10 * step) + rel * y.abs())
    b, s1 = ops.rms_norm_fp8(s, w, 1e-6)                                        # without a residual: the same operand
    assert torch.equal(b.data, a.data) and torch.equal(b.scale, a.scale) and s1 is s


def test_rows_beyond_one_launch():
    """2^26 rows of the norm and 2^28 of the quantisation are a launch's most: the rows around the border and the last ones as if they were alone"""
    M, w = (1 << 26) + 5, 1 + normal((8,), 2, F32, 0.2)
    at = torch.cat([torch.arange(3), torch.arange((1 << 26) - 8, M)]).to(DEV)
    x, res = normal((M, 8), 1, BF16), normal((M, 8), 3, BF16)
    a, s = ops.rms_norm_fp8(x, w, residual=res)
    y, s2 = ops.rms_norm(x, w, residual=res)
    a1, s1 = ops.rms_norm_fp8(x[at], w, residual=res[at])
    assert torch.equal(s[at], s1) and torch.equal(s2[at], s1) and torch.equal(y[at], ops.rms_norm(x[at], w, residual=res[at])[0])
    assert torch.equal(a.data[at], a1.data) and torch.equal(a.scale[:, at], a1.scale)
    assert torch.equal(s, x + res) and bool(torch.isfinite(y).all())
    xg = x.requires_grad_()
    dx, = torch.autograd.grad(ops.rms_norm(xg, w), [xg], res)
    xs = xg.detach()[at].requires_grad_()
    assert torch.equal(dx[at], torch.autograd.grad(ops.rms_norm(xs, w), [xs], res[at])[0])
    del x, xg, res, a, s, y, s2, dx
    M = (1 << 28) + 5
    at = torch.cat([torch.arange(3), torch.arange((1 << 28) - 8, M)]).to(DEV)
    x = torch.empty(M, 8, device=DEV, dtype=BF16).normal_(generator=gen(5))
    a = ops.fp8_quantize_block(x)
    a1 = ops.fp8_quantize_block(x[at])
    assert torch.equal(a.data[at], a1.data) and torch.equal(a.scale[:, at], a1.scale)
    del a, x
    torch.cuda.empty_cache()


# ---- cross attention ------------------------------------------------------------------------------------------------------------
def attn_inputs(B, Lq, Lk, nh, nkv, D, dtype, seed=0, std=1.0):
    q = normal((B, Lq, nh, D), seed + 1, dtype, std)
    kv = normal((B, Lk, 2, nkv, D), seed + 2, dtype, std)
    return q, kv[:, :, 0], kv[:, :, 1], normal((B, Lq, nh, D), seed + 3, dtype)


def run_attn(q, k, v, dout, **kw):
    qg, kg, vg = (t.detach().requires_grad_() for t in (q, k, v))
    o = ops.cross_attention(qg, kg, vg, **kw)
    return [o.detach(), *torch.autograd.grad(o, [qg, kg, vg], dout)]


def check_attn(q, k, v, dout, key_mask=None, k_lens=None, scale=None, what=""):
    sc = 1.0 / math.sqrt(q.shape[3]) if scale is None else scale
    got = run_attn(q, k, v, dout, key_mask=key_mask, k_lens=k_lens, scale=scale)
    want, bound = R.attention(q, k, v, sc, key_mask, k_lens, dout)
    for g, w, b, n in zip(got, want, bound, ("out", "dq", "dk", "dv")):
        R.assert_within(g, w, b, "%s %s" % (what, n))
    return got


ATTN = [  # B, Lq, Lk, nh, nkv, D
    (1, 1, 1, 1, 1, 64), (2, 1, 300, 4, 1, 64), (3, 5, 31, 4, 2, 32), (2, 33, 65, 2, 2, 64), (1, 60, 100, 12, 12, 64), (2, 130, 64, 3, 3, 64), (1, 77, 211, 12, 4, 64),
    (2, 17, 129, 4, 2, 128), (1, 200, 257, 2, 1, 128), (9, 10, 40, 2, 1, 32), (1, 257, 513, 2, 2, 64), (1, 1, 4097, 8, 2, 128), (1, 1000, 33, 2, 2, 32), (1, 1500, 1, 1, 1, 64),
    (2, 513, 1100, 4, 2, 64), (1, 900, 1201, 4, 4, 32), (2, 300, 2000, 4, 2, 128)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,Lq,Lk,nh,nkv,D", ATTN)
def test_cross_attention_plain(dtype, B, Lq, Lk, nh, nkv, D):
    check_attn(*attn_inputs(B, Lq, Lk, nh, nkv, D, dtype))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,Lq,Lk,nh,nkv,D", [(5, 9, 200, 4, 2, 64), (4, 40, 130, 2, 2, 128), (6, 1, 1100, 4, 1, 32), (3, 300, 95, 3, 3, 64), (5, 450, 1000, 4, 2, 64)])
def test_cross_attention_lengths(dtype, B, Lq, Lk, nh, nkv, D):
    """lengths of zero and one, inside and at the end of tiles, over and under the range (clamped), with NaN and infinities behind them"""
    q, k, v, dout = attn_inputs(B, Lq, Lk, nh, nkv, D, dtype)
    lens = torch.tensor([0, Lk, 1, 64, Lk + 7, -3][:B], device=DEV, dtype=torch.int32)
    for b in range(B):
        n = max(0, min(int(lens[b]), Lk))
        k[b, n:] = math.nan
        v[b, n:] = math.inf
    got = check_attn(q, k, v, dout, k_lens=lens)
    assert not got[0][0].any() and not got[1][0].any() and not got[2][0].any() and not got[3][0].any()
    again = run_attn(q, k, v, dout, k_lens=lens.long())
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,Lq,Lk,nh,nkv,D", [(4, 9, 200, 4, 2, 64), (4, 70, 60, 2, 2, 128), (4, 1, 900, 4, 1, 32), (4, 300, 1000, 4, 2, 64)])
def test_cross_attention_key_mask(dtype, B, Lq, Lk, nh, nkv, D):
    """-inf, -1e30 and the lowest fp32 remove a key with whatever it holds; finite entries weigh; a row of nothing gives zeros"""
    q, k, v, dout = attn_inputs(B, Lq, Lk, nh, nkv, D, dtype)
    mask = normal((B, Lk), 9)
    gone = torch.rand(B, Lk, generator=gen(11), device=DEV) < 0.4
    gone[:, 0] = False
    gone[1] = True
    gone[3, :Lk - 1], gone[3, Lk - 1] = True, False                              # one key left, the last
    low = torch.tensor([-math.inf, -1e30, torch.finfo(F32).min], device=DEV)[torch.randint(0, 3, (B, Lk), generator=gen(12), device=DEV)]
    mask = torch.where(gone, low, mask)
    k[gone] = math.nan
    v[gone] = -math.inf
    got = check_attn(q, k, v, dout, key_mask=mask)
    assert not got[0][1].any() and not got[1][1].any()
    assert not got[2][gone].any() and not got[3][gone].any()
    lens = torch.tensor([Lk // 2, Lk, 3, Lk], device=DEV, dtype=torch.int32)
    check_attn(q, torch.where(gone[..., None, None], 0, k), torch.where(gone[..., None, None], 0, v), dout, key_mask=mask, k_lens=lens)
    four = run_attn(q, k, v, dout, key_mask=mask[:, None, None, :])
    assert all(torch.equal(a, b) for a, b in zip(got, four))


def test_cross_attention_small_penalties_only_weigh():
    """-10000 on every key (the encoder's additive mask over a wholly padded sequence) leaves the softmax over the scores"""
    q, k, v, dout = attn_inputs(1, 8, 50, 2, 2, 64, F32)
    got = run_attn(q, k, v, dout, key_mask=torch.full((1, 50), -10000.0, device=DEV))
    want, _ = R.attention(q, k, v, 0.125, None, None, dout)
    for g, w in zip(got, want):
        # scores near -10000 are kept to 2^-24 of it in base 2 (1.4e4): the exponent is off by at most 1e-3
        assert (g.double() - w).abs().max() < 4e-3 * max(1.0, float(w.abs().max()))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_cross_attention_large_scores_and_scale(dtype):
    q, k, v, dout = attn_inputs(1, 20, 90, 2, 1, 64, dtype, std=6.0)
    check_attn(q, k, v, dout, scale=0.5)
    check_attn(q, k, v, dout, scale=0.0)
    check_attn(q, k, v, dout, scale=-0.1)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,Lq,Lk,nh,nkv,D", [(3, 70, 1, 4, 2, 64), (2, 3, 300, 4, 4, 128), (1, 1, 5000, 4, 1, 32)])
def test_cross_attention_one_key(dtype, B, Lq, Lk, nh, nkv, D):
    """one key that takes part: out is its value, dq and dk are zero.  What is left: the weight is 1 within (2 + |x|) roundings of fp32 (score x, its
    log-sum-exp), 1 in bf16, and dp and delta are sums of D products each: of sum |dout v| at most 2 D + 2 |x| + 8 of fp32's roundings"""
    q, k, v, dout = attn_inputs(B, Lq, Lk, nh, nkv, D, dtype)
    lens = torch.ones(B, dtype=torch.int32, device=DEV)
    o, dq, dk, dv = run_attn(q, k, v, dout, k_lens=lens)
    rep = lambda t: t[:, :1].double().repeat_interleave(nh // nkv, 2).expand(B, Lq, nh, D)  # noqa: E731
    Q, K, V, dO = q.double(), rep(k), rep(v), dout.double()
    x = (Q * K).abs().sum(-1, keepdim=True) * D ** -0.5
    off = (2 * D + 2 * x + 8) * R.U[F32] * (dO * V).abs().sum(-1, keepdim=True)
    R.assert_within(o, V, (R.U[dtype] * (dtype == BF16) + (4 + 2 * x) * R.U[F32]) * V.abs(), "out")
    R.assert_within(dq, torch.zeros_like(Q), off * D ** -0.5 * K.abs(), "dq")
    R.assert_within(dk[:, :1], torch.zeros_like(dk[:, :1]).double(), (off * D ** -0.5 * Q.abs()).view(B, Lq, nkv, -1, D).sum((1, 3))[:, None], "dk")
    assert not dk[:, 1:].any() and not dv[:, 1:].any()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Lq,Lk,nh,nkv,D", [(3, 1, 4, 4, 32), (70, 300, 4, 2, 64), (900, 40, 2, 1, 64), (2, 5000, 4, 1, 128), (600, 700, 3, 3, 32)])
@pytest.mark.parametrize("drop", [0.0, 0.3])
def test_cross_attention_one_key_has_no_gradient_of_its_scores(dtype, Lq, Lk, nh, nkv, D, drop):
    """the softmax over one key is 1 whatever its score: dq and dk are zero, not what fp32 leaves of dp - delta; by length, by mask (the first key, one inside,
    the last) and by both; sequences of two keys and more beside them keep their gradients"""
    at = [0, Lk // 2, Lk - 1]
    B = len(at) + 2
    q, k, v, dout = attn_inputs(B, Lq, Lk, nh, nkv, D, dtype)
    mask = torch.full((B, Lk), -math.inf, device=DEV)
    for b, j in enumerate(at):
        mask[b, j] = 0.5
    mask[3, :2] = mask[4, :2] = 0.0
    lens = torch.tensor([Lk, Lk, Lk, 1, Lk], device=DEV, dtype=torch.int32)
    torch.manual_seed(0), ops.rng.manual_seed(3)
    for kw in (dict(key_mask=mask, k_lens=lens), dict(k_lens=torch.tensor([1, 1, 1, 1, min(2, Lk)], device=DEV))):
        o, dq, dk, dv = run_attn(q, k, v, dout, drop_p=drop, **kw)
        assert not dq[:4].any() and not dk[:4].any() and o[:4].any() and dv[:4].any()
        # one or two keys: a query's gradient of two is lost only if dropout takes both
        assert Lk < 2 or bool(dq[4].any()) and bool(dk[4, :2].any())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Lq,Lk,nh,nkv,D,left", [(3, 300, 4, 4, 32, [10, 290]), (70, 300, 4, 2, 64, range(5, 300, 32)), (2, 5000, 4, 1, 128, [10, 4990]), (2, 5000, 4, 1, 64, [4998, 4999]),
                                                 (600, 1500, 3, 3, 32, range(31, 1500, 64)), (40, 64, 2, 2, 64, [0, 33])])
def test_cross_attention_keys_far_apart(dtype, Lq, Lk, nh, nkv, D, left):
    """two keys and more, one of them at most in a tile, a split or a wave's share: none is taken for the only one"""
    q, k, v, dout = attn_inputs(2, Lq, Lk, nh, nkv, D, dtype)
    mask = torch.full((2, Lk), -1e30, device=DEV)
    mask[:, list(left)] = normal((2, len(left)), 9)
    got = check_attn(q, k, v, dout, key_mask=mask)
    assert bool(got[1].any()) and all(bool(got[2][:, j].any()) for j in left)


def test_cross_attention_views():
    """heads before positions, fused projections, expanded keys, unaligned slices (copied), a gradient that is a broadcast"""
    B, Lq, Lk, nh, D = 2, 19, 70, 4, 64
    q = normal((B, nh, Lq, D), 1, BF16).transpose(1, 2)
    kv = normal((Lk, B, nh, 2 * D), 2, BF16)
    k, v = kv.transpose(0, 1)[..., :D], kv.transpose(0, 1)[..., D:]
    dout = normal((B, Lq, nh, D), 3, BF16)
    check_attn(q, k, v, dout)
    one = normal((1, Lk, 1, D), 4, BF16).expand(B, Lk, nh, D)
    check_attn(q, one, v, dout)
    wide = normal((B, Lk, nh, D + 3), 5, BF16)[..., 3:]
    check_attn(q, wide, v, dout)
    flat = normal((B * Lk * nh * D + 1,), 6, BF16)[1:].view(B, Lk, nh, D)
    check_attn(q, flat, v, dout)
    check_attn(q, k, v, torch.ones(1, 1, 1, 1, device=DEV, dtype=BF16).expand(B, Lq, nh, D))
    base = one.detach()[:, :, :1][:1].clone().requires_grad_()
    g, = torch.autograd.grad(ops.cross_attention(q, base.expand(B, Lk, nh, D), v), [base], dout)
    want, bound = R.attention(q, base.detach().expand(B, Lk, nh, D), v, 0.125, None, None, dout)
    # autograd sums the B nh gradients in bf16: each its bound, and a rounding per addition
    R.assert_within(g, want[2].sum((0, 2), keepdim=True), bound[2].sum((0, 2), keepdim=True) + B * nh * 2.0 ** -8 * want[2].abs().sum((0, 2), keepdim=True))


def test_cross_attention_beyond_32_bit_offsets():
    """keys 5 GB apart: one row of a long buffer in 2^20 elements"""
    Lk, D = 2600, 64
    buf = torch.empty(Lk, 1 << 20, device=DEV, dtype=BF16)
    k, v = buf[:, :D].view(1, Lk, 1, D), buf[:, D:2 * D].view(1, Lk, 1, D)
    k.copy_(normal((1, Lk, 1, D), 1)), v.copy_(normal((1, Lk, 1, D), 2))
    q, dout = normal((1, 3, 2, D), 3, BF16), normal((1, 3, 2, D), 4, BF16)
    check_attn(q, k, v, dout)


def test_cross_attention_empty():
    q, k, v, dout = attn_inputs(2, 4, 0, 2, 1, 64, BF16)
    got = run_attn(q, k, v, dout)
    assert not got[0].any() and not got[1].any() and got[2].shape == (2, 0, 1, 64)
    q, k, v, dout = attn_inputs(2, 0, 5, 2, 1, 64, BF16)
    got = run_attn(q, k, v, dout)
    assert got[0].shape == (2, 0, 2, 64) and not got[2].any() and not got[3].any()
    q, k, v, dout = attn_inputs(0, 4, 5, 2, 1, 64, BF16)
    assert run_attn(q, k, v, dout)[0].shape == (0, 4, 2, 64)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_cross_attention_repeats_bit_for_bit(dtype):
    for shape in [(2, 1, 3000, 8, 2, 64), (1, 700, 40, 2, 2, 64), (2, 60, 100, 4, 4, 64)]:
        a = run_attn(*attn_inputs(*shape, dtype))
        b = run_attn(*attn_inputs(*shape, dtype))
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_cross_attention_gradient_against_differences():
    q, k, v, dout = attn_inputs(2, 5, 37, 4, 2, 32, F32)
    lens = torch.tensor([37, 20], device=DEV, dtype=torch.int32)
    _, dq, dk, dv = run_attn(q, k, v, dout, k_lens=lens)
    f = lambda a, b, c: (R.attention(a, b, c, 32 ** -0.5, None, lens)[0][0] * dout.double()).sum()  # noqa: E731
    R.U.setdefault(torch.float64, 2.0 ** -53)
    Q, K, V, t = q.double(), k.double(), v.double(), 1e-4
    for seed in range(3):
        a, b, c = (normal(x.shape, 30 + seed + i).double() for i, x in enumerate((q, k, v)))
        num = (f(Q + t * a, K + t * b, V + t * c) - f(Q - t * a, K - t * b, V - t * c)) / (2 * t)
        terms = [(dq.double() * a), (dk.double() * b), (dv.double() * c)]
        # the formula's gradients to 1e-5 of each product; t^2 times third derivatives (of order ten per output element)
        tol = 1e-5 * sum(x.abs().sum() for x in terms) + 10 * t * t * dout.numel()
        assert abs(num - sum(x.sum() for x in terms)) < tol


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,Lq,Lk", [(2, 40, 90), (3, 800, 700)])
def test_cross_attention_dropout(dtype, B, Lq, Lk):
    """the mask of the general kernels (equal head counts); its rate, and the gradients under it"""
    nh, D, p = 3, 64, 0.25
    q, k, v, dout = attn_inputs(B, Lq, Lk, nh, nh, D, dtype)
    seed = torch.tensor([12345678901], device=DEV)
    # the multipliers themselves: uniform weights (q = 0) against unit values one key at a time
    keep = torch.empty(B, nh, Lq, Lk, device=DEV)
    for j0 in range(0, Lk, D):
        n = min(D, Lk - j0)
        eye = torch.zeros(B, Lk, nh, D, device=DEV)
        eye[:, torch.arange(j0, j0 + n), :, torch.arange(n)] = 1.0
        o = ops.CrossAttentionFn.apply(torch.zeros(B, Lq, nh, D, device=DEV), k.float().contiguous(), eye, None, None, 0.125, p, seed, 7)
        keep[..., j0:j0 + n] = o.permute(0, 2, 1, 3)[..., :n] * Lk
    keep = torch.where(keep > 0.5, 1.0 / (1.0 - p), 0.0)
    rate = float((keep == 0).float().mean())
    assert abs(rate - p) < 5 * math.sqrt(p * (1 - p) / keep.numel())
    qg, kg, vg = (t.detach().requires_grad_() for t in (q, k, v))
    o = ops.CrossAttentionFn.apply(qg, kg, vg, None, None, 0.125, p, seed, 7)
    got = [o.detach(), *torch.autograd.grad(o, [qg, kg, vg], dout)]
    want, bound = R.attention(q, k, v, 0.125, None, None, dout, keep)
    for g, w, b, n in zip(got, want, bound, ("out", "dq", "dk", "dv")):
        R.assert_within(g, w, b, n)
    flat = lambda x: x.contiguous().reshape(-1, nh * D)  # noqa: E731
    og, _ = ops.AttentionGeneralFn.apply(flat(q), flat(k), flat(v), None, None, B, Lq, Lk, nh, D, p, seed, 7)
    R.assert_within(og.view(B, Lq, nh, D), want[0], bound[0] + 1e-5, "general kernel, the same mask")
    # shared heads: each head draws its own mask
    q2, k2, v2, _ = attn_inputs(1, 30, 64, 4, 1, 64, F32)
    o = ops.CrossAttentionFn.apply(torch.zeros_like(q2), k2.contiguous(), torch.eye(64, device=DEV).view(1, 64, 1, 64).contiguous(), None, None, 0.125, p, seed, 7)
    assert abs(float((o < 1e-6).float().mean()) - p) < 0.03
    assert not torch.equal(o[:, :, 0] > 0, o[:, :, 1] > 0)
    ops.rng.manual_seed(5)
    a = ops.cross_attention(q, k, v, drop_p=p)
    b = ops.cross_attention(q, k, v, drop_p=p)
    ops.rng.manual_seed(5)
    assert torch.equal(a, ops.cross_attention(q, k, v, drop_p=p)) and not torch.equal(a, b)


def test_cross_attention_dropout_sites_and_expanded_masks():
    q, k, v, _ = attn_inputs(3, 20, 50, 4, 2, 64, BF16)
    with ops.rng.scope():
        a, b, c = (ops.cross_attention(q, k, v, drop_p=0.3, site=s) for s in (1, 2, 1))
    assert torch.equal(a, c) and not torch.equal(a, b)
    mask = normal((1, 1, 1, 50), 9)
    want = ops.cross_attention(q, k, v, key_mask=mask.expand(3, 1, 1, 50).contiguous())
    assert torch.equal(ops.cross_attention(q, k, v, key_mask=mask.expand(3, 1, 1, 50)), want)
    assert torch.equal(ops.cross_attention(q, k, v, key_mask=mask[0, 0].expand(3, 50).t().contiguous().t()), want)


# ---- streams, graphs, together --------------------------------------------------------------------------------------------------
def block(x, stream, enc, lens, P):
    """a pre-norm cross-attention sublayer for inference: norm -> e4m3 query projection, e4m3 key / value projection of the states,
    attention, e4m3 output projection"""
    B, Lq, H = x.shape
    nh, nkv, D = P["nh"], P["nkv"], P["D"]
    a, s = ops.rms_norm_fp8(x.reshape(-1, H), P["gain"], 1e-6, residual=stream.reshape(-1, H))
    q = ops.gemm_fp8_block(a, P["wq8"]).view(B, Lq, nh, D)
    kv = ops.gemm_fp8_block(ops.fp8_quantize_block(enc), P["wkv8"], bias=P["bkv"]).view(B, enc.shape[1], 2, nkv, D)
    o = ops.cross_attention(q, kv[:, :, 0], kv[:, :, 1], k_lens=lens)
    return ops.gemm_fp8_block(ops.fp8_quantize_block(o.reshape(B * Lq, nh * D)), P["wo8"]), s


def block_params(H, He, nh, nkv, D):
    P = dict(nh=nh, nkv=nkv, D=D, gain=1 + normal((H,), 1, F32, 0.1), wq=normal((nh * D, H), 2, F32, 2 * H ** -0.5), wkv=normal((2 * nkv * D, He), 3, F32, He ** -0.5),
             wo=normal((H, nh * D), 4, F32, (nh * D) ** -0.5), bkv=normal((2 * nkv * D,), 5, F32, 0.1))
    for n in ("wq", "wkv", "wo"):
        P[n + "8"] = ops.fp8_quantize_weight_block(P[n])
    return P


def block64(x, stream, enc, lens, P, quant):
    B, Lq, H = x.shape
    nh, nkv, D = P["nh"], P["nkv"], P["D"]
    rows = (lambda t: R.quant_rows(t)[0]) if quant else (lambda t: t.double())
    W = lambda n: R.quant_square(P[n])[0] if quant else P[n].double()  # noqa: E731
    y, s, _ = R.rms(x.reshape(-1, H), P["gain"], 1e-6, stream.reshape(-1, H))
    q = R.mm(rows(y), W("wq").t()).view(B, Lq, nh, D)
    kv = (R.mm(rows(enc.reshape(-1, enc.shape[2])), W("wkv").t()) + P["bkv"].double()).view(B, -1, 2, nkv, D)
    R.U.setdefault(torch.float64, 2.0 ** -53)
    o = R.attention(q, kv[:, :, 0], kv[:, :, 1], D ** -0.5, None, lens)[0][0]
    return R.mm(rows(o.reshape(B * Lq, nh * D)), W("wo").t()), s


@pytest.mark.parametrize("B,Lq,Lk", [(3, 1, 50), (2, 37, 100)])
def test_the_operators_together(B, Lq, Lk):
    H, He = 768, 1000
    P = block_params(H, He, 12, 4, 64)
    x, stream, enc = normal((B, Lq, H), 6, BF16), normal((B, Lq, H), 7, BF16, 2.0), normal((B, Lk, He), 8, BF16)
    lens = torch.tensor([Lk, Lk // 3, 1][:B], device=DEV, dtype=torch.int32)
    y, s = block(x, stream, enc, lens, P)
    want, s64 = block64(x, stream, enc, lens, P, True)
    assert torch.equal(s.view_as(s64), s64)
    # Beyond bf16 roundings (2^-8 each at q, kv, o and y), a value perturbed by 2^-8 falls on the other side of an e4m3 border in about one
    # of 16 cases and moves by a step of 2^-3: 2^-3 / sqrt(16) = 0.03 of the attention output's norm at the last quantisation
    assert float((y.double() - want).norm() / want.norm()) < 0.04


class Linear64(torch.autograd.Function):
    """linear_fp8_block's definition in 64 bits: quantised products, straight-through gradients"""

    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(x, w)
        return R.mm(R.quant_rows(x.reshape(-1, x.shape[-1]))[0], R.quant_square(w)[0].t()).view(*x.shape[:-1], -1)

    @staticmethod
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        d, f = dy.reshape(-1, dy.shape[-1]), x.reshape(-1, x.shape[-1])
        return R.mm(R.quant_rows(d)[0], R.quant_square(w)[0]).view(x.shape), R.mm(d.t(), f)


def test_the_operators_train_together():
    """gradients of the sublayer on linear_fp8_block against 64-bit autograd of the same definitions.  They differ by bf16 roundings, and by the e4m3
    borders that those push values over (0.03 of a norm each, see above): at the norm's output, o, dq and dkv: 0.03 sqrt(4) = 0.06"""
    B, Lq, Lk, H, He, nh, nkv, D = 2, 40, 70, 768, 512, 12, 4, 64
    P = block_params(H, He, nh, nkv, D)
    x, enc, dy = normal((B, Lq, H), 6, BF16), normal((B, Lk, He), 8, BF16), normal((B, Lq, H), 9, BF16)
    leaves = [t.clone().requires_grad_() for t in (x, enc, P["gain"], P["wq"], P["wkv"], P["wo"])]

    def run(x, enc, gain, wq, wkv, wo, own):
        norm = ops.rms_norm(x, gain) if own else x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6) * gain
        lin = ops.linear_fp8_block if own else Linear64.apply
        q, kv = lin(norm, wq).view(B, Lq, nh, D), lin(enc, wkv).view(B, Lk, 2, nkv, D)
        if own:
            o = ops.cross_attention(q, kv[:, :, 0], kv[:, :, 1])
        else:
            t = lambda a: a.repeat_interleave(nh // nkv, 2).transpose(1, 2)  # noqa: E731
            p = torch.softmax((q.transpose(1, 2) @ t(kv[:, :, 0]).transpose(2, 3)) * D ** -0.5, -1)
            o = (p @ t(kv[:, :, 1])).transpose(1, 2)
        return x + lin(o.reshape(B, Lq, nh * D), wo)
    got = torch.autograd.grad(run(*leaves, True), leaves, dy)
    l64 = [t.detach().double().requires_grad_() for t in leaves]
    want = torch.autograd.grad(run(*l64, False), l64, dy.double())
    for g, w, n in zip(got, want, ("x", "enc", "gain", "wq", "wkv", "wo")):
        assert torch.isfinite(g).all()
        assert float((g.double() - w).norm() / w.norm()) < 0.06, n


def test_operators_on_another_stream():
    P = block_params(768, 512, 12, 4, 64)
    x, st, enc = normal((2, 9, 768), 6, BF16), normal((2, 9, 768), 7, BF16), normal((2, 30, 512), 8, BF16)
    want = block(x, st, enc, None, P)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = block(x, st, enc, None, P)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_operators_in_a_graph():
    """captured once, replayed on new inputs with eager work between: the eager results; lengths are read at each replay; a second graph has
    workspaces of its own"""
    P = block_params(768, 512, 12, 4, 64)
    x, st, enc = normal((2, 1, 768), 6, BF16), normal((2, 1, 768), 7, BF16), normal((2, 3000, 512), 8, BF16)
    lens = torch.tensor([3000, 5], device=DEV, dtype=torch.int32)
    q, k, v, dout = attn_inputs(1, 4, 2500, 8, 2, 64, BF16)
    step = lambda: block(x, st, enc, lens, P)  # noqa: E731
    train = lambda: run_attn(q, k, v, dout)  # noqa: E731
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(), train()
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = step()
    with torch.cuda.graph(g2):
        o2 = train()
    for i in range(4):
        x.copy_(normal(x.shape, 100 + i)), q.copy_(normal(q.shape, 200 + i)), lens.copy_(torch.tensor([3000 - 700 * i, 2999 * (i % 2)], dtype=torch.int32))
        g1.replay(), g2.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(o1, step())) and all(torch.equal(a, b) for a, b in zip(o2, train()))


def test_training_in_a_graph():
    """forward and backward of the sublayer's three operators captured together, gradients into .grad; replayed on new inputs with eager work between"""
    B, Lq, Lk, H, nh, nkv, D = 2, 9, 1500, 96, 4, 2, 32
    x, enc, dy = normal((B, Lq, H), 1, BF16), normal((B, Lk, H), 2, BF16), normal((B, Lq, H), 3, BF16)
    mask = torch.zeros(B, 1, 1, Lk, device=DEV)
    P = [1 + normal((H,), 4, F32, 0.1), normal((nh * D, H), 5, F32, 0.2), normal((2 * nkv * D, H), 6, F32, 0.1), normal((H, nh * D), 7, F32, 0.1), normal((H,), 8)]

    def step(leaves):
        gain, wq, wkv, wo, bo = leaves
        y, s = ops.rms_norm(x, gain, residual=x)
        kv = ops.linear_fp8_block(enc, wkv).view(B, Lk, 2, nkv, D)
        o = ops.cross_attention(ops.linear_fp8_block(y, wq).view(B, Lq, nh, D), kv[:, :, 0], kv[:, :, 1], key_mask=mask)
        out = s + ops.linear_fp8_block(o.view(B, Lq, nh * D), wo, bo)
        out.backward(dy)
        return out.detach()

    def eager():
        leaves = [p.detach().clone().requires_grad_() for p in P]
        out = step(leaves)
        return [out] + [p.grad for p in leaves]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        eager()
    torch.cuda.synchronize()
    leaves = [p.detach().requires_grad_() for p in P]                                    # no graph of theirs is alive
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(leaves)
    for i in range(4):
        x.copy_(normal(x.shape, 10 + i)), dy.copy_(normal(dy.shape, 20 + i)), mask.masked_fill_(torch.rand(mask.shape, generator=gen(i), device=DEV) < 0.1, -1e30)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip([out] + [p.grad for p in leaves], eager()))


def test_capture_beside_an_eager_graph_of_the_same_leaves_is_refused(monkeypatch):
    """(nothing is captured here: the operators are told so on another stream, and refuse before anything is launched)"""
    q, k, v, _ = attn_inputs(1, 3, 9, 2, 2, 64, BF16)
    x, xb, w, g = normal((4, 96), 1), normal((4, 96), 1, BF16), normal((8, 96), 2), torch.ones(96, device=DEV)
    side = torch.cuda.Stream()
    for f, *leaves in ((ops.cross_attention, q, k, v), (ops.rms_norm, x, g), (ops.linear_fp8_block, xb, w)):
        leaves = [t.detach().requires_grad_() for t in leaves]
        eager = f(*leaves)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            out = f(*leaves)
            own = [t.detach().requires_grad_() for t in leaves]
            out2 = f(*own)
            d = torch.ones_like(out)
            with monkeypatch.context() as m:
                m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
                with pytest.raises(_lib.Uc2Error, match="eager graph"):
                    torch.autograd.grad(out, leaves, d)
                b = torch.autograd.grad(out2, own, d)
        torch.cuda.synchronize()
        assert all(torch.equal(s, t) for s, t in zip(b, torch.autograd.grad(eager, leaves, d)))


def test_the_accumulation_of_a_leaf_is_known_whoever_made_it(monkeypatch):
    """by another operation, held by a wrapper, behind a cast: the default stream's is refused, a stream's own is not (no real capture here)"""
    w, x = normal((8, 96), 2), normal((4, 96), 1, BF16)
    side = torch.cuda.Stream()
    made = {"another operation": lambda t: t * 3, "a wrapper": lambda t: t.expand_as(t).grad_fn.next_functions[0][0], "the same operator behind a cast": lambda t: ops.linear_fp8_block(x, t.to(BF16))}
    uses = {"direct": lambda t: ops.linear_fp8_block(x, t), "behind a cast": lambda t: ops.linear_fp8_block(x, t.to(BF16)), "behind a view of a product": lambda t: ops.linear_fp8_block(x, (2 * t).view(8, 96))}
    for what, make in made.items():
        for how, use in uses.items():
            leaf = w.detach().requires_grad_()
            assert _lib.accumulation_stream(leaf) is None
            held = make(leaf)
            torch.cuda.synchronize()
            assert _lib.accumulation_stream(leaf) == 0
            with torch.cuda.stream(side):
                out = use(leaf)
                with monkeypatch.context() as m:
                    m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
                    with pytest.raises(_lib.Uc2Error, match="eager graph"):
                        torch.autograd.grad(out, [leaf], torch.ones_like(out))
            torch.cuda.synchronize()
            del held, out
            with torch.cuda.stream(side):                          # made on the stream itself: nothing to refuse
                held = make(leaf)
                out = use(leaf)
                with monkeypatch.context() as m:
                    m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
                    g, = torch.autograd.grad(out, [leaf], torch.ones_like(out))
            torch.cuda.synchronize()
            assert torch.isfinite(g).all(), (what, how)
            del held, out


def test_training_in_a_graph_behind_other_operations():
    """a captured pass whose leaves reach the operators through a cast and a product, after another operation of the same capture has used them"""
    x, w32, gain, dy = normal((9, 96), 1, BF16), normal((40, 96), 2), 1 + normal((96,), 3, F32, 0.1), normal((9, 40), 4, BF16)

    def step(w, g):
        squares = w * w
        out = ops.linear_fp8_block(ops.rms_norm(x, 2 * g), w.to(BF16))
        torch.autograd.backward([out, squares], [dy, torch.ones_like(squares)])
        return [out.detach(), w.grad, g.grad]
    leaves = lambda: [t.detach().requires_grad_() for t in (w32, gain)]  # noqa: E731
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(*leaves())
    torch.cuda.synchronize()
    own, graph = leaves(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*own)
    for i in range(4):
        x.copy_(normal(x.shape, 10 + i, BF16)), dy.copy_(normal(dy.shape, 20 + i, BF16))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step(*leaves())))


def test_saved_tensors_that_come_back_where_they_were_with_other_strides():
    buf = normal((2, 9, 3, 4, 64), 1, BF16)
    q, (_, k, v, dout) = buf[:, :, 0], attn_inputs(2, 9, 70, 4, 2, 64, BF16)[0:4]
    want = run_attn(q.clone(), k, v, dout)

    def pack(t):
        return t.clone(memory_format=torch.contiguous_format), t.data_ptr()

    def unpack(p):
        if p[1] != buf.data_ptr():
            return p[0]
        buf.view(-1)[:p[0].numel()].copy_(p[0].view(-1))
        return buf.view(-1)[:p[0].numel()].view(p[0].shape)
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        qg = q.detach().requires_grad_()
        o = ops.cross_attention(qg, k, v)
    assert torch.equal(torch.autograd.grad(o, [qg], dout)[0], want[1])


def test_saved_tensors_that_come_back_with_gaps():
    """saved-tensor hooks that bring every tensor back with a stride of two in its last dimension, or as columns: the gradients of the tensors themselves"""
    def gaps(t):
        return torch.stack([t, t], -1)[..., 0]

    def columns(t):
        return t.transpose(0, -1).contiguous().transpose(0, -1)
    q, k, v, dout = attn_inputs(2, 9, 70, 4, 2, 64, BF16)
    mask, lens = normal((2, 70), 9), torch.tensor([70, 33], device=DEV, dtype=torch.int32)
    x, w, b, dy = normal((9, 96), 1, BF16), normal((40, 96), 2), normal((40,), 3), normal((9, 40), 4, BF16)
    gain, dn = 1 + normal((96,), 5, F32, 0.1), normal((9, 96), 6, BF16)

    def run(unpack):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), unpack):
            leaves = [t.detach().requires_grad_() for t in (q, k, v, x, w, b, gain, x)]
            o16 = ops.cross_attention(*leaves[:3], key_mask=mask, k_lens=lens)
            o32 = ops.cross_attention(*(t.float() for t in leaves[:3]), key_mask=mask, k_lens=lens, drop_p=0.2)
            y = ops.linear_fp8_block(*leaves[3:6])
            n, s = ops.rms_norm(leaves[7], leaves[6], residual=x)
        return torch.autograd.grad([o16, o32, y, n, s], leaves, [dout, dout.float(), dy, dn, dn])
    ops.rng.manual_seed(4)
    want = run(lambda t: t)
    for unpack in (gaps, columns):
        ops.rng.manual_seed(4)
        assert all(torch.equal(a, c) for a, c in zip(run(unpack), want)), unpack.__name__


def test_saved_tensors_that_come_back_as_copies():
    """saved-tensor hooks (offloading): the backward reads what they bring, not the tensors of the forward"""
    q, k, v, dout = attn_inputs(2, 9, 70, 4, 2, 64, BF16)
    want = run_attn(q, k, v, dout)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(DEV)):
        qg, kg, vg = (t.detach().requires_grad_() for t in (q, k, v))
        o = ops.cross_attention(qg, kg, vg)
        x, g = normal((9, 96), 1).requires_grad_(), torch.ones(96, device=DEV, requires_grad=True)
        y, s = ops.rms_norm(x, g, residual=x.detach())
    got = torch.autograd.grad(o, [qg, kg, vg], dout)
    assert all(torch.equal(a, b) for a, b in zip(got, want[1:]))
    x2 = x.detach().clone().requires_grad_()
    y2, s2 = ops.rms_norm(x2, g, residual=x2.detach())
    assert torch.equal(torch.autograd.grad([y, s], [x], [y, s])[0], torch.autograd.grad([y2, s2], [x2], [y2, s2])[0])


def test_second_derivatives_are_refused():
    q, k, v, dout = attn_inputs(1, 3, 9, 2, 2, 64, F32)
    x, g = normal((4, 96), 1).requires_grad_(), torch.ones(96, device=DEV, requires_grad=True)
    qg = q.clone().requires_grad_()
    xb, w = normal((4, 96), 1, BF16).requires_grad_(), normal((8, 96), 2).requires_grad_()
    for out, leaf in ((ops.cross_attention(qg, k, v), qg), (ops.rms_norm(x, g), x), (ops.linear_fp8_block(xb, w).float(), xb)):
        d, = torch.autograd.grad(out.square().sum(), [leaf], create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(d.float().sum(), [leaf])


def test_refusals_on_the_device():
    q, k, v, _ = attn_inputs(2, 3, 9, 4, 2, 64, BF16)
    for bad in (dict(key_mask=torch.zeros(2, 8, device=DEV)), dict(key_mask=torch.zeros(2, 9, device=DEV, dtype=torch.bool)), dict(k_lens=torch.zeros(3, device=DEV, dtype=torch.int32)),
                dict(k_lens=torch.zeros(2, device=DEV)), dict(drop_p=1.0), dict(k_lens=[1, 2]), dict(key_mask=torch.zeros(2, 9))):
        with pytest.raises(_lib.Uc2Error):
            ops.cross_attention(q, k, v, **bad)
    for a, b, c in ((q, k, v[:, :8]), (q.float(), k, v), (q[..., :48], k[..., :48], v[..., :48]), (q[:, :, :3], k, v), (q, k[:1], v[:1]), (q[0], k, v), (q.half(), k.half(), v.half())):
        with pytest.raises(_lib.Uc2Error):
            ops.cross_attention(a, b, c)
    x, w = normal((4, 300), 1, BF16), normal((70, 300), 2)
    a, b = ops.fp8_quantize_block(x), ops.fp8_quantize_weight_block(w)
    for bad in ((ops.fp8_quantize_block(x[:, :200]), b), (a, b[:1] + (b.scale[:, :1],)), (b, a), (ops.BlockRows(a.data[:2], a.scale, 300), b), (ops.BlockRows(a.data[:, :256], a.scale, 256), b)):
        with pytest.raises(_lib.Uc2Error):
            ops.gemm_fp8_block(*bad)
    for bias in (torch.zeros(69, device=DEV), torch.zeros(70, device=DEV, dtype=BF16), torch.zeros(70)):
        with pytest.raises(_lib.Uc2Error):
            ops.gemm_fp8_block(a, b, bias=bias)
    for args in ((x.float(), w), (x, w[:, :200]), (x, w[0]), (x, w.half())):
        with pytest.raises(_lib.Uc2Error):
            ops.linear_fp8_block(*args)
    g = torch.ones(300, device=DEV)
    for args, kw in (((x, g[:200]), {}), ((x, g.to(BF16)), {}), ((x, g), dict(residual=x[:2])), ((x, g), dict(residual=x.float())), ((x.half(), g), {}),
                     ((torch.zeros(2, 16385, device=DEV), torch.zeros(16385, device=DEV)), {})):
        with pytest.raises(_lib.Uc2Error):
            ops.rms_norm(*args, **kw)
    with pytest.raises(_lib.Uc2Error):
        ops.rms_norm_fp8(x.clone().requires_grad_(), g)
