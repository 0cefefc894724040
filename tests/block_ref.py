"""Plain 64-bit forms of the block-scaled e4m3 format, the root-mean-square norm and the cross attention (tests only), each with a bound on
how far a kernel may be off: a sum of the roundings it makes, value by value.  U[t] is half a step of type t relative to the value."""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, "e4m3": 2.0 ** -4}
F64 = torch.float64


def block_exponents(amax):
    """biased byte of the smallest e with amax <= 448 2^e (search over all of them, no logarithm)"""
    e = torch.arange(1, 255, device=amax.device)
    fits = amax.double()[..., None] <= 448.0 * torch.exp2((e - 127).double())
    return 1 + fits.to(torch.int8).argmax(-1)


def e4m3(x):
    """nearest e4m3 value, halves to even; |x| <= 448"""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def quant_rows(x):
    """(values [M, K] in 64 bits, biased exponents [M, ceil(K / 128)])"""
    M, K = x.shape
    p = torch.nn.functional.pad(x.double(), (0, -K % 128)).reshape(M, -1, 128)
    e = block_exponents(p.abs().amax(-1))
    s = torch.exp2((e - 127).double())[..., None]
    return (e4m3(p / s) * s).reshape(M, -1)[:, :K], e


def quant_square(w):
    N, K = w.shape
    p = torch.nn.functional.pad(w.double(), (0, -K % 128, 0, -N % 128))
    p = p.reshape(p.shape[0] // 128, 128, -1, 128)
    e = block_exponents(p.abs().amax((1, 3)))
    s = torch.exp2((e - 127).double())[:, None, :, None]
    return (e4m3(p / s) * s).reshape(p.shape[0] * 128, -1)[:N, :K], e


def rows_values(a):
    """what a BlockRows stands for, [M, cols], and its exponents [M, blocks]"""
    M, Kp = a.data.shape
    word = a.scale.to(torch.int64) & 0xFFFFFFFF
    e = torch.stack([(word >> (8 * i)) & 255 for i in range(4)], -1).permute(1, 0, 2).reshape(M, -1)[:, :Kp // 128]
    v = a.data.view(torch.float8_e4m3fn).double().reshape(M, -1, 128) * torch.exp2((e - 127).double())[..., None]
    return v.reshape(M, Kp)[:, :a.cols], e


def weight_values(b, K):
    N, Kp = b.data.shape
    e = b.scale.to(torch.int64)
    s = torch.exp2((e - 127).double()).repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)
    return (b.data.view(torch.float8_e4m3fn).double() * s)[:, :K]


def mm(a, b):
    return torch.matmul(a, b.contiguous())


def gemm_bound(a, b, out):
    """one rounding to bf16, fp32 sums of K terms, and the matrix instruction's own arithmetic: it adds the 128 products of a block aligned to the
    largest of their group and cuts what lies below 2^-13 of that one's power of two (products 16 * 16 and -16 * 16 beside 2^-j: 2^-5 arrives, 1.75 2^-4
    arrives as 1.5 2^-4, 2^-6 is gone; what is added block after block is not cut).  So each product is off by less than 2^-13 of its group's
    largest, that is at most the product of the two operands' maxima over the block: 128 2^-13 = 2^-6 of it per block."""
    def tops(x):
        return torch.nn.functional.pad(x.abs(), (0, -x.shape[1] % 128)).reshape(x.shape[0], -1, 128).amax(-1)
    return 2 * a.shape[1] * U[torch.float32] * mm(a.abs(), b.abs().t()) + 2.0 ** -6 * mm(tops(a), tops(b).t()) + U[torch.bfloat16] * out.abs() + 1e-37


def assert_gemm(got, a, b, bias=None, what=""):
    """within gemm_bound, and as a whole: a rounding's error is spread over +-2^-8, at most 2^-8 / sqrt(3) = 2.3e-3 of the norm; the cut ones add
    up like 128 random signs of 2^-14 of a maximum that is some 8 times a product's size: sqrt(128) 2^-14 8 / sqrt(128) = 5e-4.  Together below 2^-8
    = 3.9e-3 (single values may all round the same way: from 64 values on)."""
    want = mm(a, b.t()) + (0 if bias is None else bias.double())
    assert_within(got, want, gemm_bound(a, b, want) + (0 if bias is None else U[torch.float32] * bias.abs().double()), what)
    if want.numel() >= 64:
        err = float((got.double() - want).norm() / want.norm())
        assert err < 2.0 ** -8, "%s: off by %.2e of the norm" % (what, err)


def rms(x, w, eps, residual=None):
    s = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    d = s.double()
    r = 1.0 / torch.sqrt(d.pow(2).mean(-1, keepdim=True) + eps)
    return d * r * w.double(), s, r


def rms_rel(H):
    """relative error of rstd in fp32: half of the H additions', and the division, root and reciprocal"""
    return (H / 2 + 4) * U[torch.float32]


def attention(q, k, v, scale, key_mask=None, k_lens=None, dout=None, keep=None):
    """(out, dq, dk, dv) in 64 bits and a bound for each.  keep [B, nh, Lq, Lk]: multiplier of each weight (dropout)"""
    t = q.dtype
    u, u32 = U[t], U[torch.float32]
    B, Lq, nh, D = q.shape
    Lk, nkv = k.shape[1], k.shape[2]
    G = nh // nkv
    gone = torch.zeros(B, Lk, dtype=torch.bool, device=q.device)
    bias = torch.zeros(B, Lk, dtype=F64, device=q.device)
    if k_lens is not None:
        gone |= torch.arange(Lk, device=q.device) >= k_lens.long()[:, None]
    if key_mask is not None:
        gone |= key_mask <= -1e30
        bias = key_mask.double()
    bias = torch.where(gone, torch.zeros_like(bias), bias)[:, None, None, :]
    clean = lambda x: torch.where(gone[:, :, None, None], torch.zeros_like(x), x).double().permute(0, 2, 1, 3).repeat_interleave(G, 1)  # noqa: E731
    Q, K, V = q.double().permute(0, 2, 1, 3), clean(k), clean(v)
    x = mm(Q, K.transpose(2, 3)) * scale + bias
    part = ~gone[:, None, None, :]
    x = torch.where(part, x, torch.full_like(x, -math.inf))
    top = x.amax(-1, keepdim=True) if Lk else torch.zeros(B, nh, Lq, 1, dtype=F64, device=q.device)
    p = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    z = p.sum(-1, keepdim=True)
    p = torch.where(z > 0, p / z.clamp_min(1e-300), torch.zeros_like(p))
    kp = torch.ones_like(p) if keep is None else keep.double()
    o = mm(p * kp, V)
    # relative error of a weight: its score (D products, in fp32) and exponent, twice (the maximum's / the log-sum's too), and the sum over the keys
    mag = (mm(Q.abs(), K.abs().transpose(2, 3)) * abs(scale)).amax(-1, keepdim=True) + bias.abs().amax() + 4 if Lk else torch.zeros_like(top)
    ep = (2 * (D + 8) * mag + 2 * Lk + 16) * u32
    up = u if t == torch.bfloat16 else 0.0                          # the weights' rounding in front of the second product
    tiny = 2.0 ** -125                                              # weights (and ds) below the smallest normal number, 2^-126, become zero
    eo = (up + ep + 2 * Lk * u32) * mm(p * kp, V.abs()) + u * o.abs() + tiny * V.abs().sum(2, keepdim=True)
    back = lambda y: y.permute(0, 2, 1, 3)  # noqa: E731
    res = [back(o)], [back(eo)]
    if dout is None:
        return res
    dO = dout.double().permute(0, 2, 1, 3)
    dp = mm(dO, V.transpose(2, 3)) * kp
    delta = (dO * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    # an error of ds: of p, of delta (out's bound before its rounding, and its sum over D), of dp's sum over D, and ds's own rounding
    edelta = (dO.abs() * (eo - u * o.abs() + 4 * u32 * o.abs())).sum(-1, keepdim=True) + 2 * D * u32 * (dO.abs() * o.abs()).sum(-1, keepdim=True)
    eds = p * (edelta + 2 * D * u32 * mm(dO.abs(), V.abs().transpose(2, 3)) * kp) + (ep + up) * ds.abs() + (ep * p + tiny) * (dp.abs() + delta.abs()) + tiny
    dq = mm(ds, K) * scale
    edq = mm(eds + 2 * Lk * u32 * ds.abs(), K.abs()) * abs(scale) + u * dq.abs()
    shared = lambda y: back(y.reshape(B, nkv, G, Lk, D).sum(2))  # noqa: E731
    n = 2 * Lq * G * u32
    dk, dv = mm(ds.transpose(2, 3), Q) * scale, mm((p * kp).transpose(2, 3), dO)
    edk = shared(mm((eds + n * ds.abs()).transpose(2, 3), Q.abs()) * abs(scale)) + u * shared(dk).abs()
    edv = shared(mm(((up + ep + n) * p * kp + tiny).transpose(2, 3), dO.abs())) + u * shared(dv).abs()
    return [back(o), back(dq), shared(dk), shared(dv)], [back(eo), back(edq), edk, edv]


def assert_within(got, want, bound, what="", slack=1.01):
    assert got.shape == want.shape, "%s: %s against %s" % (what, tuple(got.shape), tuple(want.shape))
    d = (got.double() - want).abs()
    assert torch.isfinite(got).all(), "%s: not finite" % what
    over = d > slack * bound + 1e-37
    if over.any():
        i = torch.argmax(d - slack * bound)
        raise AssertionError("%s: %d of %d values beyond their bound; worst %.6e for %.6e, off %.3e, bound %.3e" % (
            what, int(over.sum()), d.numel(), got.double().reshape(-1)[i], want.reshape(-1)[i], d.reshape(-1)[i], bound.reshape(-1)[i]))
