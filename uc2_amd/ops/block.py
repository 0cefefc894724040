"""e4m3 under power-of-two scales for blocks of 128 (quantisation, the product, a linear layer on them) and the root-mean-square norm that
writes such an operand.  Part of uc2_amd.ops.

Beside the per-tensor mode of ops/fp8.py: a block's scale comes from the block itself, so a call needs no history of its tensor and no
maximum pass, single tokens and first calls are as exact as any other, and an outlier costs the precision of its own 128 values only."""
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .._lib import call, dt, ptr, stream
from .base import _Timed, _require_cuda, device_guard
from .linear import colsum_accum

BLOCK = 128


class BlockRows(NamedTuple):
    """a [rows, cols] matrix as e4m3 under 1 x 128 block scales: the left operand of gemm_fp8_block"""
    data: torch.Tensor            # uint8 [rows, cols rounded up to 128], zeros behind cols
    scale: torch.Tensor           # int32 [ceil(padded cols / 512), rows]: four neighbouring blocks' exponents + 127 per word
    cols: int


class BlockWeight(NamedTuple):
    """a [rows, cols] weight as e4m3 under 128 x 128 block scales: the right operand of gemm_fp8_block"""
    data: torch.Tensor            # uint8 [rows, cols rounded up to 128], zeros behind cols
    scale: torch.Tensor           # uint8 [ceil(rows / 128), ceil(cols / 128)]: exponent + 127


def _up(n):
    return (n + BLOCK - 1) // BLOCK * BLOCK


def _float_matrix(x, what):
    """x as [rows, last dimension] with contiguous columns"""
    if not torch.is_tensor(x) or x.dim() < 1:
        raise _lib.Uc2Error("%s: a tensor of one dimension at least is needed" % what)
    _require_cuda(x)
    dt(x.dtype)
    x2 = x.reshape(-1, x.shape[-1]) if x.dim() != 2 else x
    if x2.shape[1] < 1:
        raise _lib.Uc2Error("%s: the last dimension is empty" % what)
    return x2 if x2.stride(1) == 1 and (x2.stride(0) >= x2.shape[1] or x2.shape[0] <= 1) else x2.contiguous()


def _rows_out(M, K, device):
    Kp = _up(K)
    return (torch.empty((M, Kp), dtype=torch.uint8, device=device), torch.empty(((Kp + 511) // 512, M), dtype=torch.int32, device=device))


def fp8_quantize_block(x):
    """[..., K] (fp32 or bf16, any row stride) -> BlockRows of its rows, one launch"""
    x2 = _float_matrix(x, "fp8_quantize_block")
    M, K = x2.shape
    with device_guard(x2):
        q, s = _rows_out(M, K, x2.device)
        call("uc2_fp8_quant_rows", dt(x2.dtype), M, K, ptr(x2), max(x2.stride(0), K), ptr(q), ptr(s), stream())
    return BlockRows(q, s, K)


def fp8_quantize_weight_block(w, transpose=False):
    """[N, K] weight (fp32 or bf16) -> BlockWeight; transpose: also that of W^T with the same values (the operand of the input gradient),
    both from one read"""
    if not torch.is_tensor(w) or w.dim() != 2:
        raise _lib.Uc2Error("fp8_quantize_weight_block: a weight of two dimensions is needed")
    w = _float_matrix(w, "fp8_quantize_weight_block")
    N, K = w.shape
    Np, Kp = _up(N), _up(K)
    with device_guard(w):
        new = lambda *s: torch.empty(s, dtype=torch.uint8, device=w.device)  # noqa: E731
        q, s = new(N, Kp), new(Np // BLOCK, Kp // BLOCK)
        qt, st = (new(K, Np), new(Kp // BLOCK, Np // BLOCK)) if transpose else (None, None)
        call("uc2_fp8_quant_square", dt(w.dtype), N, K, ptr(w), max(w.stride(0), K), ptr(q), ptr(s), ptr(qt), ptr(st), stream())
    return (BlockWeight(q, s), BlockWeight(qt, st)) if transpose else BlockWeight(q, s)


def _block_bias(bias, N, device):
    if bias is None:
        return None
    if bias.dtype != torch.float32 or bias.dim() != 1 or bias.shape[0] != N or bias.device != device:
        raise _lib.Uc2Error("bias must be fp32 [%d] on %s" % (N, device))
    return bias if bias.is_contiguous() else bias.contiguous()


def gemm_fp8_block(a, b, bias=None):
    """bf16 [M, N] = a b^T + bias of a = BlockRows [M, K] (fp8_quantize_block, rms_norm_fp8) and b = BlockWeight [N, K]
    (fp8_quantize_weight_block; any (data, scale) pair of that layout); fp32 sums, one rounding"""
    a8, sa = a[0], a[1]
    b8, sb = b[0], b[1]
    for t, kind, what in ((a8, torch.uint8, "a.data"), (sa, torch.int32, "a.scale"), (b8, torch.uint8, "b.data"), (sb, torch.uint8, "b.scale")):
        if t.dtype != kind or t.dim() != 2:
            raise _lib.Uc2Error("gemm_fp8_block: %s must be a two-dimensional %s tensor" % (what, kind))
        _require_cuda(t)
        if t.device != a8.device:
            raise _lib.Uc2Error("gemm_fp8_block: operands on %s and %s" % (a8.device, t.device))
    (M, Kp), N = a8.shape, b8.shape[0]
    if Kp % BLOCK or Kp == 0 or b8.shape[1] != Kp or tuple(sa.shape) != ((Kp + 511) // 512, M) or tuple(sb.shape) != ((N + BLOCK - 1) // BLOCK, Kp // BLOCK):
        raise _lib.Uc2Error("gemm_fp8_block: shapes do not match: %s with scales %s against %s with scales %s"
                            % (tuple(a8.shape), tuple(sa.shape), tuple(b8.shape), tuple(sb.shape)))
    if not (a8.is_contiguous() and sa.is_contiguous() and b8.is_contiguous() and sb.is_contiguous()):
        raise _lib.Uc2Error("gemm_fp8_block: operands must be contiguous")
    bias = _block_bias(bias, N, a8.device)
    with device_guard(a8):
        out = torch.empty((M, N), dtype=torch.bfloat16, device=a8.device)
        call("uc2_gemm_fp8_block", M, N, Kp, ptr(a8), Kp, ptr(sa), max(M, 1), ptr(b8), Kp, ptr(sb), ptr(bias), ptr(out), max(N, 1), stream())
    return out


class LinearBlockFp8Fn(torch.autograd.Function):
    """y = q(x) q(W)^T + b, gradients straight through the quantisation: dx = q(dy) q(W) on the transposed copy of the same weight values,
    dW = dy^T x and db = sum dy from the unquantised bf16 tensors (the weight gradient stays bf16, as in the per-tensor mode)"""

    @staticmethod
    def forward(ctx, x, weight, bias):
        shp = x.shape
        x2 = _float_matrix(x, "linear_fp8_block")
        need_dx = ctx.needs_input_grad[0]
        w = fp8_quantize_weight_block(weight, transpose=need_dx)
        wt = None
        if need_dx:
            w, wt = w
        y = gemm_fp8_block(fp8_quantize_block(x2), w, bias)
        ctx.save_for_backward(x2 if ctx.needs_input_grad[1] else None, *((wt.data, wt.scale) if wt is not None else (None, None)))
        ctx.cfg = (shp, tuple(weight.shape), weight.dtype, bias is not None)
        return y.view(*shp[:-1], weight.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x2, wt, st = ctx.saved_tensors
        shp, (N, K), wtype, _ = ctx.cfg
        dy2 = _float_matrix(dy, "linear_fp8_block")
        M = dy2.shape[0]
        dx = dw = db = None
        with device_guard(dy2):
            if ctx.needs_input_grad[0]:
                dx = gemm_fp8_block(fp8_quantize_block(dy2), BlockWeight(wt, st)).view(shp)
            need_db = ctx.needs_input_grad[2]
            if ctx.needs_input_grad[1] and M:
                dw = torch.empty((N, K), dtype=torch.float32, device=dy2.device)
                db = torch.empty(N, dtype=torch.float32, device=dy2.device) if need_db else None
                n = _lib.load().uc2_linear_wgrad_workspace(M, N, K)
                ws = torch.empty(n, dtype=torch.uint8, device=dy2.device) if n else None
                call("uc2_linear_wgrad", M, N, K, ptr(dy2), dy2.stride(0), ptr(x2), x2.stride(0), ptr(dw), K, ptr(db), ptr(ws), n, stream())
            else:
                if ctx.needs_input_grad[1]:
                    dw = torch.zeros((N, K), dtype=torch.float32, device=dy2.device)
                if need_db:
                    db = torch.zeros(N, dtype=torch.float32, device=dy2.device)
                    if M:
                        colsum_accum(dy2, db)
            if dw is not None and wtype != torch.float32:
                dw = dw.to(wtype)
        return dx, dw, db


def linear_fp8_block(x, weight, bias=None):
    """bf16 x [..., K], weight [N, K] (fp32 or bf16), bias fp32 [N] or None -> bf16 [..., N]: a linear layer whose forward and input-gradient
    products run on e4m3 operands with block scales.  The weight is quantised in the call (a weight that does not change: quantise it
    once with fp8_quantize_weight_block and call gemm_fp8_block)."""
    if not torch.is_tensor(x) or x.dtype != torch.bfloat16 or x.dim() < 1:
        raise _lib.Uc2Error("linear_fp8_block computes on bf16 activations")
    _require_cuda(x)
    if not torch.is_tensor(weight) or weight.dim() != 2 or weight.shape[1] != x.shape[-1] or weight.shape[0] < 1:
        raise _lib.Uc2Error("linear_fp8_block: weight [N, %d] expected, got %s" % (x.shape[-1], tuple(getattr(weight, "shape", ()))))
    if weight.device != x.device:
        raise _lib.Uc2Error("linear_fp8_block: x on %s, weight on %s" % (x.device, weight.device))
    dt(weight.dtype)
    _block_bias(bias, weight.shape[0], x.device)
    return LinearBlockFp8Fn.apply(x, weight, bias)


# ---- root-mean-square norm ----------------------------------------------------------------------------------------------------------
def _rms_args(x, weight, residual, what):
    if not torch.is_tensor(x) or x.dim() < 1:
        raise _lib.Uc2Error("%s: a tensor of one dimension at least is needed" % what)
    _require_cuda(x)
    H = x.shape[-1]
    dt(x.dtype)
    if weight.dtype != torch.float32 or tuple(weight.shape) != (H,) or weight.device != x.device:
        raise _lib.Uc2Error("%s: weight must be fp32 [%d] on %s" % (what, H, x.device))
    if not 1 <= H <= 16384:
        raise _lib.Uc2Error("%s: rows of 1 to 16384 elements, got %d" % (what, H))
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise _lib.Uc2Error("%s: residual must have the shape, type and device of x" % what)
    return H


def _rms_fwd(x, weight, eps, residual, want_y, want_rstd, want_q):
    H = x.shape[-1]
    x2 = x.reshape(-1, H).contiguous()
    r2 = None if residual is None else residual.reshape(-1, H).contiguous()
    w = weight.contiguous()
    M = x2.shape[0]
    s = torch.empty_like(x2) if r2 is not None else None
    y = torch.empty_like(x2) if want_y else None
    rstd = torch.empty(M, dtype=torch.float32, device=x.device) if want_rstd else None
    q, qs = _rows_out(M, H, x.device) if want_q else (None, None)
    with _Timed("rms_fwd", x2.element_size() * M * H * (1 + (2 if r2 is not None else 0) + int(want_y)) + (M * H if want_q else 0)):
        call("uc2_rms_fwd", dt(x2.dtype), M, H, ptr(x2), ptr(r2), ptr(w), float(eps), ptr(s), ptr(y), ptr(rstd), ptr(q), ptr(qs), stream())
    return x2 if s is None else s, y, rstd, None if q is None else BlockRows(q, qs, H)


class RMSNormFn(torch.autograd.Function):
    """(y, s) with s = x + residual (rounded to the tensors' type), y = s / sqrt(mean(s^2) + eps) * weight; (y,) without a residual"""

    @staticmethod
    def forward(ctx, x, weight, eps, residual):
        grad = any(ctx.needs_input_grad)
        with device_guard(x):
            s, y, rstd, _ = _rms_fwd(x, weight, eps, residual, True, grad, False)
        if grad:
            ctx.save_for_backward(s, weight, rstd)
        ctx.set_materialize_grads(False)
        ctx.shp, ctx.res = x.shape, residual is not None
        return (y.view(x.shape), s.view(x.shape)) if residual is not None else y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, ds=None):
        s, weight, rstd = ctx.saved_tensors
        M, H = s.shape
        if dy is None:                                   # only the stream is used
            return ds, torch.zeros_like(weight) if ctx.needs_input_grad[1] else None, None, ds
        with device_guard(s):
            dy2 = dy.reshape(-1, H).contiguous()
            ds2 = None if ds is None else ds.reshape(-1, H).contiguous()
            dx = torch.empty_like(s)
            dw = ws = None
            if ctx.needs_input_grad[1]:
                dw = torch.empty(H, dtype=torch.float32, device=s.device)
                ws = torch.empty(max(_lib.load().uc2_rms_bwd_workspace(M, H), 4), dtype=torch.uint8, device=s.device)
            with _Timed("rms_bwd", s.element_size() * M * H * (3 + (ds2 is not None))):
                call("uc2_rms_bwd", dt(s.dtype), M, H, ptr(dy2), ptr(ds2), ptr(s), ptr(weight.contiguous()), ptr(rstd), ptr(dx), ptr(dw), ptr(ws),
                     0 if ws is None else ws.numel(), stream())
        dx = dx.view(ctx.shp)
        return dx if ctx.needs_input_grad[0] else None, dw, None, dx if ctx.res and ctx.needs_input_grad[3] else None


def rms_norm(x, weight, eps=1e-6, residual=None):
    """root-mean-square norm over the last dimension (fp32 or bf16, weight fp32): y, or (y, s) with s = x + residual, the stream to carry on"""
    _rms_args(x, weight, residual, "rms_norm")
    return RMSNormFn.apply(x, weight, eps, residual)


def rms_norm_fp8(x, weight, eps=1e-6, residual=None):
    """the norm as an operand of gemm_fp8_block: (BlockRows of y [rows, H], s) with s as in rms_norm (x's values in its shape without a
    residual); y itself is never written.  No gradient: for inference (training: rms_norm, then linear_fp8_block)."""
    _rms_args(x, weight, residual, "rms_norm_fp8")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise _lib.Uc2Error("rms_norm_fp8 has no gradient: call it under torch.no_grad(), or use rms_norm and linear_fp8_block")
    with device_guard(x):
        s, _, _, q = _rms_fwd(x, weight, eps, residual, False, False, True)
    return q, x if residual is None else s.view(x.shape)
