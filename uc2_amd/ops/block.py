"""e4m3 under power-of-two scales for blocks of 128 (quantisation, the product, a linear layer on them) and the root-mean-square norm that
writes such an operand.  Part of uc2_amd.ops.

Beside the per-tensor mode of ops/fp8.py: a block's scale comes from the block itself, so a call needs no history of its tensor and no
maximum pass, single tokens and first calls are as exact as any other, and an outlier costs the precision of its own 128 values only."""
from typing import NamedTuple

import torch

from .. import _lib
from .._lib import call, dt, ptr, stream
from ..config import state
from .base import _Timed, _require_cuda, device_guard, note_leaves, once

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


def _no_gradient(what, instead, *tensors):
    """refuses tensors whose gradient would be lost without a word"""
    if torch.is_grad_enabled() and any(torch.is_tensor(t) and t.requires_grad for t in tensors):
        raise _lib.Uc2Error("%s has no gradient: call it under torch.no_grad(), or use %s" % (what, instead))


def _rows_out(M, K, x):
    Kp = _up(K)
    return x.new_empty((M, Kp), dtype=torch.uint8), x.new_empty(((Kp + 511) // 512, M), dtype=torch.int32)


def _quant_rows(x2):
    """fp8_quantize_block of a matrix as _float_matrix returns it, on its device"""
    M, K = x2.shape
    q, s = _rows_out(M, K, x2)
    call("uc2_fp8_quant_rows", dt(x2.dtype), M, K, x2.data_ptr(), max(x2.stride(0), K), q.data_ptr(), s.data_ptr(), stream())
    return BlockRows(q, s, K)


def fp8_quantize_block(x):
    """[..., K] (fp32 or bf16, any row stride) -> BlockRows of its rows, one launch.  No gradient: for inference (training: linear_fp8_block)"""
    _no_gradient("fp8_quantize_block", "linear_fp8_block", x)
    x2 = _float_matrix(x, "fp8_quantize_block")
    with device_guard(x2):
        return _quant_rows(x2)


def _quant_weight(w, transpose):
    N, K = w.shape
    Np, Kp = _up(N), _up(K)
    q, s = w.new_empty((N, Kp), dtype=torch.uint8), w.new_empty((Np // BLOCK, Kp // BLOCK), dtype=torch.uint8)
    qt, st = (w.new_empty((K, Np), dtype=torch.uint8), w.new_empty((Kp // BLOCK, Np // BLOCK), dtype=torch.uint8)) if transpose else (None, None)
    call("uc2_fp8_quant_square", dt(w.dtype), N, K, w.data_ptr(), max(w.stride(0), K), q.data_ptr(), s.data_ptr(), ptr(qt), ptr(st), stream())
    return (BlockWeight(q, s), BlockWeight(qt, st)) if transpose else BlockWeight(q, s)


def fp8_quantize_weight_block(w, transpose=False):
    """[N, K] weight (fp32 or bf16) -> BlockWeight; transpose: also that of W^T with the same values (the operand of the input gradient),
    both from one read.  No gradient: a parameter is quantised under torch.no_grad() (training: linear_fp8_block)"""
    _no_gradient("fp8_quantize_weight_block", "linear_fp8_block", w)
    if not torch.is_tensor(w) or w.dim() != 2:
        raise _lib.Uc2Error("fp8_quantize_weight_block: a weight of two dimensions is needed")
    w = _float_matrix(w, "fp8_quantize_weight_block")
    with device_guard(w):
        return _quant_weight(w, transpose)


def _block_bias(bias, N, device):
    if bias is None:
        return None
    if bias.dtype != torch.float32 or bias.dim() != 1 or bias.shape[0] != N or bias.device != device:
        raise _lib.Uc2Error("bias must be fp32 [%d] on %s" % (N, device))
    return bias if bias.is_contiguous() else bias.contiguous()


def _gemm(a8, sa, b8, sb, bias):
    (M, Kp), N = a8.shape, b8.shape[0]
    out = a8.new_empty((M, N), dtype=torch.bfloat16)
    call("uc2_gemm_fp8_block", M, N, Kp, a8.data_ptr(), Kp, sa.data_ptr(), max(M, 1), b8.data_ptr(), Kp, sb.data_ptr(), ptr(bias), out.data_ptr(), max(N, 1), stream())
    return out


def gemm_fp8_block(a, b, bias=None):
    """bf16 [M, N] = a b^T + bias of a = BlockRows [M, K] (fp8_quantize_block, rms_norm_fp8) and b = BlockWeight [N, K]
    (fp8_quantize_weight_block; any (data, scale) pair of that layout); fp32 sums, one rounding.  No gradient, that of bias neither: for inference
    (training: linear_fp8_block)"""
    _no_gradient("gemm_fp8_block", "linear_fp8_block", bias)
    a8, sa, b8, sb = a[0], a[1], b[0], b[1]
    device = a8.device
    if not (a8.dtype == b8.dtype == sb.dtype == torch.uint8 and sa.dtype == torch.int32):
        raise _lib.Uc2Error("gemm_fp8_block: a = (uint8, int32 scales), b = (uint8, uint8 scales) expected, got %s, %s, %s, %s" % (a8.dtype, sa.dtype, b8.dtype, sb.dtype))
    _require_cuda(a8)
    if not sa.device == b8.device == sb.device == device:
        raise _lib.Uc2Error("gemm_fp8_block: operands on %s, %s, %s and %s" % (device, sa.device, b8.device, sb.device))
    if not (a8.dim() == b8.dim() == sa.dim() == sb.dim() == 2):
        raise _lib.Uc2Error("gemm_fp8_block: operands and scales of two dimensions expected")
    (M, Kp), N = a8.shape, b8.shape[0]
    if Kp % BLOCK or Kp == 0 or b8.shape[1] != Kp or sa.shape != ((Kp + 511) // 512, M) or sb.shape != ((N + BLOCK - 1) // BLOCK, Kp // BLOCK):
        raise _lib.Uc2Error("gemm_fp8_block: shapes do not match: %s with scales %s against %s with scales %s"
                            % (tuple(a8.shape), tuple(sa.shape), tuple(b8.shape), tuple(sb.shape)))
    if not (a8.is_contiguous() and sa.is_contiguous() and b8.is_contiguous() and sb.is_contiguous()):
        raise _lib.Uc2Error("gemm_fp8_block: operands must be contiguous")
    bias = _block_bias(bias, N, device)
    with device_guard(a8):
        return _gemm(a8, sa, b8, sb, bias)


def _wgrad(dy2, x2, K, ws, n, db):
    """(dW [N, K] fp32) of uc2_linear_wgrad on the first K columns of x2, with db written if there is one; n bytes of workspace at ws"""
    M, N = dy2.shape
    dw = dy2.new_empty((N, K), dtype=torch.float32)
    call("uc2_linear_wgrad", M, N, K, dy2.data_ptr(), max(dy2.stride(0), N), x2.data_ptr(), max(x2.stride(0), K), dw.data_ptr(), K, ptr(db), ws, n, stream())
    return dw


def _column_sums(dy2):
    """sums over the rows in a fixed order: those of the weight gradient, beside its smallest product"""
    M, N = dy2.shape
    if M == 0:
        return torch.zeros(N, dtype=torch.float32, device=dy2.device)
    db, K = dy2.new_empty(N, dtype=torch.float32), min(N, 8)
    n = _lib.load().uc2_linear_wgrad_workspace(M, N, K)
    ws = dy2.new_empty(n, dtype=torch.uint8)
    _wgrad(dy2, dy2, K, ws.data_ptr(), n, db)
    return db


def _align(n):
    return (n + 255) & ~255


def _product(x2, b8, sb, N, bias, tmp, at):
    """bf16 [M, N] = q(x2) b8^T + bias; q(x2) goes into the buffer tmp from byte `at` on (_product_bytes of it)"""
    M, K = x2.shape
    Kp = _up(K)
    q = tmp.data_ptr() + at
    qs = q + _align(M * Kp)
    out = x2.new_empty((M, N))
    call("uc2_fp8_quant_rows", dt(x2.dtype), M, K, x2.data_ptr(), max(x2.stride(0), K), q, qs, stream())
    call("uc2_gemm_fp8_block", M, N, Kp, q, Kp, qs, max(M, 1), b8, Kp, sb, ptr(bias), out.data_ptr(), N, stream())
    return out


def _product_bytes(M, K):
    Kp = _up(K)
    return _align(M * Kp) + _align((Kp + 511) // 512 * M * 4)


class LinearBlockFp8Fn(torch.autograd.Function):
    """y = q(x) q(W)^T + b, gradients straight through the quantisation: dx = q(dy) q(W) on the transposed copy of the same weight values,
    dW = dy^T x and db = sum dy from the unquantised bf16 tensors (the weight gradient stays bf16, as in the per-tensor mode).  What only one pass
    needs lies in one buffer (an allocation costs 1.5 us, a small layer's forward and backward together some 120)."""

    @staticmethod
    def forward(ctx, x, weight, bias):
        shp = x.shape
        need_dx, need_dw = ctx.needs_input_grad[:2]
        x2, weight = _float_matrix(x, "linear_fp8_block"), _float_matrix(weight, "linear_fp8_block")
        M, (N, K) = x2.shape[0], weight.shape
        Np, Kp = _up(N), _up(K)
        blocks = Np // BLOCK * (Kp // BLOCK)
        with device_guard(x2):
            at = _align(N * Kp) + _align(blocks)
            tmp = x2.new_empty(at + _product_bytes(M, K), dtype=torch.uint8)
            wt = x2.new_empty(K * Np + blocks, dtype=torch.uint8) if need_dx else None           # W^T and its scales
            w = tmp.data_ptr()
            ws = w + _align(N * Kp)
            call("uc2_fp8_quant_square", dt(weight.dtype), N, K, weight.data_ptr(), max(weight.stride(0), K), w, ws, ptr(wt), wt.data_ptr() + K * Np if need_dx else None, stream())
            y = _product(x2, w, ws, N, bias, tmp, at)
            note_leaves(ctx)
        ctx.save_for_backward(x2 if need_dw else None, wt)
        ctx.cfg = (shp, weight.shape, weight.dtype, _lib.load().uc2_linear_wgrad_workspace(M, N, K) if need_dw else 0)
        return y if len(shp) == 2 else y.view(*shp[:-1], N)

    @staticmethod
    @once
    def backward(ctx, dy):
        x2, wt = ctx.saved_tensors
        shp, (N, K), wtype, n = ctx.cfg
        need_dx, need_dw, need_db = ctx.needs_input_grad
        dy2 = _float_matrix(dy, "linear_fp8_block")
        if need_dw:                                       # (saved-tensor hooks may bring other strides than the forward's)
            x2 = _float_matrix(x2, "linear_fp8_block")
        if need_dx:
            wt = wt.contiguous()
        M = dy2.shape[0]
        dx = dw = db = None
        with device_guard(dy2):
            at = _align(n)
            tmp = dy2.new_empty(at + (_product_bytes(M, N) if need_dx else 0), dtype=torch.uint8)
            if need_dx:
                dx = _product(dy2, wt.data_ptr(), wt.data_ptr() + K * _up(N), K, None, tmp, at)
                if len(shp) != 2:
                    dx = dx.view(shp)
            if need_dw and M:
                db = dy2.new_empty(N, dtype=torch.float32) if need_db else None
                dw = _wgrad(dy2, x2, K, tmp.data_ptr(), n, db)
            else:
                if need_dw:
                    dw = torch.zeros((N, K), dtype=torch.float32, device=dy2.device)
                if need_db:
                    db = _column_sums(dy2)
            if dw is not None and wtype != torch.float32:
                dw = dw.to(wtype)
        return dx, dw, db


def linear_fp8_block(x, weight, bias=None):
    """bf16 x [..., K], weight [N, K] (fp32 or bf16), bias fp32 [N] or None -> bf16 [..., N]: a linear layer whose forward and input-gradient
    products run on e4m3 operands with block scales.  The weight is quantised in the call (for inference, with a weight that does not change:
    quantise it once with fp8_quantize_weight_block and call gemm_fp8_block).  It pays from some ten thousand rows on: 66560 x 1024 -> 4096 in 314 us, where
    the bf16 product takes 415; 9984 x 768 -> 2304 in 40 us and its input gradient in 45, where the bf16 products take 39 each."""
    if not torch.is_tensor(x) or x.dtype != torch.bfloat16 or x.dim() < 1:
        raise _lib.Uc2Error("linear_fp8_block computes on bf16 activations")
    _require_cuda(x)
    if not torch.is_tensor(weight) or weight.dim() != 2 or weight.shape[1] != x.shape[-1] or weight.shape[0] < 1:
        raise _lib.Uc2Error("linear_fp8_block: weight [N, %d] expected, got %s" % (x.shape[-1], tuple(getattr(weight, "shape", ()))))
    if weight.device != x.device:
        raise _lib.Uc2Error("linear_fp8_block: x on %s, weight on %s" % (x.device, weight.device))
    dt(weight.dtype)
    return LinearBlockFp8Fn.apply(x, weight, _block_bias(bias, weight.shape[0], x.device))


# ---- root-mean-square norm ----------------------------------------------------------------------------------------------------------
def _rms_args(x, weight, residual, what):
    if not torch.is_tensor(x) or x.dim() < 1:
        raise _lib.Uc2Error("%s: a tensor of one dimension at least is needed" % what)
    _require_cuda(x)
    H, device = x.shape[-1], x.device
    dt(x.dtype)
    if weight.dtype != torch.float32 or weight.shape != (H,) or weight.device != device:
        raise _lib.Uc2Error("%s: weight must be fp32 [%d] on %s" % (what, H, device))
    if not 1 <= H <= 16384:
        raise _lib.Uc2Error("%s: rows of 1 to 16384 elements, got %d" % (what, H))
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != device):
        raise _lib.Uc2Error("%s: residual must have the shape, type and device of x" % what)


def _dense(x, H):
    return x.contiguous() if x.dim() == 2 else x.reshape(-1, H).contiguous()


def _rms_fwd(x, weight, eps, residual, want_y, want_rstd, want_q):
    H = x.shape[-1]
    x2 = _dense(x, H)
    r2 = None if residual is None else _dense(residual, H)
    w = weight.contiguous()
    M = x2.shape[0]
    s = torch.empty_like(x2) if r2 is not None else None
    y = torch.empty_like(x2) if want_y else None
    rstd = x2.new_empty(M, dtype=torch.float32) if want_rstd else None
    q, qs = _rows_out(M, H, x2) if want_q else (None, None)
    timed = _Timed("rms_fwd", x2.element_size() * M * H * (1 + 2 * (r2 is not None) + want_y) + M * H * want_q) if state.hbm_timer is not None else None
    call("uc2_rms_fwd", dt(x2.dtype), M, H, x2.data_ptr(), ptr(r2), w.data_ptr(), eps, ptr(s), ptr(y), ptr(rstd), ptr(q), ptr(qs), stream())
    if timed is not None:
        timed.__exit__()
    return x2 if s is None else s, y, rstd, BlockRows(q, qs, H) if want_q else None


class RMSNormFn(torch.autograd.Function):
    """(y, s) with s = x + residual (rounded to the tensors' type), y = s / sqrt(mean(s^2) + eps) * weight; (y,) without a residual"""

    @staticmethod
    def forward(ctx, x, weight, eps, residual):
        grad = True in ctx.needs_input_grad
        with device_guard(x):
            s, y, rstd, _ = _rms_fwd(x, weight, eps, residual, True, grad, False)
            note_leaves(ctx)
        if grad:
            ctx.save_for_backward(s, weight.contiguous(), rstd)
            ctx.ws = _lib.load().uc2_rms_bwd_workspace(*s.shape)
        ctx.set_materialize_grads(False)
        ctx.shp = x.shape
        if x.dim() != 2:
            y, s = y.view(x.shape), s.view(x.shape)
        return y if residual is None else (y, s)

    @staticmethod
    @once
    def backward(ctx, dy, ds=None):
        s, weight, rstd = (t.contiguous() for t in ctx.saved_tensors)       # (saved-tensor hooks may bring other strides than the forward's)
        M, H = s.shape
        if dy is None:                                   # only the stream is used
            return ds, torch.zeros_like(weight) if ctx.needs_input_grad[1] else None, None, ds
        need_dx, need_dw, _, need_dr = ctx.needs_input_grad
        with device_guard(s):
            dy2 = _dense(dy, H)
            ds2 = None if ds is None else _dense(ds, H)
            dx = torch.empty_like(s)
            dw = ws = None
            n = 0
            if need_dw:
                dw = torch.empty_like(weight)
                n = ctx.ws
                ws = s.new_empty(n, dtype=torch.uint8) if n else None
            timed = _Timed("rms_bwd", s.element_size() * M * H * (3 + (ds2 is not None))) if state.hbm_timer is not None else None
            call("uc2_rms_bwd", dt(s.dtype), M, H, dy2.data_ptr(), ptr(ds2), s.data_ptr(), weight.data_ptr(), rstd.data_ptr(), dx.data_ptr(), ptr(dw), ptr(ws), n,
                 stream())
            if timed is not None:
                timed.__exit__()
        if dx.shape != ctx.shp:
            dx = dx.view(ctx.shp)
        return dx if need_dx else None, dw, None, dx if need_dr else None


def rms_norm(x, weight, eps=1e-6, residual=None):
    """root-mean-square norm over the last dimension (fp32 or bf16, weight fp32): y, or (y, s) with s = x + residual, the stream to carry on"""
    _rms_args(x, weight, residual, "rms_norm")
    return RMSNormFn.apply(x, weight, float(eps), residual)


def rms_norm_fp8(x, weight, eps=1e-6, residual=None):
    """the norm as an operand of gemm_fp8_block: (BlockRows of y [rows, H], s) with s as in rms_norm (x's values in its shape without a
    residual); y itself is never written.  No gradient: for inference (training: rms_norm, then linear_fp8_block)."""
    _rms_args(x, weight, residual, "rms_norm_fp8")
    _no_gradient("rms_norm_fp8", "rms_norm and linear_fp8_block", x, weight, residual)
    with device_guard(x):
        s, _, _, q = _rms_fwd(x, weight, float(eps), residual, False, False, True)
    return q, x if residual is None else s.view(x.shape)
