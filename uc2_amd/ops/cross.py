"""Attention from one sequence to the states of another (cross attention with per-sequence lengths and shared key heads).  Part of
uc2_amd.ops.  Beside AttentionGeneralFn (fp32 math, one thread per row, the additive [Lq, Lk] mask of MultiheadAttention)."""
import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .._lib import check, dt, ptr, stream
from .base import _Timed, _require_cuda, device_guard, rng

_I, _F, _P, _L = ctypes.c_int, ctypes.c_float, ctypes.c_void_p, ctypes.c_longlong


class _CrossAttn(ctypes.Structure):              # Uc2CrossAttn
    _fields_ = [("dtype", _I), ("B", _I), ("Lq", _I), ("Lk", _I), ("nh", _I), ("nkv", _I), ("D", _I), ("scale", _F), ("drop_p", _F),
                ("q", _P), ("k", _P), ("v", _P), ("q_sb", _L), ("q_sl", _L), ("q_sh", _L), ("k_sb", _L), ("k_sl", _L), ("k_sh", _L),
                ("v_sb", _L), ("v_sl", _L), ("v_sh", _L), ("key_mask", _P), ("key_mask_sb", _L), ("k_lens", _P),
                ("out", _P), ("o_sb", _L), ("o_sl", _L), ("o_sh", _L), ("lse", _P), ("seed", _P), ("site", ctypes.c_uint64)]


class _CrossAttnGrad(ctypes.Structure):          # Uc2CrossAttnGrad
    _fields_ = [("dout", _P), ("dout_sb", _L), ("dout_sl", _L), ("dout_sh", _L), ("dq", _P), ("dk", _P), ("dv", _P),
                ("dq_sb", _L), ("dq_sl", _L), ("dq_sh", _L), ("dk_sb", _L), ("dk_sl", _L), ("dk_sh", _L), ("dv_sb", _L), ("dv_sl", _L), ("dv_sh", _L)]


def _rows16(x):
    """x itself where the kernels can read it in place (contiguous heads, rows of 16-byte alignment), else a contiguous copy"""
    el = 16 // x.element_size()
    if x.stride(3) == 1 and x.data_ptr() % 16 == 0 and all(x.shape[i] <= 1 or (x.stride(i) % el == 0) for i in range(3)):
        return x
    return x.clone(memory_format=torch.contiguous_format)          # (contiguous() would hand an unaligned dense tensor back)


def _strides(x):
    """batch, row and head strides; those of dimensions of one element do not matter (and need not be aligned)"""
    return tuple(x.stride(i) if x.shape[i] > 1 else 0 for i in range(3))


def _describe(q, k, v, out, key_mask, k_lens, scale, drop_p, lse, seed, site):
    B, Lq, nh, D = q.shape
    return _CrossAttn(dt(q.dtype), B, Lq, k.shape[1], nh, k.shape[2], D, scale, drop_p, ptr(q), ptr(k), ptr(v), *_strides(q), *_strides(k), *_strides(v),
                      ptr(key_mask), 0 if key_mask is None or key_mask.shape[0] <= 1 else key_mask.stride(0), ptr(k_lens), ptr(out), *_strides(out),
                      ptr(lse), ptr(seed), site)


def _xattn_ws(desc, backward, device):
    n = _lib.load().uc2_xattn_workspace(ctypes.byref(desc), backward)
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


class CrossAttentionFn(torch.autograd.Function):
    """out [B, Lq, nh, D] of uc2_xattn_fwd; gradients of q, k and v"""

    @staticmethod
    def forward(ctx, q, k, v, key_mask, k_lens, scale, drop_p, seed, site):
        with device_guard(q):
            q, k, v = _rows16(q), _rows16(k), _rows16(v)
            B, Lq, nh, D = q.shape
            grad = any(ctx.needs_input_grad[:3])
            out = torch.empty((B, Lq, nh, D), dtype=q.dtype, device=q.device)
            lse = torch.empty((B, k.shape[2], Lq, nh // k.shape[2]), dtype=torch.float32, device=q.device) if grad else None
            desc = _describe(q, k, v, out, key_mask, k_lens, scale, drop_p, lse, seed, site)
            ws = _xattn_ws(desc, 0, q.device)
            with _Timed("xattn_fwd", q.element_size() * (2 * q.numel() + k.numel() + v.numel())):
                check(_lib.load().uc2_xattn_fwd(ctypes.byref(desc), ptr(ws), 0 if ws is None else ws.numel(), stream()))
        if grad:
            ctx.save_for_backward(q, k, v, key_mask, k_lens, out, lse, seed)
            ctx.cfg = (scale, drop_p, site)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, key_mask, k_lens, out, lse, seed = ctx.saved_tensors
        scale, drop_p, site = ctx.cfg
        with device_guard(q):
            dout = _rows16(dout)
            new = lambda x: torch.empty(x.shape, dtype=x.dtype, device=x.device)  # noqa: E731
            dq, dk, dv = new(q), new(k), new(v)
            desc = _describe(q, k, v, out, key_mask, k_lens, scale, drop_p, lse, seed, site)
            grad = _CrossAttnGrad(ptr(dout), *_strides(dout), ptr(dq), ptr(dk), ptr(dv), *_strides(dq), *_strides(dk), *_strides(dv))
            ws = _xattn_ws(desc, 1, q.device)
            with _Timed("xattn_bwd", q.element_size() * (4 * q.numel() + 2 * (k.numel() + v.numel()))):
                check(_lib.load().uc2_xattn_bwd(ctypes.byref(desc), ctypes.byref(grad), ptr(ws), 0 if ws is None else ws.numel(), stream()))
        return dq, dk, dv, None, None, None, None, None, None


def cross_attention(q, k, v, key_mask=None, k_lens=None, scale=None, drop_p=0.0, site=0):
    """softmax(scale q k^T + key_mask) v over the keys that take part; q [B, Lq, nh, D], k and v [B, Lk, nkv, D] (fp32 or bf16, D 32, 64 or 128,
    nh a multiple of nkv: heads h G .. h G + G - 1 share key head h) -> [B, Lq, nh, D].  Slices of a fused projection are read in place.
      k_lens    [B] integers on the device: keys from k_lens[b] on take no part (a padded batch, a buffer longer than the states in it)
      key_mask  [B, Lk] or [B, 1, 1, Lk] additive float mask; a key whose entry is <= -1e30 takes no part, -10000 and the like only weigh
      drop_p    dropout on the weights, drawn from ops.rng like the encoder's (site: tells two calls inside one ops.rng.scope() apart)
    Keys that take no part reach nothing, whatever they hold; a query that has none gets zeros and passes no gradient.  scale defaults to
    1 / sqrt(D).  Gradients for q, k and v; results repeat bit for bit."""
    for t, what in ((q, "q"), (k, "k"), (v, "v")):
        if not torch.is_tensor(t) or t.dim() != 4:
            raise _lib.Uc2Error("cross_attention: %s must be a tensor [batch, length, heads, head dimension]" % what)
        _require_cuda(t)
        if t.dtype != q.dtype or t.device != q.device:
            raise _lib.Uc2Error("cross_attention: q, k and v must have one type and device")
    dt(q.dtype)
    B, Lq, nh, D = q.shape
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != D:
        raise _lib.Uc2Error("cross_attention: k and v must be [%d, Lk, nkv, %d], got %s and %s" % (B, D, tuple(k.shape), tuple(v.shape)))
    if D not in (32, 64, 128):
        raise _lib.Uc2Error("cross_attention: head dimensions of 32, 64 and 128, got %d" % D)
    Lk, nkv = k.shape[1], k.shape[2]
    if nkv < 1 or nh < 1 or nh % nkv:
        raise _lib.Uc2Error("cross_attention: %d query heads over %d key heads" % (nh, nkv))
    if not 0.0 <= drop_p < 1.0:
        raise _lib.Uc2Error("cross_attention: drop_p in [0, 1), got %s" % drop_p)
    if k_lens is not None:
        if not torch.is_tensor(k_lens) or k_lens.device != q.device or tuple(k_lens.shape) != (B,) or k_lens.dtype not in (torch.int32, torch.int64):
            raise _lib.Uc2Error("cross_attention: k_lens must be an int32 or int64 tensor [%d] on %s" % (B, q.device))
        k_lens = k_lens.clamp(0, Lk).to(torch.int32) if k_lens.dtype == torch.int64 else k_lens
        k_lens = k_lens.contiguous()
    if key_mask is not None:
        if not torch.is_tensor(key_mask) or key_mask.device != q.device or not key_mask.is_floating_point():
            raise _lib.Uc2Error("cross_attention: key_mask must be an additive float mask on %s" % q.device)
        if key_mask.dim() == 4 and key_mask.shape[1] == 1 and key_mask.shape[2] == 1:
            key_mask = key_mask[:, 0, 0]
        if tuple(key_mask.shape) != (B, Lk):
            raise _lib.Uc2Error("cross_attention: key_mask must be [%d, %d], got %s" % (B, Lk, tuple(key_mask.shape)))
        if key_mask.requires_grad:
            raise _lib.Uc2Error("cross_attention: key_mask takes no gradient")
        key_mask = key_mask.float()
        if key_mask.stride(1) != 1 and Lk > 1:
            key_mask = key_mask.contiguous()
    seed = rng.snapshot(q.device) if drop_p > 0.0 else None
    return CrossAttentionFn.apply(q, k, v, key_mask, k_lens, 1.0 / math.sqrt(D) if scale is None else float(scale), float(drop_p), seed, rng.site(site))
