"""Attention from one sequence to the states of another (cross attention with per-sequence lengths and shared key heads).  Part of
uc2_amd.ops.  Beside AttentionGeneralFn (fp32 math, one thread per row, the additive [Lq, Lk] mask of MultiheadAttention)."""
import struct

import torch

from .. import _lib
from .._lib import check, dt, ptr, stream
from ..config import state
from .base import _Timed, _require_cuda, device_guard, note_leaves, once, rng

# Uc2CrossAttn and Uc2CrossAttnGrad (include/uc2_hip.h), packed in native alignment: a ctypes.Structure of as many fields takes 5 us to fill
_ATTN = struct.Struct("@7i2f3P9qPqPP3qPPPQ")
_GRAD = struct.Struct("@P3q3P9q")
# its pointers q, k, v, key_mask, k_lens, out, lse, out_f32, seed and what is left of it
_PTRS = struct.Struct("@40x3P72xP8xPP24xPPPQ")


def _rows16(x):
    """x itself where the kernels can read it in place (contiguous heads, rows of 16-byte alignment less than 2^22 elements apart), else a
    contiguous copy"""
    sb, sl, sh, sd = x.stride()
    B, L, nh, _ = x.shape
    es = x.element_size()
    if (sd == 1 and x.data_ptr() % 16 == 0 and (B <= 1 or sb * es % 16 == 0) and (L <= 1 or sl * es % 16 == 0 and sl < 1 << 22)
            and (nh <= 1 or sh * es % 16 == 0 and sh < 1 << 22)):
        return x
    return x.clone(memory_format=torch.contiguous_format)          # (contiguous() would hand an unaligned dense tensor back)


def _describe(q, k, v, out, key_mask, k_lens, scale, drop_p, lse, out_f32, seed, site):
    B, Lq, nh, D = q.shape
    qs, ks, vs, os = q.stride(), k.stride(), v.stride(), (0, 0, 0) if out is None else out.stride()
    return _ATTN.pack(dt(q.dtype), B, Lq, k.shape[1], nh, k.shape[2], D, scale, drop_p, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                      qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
                      0 if key_mask is None else key_mask.data_ptr(), 0 if key_mask is None else key_mask.stride(0), 0 if k_lens is None else k_lens.data_ptr(),
                      0 if out is None else out.data_ptr(), os[0], os[1], os[2], 0 if lse is None else lse.data_ptr(),
                      0 if out_f32 is None else out_f32.data_ptr(), 0 if seed is None else seed.data_ptr(), site)


def _strides(q, k, v, key_mask):
    return q.stride(), k.stride(), v.stride(), None if key_mask is None else key_mask.stride()


def _timed(name, nbytes):
    return _Timed(name, nbytes) if state.hbm_timer is not None else None


class CrossAttentionFn(torch.autograd.Function):
    """out [B, Lq, nh, D] of uc2_xattn_fwd; gradients of q, k and v"""

    @staticmethod
    def forward(ctx, q, k, v, key_mask, k_lens, scale, drop_p, seed, site):
        lib = _lib.load()
        with device_guard(q):
            q, k, v = _rows16(q), _rows16(k), _rows16(v)
            B, Lq, nh, D = q.shape
            need = ctx.needs_input_grad
            grad = need[0] or need[1] or need[2]
            out = q.new_empty((B, Lq, nh, D))
            lse = q.new_empty((B, k.shape[2], Lq, nh // k.shape[2]), dtype=torch.float32) if grad else None
            out_f32 = q.new_empty((B, k.shape[2], Lq, nh // k.shape[2], D), dtype=torch.float32) if grad and q.dtype == torch.bfloat16 else None
            desc = _describe(q, k, v, out, key_mask, k_lens, scale, drop_p, lse, out_f32, seed, site)
            n = lib.uc2_xattn_workspace(desc, 0)
            ws = q.new_empty(n, dtype=torch.uint8) if n else None
            timed = _timed("xattn_fwd", q.element_size() * (2 * q.numel() + k.numel() + v.numel()))
            rc = lib.uc2_xattn_fwd(desc, ptr(ws), n, stream())
            if timed is not None:
                timed.__exit__()
            note_leaves(ctx)
        if rc:
            check(rc)
        if grad:
            ctx.save_for_backward(q, k, v, key_mask, k_lens, out if out_f32 is None else out_f32, lse, seed)
            # what the backward would work out again on a thread that has just been woken up: the call structure, as long as the tensors that come
            # back are the ones in it, and the workspace's size
            ctx.cfg = (scale, drop_p, site, desc, _strides(q, k, v, key_mask), lib.uc2_xattn_workspace(desc, 1))
        return out

    @staticmethod
    @once
    def backward(ctx, dout):
        saved = ctx.saved_tensors
        q, k, v, key_mask, k_lens, out, lse, seed = saved                     # (out: before its rounding, if it was rounded)
        scale, drop_p, site, desc, strides, n = ctx.cfg
        lib = _lib.load()
        with device_guard(q):
            dout = _rows16(dout)
            # saved-tensor hooks may bring copies: elsewhere, or where the tensor itself had been with other strides
            p = _PTRS.unpack(desc)
            if ((*p[:5], p[7] or p[5], p[6], p[8]) != tuple([0 if t is None else t.data_ptr() for t in saved]) or strides != _strides(q, k, v, key_mask)
                    or not (out.is_contiguous() and lse.is_contiguous() and (k_lens is None or k_lens.is_contiguous()))):
                q, k, v, lse = _rows16(q), _rows16(k), _rows16(v), lse.contiguous()
                key_mask, k_lens = (None if t is None else t.contiguous() for t in (key_mask, k_lens))
                out, out_f32 = (None, out.clone(memory_format=torch.contiguous_format)) if q.dtype == torch.bfloat16 else (_rows16(out), None)
                desc = _describe(q, k, v, out, key_mask, k_lens, scale, drop_p, lse, out_f32, seed, site)
            dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
            ws = q.new_empty(n, dtype=torch.uint8)
            gs, qs, ks = dout.stride(), dq.stride(), dk.stride()
            grad = _GRAD.pack(dout.data_ptr(), gs[0], gs[1], gs[2], dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), qs[0], qs[1], qs[2], ks[0], ks[1], ks[2],
                              ks[0], ks[1], ks[2])
            timed = _timed("xattn_bwd", q.element_size() * (4 * q.numel() + 2 * (k.numel() + v.numel())))
            rc = lib.uc2_xattn_bwd(desc, grad, ws.data_ptr(), n, stream())
            if timed is not None:
                timed.__exit__()
        if rc:
            check(rc)
        return dq, dk, dv, None, None, None, None, None, None


def cross_attention(q, k, v, key_mask=None, k_lens=None, scale=None, drop_p=0.0, site=0):
    """softmax(scale q k^T + key_mask) v over the keys that take part; q [B, Lq, nh, D], k and v [B, Lk, nkv, D] (fp32 or bf16, D 32, 64 or 128,
    nh a multiple of nkv: heads h G .. h G + G - 1 share key head h) -> [B, Lq, nh, D].  Slices of a fused projection are read in place.
      k_lens    [B] integers on the device: keys from k_lens[b] on take no part (a padded batch, a buffer longer than the states in it)
      key_mask  [B, Lk] or [B, 1, 1, Lk] additive float mask; a key whose entry is <= -1e30 takes no part, -10000 and the like only weigh
      drop_p    dropout on the weights, drawn from ops.rng like the encoder's (site: tells two calls inside one ops.rng.scope() apart)
    Keys that take no part reach nothing, whatever they hold; a query that has none gets zeros and passes no gradient.  scale defaults to
    1 / sqrt(D).  Gradients for q, k and v; results repeat bit for bit."""
    if not (torch.is_tensor(q) and torch.is_tensor(k) and torch.is_tensor(v) and q.dim() == k.dim() == v.dim() == 4):
        raise _lib.Uc2Error("cross_attention: q, k and v must be tensors [batch, length, heads, head dimension]")
    _require_cuda(q)
    device = q.device
    if k.device != device or v.device != device or not q.dtype == k.dtype == v.dtype:
        raise _lib.Uc2Error("cross_attention: q, k and v must have one type and device")
    dt(q.dtype)
    B, Lq, nh, D = q.shape
    kshape = k.shape
    if kshape != v.shape or kshape[0] != B or kshape[3] != D:
        raise _lib.Uc2Error("cross_attention: k and v must be [%d, Lk, nkv, %d], got %s and %s" % (B, D, tuple(k.shape), tuple(v.shape)))
    if D not in (32, 64, 128):
        raise _lib.Uc2Error("cross_attention: head dimensions of 32, 64 and 128, got %d" % D)
    Lk, nkv = kshape[1], kshape[2]
    if nkv < 1 or nh < 1 or nh % nkv:
        raise _lib.Uc2Error("cross_attention: %d query heads over %d key heads" % (nh, nkv))
    if not 0.0 <= drop_p < 1.0:
        raise _lib.Uc2Error("cross_attention: drop_p in [0, 1), got %s" % drop_p)
    if k_lens is not None:
        if not torch.is_tensor(k_lens) or k_lens.device != device or k_lens.shape != (B,) or k_lens.dtype not in (torch.int32, torch.int64):
            raise _lib.Uc2Error("cross_attention: k_lens must be an int32 or int64 tensor [%d] on %s" % (B, device))
        if k_lens.dtype == torch.int64:
            k_lens = k_lens.clamp(0, Lk).to(torch.int32)
        k_lens = k_lens.contiguous()
    if key_mask is not None:
        if not torch.is_tensor(key_mask) or key_mask.device != device or not key_mask.is_floating_point():
            raise _lib.Uc2Error("cross_attention: key_mask must be an additive float mask on %s" % device)
        if key_mask.dim() == 4 and key_mask.shape[1] == 1 and key_mask.shape[2] == 1:
            key_mask = key_mask[:, 0, 0]
        if key_mask.shape != (B, Lk):
            raise _lib.Uc2Error("cross_attention: key_mask must be [%d, %d], got %s" % (B, Lk, tuple(key_mask.shape)))
        if key_mask.requires_grad:
            raise _lib.Uc2Error("cross_attention: key_mask takes no gradient")
        key_mask = key_mask.float()
        if Lk > 1 and key_mask.stride(1) != 1:
            key_mask = key_mask.contiguous()
    seed = None
    if drop_p > 0.0:
        seed, site = rng.snapshot(device), rng.site(site)
    return CrossAttentionFn.apply(q, k, v, key_mask, k_lens, D ** -0.5 if scale is None else float(scale), float(drop_p), seed, site)
