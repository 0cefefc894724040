"""What the block-scaled e4m3 operators, the root-mean-square norm and the cross attention refuse before anything is launched, and the test
oracle's own arithmetic, without a GPU."""
import ctypes

import pytest
import torch

import block_ref as R
from uc2_amd import _lib, ops
from uc2_amd.ops.cross import _ATTN, _GRAD

P = 4096                        # an aligned address; no check dereferences it
I, F, A, L = ctypes.c_int, ctypes.c_float, ctypes.c_void_p, ctypes.c_longlong


class _CrossAttn(ctypes.Structure):             # Uc2CrossAttn
    _fields_ = ([(n, I) for n in "dtype B Lq Lk nh nkv D".split()] + [("scale", F), ("drop_p", F)] + [(n, A) for n in "qkv"]
                + [(n, L) for n in "q_sb q_sl q_sh k_sb k_sl k_sh v_sb v_sl v_sh".split()]
                + [("key_mask", A), ("key_mask_sb", L), ("k_lens", A), ("out", A), ("o_sb", L), ("o_sl", L), ("o_sh", L), ("lse", A), ("out_f32", A), ("seed", A), ("site", ctypes.c_uint64)])


class _CrossAttnGrad(ctypes.Structure):         # Uc2CrossAttnGrad
    _fields_ = ([("dout", A), ("dout_sb", L), ("dout_sl", L), ("dout_sh", L), ("dq", A), ("dk", A), ("dv", A)]
                + [(n, L) for n in "dq_sb dq_sl dq_sh dk_sb dk_sl dk_sh dv_sb dv_sl dv_sh".split()])


def attn(**kw):
    d = dict(dtype=1, B=2, Lq=3, Lk=5, nh=4, nkv=2, D=64, scale=0.125, drop_p=0.0, q=P, k=P, v=P, q_sb=768, q_sl=256, q_sh=64, k_sb=640, k_sl=128, k_sh=64, v_sb=640,
             v_sl=128, v_sh=64, out=P, o_sb=768, o_sl=256, o_sh=64, lse=P, out_f32=P)
    d.update(kw)
    return _CrossAttn(**d)


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(D=48), dict(D=0), dict(nkv=3), dict(nkv=0), dict(B=-1), dict(Lq=-1), dict(Lk=-2), dict(drop_p=1.0), dict(drop_p=-0.5), dict(q=0),
                                 dict(k=0), dict(out=0), dict(q=P + 2), dict(v=P + 8), dict(q_sl=257), dict(k_sh=4), dict(o_sb=-8), dict(k_sl=1 << 22), dict(Lq=1 << 30)])
def test_cross_attention_argument_errors(bad):
    lib = _lib.load()
    assert lib.uc2_xattn_fwd(ctypes.byref(attn(**bad)), None, 0, None) == -1
    assert lib.uc2_last_error()


def test_cross_attention_backward_argument_errors():
    lib = _lib.load()
    g = dict(dout=P, dout_sb=768, dout_sl=256, dout_sh=64, dq=P, dk=P, dv=P, dq_sb=768, dq_sl=256, dq_sh=64, dk_sb=640, dk_sl=128, dk_sh=64, dv_sb=640, dv_sl=128, dv_sh=64)
    many = lambda **kw: attn(Lk=5000, **kw)  # noqa: E731          (its keys are split: it needs a workspace)
    need = lib.uc2_xattn_workspace(ctypes.byref(many()), 1)
    assert need > 0 and lib.uc2_xattn_workspace(ctypes.byref(attn()), 1) == 0
    for a, gb, ws, n in ((many(lse=0), g, P, need), (many(), dict(g, dq=0), P, need), (many(), dict(g, dk=0), P, need), (many(), dict(g, dout_sl=3), P, need),
                         (many(), dict(g, dv=P + 4), P, need), (many(), g, None, need), (many(), g, P, need - 1), (many(), g, P + 4, need), (attn(lse=0), g, None, 0),
                         (attn(out_f32=0), g, None, 0), (attn(out_f32=P + 4), g, None, 0), (attn(dtype=0, out=0), g, None, 0)):
        assert lib.uc2_xattn_bwd(ctypes.byref(a), ctypes.byref(_CrossAttnGrad(**gb)), ws, n, None) == -1
    assert lib.uc2_xattn_bwd(ctypes.byref(attn()), None, P, need, None) == -1
    assert lib.uc2_xattn_fwd(None, None, 0, None) == -1
    # a long axis split over workgroups needs its workspace
    long = attn(B=1, Lq=1, Lk=100000, nkv=4, q_sl=256)
    n = lib.uc2_xattn_workspace(ctypes.byref(long), 0)
    assert n > 0 and lib.uc2_xattn_fwd(ctypes.byref(long), None, 0, None) == -1 and lib.uc2_xattn_fwd(ctypes.byref(long), P, n - 1, None) == -1
    assert lib.uc2_xattn_workspace(ctypes.byref(attn(B=4000, Lk=64)), 0) == 0
    assert lib.uc2_xattn_workspace(ctypes.byref(attn(D=7)), 0) == 0


def test_cross_attention_backward_without_queries_checks_its_keys():
    lib = _lib.load()
    g = _CrossAttnGrad(dout=P, dout_sb=768, dout_sl=256, dout_sh=64, dq=P, dk=P, dv=P, dq_sb=768, dq_sl=256, dq_sh=64, dk_sb=640, dk_sl=128, dk_sh=64, dv_sb=640, dv_sl=128, dv_sh=64)
    for bad in (dict(k=0), dict(v=0), dict(k=P + 8), dict(v=P + 2), dict(k_sl=129), dict(v_sh=1 << 22)):
        assert lib.uc2_xattn_bwd(ctypes.byref(attn(Lq=0, **bad)), ctypes.byref(g), None, 0, None) == -1, bad


def test_empty_calls_launch_nothing():
    lib = _lib.load()
    assert lib.uc2_xattn_fwd(ctypes.byref(attn(B=0)), None, 0, None) == 0
    assert lib.uc2_xattn_fwd(ctypes.byref(attn(Lq=0)), None, 0, None) == 0
    assert lib.uc2_gemm_fp8_block(0, 5, 128, None, 128, None, 0, None, 128, None, None, None, 5, None) == 0
    assert lib.uc2_fp8_quant_rows(1, 0, 128, None, 128, None, None, None) == 0
    assert lib.uc2_rms_fwd(1, 0, 128, None, None, None, 1e-6, None, None, None, None, None, None) == 0


def test_block_argument_errors():
    lib = _lib.load()
    ok = [4, 8, 256, P, 256, P, 4, P, 256, P, None, P, 8, None]
    for i, bad in ((0, -1), (1, -1), (2, 0), (3, None), (3, P + 8), (4, 128), (4, 264), (5, None), (5, P + 2), (6, 3), (7, None), (7, P + 4), (8, 128), (9, None), (11, None), (11, P + 1),
                   (12, 7), (10, P + 2)):
        a = list(ok)
        a[i] = bad
        assert lib.uc2_gemm_fp8_block(*a) == -1, (i, bad)
    for a in ((2, 4, 128, P, 128, P, P, None), (1, -1, 128, P, 128, P, P, None), (1, 4, 0, P, 128, P, P, None), (1, 4, 128, P, 127, P, P, None), (1, 4, 128, None, 128, P, P, None),
              (1, 4, 128, P, 128, P + 4, P, None), (1, 4, 128, P, 128, P, P + 1, None)):
        assert lib.uc2_fp8_quant_rows(*a) == -1
    for a in ((3, 4, 128, P, 128, P, P, None, None, None), (1, 4, 128, P, 100, P, P, None, None, None), (1, 4, 128, P, 128, P, P, P, None, None), (1, 4, 128, P, 128, P, None, None, None, None),
              (1, 4, 128, P, 128, P + 1, P, None, None, None), (1, 1 << 24, 128, P, 128, P, P, None, None, None)):
        assert lib.uc2_fp8_quant_square(*a) == -1


def test_rms_argument_errors():
    lib = _lib.load()
    ok = [1, 4, 128, P, P, P, 1e-6, P, P, P, P, P, None]
    for i, bad in ((0, 5), (1, -1), (2, 0), (2, 16385), (3, None), (4, None), (5, None), (6, -1.0), (7, None), (10, None), (11, None), (10, P + 4), (11, P + 2)):
        a = list(ok)
        a[i] = bad
        assert lib.uc2_rms_fwd(*a) == -1, (i, bad)
    assert lib.uc2_rms_fwd(1, 4, 128, P, None, P, 1e-6, None, None, None, None, None, None) == -1     # no output at all
    n = lib.uc2_rms_bwd_workspace(400, 128)
    ok = [1, 400, 128, P, P, P, P, P, P, P, P, n, None]
    for i, bad in ((0, 5), (1, -1), (2, 16385), (3, None), (5, None), (6, None), (7, None), (8, None), (9, P + 2), (10, None), (10, P + 2), (11, n - 1)):
        a = list(ok)
        a[i] = bad
        assert lib.uc2_rms_bwd(*a) == -1, (i, bad)
    assert n > 0 and lib.uc2_rms_bwd_workspace(8, 128) == 0      # (few rows: one workgroup)
    assert lib.uc2_rms_bwd_workspace(0, 128) == 0 and lib.uc2_rms_bwd_workspace(4, 20000) == 0


def test_linear_wgrad_argument_errors():
    lib = _lib.load()
    n = lib.uc2_linear_wgrad_workspace(4000, 40, 72)
    assert n > 0 and lib.uc2_linear_wgrad_workspace(200, 40, 72) == 0             # (few rows are not split)
    ok = [4000, 40, 72, P, 40, P, 72, P, 72, P, P, n, None]
    for i, bad in ((0, 0), (0, -1), (1, 0), (2, 0), (3, None), (3, P + 1), (4, 39), (5, None), (5, P + 1), (6, 71), (7, None), (7, P + 2), (8, 71), (9, P + 2), (10, None), (10, P + 8),
                   (11, n - 1)):
        a = list(ok)
        a[i] = bad
        assert lib.uc2_linear_wgrad(*a) == -1, (i, bad)
    assert lib.uc2_linear_wgrad_workspace(0, 40, 72) == 0 and lib.uc2_linear_wgrad_workspace(4000, 1 << 30, 1 << 30) == 0


def test_sizes_beyond_a_launch_are_argument_errors():
    """2^32 work items along a dimension, 65535 workgroups along the second: refused before a launch that cannot be"""
    lib = _lib.load()
    g = dict(dout=P, dout_sb=64, dq=P, dk=P, dv=P, dq_sb=64, dk_sb=65 * 64, dk_sl=64, dv_sb=65 * 64, dv_sl=64)
    many = attn(B=1 << 23, Lq=1, Lk=65, nh=1, nkv=1, q_sb=64, k_sb=65 * 64, k_sl=64, v_sb=65 * 64, v_sl=64, o_sb=64)
    assert lib.uc2_xattn_workspace(ctypes.byref(many), 1) == 0
    assert lib.uc2_xattn_bwd(ctypes.byref(many), ctypes.byref(_CrossAttnGrad(**g)), None, 0, None) == -1
    assert lib.uc2_xattn_fwd(ctypes.byref(attn(B=(1 << 24) - 1, Lq=300, nh=1, nkv=1)), None, 0, None) == -1
    assert lib.uc2_fp8_quant_square(1, 65535 * 128 + 1, 128, P, 128, P, P, None, None, None) == -1
    assert lib.uc2_gemm_fp8_block((1 << 31) - 1, 8, 128, P, 128, P, (1 << 31) - 1, P, 128, P, None, P, 8, None) == -1
    assert lib.uc2_linear_wgrad((1 << 31) - 1, 8, 8, P, 8, P, 8, P, 8, None, P, 1 << 40, None) == -1


def test_a_leaf_remembers_the_stream_of_its_first_graph(monkeypatch):
    """note_leaves and refuse_foreign_capture on the streams and captures they are told of"""
    from uc2_amd.ops.base import note_leaves, once
    now = [0, False]                                       # (0: the default stream)
    monkeypatch.setattr(_lib, "stream", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now[1])

    class Twice(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, y):
            note_leaves(ctx)
            return x + 2 * y

        @staticmethod
        @once
        def backward(ctx, d):
            return d, 2 * d
    x, y = torch.ones(3, requires_grad=True), torch.ones(3, requires_grad=True)
    eager = Twice.apply(x, y)
    now[:] = [7, True]
    with pytest.raises(_lib.Uc2Error, match="eager graph"):
        Twice.apply(x, x.detach().clone()).sum().backward()
    with pytest.raises(_lib.Uc2Error, match="eager graph"):
        torch.autograd.grad(Twice.apply(torch.ones(3), y).sum(), [y])
    Twice.apply(x.detach().requires_grad_(), x.detach()).sum().backward()
    now[1] = False
    Twice.apply(x, y).sum().backward()                     # eager on another stream: torch joins the streams
    del eager
    now[1] = True
    x.grad = y.grad = None
    Twice.apply(x, y).sum().backward()                     # a graph of its own
    x.grad = y.grad = None
    now[:] = [5, False]
    warm = Twice.apply(x, y)                               # a warm-up on another stream, whose outputs are kept
    now[:] = [7, True]
    Twice.apply(x, y).sum().backward()
    del warm
    assert bool((x.grad == 1).all()) and bool((y.grad == 2).all())


def test_the_accumulations_below_other_operations_are_looked_at(monkeypatch):
    """a capture is refused for a leaf behind other operations too; what has been looked at is not walked again"""
    from uc2_amd.ops import base
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    streams, asked = {}, []

    def stream_of(node):
        asked.append(node.variable)
        return streams.get(id(node.variable), 7)
    monkeypatch.setattr(base, "_accumulation_stream", stream_of)

    class Twice(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return 2 * x

        @staticmethod
        @base.once
        def backward(ctx, d):
            return 2 * d
    x, y = torch.ones(3, requires_grad=True), torch.ones(3, requires_grad=True)
    f = lambda: Twice.apply(Twice.apply((x.double() * y.view(3)).float())).sum()  # noqa: E731
    f().backward()
    assert len(asked) == 2 and bool((x.grad == 4).all())
    streams[id(y)] = 0
    out = f()
    for _ in range(3):                                     # (a pass that is asked for again is refused again)
        with pytest.raises(_lib.Uc2Error, match="eager graph"):
            out.backward(retain_graph=True)


def test_the_module_that_knows_the_accumulations_is_built():
    x = torch.ones(3, requires_grad=True)
    y = 2 * x
    assert _lib.accumulation_stream(x) is None and y.requires_grad          # (the CPU has no streams; without the module this raises)


def test_cpu_tensors_are_refused():
    x, w, g = torch.zeros(4, 128, dtype=torch.bfloat16), torch.zeros(8, 128), torch.ones(128)
    q = torch.zeros(1, 2, 4, 64)
    for f in (lambda: ops.fp8_quantize_block(x), lambda: ops.fp8_quantize_weight_block(w), lambda: ops.linear_fp8_block(x, w), lambda: ops.rms_norm(x, g), lambda: ops.rms_norm_fp8(x, g),
              lambda: ops.cross_attention(q, q, q), lambda: ops.fp8_quantize_weight_block(g),
              lambda: ops.gemm_fp8_block(ops.BlockRows(torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(1, 4, dtype=torch.int32), 128),
                                         ops.BlockWeight(torch.zeros(8, 128, dtype=torch.uint8), torch.zeros(1, 1, dtype=torch.uint8)))):
        with pytest.raises(_lib.Uc2Error):
            f()


def test_gradients_are_refused_where_they_would_be_lost():
    """quantisation and its product run outside autograd: an argument that wants a gradient raises, under no_grad it is a constant"""
    x, w, bias = torch.zeros(4, 128, dtype=torch.bfloat16, requires_grad=True), torch.zeros(8, 128, requires_grad=True), torch.zeros(8, requires_grad=True)
    a = ops.BlockRows(torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(1, 4, dtype=torch.int32), 128)
    b = ops.BlockWeight(torch.zeros(8, 128, dtype=torch.uint8), torch.zeros(1, 1, dtype=torch.uint8))
    for f in (lambda: ops.fp8_quantize_block(x), lambda: ops.fp8_quantize_block(2 * x), lambda: ops.fp8_quantize_weight_block(w), lambda: ops.fp8_quantize_weight_block(w, transpose=True),
              lambda: ops.gemm_fp8_block(a, b, bias=bias)):
        with pytest.raises(_lib.Uc2Error, match="has no gradient"):
            f()
        with torch.no_grad(), pytest.raises(_lib.Uc2Error, match="GPU only"):            # (the next check)
            f()


def test_structures_match_the_header(tmp_path):
    """the binding's packed structures, these here and a C compiler's: the same sizes, and each field at the same place"""
    import os
    import subprocess
    fields = [(t, n) for t, c in (("Uc2CrossAttn", _CrossAttn), ("Uc2CrossAttnGrad", _CrossAttnGrad)) for n, _ in c._fields_]
    src = tmp_path / "s.c"
    src.write_text('#include "uc2_hip.h"\n#include <stdio.h>\nint main(void) {\n' + "".join('printf("%%zu ", offsetof(%s, %s));\n' % f for f in fields)
                   + 'printf("%zu %zu", sizeof(Uc2CrossAttn), sizeof(Uc2CrossAttnGrad)); return 0; }\n')
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "s")])
    want = [int(x) for x in subprocess.check_output([str(tmp_path / "s")]).split()]
    here = [getattr(c, n).offset for c in (_CrossAttn, _CrossAttnGrad) for n, _ in c._fields_] + [ctypes.sizeof(_CrossAttn), ctypes.sizeof(_CrossAttnGrad)]
    assert want == here and [_ATTN.size, _GRAD.size] == here[-2:]
    packed = _CrossAttn.from_buffer_copy(_ATTN.pack(*range(1, 8), 0.5, 0.25, *range(10, 33)))
    got = [getattr(packed, n) for n, _ in _CrossAttn._fields_]
    assert got == [*range(1, 8), 0.5, 0.25, *range(10, 33)]
    packed = _CrossAttnGrad.from_buffer_copy(_GRAD.pack(*range(1, 17)))
    assert [getattr(packed, n) for n, _ in _CrossAttnGrad._fields_] == list(range(1, 17))


def test_oracle_rounds_as_torch_does():
    """block_ref's e4m3 against torch's own cast, and its exponents against their definition"""
    x = torch.randn(4000, dtype=torch.float64) * torch.exp(2 * torch.randn(4000, dtype=torch.float64))
    x = x[x.abs() <= 448].float()
    assert torch.equal(R.e4m3(x.double()), x.to(torch.float8_e4m3fn).double())
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    every = every[torch.isfinite(every)]
    assert torch.equal(R.e4m3(every), every)
    e = R.block_exponents(torch.tensor([448.0, 448.1, 224.0, 1.75, 1.76, 0.0]))
    assert e.tolist() == [127, 128, 126, 119, 120, 1]


def test_oracle_attention_is_softmax():
    q, k, v = torch.randn(2, 5, 4, 32), torch.randn(2, 7, 2, 32), torch.randn(2, 7, 2, 32)
    dout = torch.randn(2, 5, 4, 32)
    leaves = [t.double().requires_grad_() for t in (q, k, v)]
    t = lambda a: a.repeat_interleave(4 // a.shape[2], 2).transpose(1, 2)  # noqa: E731
    o = (torch.softmax(t(leaves[0]) @ t(leaves[1]).transpose(2, 3) * 0.2, -1) @ t(leaves[2])).transpose(1, 2)
    want = [o, *torch.autograd.grad(o, leaves, dout.double())]
    got, _ = R.attention(q, k, v, 0.2, None, None, dout)
    for a, b in zip(got, want):
        assert torch.allclose(a, b.detach(), atol=1e-12)


def test_saved_pointers_are_read_from_the_call_structure():
    from uc2_amd.ops.cross import _PTRS
    names = [n for n, _ in _CrossAttn._fields_]
    packed = _ATTN.pack(*range(1, 8), 0.5, 0.25, *range(10, 33))
    value = dict(zip(names, (*range(1, 8), 0.5, 0.25, *range(10, 33))))
    assert _PTRS.size == _ATTN.size
    assert _PTRS.unpack(packed) == tuple(value[n] for n in ("q", "k", "v", "key_mask", "k_lens", "out", "lse", "out_f32", "seed", "site"))
