"""The block-scaled e4m3 projections, the root-mean-square norm before them and the cross attention after them, as timed cases.

Each case names one call that a decoder-style block over an encoder's states makes: the norm of a residual stream (with its
gradient, or with an e4m3 output that feeds a projection), a linear layer whose operands are e4m3 with a power-of-two scale for each
block of 128, and attention from one sequence to the states of another."""
import math

import torch

own = False

BLOCK, E4M3_MAX = 128, 448.0
EPS = 1e-6
BF16, F32 = torch.bfloat16, torch.float32


def listed():
    return [
        # one optimizer step's norm over 512 image-text pairs of 130 positions at hidden size 1024: reads and writes only
        dict(name="norm_train_pairs", op="norm", rows=66560, width=1024, type="bf16"),
        # the parity mode's norm at a width that is no multiple of a wave's share
        dict(name="norm_train_fp32_odd", op="norm", rows=4099, width=1000, type="fp32"),
        # eight sequences that answer a token each: the norm in front of the widening projection
        dict(name="norm_linear_tokens", op="norm_linear", rows=8, width=1024, out=4096),
        # the same pair of calls over a batch of prompts
        dict(name="norm_linear_prompts", op="norm_linear", rows=33280, width=1024, out=4096),
        # one token through the narrowing projection: the weight's bytes are the work
        dict(name="linear_token", op="linear", rows=1, width=4096, out=1024, train=False),
        # a ragged batch on sizes that fill no tile
        dict(name="linear_odd", op="linear", rows=1237, width=1000, out=777, train=False),
        # a large batch: the matrix pipes are the bound
        dict(name="linear_batch", op="linear", rows=66560, width=1024, out=4096, train=False),
        # a training micro-batch of 104 pairs of 96 positions through a fused projection, weights quantised anew as after every step
        dict(name="linear_train", op="linear", rows=9984, width=768, out=2304, train=True),
        # single tokens against long encoder states whose key / value heads are shared by four query heads
        dict(name="attend_token", op="attend", batch=16, queries=1, keys=16384, heads=16, shared=4, dim=64, type="bf16", mask="lens", train=False),
        # text positions over the image regions of their pair, 10 to 100 of them
        dict(name="attend_regions", op="attend", batch=104, queries=60, keys=100, heads=12, shared=1, dim=64, type="bf16", mask="lens", train=True),
        # long text over long encoder states
        dict(name="attend_long", op="attend", batch=2, queries=2048, keys=4096, heads=16, shared=1, dim=64, type="bf16", mask="none", train=True),
        # the parity mode with an additive mask on odd lengths
        dict(name="attend_fp32", op="attend", batch=8, queries=77, keys=211, heads=12, shared=3, dim=64, type="fp32", mask="added", train=True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "norm_linear", "linear", "linear", "attend", "attend", "attend"])
    if op == "norm":
        width = rng.choice([768, 1024, rng.randint(64, 4096)])
        return dict(op=op, rows=min(_spread(rng, 1, 66560), 60_000_000 // width), width=width, type=rng.choice(["bf16", "bf16", "fp32"]))
    if op == "norm_linear":
        width, out = rng.choice([768, 1024, rng.randint(100, 2048)]), _spread(rng, 64, 4096)
        return dict(op=op, rows=min(_spread(rng, 1, 33280), int(1.2e11) // (width * out)), width=width, out=out)
    if op == "linear":
        width, out = rng.choice([768, 1024, 4096, _spread(rng, 16, 4096)]), rng.choice([1024, 4096, _spread(rng, 16, 4096)])
        train = rng.random() < 0.5
        return dict(op=op, rows=max(1, min(_spread(rng, 1, 66560), int(2.5e11 if not train else 5e10) // (width * out))), width=width, out=out, train=train)
    train = rng.random() < 0.6
    kind = rng.choice(["bf16", "bf16", "fp32"])
    dim, kv, shared = rng.choice([32, 64, 64, 128]), rng.choice([1, 4, 12]), rng.choice([1, 1, 2, 4])
    queries = rng.choice([1, _spread(rng, 1, 2048), _spread(rng, 16, 512)])
    keys = _spread(rng, 1, 4096) if train else _spread(rng, 1, 16384)
    most = int(6e9 if train else 3e9) // (4 if kind == "fp32" else 1)
    batch = max(1, min(_spread(rng, 1, 64), most // (queries * keys * kv * shared * dim), 200_000_000 // (keys * kv * dim)))
    return dict(op=op, batch=batch, queries=queries, keys=keys, heads=kv * shared, shared=shared, dim=dim, type=kind,
                mask=rng.choice(["none", "lens", "added"]), train=train)


def _type(case):
    return F32 if case.get("type") == "fp32" else BF16


# ---- the e4m3 format: values over 2^e with one e for each block, kept as e + 127 in a byte -------------------------------------------
def _exponents(amax):
    """the smallest e with amax <= 448 * 2^e, as the biased byte (1 at least)"""
    mant, exp = torch.frexp(amax.double())                       # amax = mant 2^exp, mant in [0.5, 1)
    e = exp.to(torch.int64) - 9 + (mant > 0.875).to(torch.int64)  # 448 = 0.875 * 2^9
    return torch.where(amax > 0, (e + 127).clamp(1, 254), torch.ones_like(e))


def _pad(x, rows, cols):
    return torch.nn.functional.pad(x, (0, -x.shape[1] % cols, 0, -x.shape[0] % rows))


def _row_blocks(x):
    """(the e4m3 values over the block's 2^e, in x's own scale and type) for blocks of 128 along a row"""
    p = _pad(x, 1, BLOCK)
    p = p.reshape(p.shape[0], -1, BLOCK)
    s = torch.exp2((_exponents(p.abs().amax(-1, keepdim=True)) - 127).to(x.dtype))
    q = (p / s).float().to(torch.float8_e4m3fn).to(x.dtype) * s
    return q.reshape(x.shape[0], -1)[:, :x.shape[1]]


def _square_blocks(w):
    """(bytes [rows, cols padded to 128], exponents [row blocks, column blocks]) for blocks of 128 x 128"""
    n, k = w.shape
    p = _pad(w.float(), BLOCK, BLOCK)
    p = p.reshape(p.shape[0] // BLOCK, BLOCK, -1, BLOCK)
    e = _exponents(p.abs().amax((1, 3)))
    q = (p * torch.exp2((127 - e).float())[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.view(torch.uint8).reshape(-1, p.shape[2] * BLOCK)[:n].contiguous(), e.to(torch.uint8)


def _square_values(q, e, k, kind=F32):
    v = _pad(q.view(torch.float8_e4m3fn).to(kind), BLOCK, BLOCK)
    v = v.reshape(e.shape[0], BLOCK, e.shape[1], BLOCK) * torch.exp2((e.to(torch.int64) - 127).to(kind))[:, None, :, None]
    return v.reshape(e.shape[0] * BLOCK, -1)[:q.shape[0], :k]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t = _type(case)

    def normal(*shape, std=1.0, kind=t):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(kind)

    s = dict(case=case)
    if case["op"] in ("norm", "norm_linear"):
        m, h = case["rows"], case["width"]
        s.update(x=normal(m, h), residual=normal(m, h, std=2.0), gain=1 + normal(h, std=0.1, kind=F32))
        if case["op"] == "norm":
            s.update(dy=normal(m, h), ds=normal(m, h))
        else:
            s["weight"] = _square_blocks(normal(case["out"], h, std=h ** -0.5, kind=F32))
    elif case["op"] == "linear":
        m, k, n = case["rows"], case["width"], case["out"]
        # activations whose columns differ in size, as those behind a gain do
        s.update(x=(normal(m, k, kind=F32) * torch.exp(normal(k, kind=F32))).to(BF16), bias=normal(n, std=0.1, kind=F32))
        w = normal(n, k, std=k ** -0.5, kind=F32)
        if case["train"]:
            s.update(w=w, dy=normal(m, n))
        else:
            s["weight"] = _square_blocks(w)
    else:
        b, lq, lk, nh, d = case["batch"], case["queries"], case["keys"], case["heads"], case["dim"]
        kv = normal(b, lk, 2, nh // case["shared"], d)           # one projection's output: keys and values side by side
        s.update(q=normal(b, lq, nh, d), k=kv[:, :, 0], v=kv[:, :, 1], lens=None, added=None)
        if case["mask"] == "lens":
            s["lens"] = torch.randint(max(1, lk // 10), lk + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        elif case["mask"] == "added":
            gone = torch.rand(b, lk, generator=g, device="cuda") < 0.2
            gone[:, 0] = False
            s["added"] = normal(b, lk, kind=F32).masked_fill(gone, -math.inf)
        if case["train"]:
            s["dout"] = normal(b, lq, nh, d)
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------------------------------
def _norm(s, kind):
    t = s["x"].dtype
    total = (s["x"].to(kind) + s["residual"].to(kind)).to(t)     # the stream that is carried on
    f = total.to(kind)
    r = torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS)
    return total, f * r, r


def _norm_train(s, kind):
    total, hat, r = _norm(s, kind)
    gain, dy = s["gain"].to(kind), s["dy"].to(kind)
    g = dy * gain
    dx = r * (g - hat * (g * hat).mean(-1, keepdim=True)) + s["ds"].to(kind)
    return [hat * gain, total, dx, (dy * hat).sum(0)]


def _linear(s, kind):
    return _row_blocks(s["x"].to(kind)) @ _square_values(*s["weight"], s["x"].shape[1], kind).t() + s["bias"].to(kind)


def _linear_train(s, kind):
    x, dy = s["x"].to(kind), s["dy"].to(kind)
    w = _square_values(*_square_blocks(s["w"]), x.shape[1], kind)
    return [_row_blocks(x) @ w.t() + s["bias"].to(kind), _row_blocks(dy) @ w, dy.t() @ x, dy.sum(0)]


def _scores(s, kind):
    """rows of a shared head side by side: queries [b, kv, lq g, d], keys and values [b, kv, lk, d], and the masked scores"""
    c = s["case"]
    b, lq, g, d = c["batch"], c["queries"], c["shared"], c["dim"]
    rows = lambda x: x.to(kind).reshape(b, lq, -1, g, d).permute(0, 2, 1, 3, 4).reshape(b, -1, lq * g, d)  # noqa: E731
    q, k, v = rows(s["q"]), s["k"].to(kind).transpose(1, 2).contiguous(), s["v"].to(kind).transpose(1, 2).contiguous()
    x = q @ k.transpose(2, 3).contiguous() * d ** -0.5
    if s["lens"] is not None:
        x = x.masked_fill(torch.arange(c["keys"], device=x.device) >= s["lens"][:, None, None, None], -math.inf)
    if s["added"] is not None:
        x = x + s["added"].to(kind)[:, None, None, :]
    return rows, q, k, v, x


def _attend(s, kind):
    c = s["case"]
    b, lq, g, d = c["batch"], c["queries"], c["shared"], c["dim"]
    back = lambda x: x.reshape(b, -1, lq, g, d).permute(0, 2, 1, 3, 4).reshape(b, lq, -1, d)  # noqa: E731
    rows, q, k, v, x = _scores(s, kind)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = p @ v
    if not c["train"]:
        return [back(o)]
    do = rows(s["dout"])
    dp = do @ v.transpose(2, 3).contiguous()
    dx = p * (dp - (do * o).sum(-1, keepdim=True)) * d ** -0.5
    dk, dv = dx.transpose(2, 3).contiguous() @ q, p.transpose(2, 3).contiguous() @ do
    return [back(o), back(dx @ k), dk.transpose(1, 2), dv.transpose(1, 2)]


def _types(case):
    t = _type(case)
    return {"norm": [t, t, t, F32], "norm_linear": [BF16, BF16], "linear": [BF16, BF16, F32, F32], "attend": [t] * 4}[case["op"]]


def _plain(s, kind):
    c = s["case"]
    if c["op"] == "norm":
        return _norm_train(s, kind)
    if c["op"] == "norm_linear":
        total, hat, _ = _norm(s, kind)
        return [_row_blocks(hat * s["gain"].to(kind)) @ _square_values(*s["weight"], c["width"], kind).t(), total]
    if c["op"] == "linear":
        return _linear_train(s, kind) if c["train"] else [_linear(s, kind)]
    return _attend(s, kind)


# ---- the framework's calls ----------------------------------------------------------------------------------------------------------
def _run_own(s):
    from uc2_amd import ops
    c = s["case"]
    if c["op"] == "norm":
        x, r, w = (s[n].detach().requires_grad_() for n in ("x", "residual", "gain"))
        y, total = ops.rms_norm(x, w, EPS, residual=r)
        dx, dw = torch.autograd.grad([y, total], [x, w], [s["dy"], s["ds"]])
        return [y.detach(), total.detach(), dx, dw]
    if c["op"] == "norm_linear":
        a, total = ops.rms_norm_fp8(s["x"], s["gain"], EPS, residual=s["residual"])
        return [ops.gemm_fp8_block(a, s["weight"]), total]
    if c["op"] == "linear":
        if not c["train"]:
            return [ops.gemm_fp8_block(ops.fp8_quantize_block(s["x"]), s["weight"], bias=s["bias"])]
        x, w, b = (s[n].detach().requires_grad_() for n in ("x", "w", "bias"))
        y = ops.linear_fp8_block(x, w, b)
        return [y.detach(), *torch.autograd.grad(y, [x, w, b], s["dy"])]
    if not c["train"]:
        return [ops.cross_attention(s["q"], s["k"], s["v"], key_mask=s["added"], k_lens=s["lens"])]
    q, k, v = (s[n].detach().requires_grad_() for n in ("q", "k", "v"))
    o = ops.cross_attention(q, k, v, key_mask=s["added"], k_lens=s["lens"])
    return [o.detach(), *torch.autograd.grad(o, [q, k, v], s["dout"])]


def run(state):
    if own:
        return _run_own(state)
    return [x.to(t) for x, t in zip(_plain(state, F32), _types(state["case"]))]


def work(case):
    e = 4 if case.get("type") == "fp32" else 2
    if case["op"] == "norm":                                     # x, residual, dy, ds in; y, stream, dx out; the stream again in the backward
        return {"bytes": 7.0 * case["rows"] * case["width"] * e + 8 * case["width"], "flops": 14.0 * case["rows"] * case["width"]}
    if case["op"] in ("norm_linear", "linear"):
        m, k, n = case["rows"], case["width"], case["out"]
        if case.get("train"):                                    # x, w, dy in; y, dx, dw out
            return {"bytes": 4.0 * m * k + 4.0 * m * n + 8.0 * n * k, "flops": 6.0 * m * n * k}
        norm = case["op"] == "norm_linear"
        return {"bytes": (6.0 if norm else 2.0) * m * k + 1.0 * n * k + 2.0 * m * n, "flops": 2.0 * m * n * k}
    b, lq, nh, d, kv = case["batch"], case["queries"], case["heads"], case["dim"], case["heads"] // case["shared"]
    lk = case["keys"] * (0.55 if case["mask"] == "lens" else 1.0)
    rows, keys = 1.0 * b * lq * nh * d * e, 1.0 * b * lk * kv * d * e
    passes, products = ((4, 4), 14) if case["train"] else ((2, 2), 4)
    return {"bytes": passes[0] * rows + passes[1] * keys, "flops": 1.0 * products * b * nh * lq * lk * d}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------------------
def _cut64(v, size, dims):
    """v rounded to the 4-bit significands of e4m3 under one power of two for each block of `size` along `dims`"""
    pads = [0, 0, 0, 0]
    for d in dims:
        pads[2 * (1 - d) + 1] = -v.shape[d] % size
    p = torch.nn.functional.pad(v, pads)
    r, c = (size if 0 in dims else 1), (size if 1 in dims else 1)
    p = p.reshape(p.shape[0] // r, r, p.shape[1] // c, c)
    top = p.abs().amax((1, 3), keepdim=True)
    unit = torch.exp2(torch.ceil(torch.log2(top.clamp_min(1e-300) / E4M3_MAX)).clamp_min(-126))
    unit = torch.where(top > E4M3_MAX * unit, unit * 2, torch.where(top <= E4M3_MAX * unit / 2, unit / 2, unit)).clamp_min(2.0 ** -126)
    x = p / unit
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)  # spacing 2^(e-3), 2^-9 below 2^-6
    x = torch.round(x / step) * step * unit                     # torch.round: halves to even
    return x.reshape(p.shape[0] * r, -1)[:v.shape[0], :v.shape[1]]


def exact(case, seed):
    s = prepare(case, seed)
    f = lambda n: s[n].double()  # noqa: E731
    if case["op"] in ("norm", "norm_linear"):
        total = (s["x"].float() + s["residual"].float()).to(s["x"].dtype)   # the rounding is part of the definition
        z = total.double()
        inv = 1.0 / torch.sqrt(z.pow(2).sum(-1, keepdim=True) / z.shape[1] + EPS)
        y = z * inv * f("gain")
        if case["op"] == "norm_linear":
            q, e = s["weight"]
            w = torch.ldexp(q.view(torch.float8_e4m3fn).double(), e.repeat_interleave(BLOCK, 0)[:q.shape[0]].repeat_interleave(BLOCK, 1).int() - 127)
            return [_cut64(y, BLOCK, (1,)) @ w[:, :case["width"]].t(), z]
        a = f("dy") * f("gain")
        dx = a * inv - z * inv.pow(3) * (a * z).sum(-1, keepdim=True) / z.shape[1] + f("ds")
        return [y, z, dx, torch.einsum("mh,mh->h", f("dy"), z * inv)]
    if case["op"] == "linear":
        x = f("x")
        if not case["train"]:
            q, e = s["weight"]
            w = torch.ldexp(q.view(torch.float8_e4m3fn).double(), e.repeat_interleave(BLOCK, 0)[:q.shape[0]].repeat_interleave(BLOCK, 1).int() - 127)
            return [torch.addmm(f("bias"), _cut64(x, BLOCK, (1,)), w[:, :case["width"]].t())]
        w, dy = _cut64(f("w"), BLOCK, (0, 1)), f("dy")
        return [torch.addmm(f("bias"), _cut64(x, BLOCK, (1,)), w.t()), torch.mm(_cut64(dy, BLOCK, (1,)), w), torch.mm(dy.t(), x), dy.sum(0)]
    g, lk = case["shared"], case["keys"]
    if case["batch"] * case["heads"] * case["queries"] * lk > 600_000_000:
        return None
    heads = lambda x, n: x.double().repeat_interleave(n, 2).permute(0, 2, 1, 3).contiguous()  # noqa: E731
    q, k, v = heads(s["q"], 1), heads(s["k"], g), heads(s["v"], g)
    logits = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(case["dim"])
    if s["added"] is not None:
        logits += s["added"].double()[:, None, None, :]
    if s["lens"] is not None:
        logits = torch.where(torch.arange(lk, device="cuda")[None, None, None, :] < s["lens"].long()[:, None, None, None], logits, -math.inf)
    p = (logits - torch.logsumexp(logits, -1, keepdim=True)).exp()
    o = torch.matmul(p, v)
    whole = lambda x: x.permute(0, 2, 1, 3)  # noqa: E731
    if not case["train"]:
        return [whole(o)]
    do = heads(s["dout"], 1)
    dp = torch.matmul(do, v.transpose(-1, -2))
    dl = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(case["dim"])
    one = lambda x: whole(x.reshape(x.shape[0], -1, g, *x.shape[2:]).sum(2))  # noqa: E731
    return [whole(o), whole(torch.matmul(dl, k)), one(torch.matmul(dl.transpose(-1, -2), q)), one(torch.matmul(p.transpose(-1, -2), do))]
