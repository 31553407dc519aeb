"""The operators of a residual block in 8 bits, as they are measured: products in 8-bit integers and the norms around a block.

`listed()` is the fixed set, `draw(rng)` one more case of the same ranges, `prepare(case, seed)` what a program holds before the
call, `run(state)` one pass -- in elementary torch operations in 32 bits, or, where `own` is true, through the library's entry
points -- `work(case)` what a pass cannot do without and `exact(case, seed)` its result in 64 bits.

kind "linear": out = act((q . w^T) * x_scale * w_scale + bias) with q int8 rows; floating rows are quantised on the way:
    a = max|x|, q = rint(x * min(127 / a, FLT_MAX)), x_scale = a / 127 (NaN where a is not finite).
kind "norm": s = residual_scale * r + branch_scale * gate * N1(y), o = N2(s), N one of none, layer, rms.
kind "norm_grad": the gradients of all inputs of "norm" for given gradients of s and o.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
EPS = 1e-5
FLT_MAX = torch.finfo(torch.float32).max


def listed():
    return [
        # the first MLP product of one token at the library's BERT width: a server answering one request at a time
        dict(name="linear_1x768x3072_f16", kind="linear", rows=1, inner=768, cols=3072, dtype="float16", out="float16", act="gelu", bias=True),
        # the second MLP product of a handful of tokens
        dict(name="linear_7x3072x768_bf16", kind="linear", rows=7, inner=3072, cols=768, dtype="bfloat16", out="bfloat16", act="none", bias=True),
        # the MLP of a Swin block on one 14 x 14 image
        dict(name="linear_196x512x2048_f16", kind="linear", rows=196, inner=512, cols=2048, dtype="float16", out="float16", act="gelu", bias=True),
        # sizes that divide by nothing: ragged tokens, a classifier's width, fp32 in and out
        dict(name="linear_1571x1001x1003_f32", kind="linear", rows=1571, inner=1001, cols=1003, dtype="float32", out="float32", act="relu", bias=True),
        # the first MLP product of the benchmark's 64 sequences of 128 tokens
        dict(name="linear_8192x768x3072_f16", kind="linear", rows=8192, inner=768, cols=3072, dtype="float16", out="float16", act="gelu", bias=True),
        # the largest: rows that are in 8 bits already (a norm left them so), wide layers, no bias
        dict(name="linear_8192x4096x4096_i8", kind="linear", rows=8192, inner=4096, cols=4096, dtype="int8", out="bfloat16", act="none", bias=False),
        # LayerNorm of residual and branch for one token at the BERT width
        dict(name="norm_1x768_f16", kind="norm", rows=1, cols=768, dtype="float16", params="float16", n1="none", n2="layer", gates=0, alpha=1.0, beta=1.0),
        # between the blocks of 64 sequences of 128 tokens: a learned scale per channel on the branch, LayerNorm in front of the next one
        dict(name="norm_8192x768_f16", kind="norm", rows=8192, cols=768, dtype="float16", params="float16", n1="none", n2="layer", gates=1, alpha=1.0, beta=1.0),
        # norm behind the branch, gates per image, norm in front of the next block: four images of 56 x 56 tokens, fp32
        dict(name="norm_12544x128_f32", kind="norm", rows=12544, cols=128, dtype="float32", params="float32", n1="layer", n2="layer", gates=4, alpha=1.0, beta=1.0),
        # root-mean-square norms on both sides of a wide block with a scaled residual, an odd number of tokens
        dict(name="norm_4095x4096_bf16", kind="norm", rows=4095, cols=4096, dtype="bfloat16", params="float32", n1="rms", n2="rms", gates=0, alpha=1.25, beta=0.22),
        # training at small and odd sizes: both norms, gates per sample
        dict(name="grad_1001x513_f32", kind="norm_grad", rows=1001, cols=513, dtype="float32", params="float32", n1="layer", n2="layer", gates=7, alpha=0.9, beta=1.0),
        # training at the benchmark's rows, gates per sequence
        dict(name="grad_8192x768_f16", kind="norm_grad", rows=8192, cols=768, dtype="float16", params="float32", n1="layer", n2="layer", gates=64, alpha=1.0, beta=1.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("linear", "linear", "norm", "norm_grad"))
    dtype = rng.choice(("float16", "bfloat16", "float32"))
    if kind == "linear":
        given = rng.random() < 0.25
        return dict(kind="linear", rows=_log_int(rng, 1, 8192), inner=_log_int(rng, 48, 4096), cols=_log_int(rng, 48, 4096),
                    dtype="int8" if given else dtype, out=dtype, act=rng.choice(("none", "relu", "gelu")), bias=rng.random() < 0.75)
    gates = rng.choice((0, 1, 2, 16, 64))
    rows = _log_int(rng, 1, 8192)
    if gates > 1:
        rows = max(1, rows // gates) * gates          # as many rows for each gate
    n1, n2 = rng.choice((("none", "layer"), ("none", "rms"), ("layer", "layer"), ("rms", "rms"), ("layer", "none")))
    return dict(kind=kind, rows=rows, cols=_log_int(rng, 33, 4096), dtype=dtype, params=rng.choice((dtype, "float32")), n1=n1, n2=n2,
                gates=gates, alpha=rng.choice((1.0, 0.9)), beta=rng.choice((1.0, 0.22)))


def _quantise(x, most=127.0):
    """Rows of x in 8-bit integers and their scales, in the type of x."""
    a = x.abs().amax(dim=-1, keepdim=True)
    most = torch.full_like(a, most)                # quotients of two tensors: a number's would be a product with its reciprocal
    inv = (most / a).clamp(max=FLT_MAX)
    fine = torch.isfinite(a)
    q = torch.where(fine, torch.round(x * inv), torch.zeros_like(x))
    return q, torch.where(fine, a / most, torch.full_like(a, math.nan))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * std

    s = dict(case)
    if case["kind"] == "linear":
        M, K, N = case["rows"], case["inner"], case["cols"]
        # activations with a few strong channels, tokens of different loudness and, in larger batches, silent padding tokens
        x = randn(M, K) * torch.exp(randn(K, std=0.5)) * torch.exp(randn(M, 1, std=0.5))
        if M >= 64:
            x[-3:] = 0
        w, s["w_scale"] = _quantise(randn(N, K, std=0.03))
        s["w_scale"] = s["w_scale"].reshape(N).contiguous()
        s["w"] = _padded_int8(w)
        s["b"] = randn(N, std=0.1).to(DTYPES[case["out"]]) if case["bias"] else None
        if case["dtype"] == "int8":
            q, sc = _quantise(x)
            s["x"], s["x_scale"] = _padded_int8(q), sc.reshape(M).contiguous()
        else:
            s["x"], s["x_scale"] = x.to(DTYPES[case["dtype"]]), None
        return s
    M, N, G = case["rows"], case["cols"], case["gates"]
    t, p = DTYPES[case["dtype"]], DTYPES[case["params"]]
    s["r"], s["y"] = randn(M, N, std=2.0).to(t), (randn(M, N) + 0.3).to(t)
    s["g"] = (0.5 + randn(G, N, std=0.2)).to(p) if G else None
    for k in ("n1", "n2"):
        s["w_" + k] = (1 + randn(N, std=0.1)).to(p) if case[k] != "none" else None
        s["b_" + k] = randn(N, std=0.1).to(p) if case[k] == "layer" else None
    if case["kind"] == "norm_grad":
        s["ds"] = randn(M, N, std=0.5).to(t)
        s["do"] = randn(M, N).to(t) if case["n2"] != "none" else None
    return s


def _padded_int8(q):
    """int8 rows that begin on 16-byte boundaries, as the library lays quantised rows out."""
    rows, cols = q.shape
    buf = torch.zeros(rows, (cols + 15) // 16 * 16, dtype=torch.int8, device=q.device)
    buf[:, :cols] = q.to(torch.int8)
    return buf[:, :cols]


def run(s):
    if own:
        return _run_own(s)
    return _linear(s) if s["kind"] == "linear" else _norm(s) if s["kind"] == "norm" else _norm_grad(s)


def _run_own(s):
    if s["kind"] == "linear":
        from souffle_models_b200 import int8
        return int8.int8_linear(s["x"], s["w"], s["w_scale"], bias=s["b"], activation=s["act"], x_scale=s["x_scale"], out_dtype=DTYPES[s["out"]])
    from souffle_models_b200 import residual_norm as rn
    kw = dict(branch_norm=s["n1"], branch_weight=s["w_n1"], branch_bias=s["b_n1"], gate=s["g"], out_norm=s["n2"], out_weight=s["w_n2"],
              residual_scale=s["alpha"], branch_scale=s["beta"], branch_eps=EPS, out_eps=EPS)
    if s["kind"] == "norm":
        return rn.residual_norm(s["r"], s["y"], out_bias=s["b_n2"], **kw)
    return rn.residual_norm_backward(s["ds"], s["do"], s["r"], s["y"], **kw)


# ---- the plain form: 32 bits throughout, rounded once at the end -------------------------------------------------

def _f(t):
    return None if t is None else t.float()


def _linear(s):
    if s["x_scale"] is None:
        q, sx = _quantise(s["x"].float())
    else:
        q, sx = s["x"].float(), s["x_scale"][:, None]
    v = (q @ s["w"].float().t()) * sx * s["w_scale"][None, :]
    if s["b"] is not None:
        v = v + s["b"].float()
    if s["act"] == "relu":
        v = torch.where(v < 0, torch.zeros_like(v), v)
    elif s["act"] == "gelu":
        v = 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    return v.to(DTYPES[s["out"]])


def _hat(x, kind):
    """The normalised rows and the reciprocal of their deviation."""
    if kind == "layer":
        x = x - x.mean(dim=-1, keepdim=True)
    rstd = torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS)
    return x * rstd, rstd


def _affine(h, w, b):
    h = h * w
    return h if b is None else h + b


def _per_row(g, rows):
    """Gates [G, C] as [G, 1, C] against rows [G, rows / G, C]."""
    return g.float()[:, None, :]


def _gated(u, g):
    return u if g is None else (u.view(g.shape[0], -1, u.shape[1]) * _per_row(g, u.shape[0])).view_as(u)


def _norm(s):
    u = s["y"].float()
    if s["n1"] != "none":
        u = _affine(_hat(u, s["n1"])[0], _f(s["w_n1"]), _f(s["b_n1"]))
    h = s["alpha"] * s["r"].float() + s["beta"] * _gated(u, s["g"])
    o = None
    if s["n2"] != "none":
        o = _affine(_hat(h, s["n2"])[0], _f(s["w_n2"]), _f(s["b_n2"])).to(s["y"].dtype)
    return h.to(s["y"].dtype), o


def _norm_back(d, hat, rstd, w, kind):
    """(gradient of the norm's input, of its weight, of its bias)."""
    a = d * w
    back = a - hat * (a * hat).mean(dim=-1, keepdim=True)
    if kind == "layer":
        back = back - a.mean(dim=-1, keepdim=True)
    return back * rstd, (d * hat).sum(0), d.sum(0) if kind == "layer" else None


def _norm_grad(s):
    y, p = s["y"].float(), DTYPES[s["params"]]
    u, out = y, dict.fromkeys(("branch_weight", "branch_bias", "gate", "out_weight", "out_bias"))
    if s["n1"] != "none":
        yhat, yr = _hat(y, s["n1"])
        u = _affine(yhat, _f(s["w_n1"]), _f(s["b_n1"]))
    d = s["ds"].float()
    if s["n2"] != "none":
        hhat, hr = _hat(s["alpha"] * s["r"].float() + s["beta"] * _gated(u, s["g"]), s["n2"])
        dh, out["out_weight"], out["out_bias"] = _norm_back(s["do"].float(), hhat, hr, _f(s["w_n2"]), s["n2"])
        d = d + dh
    out["residual"] = (s["alpha"] * d).to(s["r"].dtype)
    if s["g"] is not None:
        out["gate"] = s["beta"] * (d * u).view(s["g"].shape[0], -1, d.shape[1]).sum(1)
    du = s["beta"] * _gated(d, s["g"])
    if s["n1"] != "none":
        du, out["branch_weight"], out["branch_bias"] = _norm_back(du, yhat, yr, _f(s["w_n1"]), s["n1"])
    out["branch"] = du.to(s["y"].dtype)
    return {k: v if v is None or k in ("residual", "branch") else v.to(p) for k, v in out.items()}


# ---- the bytes and operations of one pass ------------------------------------------------------------------------

def work(case):
    size = {"float16": 2, "bfloat16": 2, "float32": 4, "int8": 1}
    if case["kind"] == "linear":
        M, K, N = case["rows"], case["inner"], case["cols"]
        return {"bytes": M * K * size[case["dtype"]] + (4 * M if case["dtype"] == "int8" else 0) + N * K + 4 * N +
                (N + M * N if case["bias"] else M * N) * size[case["out"]], "flops": 2 * M * N * K}
    M, N, e, p = case["rows"], case["cols"], size[case["dtype"]], size[case["params"]]
    vectors = case["gates"] + sum({"none": 0, "rms": 1, "layer": 2}[case[k]] for k in ("n1", "n2"))
    normed = case["n2"] != "none"
    if case["kind"] == "norm":
        return {"bytes": (3 + normed) * M * N * e + vectors * N * p, "flops": 20 * M * N}
    return {"bytes": (5 + normed) * M * N * e + 2 * vectors * N * p, "flops": 50 * M * N}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    if case["kind"] == "linear":
        q, sx = d["x"].double(), d["x_scale"]
        if sx is None:
            sx = q.abs().amax(dim=1)
            q = torch.where(sx[:, None] > 0, torch.round(q * (127 / sx)[:, None]), torch.zeros_like(q))
            sx = sx / 127
        v = torch.einsum("mk,nk->mn", q, d["w"].double()) * torch.outer(sx, d["w_scale"])
        v = v if d["b"] is None else v + d["b"]
        if case["act"] == "relu":
            v = v.clamp(min=0)
        elif case["act"] == "gelu":
            v = v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * v * (1 + 0.044715 * v ** 2))
        return v
    names = {"residual": "r", "branch": "y", "gate": "g", "branch_weight": "w_n1", "branch_bias": "b_n1", "out_weight": "w_n2", "out_bias": "b_n2"}
    leaf = {k: d[n].requires_grad_(case["kind"] == "norm_grad") for k, n in names.items() if d[n] is not None}

    def norm(x, kind, w, b):
        if kind == "none":
            return x
        m = x.mean(1, keepdim=True) if kind == "layer" else 0.0
        x = (x - m) / torch.sqrt(((x - m) ** 2).mean(1, keepdim=True) + EPS)
        return x * leaf[w] + (leaf[b] if b in leaf else 0.0)

    u = norm(leaf["branch"], case["n1"], "branch_weight", "branch_bias")
    if case["gates"]:
        u = u * leaf["gate"].repeat_interleave(case["rows"] // case["gates"], dim=0)
    h = case["alpha"] * leaf["residual"] + case["beta"] * u
    o = norm(h, case["n2"], "out_weight", "out_bias") if case["n2"] != "none" else None
    if case["kind"] == "norm":
        return h, o
    total = (h * d["ds"]).sum() + (0.0 if o is None else (o * d["do"]).sum())
    grads = torch.autograd.grad(total, list(leaf.values()))
    got = dict(zip(leaf, grads))
    return {k: got.get(k) for k in names}
