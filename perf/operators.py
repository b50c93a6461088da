"""The operators of an 8-bit transformer block, as they are measured.

Three operators that follow one another in a block whose linear layers run on
8-bit integers:

  residual_norm   x' = residual_scale * x + gate * postnorm(branch), then
                  y = prenorm(x') * (1 + scale) + shift, in 16 or 32 bits or as
                  int8 with one scale per row
  quantize_rows   a 16- or 32-bit matrix as int8 with one scale per row (token)
  linear_w8a8     the product of two int8 matrices with a scale per token and
                  one per output channel, and an epilogue

`run` computes them in plain torch operations, or, where `own` is true, with
naivediffusion_b200.ops. `exact` is their definition in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "i8": torch.int8}
BYTES = {"bf16": 2, "f16": 2, "f32": 4, "i8": 1}
EPS = 1e-6
GATED = ("swiglu", "geglu")


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # One token through a text tower's block: the norm between attention and MLP.
        {"name": "norm 1x1024 rms", "op": "norm", "rows": 1, "width": 1024, "branch": "bf16", "post": "none", "gate": False,
         "pre": "rms", "weight": True, "modulate": False, "vecs": 1, "out": "bf16"},
        # A single-stream DiT's sandwich norms at 1024 x 1024: image and text rows, two sets of vectors.
        {"name": "norm 4352x4096 sandwich", "op": "norm", "rows": 4352, "width": 4096, "branch": "bf16", "post": "rms",
         "gate": True, "pre": "rms", "weight": True, "modulate": True, "vecs": 2, "out": "bf16"},
        # A DiT at batch 2, LayerNorm with adaLN vectors per batch item, straight to int8 for the next product.
        {"name": "norm 8192x2048 to int8", "op": "norm", "rows": 8192, "width": 2048, "branch": "f16", "post": "none",
         "gate": True, "pre": "layer", "weight": False, "modulate": True, "vecs": 2, "out": "i8"},
        # An odd width and ragged rows, everything in 32 bits.
        {"name": "norm 333x1155 fp32", "op": "norm", "rows": 333, "width": 1155, "branch": "f32", "post": "layer", "gate": True,
         "pre": "layer", "weight": True, "modulate": True, "vecs": 3, "out": "f32"},
        # A prompt's 77 encoder rows before the key / value product.
        {"name": "quantize 77x2048 f16", "op": "quantize", "rows": 77, "width": 2048, "in": "f16"},
        # The MLP's hidden rows before the down product.
        {"name": "quantize 4352x12288 bf16", "op": "quantize", "rows": 4352, "width": 12288, "in": "bf16"},
        # Odd sizes, 32-bit input.
        {"name": "quantize 1001x5121 f32", "op": "quantize", "rows": 1001, "width": 5121, "in": "f32"},
        # One token: the product is a matrix times a vector, bound by reading the weights.
        {"name": "w8a8 1x4096x12288", "op": "linear", "rows": 1, "in": 4096, "out": 12288, "epilogue": "silu", "bias": True,
         "type": "bf16"},
        # Two prompts' 77 rows to the keys and values of a cross attention.
        {"name": "w8a8 154x2048x2560 f16", "op": "linear", "rows": 154, "in": 2048, "out": 2560, "epilogue": "store", "bias": False,
         "type": "f16"},
        # The fused gate and up product of a SwiGLU MLP, the block's largest.
        {"name": "w8a8 4352x4096x12288 swiglu", "op": "linear", "rows": 4352, "in": 4096, "out": 12288, "epilogue": "swiglu",
         "bias": False, "type": "bf16"},
        # Its down product.
        {"name": "w8a8 4352x12288x4096", "op": "linear", "rows": 4352, "in": 12288, "out": 4096, "epilogue": "store", "bias": True,
         "type": "bf16"},
        # Odd sizes in every direction, 32-bit output.
        {"name": "w8a8 1003x1155x999 f32", "op": "linear", "rows": 1003, "in": 1155, "out": 999, "epilogue": "store", "bias": True,
         "type": "f32"},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("norm", "quantize", "linear", "linear"))
    if op == "norm":
        width = _log(rng, 64, 8192)
        if rng.random() < 0.6:
            width = -(-width // 64) * 64
        rows = _log(rng, 1, min(32768, 36_000_000 // width))
        pre = rng.choice(("rms", "layer"))
        return {"op": op, "rows": rows, "width": width, "branch": rng.choice(("bf16", "f16", "f32")),
                "post": rng.choice(("none", "rms", "layer")), "gate": rng.random() < 0.7, "pre": pre, "weight": rng.random() < 0.5,
                "modulate": rng.random() < 0.6, "vecs": rng.choice((1, 2, 4)), "out": rng.choice(("bf16", "f16", "f32", "i8"))}
    if op == "quantize":
        width = _log(rng, 64, 16384)
        if rng.random() < 0.6:
            width = -(-width // 64) * 64
        return {"op": op, "rows": _log(rng, 1, min(32768, 50_000_000 // width)), "width": width,
                "in": rng.choice(("bf16", "f16", "f32"))}
    k, n = _log(rng, 64, 12288), _log(rng, 64, 12288)
    if rng.random() < 0.7:
        k, n = -(-k // 64) * 64, -(-n // 64) * 64
    epilogue = rng.choice(("store", "store", "gelu_tanh", "gelu_erf", "silu", "swiglu", "geglu"))
    if epilogue in GATED:
        n = -(-n // 128) * 128
    kind = rng.choice(("bf16", "f16", "f32")) if epilogue == "store" else rng.choice(("bf16", "f16"))
    return {"op": op, "rows": _log(rng, 1, 8192), "in": k, "out": n, "epilogue": epilogue, "bias": rng.random() < 0.6, "type": kind}


# ------------------------------------------------------------------ the inputs

def _padded(t, multiple):
    """`t` [rows, cols] in rows that are a multiple of `multiple` elements apart."""
    rows, cols = t.shape
    wide = torch.zeros(rows, -(-cols // multiple) * multiple, device=t.device, dtype=t.dtype)
    wide[:, :cols] = t
    return wide[:, :cols]


def _int8(t):
    peak = t.abs().amax(1, keepdim=True)
    return _padded((t * (127 / peak)).round().clamp(-127, 127).to(torch.int8), 16), (peak[:, 0] / 127).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = dict(case)
    if case["op"] == "norm":
        rows, width, vecs = case["rows"], case["width"], case["vecs"]
        # A residual stream has a few channels far above the others, and an offset.
        loud = 1 + 8 * (torch.rand(width, generator=g, device="cuda") < 0.01)
        s["x"] = normal(rows, width) * 3 * loud + 0.5
        s["branch_rows"] = (normal(rows, width) * (0.5 + torch.rand(rows, 1, generator=g, device="cuda"))).to(DTYPES[case["branch"]])
        s["rows_per_vec"] = -(-rows // vecs)
        s["post_weight"] = 1 + 0.1 * normal(width) if case["post"] != "none" else None
        s["pre_weight"] = 1 + 0.1 * normal(width) if case["weight"] else None
        # The block's vectors come out of one product: slices of its rows.
        all_vecs = 0.3 * normal(vecs, 3, width)
        s["gate_vec"] = all_vecs[:, 0] if case["gate"] else None
        s["scale_vec"], s["shift_vec"] = (all_vecs[:, 1], all_vecs[:, 2]) if case["modulate"] else (None, None)
    elif case["op"] == "quantize":
        rows, width = case["rows"], case["width"]
        loud = 1 + 6 * (torch.rand(width, generator=g, device="cuda") < 0.01)
        x = normal(rows, width) * loud * (0.1 + torch.rand(rows, 1, generator=g, device="cuda"))
        s["x"] = x.to(DTYPES[case["in"]])
    else:
        rows, k, n = case["rows"], case["in"], case["out"] * (2 if case["epilogue"] in GATED else 1)
        s["x"], s["x_scale"] = _int8(normal(rows, k))
        s["weight"], s["w_scale"] = _int8(normal(n, k) / math.sqrt(k))
        s["bias_vec"] = 0.1 * normal(n) if case["bias"] else None
    return s


# ------------------------------------------------------------------ one pass

def run(s):
    return {"norm": _norm, "quantize": _quantize, "linear": _linear}[s["op"]](s)


def _values(q, scale, dtype):
    """What int8 rows stand for, rounded to `dtype`."""
    out = torch.empty(q.shape, device=q.device, dtype=dtype)
    return torch.mul(q, scale[:, None], out=out)


def _plain_norm(x, kind):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(1, keepdim=True)
    return x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPS)


def _rows_of(vec, rows, per):
    """Row r's vector: vec[min(r / per, vecs - 1)]."""
    return vec[(torch.arange(rows, device=vec.device) // per).clamp(max=vec.shape[0] - 1)]


def _norm(s):
    rows, per = s["rows"], s["rows_per_vec"]
    if own:
        from naivediffusion_b200 import _lib, ops
        kinds = {"none": _lib.ND_NORM_NONE, "rms": _lib.ND_NORM_RMS, "layer": _lib.ND_NORM_LAYER}
        got = ops.residual_norm(s["x"], s["branch_rows"], x_out=torch.empty_like(s["x"]), post_norm=kinds[s["post"]],
                                post_weight=s["post_weight"], gate=s["gate_vec"], residual_scale=0.75, pre_norm=kinds[s["pre"]],
                                pre_weight=s["pre_weight"], scale=s["scale_vec"], shift=s["shift_vec"], rows_per_vec=per, eps=EPS,
                                out_dtype=DTYPES[s["out"]])
        if s["out"] == "i8":
            return {"x": got[0], "y": ops.dequantize(got[1].contiguous(), got[2], 0, torch.bfloat16), "scale": got[2]}
        return {"x": got[0], "y": got[1]}
    b = _plain_norm(s["branch_rows"].float(), s["post"])
    if s["post_weight"] is not None:
        b = b * s["post_weight"]
    if s["gate_vec"] is not None:
        b = b * _rows_of(s["gate_vec"], rows, per)
    x = 0.75 * s["x"] + b
    y = _plain_norm(x, s["pre"])
    if s["pre_weight"] is not None:
        y = y * s["pre_weight"]
    if s["scale_vec"] is not None:
        y = y * (1 + _rows_of(s["scale_vec"], rows, per)) + _rows_of(s["shift_vec"], rows, per)
    if s["out"] == "i8":
        peak = y.abs().amax(1, keepdim=True)
        q = (y * 127 / peak).round()
        return {"x": x, "y": _values(q, peak[:, 0] / 127, torch.bfloat16), "scale": peak[:, 0] / 127}
    return {"x": x, "y": y.to(DTYPES[s["out"]])}


def _quantize(s):
    to = torch.bfloat16 if s["in"] == "f32" else s["x"].dtype
    if own:
        from naivediffusion_b200 import ops
        q, scale = ops.quantize_rows(s["x"])
        return {"values": ops.dequantize(q.contiguous(), scale, 0, to), "scale": scale}
    else:
        x = s["x"].double()  # values next to a half are rounded by their exact quotient
        peak = x.abs().amax(1, keepdim=True)
        q = (x * 127 / peak).round().float()
        scale = (peak[:, 0] / 127).float()
    return {"values": _values(q, scale, to), "scale": scale}


def _plain_act(v, epilogue):
    if epilogue == "gelu_tanh":
        return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v))
    if epilogue == "gelu_erf":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if epilogue == "silu":
        return v * torch.sigmoid(v)
    if epilogue == "swiglu":
        f = v.shape[1] // 2
        return _plain_act(v[:, :f], "silu") * v[:, f:]
    if epilogue == "geglu":
        f = v.shape[1] // 2
        return v[:, :f] * _plain_act(v[:, f:], "gelu_erf")
    return v


def _linear(s):
    if own:
        from naivediffusion_b200 import _lib, ops
        if s["type"] == "f32":
            epilogue = _lib.ND_EPI_STORE_F32
        else:
            epilogue = {"store": _lib.ND_EPI_STORE, "gelu_tanh": _lib.ND_EPI_GELU_TANH, "gelu_erf": _lib.ND_EPI_GELU_ERF,
                        "silu": _lib.ND_EPI_SILU, "swiglu": _lib.ND_EPI_SWIGLU, "geglu": _lib.ND_EPI_GEGLU}[s["epilogue"]]
        return ops.linear_w8a8(s["x"], s["x_scale"], s["weight"], s["w_scale"], s["bias_vec"], epilogue=epilogue,
                               out_dtype=DTYPES[s["type"]])
    v = (s["x"].float() @ s["weight"].float().t()) * s["x_scale"][:, None] * s["w_scale"]
    if s["bias_vec"] is not None:
        v = v + s["bias_vec"]
    return _plain_act(v, s["epilogue"]).to(DTYPES[s["type"]])


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    if case["op"] == "norm":
        rows, width, vecs = case["rows"], case["width"], case["vecs"]
        each = 4 + 4 + BYTES[case["branch"]] + BYTES[case["out"]]
        vectors = (case["post"] != "none") + case["weight"] + vecs * (case["gate"] + 2 * case["modulate"])
        return {"bytes": rows * width * each + 4 * width * vectors + (4 * rows if case["out"] == "i8" else 0),
                "flops": 12 * rows * width}
    if case["op"] == "quantize":
        return {"bytes": case["rows"] * (case["width"] * (BYTES[case["in"]] + 1) + 4), "flops": 3 * case["rows"] * case["width"]}
    rows, k, n = case["rows"], case["in"], case["out"]
    wide = n * (2 if case["epilogue"] in GATED else 1)
    return {"bytes": rows * k + wide * k + rows * n * BYTES[case["type"]] + 4 * rows + 4 * wide * (1 + case["bias"]),
            "flops": 2 * rows * k * wide}


# ------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in s.items()}

    def quantized(m):
        top = torch.max(m.abs(), dim=1).values
        return torch.round(m * 127.0 / top.unsqueeze(1)) * (top / 127.0).unsqueeze(1), top / 127.0

    def normed(m, kind):
        if kind == "layer":
            m = m - m.sum(1, keepdim=True) / m.shape[1]
        if kind != "none":
            m = m / torch.sqrt((m * m).sum(1, keepdim=True) / m.shape[1] + EPS)
        return m

    if case["op"] == "quantize":
        values, scale = quantized(d["x"])
        return {"values": values, "scale": scale}
    if case["op"] == "norm":
        which = torch.div(torch.arange(case["rows"], device="cuda"), s["rows_per_vec"], rounding_mode="floor")
        which = torch.minimum(which, torch.full_like(which, case["vecs"] - 1))
        b = normed(d["branch_rows"], case["post"])
        if case["post"] != "none":
            b = torch.einsum("rc,c->rc", b, d["post_weight"])
        if case["gate"]:
            b = d["gate_vec"].index_select(0, which) * b
        x = 3.0 * d["x"] / 4.0 + b
        y = normed(x, case["pre"])
        if case["weight"]:
            y = torch.einsum("rc,c->rc", y, d["pre_weight"])
        if case["modulate"]:
            y = y + d["scale_vec"].index_select(0, which) * y + d["shift_vec"].index_select(0, which)
        if case["out"] == "i8":
            values, scale = quantized(y)
            return {"x": x, "y": values, "scale": scale}
        return {"x": x, "y": y}
    # Sums of products of 8-bit integers are exact in 64 bits.
    v = torch.einsum("rk,nk->rn", d["x"], d["weight"])
    v = v * torch.outer(d["x_scale"], d["w_scale"])
    if case["bias"]:
        v = v + d["bias_vec"].unsqueeze(0)

    def silu(t):
        return t / (1 + torch.exp(-t))

    def erf_gelu(t):
        return t * torch.special.ndtr(t)

    kind, half = case["epilogue"], case["out"]
    if kind == "silu":
        return silu(v)
    if kind == "gelu_erf":
        return erf_gelu(v)
    if kind == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    if kind == "swiglu":
        return silu(v[:, :half]) * v[:, half:]
    if kind == "geglu":
        return v[:, :half] * erf_gelu(v[:, half:])
    return v
