"""Op-level host API over torch device tensors (torch is only the allocator
and stream here; every op runs the library's sm_100a kernels through the C
ABI in include/nd_denoise.h).

These mirror the operator checks of the reference's smoke command
(src/NaiveDiffusion.Cli/SmokeTest.cs) and the layer helpers they exercise
(src/NaiveDiffusion/Graph/Layers.cs, Graph/Transformer.cs).
"""
from __future__ import annotations

import ctypes as C
import struct

import torch

from . import _lib
from ._lib import (AttentionArgs, GemvArgs, LinearArgs, LinearW8A8Args, ModulateArgs, ResidualNormArgs, RmsNormArgs,
                   check, lib)

_DT = {torch.bfloat16: _lib.ND_BF16, torch.float16: _lib.ND_F16, torch.float32: _lib.ND_F32}
_DT8 = {**_DT, torch.int8: _lib.ND_I8}
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _check_out(what: str, t: torch.Tensor, rows: int, cols: int, dtypes, device) -> None:
    """A caller's output tensor must hold what the op writes: the C ABI sees
    only its pointer and row stride."""
    if (t.dim() != 2 or t.shape[0] < rows or t.shape[1] < cols or t.stride(1) != 1 or t.dtype not in dtypes
            or t.device != device):
        raise ValueError(f"{what} must be a 2-D {'/'.join(str(d) for d in dtypes)} tensor of at least "
                         f"[{rows}, {cols}] with unit column stride on {device}, got {tuple(t.shape)} {t.dtype}")


def _check_vec(what: str, t: torch.Tensor | None, n: int, device) -> None:
    if t is not None and (t.dtype != torch.float32 or not t.is_contiguous() or t.numel() < n or t.device != device):
        raise ValueError(f"{what} must be a contiguous float32 tensor of at least {n} values on {device}")


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def sync() -> None:
    """Synchronize the current stream and raise on a kernel's timed-out wait."""
    check(lib().nd_op_sync(C.c_void_p(_stream())))


def wait_probe(limit_ns: int, ctas: int = 1, armed: bool = False) -> None:
    """Launch the bounded-wait probe (nd_op_wait_probe) on the current stream.
    Unarmed, its wait runs out after limit_ns and the next sync() raises
    NdError with ND_ERR_TIMEOUT; armed, it completes at once."""
    check(lib().nd_op_wait_probe(C.c_uint64(limit_ns), ctas, int(armed), C.c_void_p(_stream())))


def to_pairs(t: torch.Tensor) -> torch.Tensor:
    """fp32 [rows, cols] -> the ND_BF16X2 pair [rows, 2 * cols] (hi = bf16(t),
    lo = bf16(t - hi)), the operand format of fp32-compute GEMMs."""
    hi = t.float().bfloat16()
    lo = (t.float() - hi.float()).bfloat16()
    return torch.cat([hi, lo], dim=1).contiguous()


def from_pairs(p: torch.Tensor) -> torch.Tensor:
    """The fp32 value hi + lo of an ND_BF16X2 pair [rows, 2 * cols]."""
    c = p.shape[1] // 2
    return p[:, :c].float() + p[:, c:].float()


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
           epilogue: int = _lib.ND_EPI_STORE, out: torch.Tensor | None = None,
           residual: torch.Tensor | None = None, gate: torch.Tensor | None = None,
           group_split: int | None = None, qk_norm: torch.Tensor | None = None,
           rope_cos: torch.Tensor | None = None, rope_sin: torch.Tensor | None = None,
           qk_cols: int = 0, eps: float = 1e-6, scales: torch.Tensor | None = None,
           quant_group: int = 32, norm_span: int = 0, rope_period: int = 0,
           gate_stride: int = 0, pairs: bool = False, shared_weights: bool = False) -> torch.Tensor:
    """y = x . W^T + bias with a fused epilogue (Layers.Linear, Graph/Layers.cs:131-160).

    weight is [groups * out, in]; rows >= group_split use the second group.
    Residual epilogues update `residual` (fp32) in place and return it.
    An int8 weight (with `scales`, fp16 or fp32, `quant_group` 32 or 0 = per
    output channel) is widened inside the GEMM (BlockQuantizer's scheme).
    pairs=True: fp32 compute on ND_BF16X2 operands (x [rows, 2 * in], weight
    [groups * out, 2 * in]); the output is a pair [rows, 2 * out], or fp32
    [rows, out] for QK_NORM_ROPE.
    ND_EPI_SWIGLU: weight is the fused [gate; up] matrix [2F, in]; the output
    is [rows, F]. shared_weights=True: one weight matrix for every row, the
    bias / gate vectors chosen per row by group_split (any row).
    """
    rows, k = x.shape
    if pairs:
        k //= 2
    groups = 1 if shared_weights or group_split is None or group_split >= rows else 2
    n = weight.shape[0] // groups
    if epilogue in (_lib.ND_EPI_SWIGLU, _lib.ND_EPI_GEGLU):
        n //= 2
    resid_epi = epilogue in (_lib.ND_EPI_RESIDUAL_GATE, _lib.ND_EPI_RESIDUAL_ADD, _lib.ND_EPI_STORE_F32)
    if resid_epi:
        if residual is None:
            residual = torch.empty(rows, n, device=x.device, dtype=torch.float32)
        else:
            _check_out("linear: residual", residual, rows, n, (torch.float32,), x.device)
    elif out is not None:
        if pairs and epilogue == _lib.ND_EPI_QK_NORM_ROPE:
            _check_out("linear: out", out, rows, n, (torch.float32,), x.device)
        elif pairs:
            _check_out("linear: out", out, rows, 2 * n, (torch.bfloat16,), x.device)
        else:
            _check_out("linear: out", out, rows, n, (torch.float16, torch.bfloat16), x.device)
    if out is None and not resid_epi:
        if pairs and epilogue == _lib.ND_EPI_QK_NORM_ROPE:
            out = torch.empty(rows, n, device=x.device, dtype=torch.float32)
        elif pairs:
            out = torch.empty(rows, 2 * n, device=x.device, dtype=torch.bfloat16)
        else:
            out = torch.empty(rows, n, device=x.device, dtype=x.dtype)
    a = LinearArgs()
    a.dtype = _lib.ND_BF16X2 if pairs else _DT[x.dtype]
    a.epilogue = epilogue
    a.rows, a.in_features, a.out_features = rows, k, n
    a.x, a.ldx = x.data_ptr(), x.stride(0)
    a.weight = weight.data_ptr()
    a.bias = _ptr(bias)
    a.group_split = group_split if group_split is not None else rows
    a.y = _ptr(out)
    a.ldy = out.stride(0) if out is not None else 0
    a.residual = _ptr(residual)
    a.ldr = residual.stride(0) if residual is not None else 0
    a.gate = _ptr(gate)
    a.qk_norm = _ptr(qk_norm)
    a.rope_cos = _ptr(rope_cos)
    a.rope_sin = _ptr(rope_sin)
    a.qk_cols = qk_cols
    a.eps = eps
    a.norm_span = norm_span
    a.rope_period = rope_period
    a.gate_stride = gate_stride
    a.shared_weights = 1 if shared_weights else 0
    if weight.dtype == torch.int8:
        a.weight_dtype = _lib.ND_I8
        a.scales = scales.data_ptr()
        a.scale_dtype = _DT[scales.dtype]
        a.quant_group = quant_group
    check(lib().nd_op_linear(C.byref(a), C.c_void_p(_stream())))
    return residual if resid_epi else out


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, heads: int, *,
              out: torch.Tensor | None = None, batch: int = 1, key_limit: int = 0,
              causal: bool = False, scale: float = 0.0, head_dim: int = 128,
              out_pairs: bool = False, kv_heads: int = 0,
              workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Flash attention over packed heads (Layers.Attend, Graph/Layers.cs:260-279).

    q: [batch * q_rows, >= heads*128] (row stride q.stride(0)); k, v likewise
    with kv_rows per item. Returns out [batch * q_rows, heads * 128].
    fp32 q/k/v run the fp32 attention; out_pairs then writes an ND_BF16X2 pair.
    kv_heads < heads: grouped-query attention (k, v [rows, kv_heads * head_dim]).
    workspace: a zeroed uint8 tensor from attention_workspace(); with it the
    last partial wave of query tiles is split along the keys.
    """
    q_rows = q.shape[0] // batch
    kv_rows = k.shape[0] // batch
    if out is not None:
        _check_out("attention: out", out, q.shape[0], (2 if out_pairs else 1) * heads * head_dim,
                   (torch.bfloat16,) if out_pairs else (q.dtype,), q.device)
    if out is None:
        if out_pairs:
            out = torch.empty(q.shape[0], 2 * heads * head_dim, device=q.device, dtype=torch.bfloat16)
        else:
            out = torch.empty(q.shape[0], heads * head_dim, device=q.device, dtype=q.dtype)
    a = AttentionArgs()
    a.dtype = _DT[q.dtype]
    a.out_dtype = _lib.ND_BF16X2 if out_pairs else 0
    a.heads, a.head_dim, a.batch = heads, head_dim, batch
    a.q_rows, a.kv_rows, a.key_limit, a.causal = q_rows, kv_rows, key_limit, int(causal)
    a.q, a.ldq = q.data_ptr(), q.stride(0)
    a.k, a.ldk = k.data_ptr(), k.stride(0)
    a.v, a.ldv = v.data_ptr(), v.stride(0)
    a.out, a.ldo = out.data_ptr(), out.stride(0)
    a.scale = scale
    a.kv_heads = kv_heads
    if workspace is not None:
        if workspace.device != q.device or workspace.dtype != torch.uint8 or not workspace.is_contiguous():
            raise ValueError("attention: workspace must be a contiguous uint8 tensor on q's device")
        a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel()
    check(lib().nd_op_attention(C.byref(a), C.c_void_p(_stream())))
    return out


def attention_workspace(head_dim: int = 128, device="cuda") -> torch.Tensor:
    """A zeroed workspace for attention(..., workspace=) on `device` (one per
    stream; the kernel leaves it zeroed)."""
    n = int(lib().nd_attention_workspace_bytes(head_dim))
    if n <= 0:
        raise ValueError(f"attention_workspace: no workspace for head_dim {head_dim}")
    return torch.zeros(n, dtype=torch.uint8, device=device)


def modulate(x: torch.Tensor, shift: torch.Tensor | None, scale: torch.Tensor, *,
             out_dtype=torch.bfloat16, group_split: int | None = None, eps: float = 1e-6,
             out: torch.Tensor | None = None) -> torch.Tensor:
    """LayerNorm(x) * (1 + scale) + shift (Transformer.Modulate, Graph/Transformer.cs:72-80).
    scale/shift: [width] or [2, width] (second row for rows >= group_split)."""
    rows, width = x.shape
    pairs = out_dtype == "pairs"
    groups = 2 if group_split is not None and group_split < rows else 1
    _check_vec("modulate: scale", scale, groups * width, x.device)
    _check_vec("modulate: shift", shift, groups * width, x.device)
    if out is None:
        out = torch.empty(rows, 2 * width if pairs else width, device=x.device,
                          dtype=torch.bfloat16 if pairs else out_dtype)
    else:
        _check_out("modulate: out", out, rows, 2 * width if pairs else width,
                   (torch.bfloat16,) if pairs else (torch.float32, torch.float16, torch.bfloat16), x.device)
    a = ModulateArgs()
    a.x, a.ldx = x.data_ptr(), x.stride(0)
    a.y, a.ldy, a.out_dtype = out.data_ptr(), out.stride(0), (_lib.ND_BF16X2 if pairs else _DT[out.dtype])
    a.rows, a.width = rows, width
    a.shift = _ptr(shift)
    a.scale = scale.data_ptr()
    a.vec_stride = width
    a.group_split = group_split if group_split is not None else rows
    a.eps = eps
    check(lib().nd_op_modulate(C.byref(a), C.c_void_p(_stream())))
    return out


# The wrappers from here to linear_w8a8 run before kernels of a few
# microseconds, so they read each tensor attribute once and pack the C struct
# in one call (filling a ctypes Structure takes four times as long).
def _packer(args):
    """struct's pack for a ctypes Structure's fields, in their native layout."""
    fmt = struct.Struct("@" + "".join({C.c_int: "i", C.c_int64: "q", C.c_float: "f", C.c_void_p: "P"}[t]
                                      for _, t in args._fields_))
    pad = C.sizeof(args) - fmt.size
    return fmt.pack if pad == 0 else lambda *values: fmt.pack(*values) + bytes(pad)


_pack_residual_norm, _pack_linear_w8a8 = _packer(ResidualNormArgs), _packer(LinearW8A8Args)


def _round_up(n: int, multiple: int) -> int:
    return (n + multiple - 1) // multiple * multiple


def _matrix(what: str, t: torch.Tensor, dtypes, device, multiple: int = 1) -> tuple[int, int, int]:
    """Rows, columns and row stride of a matrix with unit column stride. A single row's stride is never used and may
    be anything: the next multiple of `multiple` then."""
    if t.dtype in dtypes and t.device == device:
        stride = t.stride()
        if len(stride) == 2:
            rows, cols = t.shape
            if stride[1] == 1 or cols == 1:
                return rows, cols, stride[0] if rows > 1 else _round_up(cols, multiple)
    raise ValueError(f"{what} must be a 2-D {'/'.join(str(d) for d in dtypes)} tensor with unit column stride on "
                     f"{device}, got {tuple(t.shape)} {t.dtype} on {t.device}")


def _vector(what: str, t: torch.Tensor | None, n: int, device) -> int:
    """The address of a vector that holds n values (0 for None)."""
    if t is None:
        return 0
    if t.dtype is _F32 and t.device == device and t.numel() >= n and t.is_contiguous():
        return t.data_ptr()
    _check_vec(what, t, n, device)
    return t.data_ptr()


def _output(what: str, t: torch.Tensor, rows: int, cols: int, dtypes, device, multiple: int = 1) -> int:
    """The row stride of a caller's output, which must hold [rows, cols]."""
    have, wide, ld = _matrix(what, t, dtypes, device, multiple)
    if have < rows or wide < cols:
        raise ValueError(f"{what} must be at least [{rows}, {cols}], got {tuple(t.shape)}")
    return ld


def _padded(rows: int, cols: int, multiple: int, device, dtype) -> tuple[torch.Tensor, int]:
    """An uninitialised [rows, cols] matrix whose row stride is a multiple of `multiple`, and that stride."""
    wide = _round_up(cols, multiple)
    t = torch.empty(rows, wide, device=device, dtype=dtype)
    return (t if wide == cols else t[:, :cols]), wide


def _launch(what: str, device, fn, *args) -> None:
    """Call an op on the current stream of the tensors' device."""
    if device.type != "cuda":
        raise ValueError(f"{what}: the tensors must be on a CUDA device, got {device}")
    stream = torch._C._cuda_getCurrentRawStream(device.index)  # what current_stream(device).cuda_stream reads
    if device.index == torch.cuda.current_device():
        code = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            code = fn(*args, stream)
    if code:
        check(code)


_F32, _I8 = torch.float32, torch.int8
_RESIDUAL_EPI = (_lib.ND_EPI_RESIDUAL_GATE, _lib.ND_EPI_RESIDUAL_ADD, _lib.ND_EPI_STORE_F32)
_GATED_EPI = (_lib.ND_EPI_SWIGLU, _lib.ND_EPI_GEGLU)
_VECTORS = ("residual_norm: gate", "residual_norm: scale", "residual_norm: shift")
_FP32, _INT8, _HALVES = (_F32,), (_I8,), (torch.bfloat16, torch.float16)


def residual_norm(x: torch.Tensor, branch: torch.Tensor | None = None, *, x_out: torch.Tensor | None = None,
                  post_norm: int = _lib.ND_NORM_NONE, post_weight: torch.Tensor | None = None,
                  gate: torch.Tensor | None = None, residual_scale: float = 1.0,
                  pre_norm: int | None = None, pre_weight: torch.Tensor | None = None,
                  scale: torch.Tensor | None = None, shift: torch.Tensor | None = None, rows_per_vec: int = 0,
                  plus_one: bool = False, eps: float = 1e-6, out_dtype=torch.bfloat16,
                  out: torch.Tensor | None = None, out_scale: torch.Tensor | None = None):
    """x' = residual_scale * x + gate * post(branch), then y = pre(x') * (1 + scale) + shift, in one pass.

    x: fp32 [rows, width], updated in place unless x_out is given (without a
    branch and a residual_scale x' is x, and is only stored into x_out).
    post_norm / pre_norm: ND_NORM_NONE, _RMS or _LAYER, times post_weight /
    pre_weight [width] (+ 1 with plus_one); pre_norm is _LAYER unless given,
    where y is made. gate, scale, shift: [width], or
    [vecs, width] of one row stride: row r reads set min(r // rows_per_vec,
    vecs - 1). out_dtype None: x' only; torch.int8: one scale per row.
    Returns (x', y), (x', q, y_scale) for int8, or (x', None).
    """
    device = x.device
    rows, width, ldx = _matrix("residual_norm: x", x, _FP32, device)
    x_ptr = x.data_ptr()
    b_ptr = ldb = b_type = 0
    if branch is not None:
        have, wide, ldb = _matrix("residual_norm: branch", branch, _FLOATS, device)
        if have != rows or wide != width:
            raise ValueError(f"residual_norm: branch must be [{rows}, {width}], got {tuple(branch.shape)}")
        b_ptr, b_type = branch.data_ptr(), _DT[branch.dtype]
    post_ptr = _vector("residual_norm: post_weight", post_weight, width, device)
    pre_ptr = _vector("residual_norm: pre_weight", pre_weight, width, device)
    vecs, vec_stride, ptrs = 0, width, [0, 0, 0]
    for i, t in enumerate((gate, scale, shift)):
        if t is None:
            continue
        name = _VECTORS[i]
        sets, wide, stride = _matrix(name, t if t.dim() != 1 else t[None], _FP32, device)
        if vecs == 0:
            vecs, vec_stride = sets, stride
        if wide != width or sets == 0 or sets != vecs or stride != vec_stride:
            raise ValueError(f"{name} must be [{width}] or [vecs, {width}] with the others' number of sets and row stride, "
                             f"got {tuple(t.shape)} with stride {stride}")
        ptrs[i] = t.data_ptr()
    if vecs > 1 and rows_per_vec <= 0:
        raise ValueError("residual_norm: several vector sets need rows_per_vec")
    x_new, xo_ptr, ldo = x, 0, 0
    if x_out is not None:
        ldo = _output("residual_norm: x_out", x_out, rows, width, _FP32, device)
        x_new, xo_ptr = x_out, x_out.data_ptr()
    elif branch is not None or residual_scale != 1.0:
        xo_ptr, ldo = x_ptr, ldx
    y_ptr = ldy = y_type = q_ptr = 0
    if out is not None:
        ldy = _output("residual_norm: out", out, rows, width, (*_FLOATS, _I8), device)
        out_dtype = out.dtype
    elif out_dtype is not None:
        if out_dtype not in _DT8:
            raise ValueError(f"residual_norm: out_dtype must be a float type, torch.int8 or None, got {out_dtype}")
        out, ldy = _padded(rows, width, 16 if out_dtype is _I8 else 1, device, out_dtype)
    int8 = out_dtype is _I8
    if int8:
        if out_scale is None:
            out_scale = torch.empty(rows, device=device, dtype=_F32)
        q_ptr = _vector("residual_norm: out_scale", out_scale, rows, device)
    elif out_scale is not None:
        raise ValueError("residual_norm: out_scale goes with an int8 output")
    if out is not None:
        y_ptr, y_type = out.data_ptr(), _DT8[out_dtype]
    if pre_norm is None:
        pre_norm = _lib.ND_NORM_NONE if out is None else _lib.ND_NORM_LAYER
    a = _pack_residual_norm(rows, width, x_ptr, ldx, xo_ptr, ldo, b_ptr, ldb, b_type, post_norm, post_ptr, ptrs[0],
                            residual_scale, pre_norm, pre_ptr, ptrs[1], ptrs[2], vecs or 1, vec_stride, rows_per_vec,
                            1 if plus_one else 0, eps, y_ptr, ldy, y_type, q_ptr)
    _launch("residual_norm", device, lib().nd_op_residual_norm, a)
    return (x_new, out, out_scale) if int8 else (x_new, out)


def quantize_rows(x: torch.Tensor, *, out: torch.Tensor | None = None,
                  scale: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows (tokens) as int8 with one scale each: scale = max |x| / 127 over the row, q = rint(x * 127 / max |x|),
    the quotient rounded as if exact. Returns (q [rows, cols], scale [rows]); q's rows are a multiple of 16 bytes
    apart, as linear_w8a8 reads them: its x, or a weight with any number of inputs. A row with an infinity or a NaN gets scale NaN and q 0."""
    device = x.device
    rows, cols, ldx = _matrix("quantize_rows: x", x, _FLOATS, device)
    if out is None:
        out, ldq = _padded(rows, cols, 16, device, torch.int8)
    else:
        ldq = _output("quantize_rows: out", out, rows, cols, _INT8, device, 16)
    if scale is None:
        scale = torch.empty(rows, device=device, dtype=_F32)
    _launch("quantize_rows", device, lib().nd_op_quantize_rows, x.data_ptr(), _DT[x.dtype], rows, cols, ldx,
            out.data_ptr(), ldq, _vector("quantize_rows: scale", scale, rows, device))
    return out, scale


def linear_w8a8(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, w_scale: torch.Tensor,
                bias: torch.Tensor | None = None, *, epilogue: int = _lib.ND_EPI_STORE, out_dtype=None,
                out: torch.Tensor | None = None, residual: torch.Tensor | None = None,
                gate: torch.Tensor | None = None, group_split: int | None = None, shared_weights: bool = False,
                addend: torch.Tensor | None = None) -> torch.Tensor:
    """epilogue(x_scale[r] * w_scale[c] * (x . W^T) + bias) with int8 x and int8 weight, the sum exact.

    x [rows, in] and x_scale [rows] as quantize_rows or residual_norm write
    them; weight [groups * out, in] int8 (row stride a multiple of 16) with
    w_scale, one per weight row: quantize(w, quant_group=0,
    scale_dtype=torch.float32) where in is a multiple of 16, quantize_rows(w)
    for any. rows >= group_split use the second group of
    weight rows, or with shared_weights only the second bias / gate. Residual
    epilogues update `residual` (fp32) in place and return it; STORE_F32 makes
    one if none is given; the others write `out`, or a new matrix of out_dtype
    (bfloat16 unless given). SWIGLU / GEGLU: weight [2F, in], output [rows, F].
    gate goes with RESIDUAL_GATE, addend with ADD_STORE.
    """
    device = x.device
    rows, k, ldx = _matrix("linear_w8a8: x", x, _INT8, device, 16)
    w_rows, w_cols, ldw = _matrix("linear_w8a8: weight", weight, _INT8, device, 16)
    split = group_split is not None and group_split < rows
    groups = 2 if split and not shared_weights else 1
    gated = epilogue in _GATED_EPI
    each = w_rows // groups
    n = each // 2 if gated else each
    if w_cols != k or each * groups != w_rows or (gated and each % 2):
        raise ValueError(f"linear_w8a8: weight must be [{groups} * {'2 * ' if gated else ''}out, {k}], got {tuple(weight.shape)}")
    sx_ptr = _vector("linear_w8a8: x_scale", x_scale, rows, device)
    sw_ptr = _vector("linear_w8a8: w_scale", w_scale, w_rows, device)
    bias_ptr = _vector("linear_w8a8: bias", bias, (2 if split else 1) * each, device)
    gate_ptr = _vector("linear_w8a8: gate", gate, (2 if split else 1) * n, device)
    if (gate is not None) != (epilogue == _lib.ND_EPI_RESIDUAL_GATE):
        raise ValueError("linear_w8a8: gate goes with RESIDUAL_GATE, and RESIDUAL_GATE with a gate")
    if (addend is not None) != (epilogue == _lib.ND_EPI_ADD_STORE):
        raise ValueError("linear_w8a8: addend goes with ADD_STORE, and ADD_STORE with an addend")
    y_ptr = ldy = r_ptr = ldr = a_ptr = lda = 0
    if epilogue in _RESIDUAL_EPI:
        if out is not None or (out_dtype is not None and out_dtype is not _F32):
            raise ValueError("linear_w8a8: this epilogue writes residual in float32, and takes no out nor another out_dtype")
        if residual is not None:
            ldr = _output("linear_w8a8: residual", residual, rows, n, _FP32, device, 4)
        elif epilogue == _lib.ND_EPI_STORE_F32:
            residual, ldr = _padded(rows, n, 4, device, _F32)
        else:
            raise ValueError("linear_w8a8: this epilogue adds to residual, and none is given")
        result, r_ptr, out_dtype = residual, residual.data_ptr(), torch.bfloat16
    else:
        if residual is not None:
            raise ValueError("linear_w8a8: this epilogue writes out, and takes no residual")
        if out is not None:
            ldy = _output("linear_w8a8: out", out, rows, n, _HALVES, device, 8)
            if out_dtype is not None and out_dtype != out.dtype:
                raise ValueError(f"linear_w8a8: out_dtype is {out_dtype}, out is {out.dtype}")
            out_dtype = out.dtype
        else:
            if out_dtype is None:
                out_dtype = torch.bfloat16
            if out_dtype not in _HALVES:
                raise ValueError(f"linear_w8a8: out_dtype must be float16 or bfloat16 (STORE_F32 for fp32), got {out_dtype}")
            out, ldy = _padded(rows, n, 8, device, out_dtype)
        result, y_ptr = out, out.data_ptr()
    if addend is not None:
        lda = _output("linear_w8a8: addend", addend, rows, n, (out_dtype,), device)
        a_ptr = addend.data_ptr()
    a = _pack_linear_w8a8(_DT[out_dtype], epilogue, rows, k, n, x.data_ptr(), ldx, sx_ptr, weight.data_ptr(), ldw, sw_ptr,
                          bias_ptr, rows if group_split is None else group_split, 1 if shared_weights else 0, y_ptr, ldy,
                          r_ptr, ldr, gate_ptr, 0, a_ptr, lda)
    _launch("linear_w8a8", device, lib().nd_op_linear_w8a8, a)
    return result


def rmsnorm(x: torch.Tensor, weight: torch.Tensor | None, *, out_dtype=None, plus_one=False,
            eps: float = 1e-6, silu: bool = False) -> torch.Tensor:
    """x * rsqrt(mean(x^2) + eps) * (weight [+ 1]) over rows (CpuMath.RmsNorm),
    then SiLU when silu=True."""
    rows, width = x.shape
    out = torch.empty(rows, width, device=x.device, dtype=out_dtype or x.dtype)
    a = RmsNormArgs()
    a.x, a.ldx, a.in_dtype = x.data_ptr(), x.stride(0), _DT[x.dtype]
    a.y, a.ldy, a.out_dtype = out.data_ptr(), out.stride(0), _DT[out.dtype]
    a.rows, a.width = rows, width
    a.weight = _ptr(weight)
    a.plus_one = int(plus_one)
    a.eps = eps
    a.silu = int(silu)
    check(lib().nd_op_rmsnorm(C.byref(a), C.c_void_p(_stream())))
    return out


def head_norm_rope(x: torch.Tensor, heads: int, head_dim: int, weight: torch.Tensor,
                   cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, eps: float = 1e-6) -> torch.Tensor:
    """In place: per-head RMSNorm * weight then rotate-half RoPE with row r's
    angles (Transformer.HeadNorm + Transformer.Rotate) over x [rows, >= heads * head_dim]."""
    check(lib().nd_op_head_norm_rope(C.c_void_p(x.data_ptr()), _DT[x.dtype], x.stride(0), x.shape[0], heads, head_dim,
                                     C.c_void_p(weight.data_ptr()), _ptr(cos), _ptr(sin), C.c_float(eps),
                                     C.c_void_p(_stream())))
    return x


def gemv(w: torch.Tensor, x: torch.Tensor, bias: torch.Tensor | None = None, *,
         pre_silu: bool = False, act: int = 0, w_pairs: bool = False, x_rows_per_vec: int = 0,
         bias_period: int = 0) -> torch.Tensor:
    """y[b] = act(W . pre(x[b]) + bias) for 1-4 fp32 rows x; W bf16/f16 [n, k]
    (w_pairs: an ND_BF16X2 pair [n, 2k]). x_rows_per_vec > 0: output row j
    reads input vector j // x_rows_per_vec (x holds ceil(n / x_rows_per_vec)
    vectors; y is [1, n]); bias_period > 0: bias index j % bias_period."""
    n, k = w.shape
    if w_pairs:
        k //= 2
    x = x.reshape(-1, k).contiguous()
    y = torch.empty(1 if x_rows_per_vec else x.shape[0], n, device=w.device, dtype=torch.float32)
    a = GemvArgs()
    a.w, a.w_dtype, a.n, a.k = w.data_ptr(), (_lib.ND_BF16X2 if w_pairs else _DT[w.dtype]), n, k
    a.x, a.batch, a.pre_silu = x.data_ptr(), 1 if x_rows_per_vec else x.shape[0], int(pre_silu)
    a.bias, a.act, a.y = _ptr(bias), act, y.data_ptr()
    a.x_rows_per_vec, a.bias_period = x_rows_per_vec, bias_period
    check(lib().nd_op_gemv(C.byref(a), C.c_void_p(_stream())))
    return y


def patchify(latent: torch.Tensor, patch: int, out_dtype=torch.bfloat16) -> torch.Tensor:
    """[B, C, H, W] fp32 -> [B*(H/p)*(W/p), C*p*p] (AnimaDit.Patchify order)."""
    b, c, h, w = latent.shape
    tok = torch.empty(b * (h // patch) * (w // patch), c * patch * patch, device=latent.device,
                      dtype=out_dtype)
    check(lib().nd_op_patchify(latent.data_ptr(), tok.data_ptr(), _DT[out_dtype], b, c, h, w, patch,
                               tok.stride(0), C.c_void_p(_stream())))
    return tok


def unpatchify(tokens: torch.Tensor, shape, patch: int) -> torch.Tensor:
    b, c, h, w = shape
    lat = torch.empty(b, c, h, w, device=tokens.device, dtype=torch.float32)
    check(lib().nd_op_unpatchify(tokens.data_ptr(), tokens.stride(0), lat.data_ptr(), b, c, h, w,
                                 patch, C.c_void_p(_stream())))
    return lat


def tile_gather(latent: torch.Tensor, rows, cols, tile: int) -> torch.Tensor:
    """latent [C, H, W] fp32 -> tiles [len(rows) * len(cols), C, tile, tile],
    tile (i, j) starting at (rows[i], cols[j]) (TiledVae.CopyTile)."""
    if latent.dim() != 3 or latent.dtype != torch.float32:
        raise ValueError("tile_gather: latent must be a float32 [C, H, W] tensor")
    latent = latent.contiguous()
    c, h, w = latent.shape
    r = (C.c_int32 * len(rows))(*rows)
    q = (C.c_int32 * len(cols))(*cols)
    tiles = torch.empty(len(rows) * len(cols), c, tile, tile, device=latent.device, dtype=torch.float32)
    check(lib().nd_op_tile_gather(latent.data_ptr(), c, h, w, r, len(rows), q, len(cols), tile, tiles.data_ptr(),
                                  C.c_void_p(_stream())))
    return tiles


def tile_blend(tiles: torch.Tensor, rows, cols, vertical: torch.Tensor, horizontal: torch.Tensor, height: int,
               width: int, out: torch.Tensor | None = None) -> torch.Tensor:
    """Decoded tiles [len(rows) * len(cols), C, side, side] crossfaded into
    out [C, height, width] (TiledVae.BlendTile + DivideByWeights); rows / cols
    in the tiles' own units, vertical / horizontal the two axes' ramps."""
    if tiles.dim() != 4 or tiles.dtype != torch.float32 or not tiles.is_contiguous():
        raise ValueError("tile_blend: tiles must be a contiguous float32 [tiles, C, side, side] tensor")
    t, c, side, _ = tiles.shape
    if t != len(rows) * len(cols) or tiles.shape[3] != side:
        raise ValueError(f"tile_blend: {len(rows)} x {len(cols)} square tiles expected, got {tuple(tiles.shape)}")
    for ramp in (vertical, horizontal):
        if ramp.dtype != torch.float32 or ramp.numel() != side or ramp.device != tiles.device:
            raise ValueError(f"tile_blend: the ramps must be float32 vectors of {side} on the tiles' device")
    if out is None:
        out = torch.empty(c, height, width, device=tiles.device, dtype=torch.float32)
    elif (tuple(out.shape) != (c, height, width) or out.dtype != torch.float32 or not out.is_contiguous()
          or out.device != tiles.device):
        raise ValueError(f"tile_blend: out must be a contiguous float32 [{c}, {height}, {width}] tensor")
    r = (C.c_int32 * len(rows))(*rows)
    q = (C.c_int32 * len(cols))(*cols)
    check(lib().nd_op_tile_blend(tiles.data_ptr(), c, side, r, len(rows), q, len(cols), vertical.data_ptr(),
                                 horizontal.data_ptr(), out.data_ptr(), height, width, C.c_void_p(_stream())))
    return out


def dequantize(q: torch.Tensor, scales: torch.Tensor, quant_group: int = 32,
               out_dtype=torch.bfloat16) -> torch.Tensor:
    """w = round(q * scale) in out_dtype (DmlOps.Dequantize, Dml/DmlOps.cs:208-228)."""
    rows, cols = q.shape
    if not q.is_contiguous():
        raise ValueError("dequantize: q must be contiguous")
    device = q.device
    out = torch.empty(rows, cols, device=device, dtype=out_dtype)
    _launch("dequantize", device, lib().nd_op_dequantize, q.data_ptr(), scales.data_ptr(), _DT[scales.dtype], quant_group,
            rows, cols, out.data_ptr(), _DT[out_dtype])
    return out


def quantize(w: torch.Tensor, quant_group: int = 32, scale_dtype=torch.float16):
    """BlockQuantizer on the device: (q int8 [rows, cols], scales [rows, cols / group] or [rows])."""
    rows, cols = w.shape
    g = quant_group or cols
    q = torch.empty(rows, cols, device=w.device, dtype=torch.int8)
    s = torch.empty(rows, cols // g, device=w.device, dtype=scale_dtype)
    check(lib().nd_op_quantize(w.data_ptr(), _DT[w.dtype], rows, cols, quant_group, _DT[scale_dtype],
                               q.data_ptr(), s.data_ptr(), C.c_void_p(_stream())))
    return q, s


_EPI_CONV = {"store": 0, "silu": 3, "store_f32": 5, "add_store": 8}


def conv2d(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, stride: int = 1,
           epilogue: str = "store", addend: torch.Tensor | None = None,
           per_batch_bias: bool = False) -> torch.Tensor:
    """3x3 convolution, padding 1, over NHWC activations x [B, H, W, Cin] with
    weight [Cout, 3, 3, Cin rounded up to 64, the pad zero] (Layers.Conv2d,
    Graph/Layers.cs:115-128).
    bias: [Cout] fp32, or [B, Cout] with per_batch_bias."""
    b, h, w, cin = x.shape
    cout = weight.shape[0]
    ho, wo = (h + 2 - 3) // stride + 1, (w + 2 - 3) // stride + 1
    a = _lib.ConvArgs()
    a.dtype = _DT[x.dtype]
    a.epilogue = _EPI_CONV[epilogue]
    a.batch, a.height, a.width, a.in_channels, a.out_channels, a.stride = b, h, w, cin, cout, stride
    a.x, a.weight, a.bias = x.data_ptr(), weight.data_ptr(), _ptr(bias)
    a.per_batch_bias = 1 if per_batch_bias else 0
    a.bias_stride = bias.stride(0) if per_batch_bias else 0
    if epilogue == "store_f32":
        y = torch.empty(b, ho, wo, cout, device=x.device, dtype=torch.float32)
        a.y_f32 = y.data_ptr()
    else:
        y = torch.empty(b, ho, wo, cout, device=x.device, dtype=x.dtype)
        a.y = y.data_ptr()
    a.addend = _ptr(addend)
    check(lib().nd_op_conv2d(C.byref(a), C.c_void_p(_stream())))
    return y


def group_norm(x: torch.Tensor, groups: int, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
               eps: float = 1e-5, silu: bool = False) -> torch.Tensor:
    """GroupNorm over NHWC x [B, pixels, C] (Layers.GroupNorm, Graph/Layers.cs:166-185),
    optionally followed by SiLU."""
    b, p, c = x.shape
    y = torch.empty_like(x)
    check(lib().nd_op_group_norm(x.data_ptr(), y.data_ptr(), _DT[x.dtype], b, p, c, groups, weight.data_ptr(),
                                 _ptr(bias), eps, 1 if silu else 0, C.c_void_p(_stream())))
    return y


def geglu(x: torch.Tensor) -> torch.Tensor:
    """[rows, 2F] -> [rows, F] = x[:, :F] * gelu(x[:, F:]) (UNetLayers.Geglu, Models/Sdxl/UNetLayers.cs:30-46)."""
    rows, two_f = x.shape
    y = torch.empty(rows, two_f // 2, device=x.device, dtype=x.dtype)
    check(lib().nd_op_geglu(x.data_ptr(), y.data_ptr(), _DT[x.dtype], rows, two_f // 2, C.c_void_p(_stream())))
    return y


def sampler_step(sampler: int, prediction: int, out: torch.Tensor, sample: torch.Tensor, *,
                 guidance: float = 1.0, last: torch.Tensor | None = None, noise: torch.Tensor | None = None,
                 denoised_out: torch.Tensor | None = None, next_input: torch.Tensor | None = None,
                 next_input_scale: float = 1.0, sigma: float, sigma_next: float, up: float = 0.0,
                 down: float = 0.0, rescale: float = 1.0, noise_scale: float = 0.0, shrink: float = 0.0,
                 weight: float = 0.0, second_order: bool = False) -> torch.Tensor:
    """Guidance combine + one solver step in place on `sample` (fp32, device),
    bit-identical to the reference's CPU step (Sampling/Schedulers.cs).
    out: [n] or [2, n] (uncond then cond)."""
    n = sample.numel()
    branches = out.numel() // n
    if branches not in (1, 2) or out.numel() != branches * n:
        raise ValueError(f"sampler_step: out must hold 1 or 2 branches of {n} values")
    for what, t in (("out", out), ("sample", sample), ("last", last), ("noise", noise),
                    ("denoised_out", denoised_out), ("next_input", next_input)):
        _check_vec(f"sampler_step: {what}", t, branches * n if what == "out" else n, sample.device)
    a = _lib.SamplerArgs()
    a.sampler, a.prediction, a.n, a.branches = sampler, prediction, n, branches
    a.out, a.guidance, a.sample = out.data_ptr(), guidance, sample.data_ptr()
    a.last_denoised, a.noise, a.denoised_out, a.next_input = _ptr(last), _ptr(noise), _ptr(denoised_out), _ptr(next_input)
    a.next_input_scale, a.sigma, a.sigma_next = next_input_scale, sigma, sigma_next
    a.up, a.down, a.rescale, a.noise_scale, a.shrink, a.weight = up, down, rescale, noise_scale, shrink, weight
    a.second_order = int(bool(second_order))
    check(lib().nd_op_sampler_step(C.byref(a), C.c_void_p(_stream())))
    return sample
