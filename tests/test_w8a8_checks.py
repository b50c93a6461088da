"""residual_norm, quantize_rows and linear_w8a8 refuse what they cannot run:
the wrappers before anything is launched (CPU tensors here), the C entry
points by status and message. No GPU."""
import ctypes as C

import pytest
import torch

from naivediffusion_b200 import _lib, ops

I8 = torch.int8


def test_wrappers_refuse_cpu_tensors():
    x = torch.zeros(4, 32)
    with pytest.raises(ValueError, match="residual_norm: the tensors must be on a CUDA device"):
        ops.residual_norm(x)
    with pytest.raises(ValueError, match="quantize_rows: the tensors must be on a CUDA device"):
        ops.quantize_rows(x)
    q, s = torch.zeros(4, 32, dtype=I8), torch.zeros(4)
    with pytest.raises(ValueError, match="linear_w8a8: the tensors must be on a CUDA device"):
        ops.linear_w8a8(q, s, q, s)


def test_residual_norm_refuses_wrong_operands():
    x = torch.zeros(8, 64)
    for match, kw in (("x_out", dict(x_out=torch.zeros(7, 64))), ("x_out", dict(x_out=torch.zeros(8, 64, dtype=torch.float16))),
                      ("branch", dict(branch=torch.zeros(8, 63))), ("branch", dict(branch=torch.zeros(8, 64, dtype=I8))),
                      ("post_weight", dict(post_weight=torch.zeros(63))), ("pre_weight", dict(pre_weight=torch.zeros(64).half())),
                      ("gate", dict(gate=torch.zeros(63))), ("gate", dict(gate=torch.zeros(2, 128)[:, ::2], rows_per_vec=4)),
                      ("shift", dict(scale=torch.zeros(2, 64), shift=torch.zeros(1, 64), rows_per_vec=4)),
                      ("shift", dict(scale=torch.zeros(2, 64), shift=torch.zeros(2, 128)[:, :64], rows_per_vec=4)),
                      ("rows_per_vec", dict(scale=torch.zeros(2, 64))),
                      ("out_dtype", dict(out_dtype=torch.float64)), ("out_scale", dict(out_scale=torch.zeros(8))),
                      ("out_scale", dict(out_dtype=I8, out_scale=torch.zeros(7))),
                      ("out must", dict(out=torch.zeros(8, 63, dtype=torch.bfloat16))),
                      ("out must", dict(out=torch.zeros(8, 64, dtype=torch.int16)))):
        with pytest.raises(ValueError, match=match):
            ops.residual_norm(x, **kw)
    for bad in (torch.zeros(8, 64, dtype=torch.bfloat16), torch.zeros(64, 8).t(), torch.zeros(8)):
        with pytest.raises(ValueError, match="residual_norm: x"):
            ops.residual_norm(bad)


def test_quantize_rows_refuses_wrong_operands():
    x = torch.zeros(8, 64)
    for match, args, kw in (("quantize_rows: x", torch.zeros(8, 64, dtype=I8), {}), ("quantize_rows: x", torch.zeros(64, 8).t(), {}),
                            ("out", x, dict(out=torch.zeros(8, 63, dtype=I8))), ("out", x, dict(out=torch.zeros(8, 64))),
                            ("scale", x, dict(scale=torch.zeros(7)))):
        with pytest.raises(ValueError, match=match):
            ops.quantize_rows(args, **kw)


def test_linear_w8a8_refuses_wrong_operands():
    x, sx, w, sw = torch.zeros(8, 64, dtype=I8), torch.zeros(8), torch.zeros(32, 64, dtype=I8), torch.zeros(32)
    for match, args, kw in (
            ("linear_w8a8: x", (x.float(), sx, w, sw), {}), ("weight", (x, sx, w.float(), sw), {}),
            ("weight", (x, sx, w[:, :48], sw), {}), ("x_scale", (x, sx[:7], w, sw), {}), ("w_scale", (x, sx, w, sw[:31]), {}),
            ("w_scale", (x, sx, w, sw.half()), {}), ("bias", (x, sx, w, sw, torch.zeros(31)), {}),
            ("bias", (x, sx, w, sw, torch.zeros(32)), dict(group_split=4, shared_weights=True)),
            ("gate", (x, sx, w, sw), dict(epilogue=_lib.ND_EPI_RESIDUAL_GATE, gate=torch.zeros(31), residual=torch.zeros(8, 32))),
            ("residual", (x, sx, w, sw), dict(epilogue=_lib.ND_EPI_RESIDUAL_ADD)),
            ("residual", (x, sx, w, sw), dict(epilogue=_lib.ND_EPI_RESIDUAL_ADD, residual=torch.zeros(8, 31))),
            ("out_dtype", (x, sx, w, sw), dict(out_dtype=torch.float32)),
            ("out", (x, sx, w, sw), dict(out=torch.zeros(7, 32, dtype=torch.bfloat16))),
            ("addend", (x, sx, w, sw), dict(epilogue=_lib.ND_EPI_ADD_STORE, addend=torch.zeros(8, 32, dtype=torch.float16))),
            ("weight must be", (x, sx, w[:31], sw), dict(epilogue=_lib.ND_EPI_SWIGLU)),
            ("weight must be", (x, sx, w[:31], sw), dict(group_split=4))):
        with pytest.raises(ValueError, match=match):
            ops.linear_w8a8(*args, **kw)


def test_dequantize_refuses_strided_rows():
    with pytest.raises(ValueError, match="contiguous"):
        ops.dequantize(torch.zeros(8, 80, dtype=I8)[:, :72], torch.zeros(8), 0)


def _refused(rc, text):
    assert rc in (_lib.ND_ERR_INVALID, _lib.ND_ERR_UNSUPPORTED), rc
    assert text in _lib.lib().nd_last_error().decode(), _lib.lib().nd_last_error()


P = 1 << 20  # a 16-byte aligned address that is never read: every call here is refused


def test_residual_norm_entry_point_refuses():
    L = _lib.lib()
    _refused(L.nd_op_residual_norm(None, None), "null args")
    good = dict(rows=8, width=64, x=P, ldx=64, x_out=P, ldxo=64, branch=P, ldb=64, branch_dtype=_lib.ND_BF16, pre_norm=1,
                vecs=1, rows_per_vec=0, y=P, ldy=64, out_dtype=_lib.ND_BF16, residual_scale=1.0)
    for text, change in (("empty", dict(rows=0)), ("empty", dict(width=0)), ("empty", dict(rows=-1)), ("too many", dict(rows=1 << 31)),
                         ("16384", dict(width=16385, ldx=20000, ldxo=20000, ldb=20000, ldy=20000)), ("null x", dict(x=None)),
                         ("neither", dict(x_out=None, y=None, pre_norm=0)), ("stride", dict(ldx=63)), ("stride", dict(ldb=60)),
                         ("stride", dict(ldy=32)), ("in place", dict(ldxo=128)), ("unknown norm", dict(post_norm=3)),
                         ("unknown norm", dict(pre_norm=-1)), ("branch_dtype", dict(branch_dtype=_lib.ND_I8)),
                         ("needs a branch", dict(branch=None, gate=P)), ("post_weight", dict(post_weight=P)),
                         ("without y", dict(y=None)), ("pre_weight", dict(pre_norm=0, pre_weight=P)),
                         ("out_dtype", dict(out_dtype=_lib.ND_BF16X2)), ("y_scale", dict(out_dtype=_lib.ND_I8)),
                         ("vecs", dict(vecs=0)), ("rows_per_vec", dict(vecs=2)),
                         ("vec_stride", dict(vecs=2, rows_per_vec=4, gate=P, vec_stride=63))):
        _refused(L.nd_op_residual_norm(C.byref(_lib.ResidualNormArgs(**{**good, **change})), None), text)


def test_quantize_rows_entry_point_refuses():
    L = _lib.lib()
    good = [P, _lib.ND_BF16, 8, 64, 64, P, 64, P]
    for text, at, value in (("f32, f16 or bf16", 1, _lib.ND_I8), ("empty", 2, 0), ("empty", 3, -4), ("too large", 2, 1 << 31),
                            ("null", 0, None), ("null", 5, None), ("null", 7, None), ("stride", 4, 63), ("stride", 6, 63)):
        args = list(good)
        args[at] = value
        _refused(L.nd_op_quantize_rows(*args, None), text)


def test_linear_w8a8_entry_point_refuses():
    L = _lib.lib()
    _refused(L.nd_op_linear_w8a8(None, None), "null args")
    good = dict(dtype=_lib.ND_BF16, epilogue=0, rows=8, in_features=64, out_features=128, x=P, ldx=64, x_scale=P, weight=P, ldw=64,
                w_scale=P, group_split=8, y=P, ldy=128)
    resid = dict(epilogue=_lib.ND_EPI_RESIDUAL_ADD, residual=P, ldr=128)
    for text, change in (("dtype", dict(dtype=_lib.ND_F32)), ("empty", dict(rows=0)), ("empty", dict(in_features=0)),
                         ("empty", dict(out_features=-1)), ("too large", dict(rows=1 << 31)),
                         ("131071", dict(in_features=131072, ldx=131072, ldw=131072)), ("null", dict(x=None)),
                         ("null", dict(w_scale=None)), ("null", dict(x_scale=None)), ("x must be", dict(ldx=48)),
                         ("x must be", dict(ldx=72)), ("x must be", dict(x=P + 8)), ("weight must be", dict(ldw=72)),
                         ("weight must be", dict(weight=P + 1)), ("group_split", dict(group_split=0)),
                         ("group_split", dict(rows=300, group_split=100)), ("epilogue", dict(epilogue=_lib.ND_EPI_QK_NORM_ROPE)),
                         ("epilogue", dict(epilogue=11)), ("epilogue", dict(epilogue=-1)),
                         ("SWIGLU", dict(epilogue=_lib.ND_EPI_SWIGLU, out_features=64)), ("y must be", dict(y=None)),
                         ("y must be", dict(ldy=120)), ("y must be", dict(ldy=132)), ("y must be", dict(y=P + 2)),
                         ("residual", {**resid, "residual": None}), ("residual", {**resid, "ldr": 130}),
                         ("residual", {**resid, "residual": P + 4}), ("gate missing", {**resid, "epilogue": _lib.ND_EPI_RESIDUAL_GATE}),
                         ("gate_stride", {**resid, "epilogue": _lib.ND_EPI_RESIDUAL_GATE, "gate": P, "gate_stride": 127}),
                         ("addend", dict(epilogue=_lib.ND_EPI_ADD_STORE))):
        _refused(L.nd_op_linear_w8a8(C.byref(_lib.LinearW8A8Args(**{**good, **change})), None), text)


def test_struct_layouts_match_the_header(tmp_path):
    import shutil
    import subprocess
    from pathlib import Path
    cc = shutil.which("gcc") or shutil.which("cc")
    if not cc:
        pytest.skip("no C compiler")
    structs = {"nd_residual_norm_args": _lib.ResidualNormArgs, "nd_linear_w8a8_args": _lib.LinearW8A8Args}
    src, exe = tmp_path / "sizes.c", tmp_path / "sizes"
    lines = "".join(f'printf("%zu\\n", sizeof({n}));\n' + "".join(f'printf("%zu\\n", offsetof({n}, {f[0]}));\n' for f in c._fields_)
                    for n, c in structs.items())
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "nd_denoise.h"\nint main(void){\n' + lines + "return 0;}\n")
    include = Path(__file__).resolve().parent.parent / "include"
    subprocess.run([cc, "-I", str(include), str(src), "-o", str(exe)], check=True)
    sizes = iter(int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split())
    for name, cls in structs.items():
        assert C.sizeof(cls) == next(sizes), name
        for f in cls._fields_:
            assert getattr(cls, f[0]).offset == next(sizes), (name, f[0])


def test_the_norm_defaults_to_layer_norm_where_y_is_made(monkeypatch):
    """out_dtype None asks for x' only, and the call then names no norm."""
    calls = []
    monkeypatch.setattr(ops, "_launch", lambda what, device, fn, args: calls.append(_lib.ResidualNormArgs.from_buffer_copy(args)))
    x, b = torch.zeros(4, 32), torch.zeros(4, 32)
    for kw, want in (({}, _lib.ND_NORM_LAYER), (dict(out_dtype=None), _lib.ND_NORM_NONE), (dict(out_dtype=I8), _lib.ND_NORM_LAYER),
                     (dict(out=torch.zeros(4, 32), out_dtype=None), _lib.ND_NORM_LAYER), (dict(pre_norm=1), _lib.ND_NORM_RMS),
                     (dict(pre_norm=0), _lib.ND_NORM_NONE)):
        ops.residual_norm(x, b, **kw)
        assert calls[-1].pre_norm == want, kw
    assert calls[1].y is None and calls[1].x_out == x.data_ptr()


@pytest.mark.parametrize("name", ["gate", "scale", "shift"])
def test_residual_norm_refuses_no_vector_sets(name):
    x = torch.zeros(4, 32)
    with pytest.raises(ValueError, match=f"residual_norm: {name}"):
        ops.residual_norm(x, torch.zeros(4, 32), **{name: torch.zeros(0, 32)})


def test_linear_w8a8_refuses_what_it_would_not_use(monkeypatch):
    x, sx, w, sw = torch.zeros(8, 64, dtype=I8), torch.zeros(8), torch.zeros(32, 64, dtype=I8), torch.zeros(32)
    y, r, add, gate = torch.zeros(8, 32).bfloat16(), torch.zeros(8, 32), torch.zeros(8, 32).bfloat16(), torch.zeros(32)
    E = _lib
    for match, kw in (("out", dict(epilogue=E.ND_EPI_STORE_F32, out=y)), ("out", dict(epilogue=E.ND_EPI_RESIDUAL_ADD, residual=r, out=y)),
                      ("out_dtype", dict(epilogue=E.ND_EPI_STORE_F32, out_dtype=torch.float16)),
                      ("out_dtype", dict(epilogue=E.ND_EPI_RESIDUAL_ADD, residual=r, out_dtype=torch.bfloat16)),
                      ("out_dtype", dict(out=y, out_dtype=torch.float16)),
                      ("residual", dict(residual=r)), ("residual", dict(epilogue=E.ND_EPI_SILU, residual=r)),
                      ("addend", dict(addend=add)), ("addend", dict(epilogue=E.ND_EPI_STORE_F32, addend=add)),
                      ("addend", dict(epilogue=E.ND_EPI_ADD_STORE)),
                      ("gate", dict(gate=gate)), ("gate", dict(epilogue=E.ND_EPI_RESIDUAL_ADD, residual=r, gate=gate)),
                      ("gate", dict(epilogue=E.ND_EPI_RESIDUAL_GATE, residual=r))):
        with pytest.raises(ValueError, match=f"linear_w8a8: .*{match}"):
            ops.linear_w8a8(x, sx, w, sw, **kw)
    monkeypatch.setattr(ops, "_launch", lambda *args: None)
    for kw, dtype in (({}, torch.bfloat16), (dict(out_dtype=torch.float16), torch.float16), (dict(out=y), torch.bfloat16),
                      (dict(out=y, out_dtype=torch.bfloat16), torch.bfloat16), (dict(epilogue=E.ND_EPI_STORE_F32), torch.float32),
                      (dict(epilogue=E.ND_EPI_STORE_F32, out_dtype=torch.float32, residual=r), torch.float32),
                      (dict(epilogue=E.ND_EPI_ADD_STORE, addend=add), torch.bfloat16),
                      (dict(epilogue=E.ND_EPI_RESIDUAL_GATE, residual=r, gate=gate), torch.float32)):
        assert ops.linear_w8a8(x, sx, w, sw, **kw).dtype == dtype
