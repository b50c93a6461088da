"""nd_op_linear into wider matrices: an output width that ends inside 16 bytes
(where TMA clips a store) leaves what lies beside it as it was. Small whole
numbers, so every sum is exact and the results are compared bit for bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8
STORE, GATE, STORE_F32, ADD, ADD_STORE = 0, 4, 5, 7, 8


def _whole(g, low, high, *shape):
    return torch.randint(low, high + 1, shape, generator=g, device="cuda").float()


def _weights(g, rows, k, dtype):
    """Weights, their values, and what linear takes beside int8 ones."""
    w = _whole(g, -2, 2, rows, k)
    if dtype == I8:
        return w.to(I8), w * 0.5, dict(scales=torch.full((rows, 1), 0.5, device="cuda"), quant_group=0)
    return w.to(dtype), w, {}


# One-SM tiles, and CTA pairs of 128, 160 and 256 columns.
@pytest.mark.parametrize("m,n", [(1, 1), (50, 100), (300, 201), (77, 390), (130, 7), (1100, 102), (1280, 636), (4864, 1271),
                                 (2048, 157)])
@pytest.mark.parametrize("weights", [BF16, F16, I8])
def test_what_lies_beside_an_output_stays(cuda, m, n, weights):
    from naivediffusion_b200 import ops
    k, g = 64, torch.Generator(device="cuda").manual_seed(m + n)
    dtype = BF16 if weights == I8 else weights
    x = _whole(g, -3, 3, m, k).to(dtype)
    w, values, kw = _weights(g, n, k, weights)
    bias = _whole(g, -9, 9, n) if n % 4 == 0 else None
    sums = x.float() @ values.t() + (0 if bias is None else bias)  # at most 6 k + 9: exact
    gate = _whole(g, -2, 2, n) if n % 4 == 0 else None
    wide = -(-n // 8) * 8 + 32
    addend = _whole(g, -9, 9, m, wide).to(dtype)
    for epi in (STORE, ADD_STORE, STORE_F32, ADD, GATE):
        if epi == GATE and gate is None:
            continue
        f32 = epi in (STORE_F32, ADD, GATE)
        store = torch.full((m + 3, wide), 5.0, device="cuda", dtype=F32 if f32 else dtype)
        args = dict(kw, residual=store[:, :n]) if f32 else dict(kw, out=store[:, :n])
        if epi == GATE:
            args["gate"] = gate
        _linear(ops, x, w, bias, epi, addend if epi == ADD_STORE else None, args)
        ops.sync()
        want = {STORE: sums, STORE_F32: sums, ADD: sums + 5, ADD_STORE: sums + addend[:, :n].float()}.get(epi)
        if want is None:
            want = sums * gate + 5
        assert torch.equal(store[:m, :n], want.to(store.dtype)), epi
        assert store[m:].eq(5).all() and store[:m, n:].eq(5).all(), epi


def _linear(ops, x, w, bias, epi, addend, args):
    """ops.linear, and the C entry point where there is an addend (the wrapper takes none)."""
    if addend is None:
        ops.linear(x, w, bias, epilogue=epi, **args)
        return
    import ctypes as C
    from naivediffusion_b200 import _lib
    out, a = args["out"], _lib.LinearArgs()
    a.dtype, a.epilogue = ops._DT[x.dtype], epi
    a.rows, a.in_features, a.out_features = x.shape[0], x.shape[1], w.shape[0]
    a.x, a.ldx, a.weight = x.data_ptr(), x.stride(0), w.data_ptr()
    a.bias = None if bias is None else bias.data_ptr()
    a.group_split, a.y, a.ldy = x.shape[0], out.data_ptr(), out.stride(0)
    a.addend, a.ld_add = addend.data_ptr(), addend.stride(0)
    if w.dtype == I8:
        a.weight_dtype, a.scales, a.scale_dtype, a.quant_group = _lib.ND_I8, args["scales"].data_ptr(), _lib.ND_F32, 0
    _lib.check(_lib.lib().nd_op_linear(C.byref(a), C.c_void_p(torch.cuda.current_stream().cuda_stream)))


@pytest.mark.parametrize("m,split,n", [(256, 128, 100), (300, 256, 39), (1536, 1280, 642), (1536, 1152, 130)])
@pytest.mark.parametrize("weights", [BF16, F16, I8])
def test_what_lies_beside_two_groups_stays(cuda, m, split, n, weights):
    """Group 0's tiles reach into group 1's weight rows: none of those products may land beside the output."""
    from naivediffusion_b200 import ops
    k, g = 64, torch.Generator(device="cuda").manual_seed(m + n)
    dtype = BF16 if weights == I8 else weights
    x = _whole(g, 1, 3, m, k).to(dtype)
    w, values, kw = _weights(g, 2 * n, k, weights)
    sums = torch.cat([x[:split].float() @ values[:n].t(), x[split:].float() @ values[n:].t()])
    wide = -(-n // 8) * 8 + 16
    for epi in (STORE, STORE_F32, ADD):
        store = torch.full((m, wide), 5.0, device="cuda", dtype=dtype if epi == STORE else F32)
        ops.linear(x, w, epilogue=epi, group_split=split, **kw, **{"out" if epi == STORE else "residual": store[:, :n]})
        ops.sync()
        assert torch.equal(store[:, :n], (sums + (5 if epi == ADD else 0)).to(store.dtype)), epi
        assert store[:, n:].eq(5).all(), epi


@pytest.mark.parametrize("m,n", [(50, 101), (300, 202), (1100, 1023)])
def test_what_lies_beside_fp32_compute_stays(cuda, m, n):
    """The residual epilogues on bf16 pairs (hi | lo), whose fp32 output may have any width."""
    from naivediffusion_b200 import ops
    k, g = 64, torch.Generator(device="cuda").manual_seed(m)
    x, w = _whole(g, -3, 3, m, k), _whole(g, -2, 2, n, k)
    sums = x @ w.t()
    wide = -(-n // 4) * 4 + 16
    for epi in (STORE_F32, ADD):
        store = torch.full((m + 2, wide), 5.0, device="cuda")
        ops.linear(ops.to_pairs(x), ops.to_pairs(w), epilogue=epi, pairs=True, residual=store[:, :n])
        ops.sync()
        assert torch.equal(store[:m, :n], sums + (5 if epi == ADD else 0)), epi
        assert store[m:].eq(5).all() and store[:m, n:].eq(5).all(), epi
