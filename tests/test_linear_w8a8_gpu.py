"""linear_w8a8 against the product in 64 bits (rowops_reference)."""
import math

import pytest
import torch

from rowops_reference import U, act64, check, half_step, linear64, quantize64, residual_norm64

pytestmark = pytest.mark.gpu
BF16, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8
EPI = {"store": 0, "gelu_tanh": 1, "gelu_erf": 2, "silu": 3, "gate": 4, "f32": 5, "add": 7, "add_store": 8, "swiglu": 9,
       "geglu": 10}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _int8(g, rows, cols, pad=0):
    """[rows, cols] int8 over the whole range (-128 too) with its row stride a multiple of 16, and scales."""
    wide = -(-cols // 16) * 16 + pad
    t = torch.randint(-128, 128, (rows, wide), generator=g, device="cuda", dtype=torch.int32).to(I8)
    return t[:, :cols], (0.5 + torch.rand(rows, generator=g, device="cuda")) / (74 * math.sqrt(cols))


def _case(m, n, k, seed, gated=False):
    g = _gen(seed)
    x, sx = _int8(g, m, k)
    w, sw = _int8(g, n * (2 if gated else 1), k)
    sx = sx * math.sqrt(k)  # products of about one
    return g, x, sx, w, sw, 0.3 * torch.randn(w.shape[0], generator=g, device="cuda")


SHAPES = [(1, 1, 1), (1, 8, 16), (1, 4096, 1024), (2, 1000, 4096), (3, 100, 130), (4, 640, 2048), (5, 256, 64), (8, 999, 1155),
          (16, 2560, 2048), (33, 72, 5000), (77, 1280, 2048), (128, 128, 128), (129, 257, 129), (154, 2560, 2048),
          (300, 512, 96), (512, 4096, 1024), (9, 19001, 200), (27, 19500, 300), (40, 19003, 256), (64, 20000, 130),
          (20, 256, 6000), (50, 640, 9000), (90, 1000, 7000), (200, 384, 12000), (1003, 999, 1155), (1024, 1024, 640), (1300, 2050, 320), (2049, 640, 2048)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("out,bias", [(BF16, True), (F16, False), (F32, True)])
def test_store(cuda, m, n, k, out, bias):
    from naivediffusion_b200 import ops
    _, x, sx, w, sw, b = _case(m, n, k, m * 31 + n * 7 + k)
    b = b if bias else None
    y = ops.linear_w8a8(x, sx, w, sw, b, epilogue=EPI["f32"] if out == F32 else 0, out_dtype=out)
    ops.sync()
    assert y.dtype == out and tuple(y.shape) == (m, n)
    v, dv = linear64(x, sx, w, sw, b)
    check(y, v, dv + (half_step(v.abs() + dv, out) if out != F32 else 0), f"{m} {n} {k}")


@pytest.mark.parametrize("m", [1, 3, 40, 200, 1100])
@pytest.mark.parametrize("act", ["gelu_tanh", "gelu_erf", "silu", "swiglu", "geglu"])
@pytest.mark.parametrize("out", [BF16, F16])
def test_activations(cuda, m, act, out):
    from naivediffusion_b200 import ops
    n, k = 384, 500
    _, x, sx, w, sw, b = _case(m, n, k, m + 17, gated=act in ("swiglu", "geglu"))
    y = ops.linear_w8a8(x, sx, w, sw, b, epilogue=EPI[act], out_dtype=out)
    ops.sync()
    v, dv = linear64(x, sx, w, sw, b, act)
    check(y, v, dv + half_step(v.abs() + dv, out), act)


@pytest.mark.parametrize("m", [3, 12, 32, 41, 64, 100])
@pytest.mark.parametrize("act", ["swiglu", "geglu"])
@pytest.mark.parametrize("n,k", [(9600, 190), (256, 5000)])
def test_gated_wide_and_deep(cuda, m, act, n, k):
    """Few rows of many outputs, and of few outputs with the k blocks split."""
    from naivediffusion_b200 import ops
    _, x, sx, w, sw, b = _case(m, n, k, m + n, gated=True)
    y = ops.linear_w8a8(x, sx, w, sw, b, epilogue=EPI[act])
    ops.sync()
    v, dv = linear64(x, sx, w, sw, b, act)
    check(y, v, dv + half_step(v.abs() + dv, BF16), act)


@pytest.mark.parametrize("m,n,k", [(2, 64, 256), (9, 200, 300), (30, 128, 6000), (45, 256, 9000), (64, 19200, 128), (90, 256, 256)])
@pytest.mark.parametrize("act", ["silu", "gelu_erf", "gate", "add_store"])
def test_shared_weights_at_few_rows(cuda, m, n, k, act):
    """Every kernel for few rows with a split between two biases and gates."""
    from naivediffusion_b200 import ops
    g, x, sx, w, sw, _ = _case(m, n, k, m + k)
    split = m // 2
    b, gate = torch.randn(2 * n, generator=g, device="cuda"), torch.randn(2 * n, generator=g, device="cuda")
    r0 = torch.randn(m, n, generator=g, device="cuda")
    addend = torch.randn(m, n, generator=g, device="cuda").to(BF16)
    kw = dict(group_split=split, shared_weights=True, epilogue=EPI[act])
    if act == "gate":
        got = ops.linear_w8a8(x, sx, w, sw, b, residual=r0.clone(), gate=gate, **kw)
    else:
        got = ops.linear_w8a8(x, sx, w, sw, b, addend=addend if act == "add_store" else None, **kw)
    ops.sync()
    for rows, cols in ((slice(0, split), slice(0, n)), (slice(split, m), slice(n, 2 * n))):
        v, dv = linear64(x[rows], sx[rows], w, sw, b[cols], act if act in ("silu", "gelu_erf") else "store")
        if act == "gate":
            f = gate[cols].double()
            want = r0[rows].double() + v * f
            check(got[rows], want, dv * f.abs() + U * (v * f).abs() * 1.01 + U * want.abs() + 1e-30, act)
            continue
        if act == "add_store":
            v = v + addend[rows].double()
            dv = dv + U * v.abs()
        check(got[rows], v, dv + half_step(v.abs() + dv, BF16), act)


@pytest.mark.parametrize("m", [1, 4, 20, 60, 400, 1500])
def test_residual_epilogues_and_addend(cuda, m):
    from naivediffusion_b200 import ops
    n, k = 333, 770
    g, x, sx, w, sw, b = _case(m, n, k, m + 3)
    v, dv = linear64(x, sx, w, sw, b)
    base = torch.randn(m, -(-n // 4) * 4 + 4, generator=g, device="cuda")
    gate = torch.randn(n, generator=g, device="cuda")
    for epi, factor in (("add", torch.ones(n, device="cuda")), ("gate", gate)):
        r = base.clone()
        got = ops.linear_w8a8(x, sx, w, sw, b, epilogue=EPI[epi], residual=r, gate=gate if epi == "gate" else None)
        ops.sync()
        f = factor.double()
        want = base[:, :n].double() + v * f
        assert got is r and torch.equal(r[:, n:], base[:, n:])
        check(r[:, :n], want, dv * f.abs() + U * (v * f).abs() * 1.01 + U * (want.abs() + 1e-30), epi)
    addend = torch.randn(m, -(-n // 8) * 8, generator=g, device="cuda").to(F16)
    y = ops.linear_w8a8(x, sx, w, sw, b, epilogue=EPI["add_store"], addend=addend[:, :n], out_dtype=F16)
    ops.sync()
    want = v + addend[:, :n].double()
    d = dv + U * want.abs()
    check(y, want, d + half_step(want.abs() + d, F16), "add_store")


@pytest.mark.parametrize("m,split", [(256, 128), (300, 256), (1536, 1280), (1536, 1152), (130, 128)])
def test_two_weight_groups(cuda, m, split):
    """A dual-stream block: rows from group_split on take the second weights, scales, bias and gate."""
    from naivediffusion_b200 import ops
    n, k = 390, 256
    g = _gen(m + split)
    x, sx = _int8(g, m, k)
    sx = sx * math.sqrt(k)
    w, sw = _int8(g, 2 * n, k)
    b, gate = torch.randn(2 * n, generator=g, device="cuda"), torch.randn(2 * n, generator=g, device="cuda")
    parts = [(slice(0, split), slice(0, n)), (slice(split, m), slice(n, 2 * n))]
    y = ops.linear_w8a8(x, sx, w, sw, b, group_split=split)
    r0 = torch.randn(m, -(-n // 4) * 4, generator=g, device="cuda")
    r = r0.clone()
    ops.linear_w8a8(x, sx, w, sw, b, group_split=split, epilogue=EPI["gate"], gate=gate, residual=r)
    ops.sync()
    for rows, cols in parts:
        v, dv = linear64(x[rows], sx[rows], w[cols], sw[cols], b[cols])
        check(y[rows], v, dv + half_step(v.abs() + dv, BF16))
        f = gate[cols].double()
        want = r0[rows, :n].double() + v * f
        check(r[rows, :n], want, dv * f.abs() + U * (v * f).abs() * 1.01 + U * want.abs() + 1e-30)


@pytest.mark.parametrize("m,split", [(2, 1), (300, 77), (1500, 1003)])
def test_shared_weights_with_two_biases(cuda, m, split):
    from naivediffusion_b200 import ops
    n, k = 256, 192
    g, x, sx, w, sw, _ = _case(m, n, k, m, gated=True)
    b = torch.randn(2 * 2 * n, generator=g, device="cuda")
    y = ops.linear_w8a8(x, sx, w, sw, b, epilogue=EPI["swiglu"], group_split=split, shared_weights=True)
    z = ops.linear_w8a8(x, sx, w, sw, b, group_split=split, shared_weights=True)
    ops.sync()
    for rows, bias in ((slice(0, split), b[:2 * n]), (slice(split, m), b[2 * n:])):
        for got, act in ((y, "swiglu"), (z, "store")):
            v, dv = linear64(x[rows], sx[rows], w, sw, bias, act)
            check(got[rows], v, dv + half_step(v.abs() + dv, BF16), act)


@pytest.mark.parametrize("m,n,k", [(1, 512, 8192), (4, 300, 20000), (100, 256, 131071), (1100, 512, 40000)])
def test_largest_sums_are_exact(cuda, m, n, k):
    """Every product 127 * 127 or 128 * 128: sums past 2^24, up to just under 2^31, come out as fp32 rounds them."""
    from naivediffusion_b200 import ops
    x = torch.full((m, -(-k // 16) * 16), -128, device="cuda", dtype=I8)[:, :k]
    w = torch.full((n, -(-k // 16) * 16), -128, device="cuda", dtype=I8)[:, :k]
    w[1::2] = 127
    one_m, one_n = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
    y = ops.linear_w8a8(x, one_m, w, one_n, epilogue=EPI["f32"])
    ops.sync()
    want = torch.tensor([128 * 128 * k, -128 * 127 * k], device="cuda", dtype=torch.float64).float().repeat((n + 1) // 2)[:n]
    assert torch.equal(y, want.expand(m, n))


@pytest.mark.parametrize("m", [1, 20, 50, 1200])
@pytest.mark.parametrize("n", [200, 201, 7, 33, 389, 510])
def test_what_lies_beside_stays(cuda, m, n):
    """Rows and columns past the output, and int8 columns past in_features, are neither written nor read."""
    from naivediffusion_b200 import ops
    k = 250
    g = _gen(m + n)
    x, sx = _int8(g, m, k, pad=16)
    w, sw = _int8(g, n, k, pad=32)
    v, dv = linear64(x, sx, w, sw)
    for epi, dtype in (("f32", F32), ("add", F32), ("store", BF16), ("gelu_tanh", F16)):
        # negative zeros beside: adding nothing to them would show too
        store = torch.full((m + 3, -(-n // 8) * 8 + 32), -0.0, device="cuda", dtype=dtype)
        ops.linear_w8a8(x, sx, w, sw, epilogue=EPI[epi], **(dict(residual=store[:, :n]) if dtype == F32 else dict(out=store[:, :n])))
        ops.sync()
        y, dy = act64(v, dv, epi) if epi == "gelu_tanh" else (v, dv)
        check(store[:m, :n], y, dy + (half_step(y.abs() + dy, dtype) if dtype != F32 else U * y.abs()), epi)
        beside = torch.cat([store[m:].flatten(), store[:m, n:].flatten()])
        assert beside.eq(0).all() and torch.signbit(beside).all(), epi


@pytest.mark.parametrize("m", [2, 17, 90, 1100])
def test_special_scales(cuda, m):
    """A row quantized from NaN or infinity has scale NaN and its outputs are NaN; a row of zeros gives the bias."""
    from naivediffusion_b200 import ops
    n, k = 136, 128
    g = _gen(m)
    h = torch.randn(m, k, generator=g, device="cuda")
    h[0] = 0
    h[1, 3] = math.inf
    q, sx = ops.quantize_rows(h)
    w, sw = _int8(g, n, k)
    b = torch.randn(n, generator=g, device="cuda")
    y = ops.linear_w8a8(q, sx, w, sw, b, epilogue=EPI["f32"])
    ops.sync()
    assert torch.equal(y[0], b) and torch.isnan(y[1]).all() and torch.isfinite(y[2:]).all()


@pytest.mark.parametrize("m", [1, 24, 150, 1400])
def test_streams_and_graphs(cuda, m):
    """Two products at once on two streams, and a captured one replayed on other values."""
    from naivediffusion_b200 import ops
    _, x, sx, w, sw, b = _case(m, 2560, 2048, m)
    _, x2, sx2, w2, sw2, b2 = _case(m, 1280, 1024, m + 1)
    want, want2 = ops.linear_w8a8(x, sx, w, sw, b), ops.linear_w8a8(x2, sx2, w2, sw2, b2)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got, got2 = [], []
    for _ in range(10):
        with torch.cuda.stream(s1):
            got.append(ops.linear_w8a8(x, sx, w, sw, b))
        with torch.cuda.stream(s2):
            got2.append(ops.linear_w8a8(x2, sx2, w2, sw2, b2))
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in got) and all(torch.equal(t, want2) for t in got2)
    xs = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.linear_w8a8(xs, sx, w, sw, b)
        y2 = ops.linear_w8a8(x2, sx2, w2, sw2, b2)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(y2, want2)
    xs.zero_()
    graph.replay()
    ops.sync()
    assert torch.equal(y, b.to(BF16).expand(m, -1))


@pytest.mark.parametrize("m", [1, 20, 100, 300, 1200])
def test_the_addend_may_be_the_output(cuda, m):
    from naivediffusion_b200 import ops
    n, k = 1000, 640
    g, x, sx, w, sw, b = _case(m, n, k, m + 5)
    base = torch.randn(m, n, generator=g, device="cuda").to(BF16)
    want = ops.linear_w8a8(x, sx, w, sw, b, epilogue=EPI["add_store"], addend=base)
    y = base.clone()
    got = ops.linear_w8a8(x, sx, w, sw, b, epilogue=EPI["add_store"], addend=y, out=y)
    ops.sync()
    assert got is y and torch.equal(y, want)


@pytest.mark.parametrize("m", [1, 2, 20, 60, 1100])
def test_every_kernel_repeats_itself(cuda, m):
    """The same call twice gives the same bits: integer sums, and no order that varies."""
    from naivediffusion_b200 import ops
    _, x, sx, w, sw, b = _case(m, 768, 9000, m)
    y = [ops.linear_w8a8(x, sx, w, sw, b, epilogue=EPI["gelu_erf"]) for _ in range(4)]
    ops.sync()
    assert all(torch.equal(t, y[0]) for t in y)


def test_a_block_of_them(cuda):
    """A transformer block's MLP as it runs on 8 bits: norm to int8, gate and up product, its rows to int8, down
    product, gated residual and the next norm. Each step against 64 bits on what the step before stored, and the
    whole against the same block without 8-bit rounding."""
    from naivediffusion_b200 import ops
    rows, width, hidden = 1300, 640, 1792
    g = _gen(2)
    x = torch.randn(rows, width, generator=g, device="cuda") * 2
    vec = 0.3 * torch.randn(2, 3, width, generator=g, device="cuda")
    per = 1024
    wf = [torch.randn(2 * hidden, width, generator=g, device="cuda") / math.sqrt(width),
          torch.randn(width, hidden, generator=g, device="cuda") / math.sqrt(hidden)]
    weights = [ops.quantize(t, quant_group=0, scale_dtype=F32) for t in wf]
    (wu, su), (wd, sd) = [(q, s.reshape(-1)) for q, s in weights]
    norm = dict(scale=vec[:, 0], shift=vec[:, 1], rows_per_vec=per)
    x0 = x.clone()
    _, q, s = ops.residual_norm(x, **norm, out_dtype=I8)
    h = ops.linear_w8a8(q, s, wu, su, epilogue=EPI["swiglu"])
    qh, sh = ops.quantize_rows(h)
    d = ops.linear_w8a8(qh, sh, wd, sd)
    xn, y = ops.residual_norm(x, d, post_norm=1, gate=vec[:, 2], rows_per_vec=per, pre_norm=1, out_dtype=BF16)
    ops.sync()

    _, _, y1, dy1 = residual_norm64(x0, pre=2, **norm)
    st = s.double()[:, None]
    check(q.double() * st, y1, st * 0.5 + dy1 + 8 * U * (y1.abs() + st), "norm")
    v, dv = linear64(q, s, wu, su, None, "swiglu")
    check(h, v, dv + half_step(v.abs() + dv, BF16), "gate and up")
    want, ws = quantize64(h)
    assert torch.equal(qh, want) and torch.equal(sh, ws)
    v, dv = linear64(qh, sh, wd, sd)
    check(d, v, dv + half_step(v.abs() + dv, BF16), "down")
    x64, dx, y64, dy = residual_norm64(x0, d, post=1, gate=vec[:, 2], rows_per_vec=per, pre=1)
    assert xn is x
    check(x, x64, dx, "x'")
    check(y, y64, dy + half_step(y64.abs() + dy, BF16), "y")

    u, _ = act64(y1 @ wf[0].double().t()[:, :hidden], torch.zeros((), device="cuda"), "silu")
    full = (u * (y1 @ wf[0].double().t()[:, hidden:])) @ wf[1].double().t()
    cos = torch.nn.functional.cosine_similarity(d.double().flatten(), full.flatten(), dim=0).item()
    # Four 8-bit roundings (two of rows, two of weights). A row's or channel's peak is below 5.5 deviations, so a step
    # is below 5.5 / 127 and its rounding adds at most step^2 / 12 = 1.6e-4 of the variance; the gated product passes a
    # factor's relative error on with a slope below 2 (variance 4) from each of its factors, and the hidden rows' peak is
    # below 40 of their deviations: 8.3e-3. Together under 1.5e-2 of the variance: cosine above 1 - 0.75e-2.
    assert cos > 0.9925, cos


@pytest.mark.parametrize("m", [1, 3, 20, 100, 300, 1100])
@pytest.mark.parametrize("act", ["gelu_tanh", "gelu_erf", "silu", "swiglu", "geglu"])
def test_activations_of_infinities(cuda, m, act):
    """An infinite bias, and a scaled sum that overflows: +inf stays +inf and what the definition makes NaN is NaN."""
    from naivediffusion_b200 import ops
    n, k = 256, 320
    _, x, sx, w, sw, b = _case(m, n, k, m + 23, gated=act in ("swiglu", "geglu"))
    b[5::16], b[6::32] = math.inf, -math.inf
    sx[m // 2] = 3e38
    sw[9::16] = 1e3
    y = ops.linear_w8a8(x, sx, w, sw, b, epilogue=EPI[act])
    ops.sync()
    v = (linear64(x, sx, w, sw, b)[0]).float().double()  # overflows where fp32 does
    f = n if act in ("swiglu", "geglu") else v.shape[1]
    zero = torch.zeros((), device="cuda", dtype=torch.float64)
    if act == "swiglu":
        want = act64(v[:, :f], zero, "silu")[0] * v[:, f:]
    elif act == "geglu":
        want = v[:, :f] * act64(v[:, f:], zero, "gelu_erf")[0]
    else:
        want = act64(v, zero, act)[0]
    far = torch.isinf(want)
    assert far.any() and torch.equal(torch.isnan(y), torch.isnan(want))
    assert torch.equal(y[far].double(), want[far])


@pytest.mark.parametrize("m,splits", [(3, (1, 2)), (30, (7, 16)), (200, (33, 77)), (1500, (130, 1003))])
@pytest.mark.parametrize("act", ["f32", "store", "gate", "gelu_erf", "swiglu"])
def test_a_split_changes_no_row(cuda, m, splits, act):
    """With shared weights a row's bits do not depend on where the two groups meet: they are those of its own group's
    vectors alone."""
    from naivediffusion_b200 import ops
    n, k = 256, 384
    g, x, sx, w, sw, _ = _case(m, n, k, m + 41, gated=act == "swiglu")
    b = torch.randn(2, w.shape[0], generator=g, device="cuda")
    gate = torch.randn(2, n, generator=g, device="cuda") if act == "gate" else None
    r0 = torch.randn(m, n, generator=g, device="cuda")

    def run(bias, gates, **kw):
        if act == "gate":
            kw.update(gate=gates, residual=r0.clone())
        return ops.linear_w8a8(x, sx, w, sw, bias, epilogue=EPI[act], **kw)

    alone = [run(b[i], None if gate is None else gate[i]) for i in range(2)]
    for split in splits:
        y = run(b, gate, group_split=split, shared_weights=True)
        ops.sync()
        assert torch.equal(y[:split], alone[0][:split]) and torch.equal(y[split:], alone[1][split:]), split


def test_more_gated_outputs_than_warps_count_in_32_bits(cuda):
    """One row, 2^27 + 128 outputs: a warp each, whose threads' numbers pass 2^32."""
    from naivediffusion_b200 import ops
    n, k = (1 << 27) + 128, 16
    x, sx = torch.ones(1, k, device="cuda", dtype=I8), torch.ones(1, device="cuda")
    w = torch.ones(2 * n, k, device="cuda", dtype=I8)
    sw = torch.full((2 * n,), 1 / 16, device="cuda")
    sw[n - 100:n], sw[n:n + 50] = 1 / 8, 1 / 4  # first factors 2 at the end, second factors 4 at the start
    out = torch.full((1, n), math.nan, device="cuda", dtype=BF16)
    ops.linear_w8a8(x, sx, w, sw, epilogue=EPI["swiglu"], out=out)
    ops.sync()
    one, two = (1 / (1 + math.exp(-1))), 2 / (1 + math.exp(-2))
    want = torch.full((n,), one, device="cuda", dtype=F32)
    want[:50], want[n - 100:] = 4 * one, two
    # two fp32 roundings of the factors, ex2 and rcp a few ulp each, and the store's half step
    assert (out[0].float() - want).abs().le(want * (2.0 ** -8 + 16 * U)).all()


@pytest.mark.parametrize("m,n,k", [(1, 96, 77), (20, 130, 1155), (200, 64, 333), (1100, 512, 71)])
def test_weights_of_any_width(cuda, m, n, k):
    """quantize_rows makes weights too, of any in_features: rows a multiple of 16 bytes apart, a scale per channel."""
    from naivediffusion_b200 import ops
    g = _gen(m + k)
    wf = torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)
    x, sx = ops.quantize_rows(torch.randn(m, k, generator=g, device="cuda"))
    w, sw = ops.quantize_rows(wf)
    y = ops.linear_w8a8(x, sx, w, sw)
    ops.sync()
    check(w.double() * sw.double()[:, None], wf.double(), sw.double()[:, None] * 0.5 + 2 * U * wf.abs())
    v, dv = linear64(x, sx, w, sw)
    check(y, v, dv + half_step(v.abs() + dv, BF16))
