"""residual_norm and quantize_rows against plain 64-bit forms (rowops_reference)."""
import math

import pytest
import torch

from rowops_reference import U, check, half_step, quantize64, residual_norm64

pytestmark = pytest.mark.gpu
NONE, RMS, LAYER = 0, 1, 2
BF16, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _inputs(rows, width, btype, vecs, seed):
    g = _gen(seed)
    x = _randn(g, rows, width) * 2 + 0.5
    b = None if btype is None else (_randn(g, rows, width) * 1.5 - 0.25).to(btype)
    v = 0.3 * _randn(g, vecs, 3, width)
    return x, b, v, 1 + 0.1 * _randn(g, width), 0.1 * _randn(g, width)


def _check_y(got, y, dy, out):
    if out == I8:
        _, q, scale = got
        peak = y.abs().amax(1)
        dpeak = dy.amax(1)
        check(scale, peak / 127, dpeak / 127 + 2 * U * (peak + dpeak) / 127, "scale")
        # q is the nearest integer to y's fp32 form over the stored scale (its product with 127 / peak is 2 U off)
        s = scale.double()[:, None]
        check(q.double() * s, y, s * 0.5 + dy + 8 * U * (y.abs() + s), "q")
        assert q.abs().amax(1).eq(127).logical_or(peak.eq(0)).all()
    else:
        assert got[1].dtype == out
        check(got[1], y, dy + (half_step(y.abs() + dy, out) if out != F32 else U * y.abs()), "y")


@pytest.mark.parametrize("rows,width", [(1, 1), (1, 1024), (3, 4), (5, 130), (37, 512), (129, 1155), (64, 2048), (33, 3584),
                                        (7, 4100), (4, 8192), (3, 12289), (2, 16384), (1400, 1028), (2500, 333), (1501, 1),
                                        (1187, 2047), (305, 3001), (301, 8191), (310, 4104)])
@pytest.mark.parametrize("btype,out,post,pre", [(BF16, BF16, RMS, RMS), (F16, I8, NONE, LAYER), (F32, F32, LAYER, LAYER),
                                                (None, F16, NONE, RMS)])
def test_against_64_bits(cuda, rows, width, btype, out, post, pre):
    from naivediffusion_b200 import ops
    x, b, v, w1, w2 = _inputs(rows, width, btype, 2, rows * 1000 + width)
    per = (rows + 1) // 2
    kw = dict(post_norm=post, post_weight=w1 if post else None, gate=None if b is None else v[:, 0], residual_scale=0.75,
              pre_norm=pre, pre_weight=w2, scale=v[:, 1], shift=v[:, 2], rows_per_vec=per, plus_one=False, eps=1e-5)
    new = torch.empty_like(x)
    got = ops.residual_norm(x, b, x_out=new, out_dtype=out, **kw)
    ops.sync()
    assert got[0] is new
    kw["post"], kw["pre"] = kw.pop("post_norm"), kw.pop("pre_norm")
    xn, dx, y, dy = residual_norm64(x, b, **kw)
    check(new, xn, dx, "x'")
    _check_y(got, y, dy, out)


@pytest.mark.parametrize("rows,width,btype,out,post,pre,vecs", [
    (8200, 1024, BF16, BF16, RMS, RMS, 3), (16500, 512, F16, F16, NONE, LAYER, 1), (4100, 2048, F32, I8, LAYER, RMS, 2),
    (2100, 4096, BF16, I8, RMS, LAYER, 2), (1100, 8192, F32, F32, LAYER, LAYER, 2), (8200, 1032, None, BF16, NONE, LAYER, 4),
    (30000, 296, BF16, F32, RMS, LAYER, 3000), (4300, 2047, BF16, F16, LAYER, LAYER, 5), (2300, 4095, F32, I8, NONE, RMS, 1)])
def test_many_rows(cuda, rows, width, btype, out, post, pre, vecs):
    """The rows that persistent blocks work through, in place, with many vector sets too."""
    from naivediffusion_b200 import ops
    x, b, v, w1, w2 = _inputs(rows, width, btype, vecs, rows + width)
    per = -(-rows // vecs)
    kw = dict(post_weight=w1 if post else None, gate=None if b is None else v[:, 0], residual_scale=1.0 if b is None else 0.5,
              pre_weight=w2 if pre == RMS else None, scale=v[:, 1], shift=v[:, 2], rows_per_vec=per)
    xn, dx, y, dy = residual_norm64(x, b, post=post, pre=pre, **kw)
    got = ops.residual_norm(x, b, post_norm=post, pre_norm=pre, out_dtype=out, **kw)
    ops.sync()
    check(x, xn, dx, "x'")
    _check_y(got, y, dy, out)


def test_every_norm_pair_plus_one_and_in_place(cuda):
    from naivediffusion_b200 import ops
    for post in (NONE, RMS, LAYER):
        for pre in (NONE, RMS, LAYER):
            x, b, v, w1, w2 = _inputs(19, 640, BF16, 1, 10 * post + pre)
            kw = dict(post_weight=w2 if post else None, gate=v[0, 0], pre_weight=w2 if pre else None, plus_one=True)
            xn, dx, y, dy = residual_norm64(x, b, post=post, pre=pre, **kw)
            again = x.clone()
            got = ops.residual_norm(x, b, post_norm=post, pre_norm=pre, out_dtype=F32, **kw)
            assert got[0] is x
            first = [t.clone() for t in got]
            second = ops.residual_norm(again, b, post_norm=post, pre_norm=pre, out_dtype=F32, **kw)
            ops.sync()
            check(x, xn, dx, f"x' {post} {pre}")
            check(got[1], y, dy + U * y.abs(), f"y {post} {pre}")
            assert all(torch.equal(a, c) for a, c in zip(first, second))


def test_parts_alone(cuda):
    """Only x', only a norm (x untouched), and a residual scale without a branch."""
    from naivediffusion_b200 import ops
    x, b, v, w1, _ = _inputs(40, 1280, F16, 1, 5)
    keep = x.clone()
    new, none = ops.residual_norm(x, b, x_out=torch.empty_like(x), gate=v[0, 0], pre_norm=NONE, out_dtype=None)
    assert none is None
    xn, dx, _, _ = residual_norm64(x, b, gate=v[0, 0])
    same, y = ops.residual_norm(x, pre_norm=RMS, pre_weight=w1, out_dtype=BF16)
    _, _, y64, dy = residual_norm64(x, pre=RMS, pre_weight=w1)
    ops.sync()
    check(new, xn, dx)
    assert same is x and torch.equal(x, keep)
    check(y, y64, dy + half_step(y64.abs() + dy, BF16))
    half, _ = ops.residual_norm(x, residual_scale=0.5, pre_norm=NONE, out_dtype=None)
    ops.sync()
    assert half is x and torch.equal(x, keep * 0.5)


@pytest.mark.parametrize("rows,width,offset,stride", [(21, 1280, 0, 1284), (21, 1280, 1, 1283), (21, 1280, 4, 1300),
                                                      (21, 1280, 3, 1290), (6600, 1280, 8, 1296), (1300, 1280, 3, 1281),
                                                      (1201, 517, 5, 517), (250001, 3, 1, 3), (90001, 7, 7, 9),
                                                      (1250, 1030, 2, 1037), (600003, 1, 1, 1)])
def test_strides_and_alignment(cuda, rows, width, offset, stride):
    """Rows of wider matrices, starting anywhere; what lies beside them stays."""
    from naivediffusion_b200 import ops
    g = _gen(offset + stride)

    def view(t):
        return t.as_strided((rows, width), (stride, 1), offset)

    size = rows * stride + 16
    xs, bs = _randn(g, size), _randn(g, size).to(BF16)
    v = 0.3 * _randn(g, 3, 4, width + 1)
    gate, scale, shift = (v[:, i, :width] for i in range(3))
    outs = {t: torch.full((size,), 7, device="cuda", dtype=t) for t in (F32, BF16, I8)}
    x2 = torch.full((size,), 7.0, device="cuda")
    xn, dx, y, dy = residual_norm64(view(xs), view(bs), post=RMS, gate=gate, pre=LAYER, scale=scale, shift=shift,
                                    rows_per_vec=(rows + 2) // 3)
    for dtype, store in outs.items():
        got = ops.residual_norm(view(xs), view(bs), x_out=view(x2), post_norm=RMS, gate=gate, scale=scale, shift=shift,
                                rows_per_vec=(rows + 2) // 3, out=view(store))
        ops.sync()
        check(view(x2), xn, dx)
        _check_y(got, y, dy, dtype)
        inside = torch.zeros(size, dtype=torch.bool, device="cuda")
        view(inside).fill_(True)
        assert store[~inside].eq(7).all() and x2[~inside].eq(7).all()


def test_more_rows_than_the_last_vector_set(cuda):
    """Rows past the last set's share keep the last set."""
    from naivediffusion_b200 import ops
    x, b, v, _, _ = _inputs(100, 256, BF16, 3, 9)
    kw = dict(gate=v[:, 0], scale=v[:, 1], shift=v[:, 2], rows_per_vec=10)
    new, y = ops.residual_norm(x, b, x_out=torch.empty_like(x), out_dtype=F32, **kw)
    ops.sync()
    xn, dx, y64, dy = residual_norm64(x, b, pre=LAYER, **kw)
    check(new, xn, dx)
    check(y, y64, dy + U * y64.abs())


@pytest.mark.parametrize("width", [96, 1155, 2048])
def test_rows_of_zeros_and_not_finite(cuda, width):
    from naivediffusion_b200 import ops
    x, b, _, _, _ = _inputs(6, width, F32, 1, width)
    x[1], b[1] = 0, 0
    x[2, width // 2], b[3, 0], x[4, -1] = math.inf, math.nan, -math.inf
    new, q, scale = ops.residual_norm(x, b, x_out=torch.empty_like(x), pre_norm=RMS, out_dtype=I8)
    _, y = ops.residual_norm(x, b, x_out=torch.empty_like(x), pre_norm=RMS, out_dtype=BF16)
    ops.sync()
    assert scale[1] == 0 and q[1].eq(0).all() and y[1].eq(0).all()
    assert torch.isnan(scale[2:5]).all() and q[2:5].eq(0).all()
    assert torch.isnan(y[3]).all() and torch.isnan(y[2, width // 2]) and torch.isnan(y[4, -1])
    assert torch.isfinite(scale[[0, 5]]).all() and torch.isfinite(y[[0, 1, 5]]).all()
    assert new[2, width // 2] == math.inf and new[4, -1] == -math.inf and torch.isnan(new[3, 0])


def test_values_far_from_one(cuda):
    """A large offset under LayerNorm (two passes keep it), tiny and large rows to int8."""
    from naivediffusion_b200 import ops
    g = _gen(11)
    x = _randn(g, 16, 1024) + 1000
    _, y = ops.residual_norm(x, out_dtype=F32)
    ops.sync()
    _, _, y64, dy = residual_norm64(x, pre=LAYER)
    check(y, y64, dy + U * y64.abs())
    for size in (1e-38, 3e-33, 1e30):
        x = _randn(g, 5, 512) * size
        _, q, scale = ops.residual_norm(x, pre_norm=NONE, out_dtype=I8)
        ops.sync()
        want, ws = quantize64(x)
        assert (q.int() - want.int()).abs().max() <= 1
        check(scale, ws, 2 * U * ws.double() + 2.0 ** -149)


@pytest.mark.parametrize("rows,width", [(1, 1), (1, 77), (77, 2048), (5, 130), (300, 513), (33, 4096), (17, 5121), (3, 12288),
                                        (2, 20001), (1, 40000), (40, 1), (41, 2), (19, 3), (500, 511), (130, 2047), (9, 4095),
                                        (1200, 8191), (3, 16383)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_quantize_rows_is_exact(cuda, rows, width, dtype):
    from naivediffusion_b200 import ops
    g = _gen(rows * 7 + width)
    x = (_randn(g, rows, width) * (0.1 + torch.rand(rows, 1, generator=g, device="cuda"))).to(dtype)
    q, scale = ops.quantize_rows(x)
    ops.sync()
    want, ws = quantize64(x)
    assert torch.equal(q, want) and torch.equal(scale, ws)
    assert rows == 1 or q.stride(0) % 16 == 0


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_quantize_rows_rounds_halves_to_even(cuda, dtype):
    """Quotients that are a half, or one step of x from it: x = peak * (k + 1/2) / 127 where it has such a value."""
    from naivediffusion_b200 import ops
    g = _gen(3)
    peaks = torch.cat([127.0 * 2.0 ** torch.arange(-6, 6), torch.tensor([1.0, 3.0, 0.37, 254.0])]).to("cuda").to(dtype)
    near = (peaks[:, None].double() * (torch.arange(-127, 127, device="cuda") + 0.5) / 127).to(dtype)
    rows = torch.cat([near, torch.nextafter(near.float(), torch.full_like(near, 1e4).float()).to(dtype), peaks[:, None]], 1)
    if dtype != F32:
        step = near.view(torch.int16)
        rows = torch.cat([rows, (step + 1).view(dtype), (step - 1).view(dtype)], 1)
        rows = torch.where(rows.abs() > peaks[:, None], peaks[:, None], rows)
    rows = rows[:, torch.randperm(rows.shape[1], generator=g, device="cuda")].contiguous()
    q, scale = ops.quantize_rows(rows)
    ops.sync()
    want, ws = quantize64(rows)
    assert torch.equal(q, want) and torch.equal(scale, ws)


def test_quantize_rows_special_rows_and_strides(cuda):
    from naivediffusion_b200 import ops
    g = _gen(4)
    for width, offset, stride in ((128, 0, 160), (1155, 1, 1160), (1156, 2, 1161)):
        store = _randn(g, 12 * stride + 4)
        x = store.as_strided((12, width), (stride, 1), offset)
        x[1] = 0
        x[2, 0], x[3, width - 1], x[4, 5] = math.inf, math.nan, -math.inf
        x[5] *= 1e-40
        x[6] *= 1e37
        out = torch.full((12, width + 9), 55, device="cuda", dtype=I8)
        q, scale = ops.quantize_rows(x, out=out)
        ops.sync()
        want, ws = quantize64(x)
        assert torch.equal(q[:, :width], want) and q[:, width:].eq(55).all()
        assert torch.equal(torch.isnan(scale), torch.isnan(ws)) and torch.equal(scale.nan_to_num(9), ws.nan_to_num(9))


@pytest.mark.parametrize("rows,cols", [(1, 1), (77, 2048), (3000, 640), (1001, 5121), (9, 40000), (5000, 48), (700, 17),
                                       (33, 21), (3, 5), (1, 16), (257, 1155)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_values_of_int8_rows(cuda, rows, cols, dtype):
    """dequantize gives back what a quantized row stands for, rounded once: within half a step of x and of dtype."""
    from naivediffusion_b200 import ops
    x = _randn(_gen(rows + cols), rows, cols)
    q, scale = ops.quantize_rows(x)
    got = ops.dequantize(q.contiguous(), scale, 0, dtype)
    ops.sync()
    assert torch.equal(got, (q.float() * scale[:, None]).to(dtype))
    v, s = x.double(), scale.double()[:, None]
    check(got, v, s * 0.5 + 2 * U * v.abs() + half_step(v.abs() + s, dtype))


@pytest.mark.parametrize("rows,cols,group", [(300, 512, 32), (301, 264, 24), (77, 340, 20), (5, 51, 17), (129, 96, 16),
                                             (64, 640, 8), (3, 15, 5), (2000, 2560, 64), (1, 33, 33)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_values_of_groups(cuda, rows, cols, group, dtype):
    """Groups that runs of 16 values straddle, and matrices off a 16-byte address, bit for bit."""
    from naivediffusion_b200 import ops
    g = _gen(rows + cols)
    q = torch.randint(-127, 128, (rows * cols + 3,), generator=g, device=g.device, dtype=I8).cuda()
    scale = _randn(g, rows, cols // group).cuda().abs()
    for start, sdt in ((0, F32), (0, F16), (3, F32)):
        part, s = q[start:start + rows * cols].view(rows, cols), scale.to(sdt)
        got = ops.dequantize(part, s, group, dtype)
        ops.sync()
        want = (part.float().view(rows, -1, group) * s.float()[:, :, None]).to(dtype)
        assert torch.equal(got, want.view(rows, cols))


def test_streams_and_graphs(cuda):
    """On a side stream, and captured: a replay reads the inputs' values of that moment."""
    from naivediffusion_b200 import ops
    x, b, v, _, _ = _inputs(50, 1024, BF16, 1, 21)
    new = torch.empty_like(x)
    want = [t.clone() for t in ops.residual_norm(x, b, x_out=new, gate=v[0, 0], out_dtype=I8)]
    qw = [t.clone() for t in ops.quantize_rows(b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.residual_norm(x, b, x_out=torch.empty_like(x), gate=v[0, 0], out_dtype=I8)
        q = ops.quantize_rows(b)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(got, want)) and all(torch.equal(a, c) for a, c in zip(q, qw))
    x2, b2 = x.clone(), b.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.residual_norm(x2, b2, x_out=torch.empty_like(x2), gate=v[0, 0], out_dtype=I8)
        q = ops.quantize_rows(b2)
    for _ in range(2):
        x2.copy_(x), b2.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(got, want)) and all(torch.equal(a, c) for a, c in zip(q, qw))
        x2.zero_(), b2.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert got[1].eq(0).all() and q[1].eq(0).all()


@pytest.mark.parametrize("rows,width", [(5000, 2048), (3000, 2047)])
def test_many_rows_in_place_on_two_streams_and_captured(cuda, rows, width):
    """Persistent blocks of two calls at once share nothing; a captured in-place call goes on from what it left."""
    from naivediffusion_b200 import ops
    cases = [_inputs(rows, width, BF16, 2, seed) for seed in (1, 2)]
    kw = [dict(gate=v[:, 0], scale=v[:, 1], shift=v[:, 2], rows_per_vec=rows // 2, post_norm=RMS, out_dtype=BF16) for _, _, v, _, _ in cases]
    want = []
    for (x, b, _, _, _), k in zip(cases, kw):
        x = x.clone()
        want.append([[t.clone() for t in ops.residual_norm(x, b, **k)] for _ in range(3)])
    torch.cuda.synchronize()
    xs = [c[0].clone() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append([t.clone() for t in ops.residual_norm(xs[i], cases[i][1], **kw[i])])
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(p, q) for a, b in zip(w, g) for p, q in zip(a, b))
    x = cases[0][0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new, y = ops.residual_norm(x, cases[0][1], **kw[0])
    x.copy_(cases[0][0])
    for step in range(3):
        graph.replay()
        ops.sync()
        assert new is x and torch.equal(x, want[0][step][0]) and torch.equal(y, want[0][step][1])


@pytest.mark.parametrize("rows,width", [(1, 1), (9, 4), (40, 130), (33, 512), (30, 1024), (20, 1155), (64, 2048), (7, 4100), (5, 8192),
                                        (2, 12289), (2, 16384), (5000, 2048), (3000, 2047), (17000, 512), (1100, 8192)])
@pytest.mark.parametrize("pre", [NONE, RMS, LAYER])
def test_int8_rows_are_those_of_the_quantizer(cuda, rows, width, pre):
    """An int8 y is what quantize_rows makes of the fp32 y, bit for bit; every quotient a half or near one without a norm."""
    from naivediffusion_b200 import ops
    g = _gen(rows + width + pre)
    if pre == NONE:  # peak 381 2^j, so y * 127 / peak = y 2^-j / 3: thirds of odd halves, and their neighbours
        x = (torch.randint(-762, 763, (rows, width), generator=g, device="cuda").float() / 2)
        x[:, 0] = 381
        near = torch.nextafter(x, torch.where(x > 0, math.inf, -math.inf).to(x))
        x = torch.where(torch.rand(rows, width, generator=g, device="cuda") < 0.25, near.clamp(-381, 381), x)
        x = x * 2.0 ** torch.randint(-120, 110, (rows, 1), generator=g, device="cuda")
    else:
        x = _randn(g, rows, width) * 2 + 0.5
    x[rows // 2] = 0
    _, y = ops.residual_norm(x, pre_norm=pre, out_dtype=F32)
    _, q, scale = ops.residual_norm(x, pre_norm=pre, out_dtype=I8)
    want, ws = ops.quantize_rows(y)
    ops.sync()
    assert torch.equal(scale, ws)
    assert torch.equal(q, want), (q != want).sum()


def test_an_exact_half_goes_to_even(cuda):
    from naivediffusion_b200 import ops
    x = torch.tensor([[381.0, 1.5, -1.5, 4.5, -4.5, 7.5]], device="cuda")
    _, q, scale = ops.residual_norm(x, pre_norm=NONE, out_dtype=I8)
    ops.sync()
    assert q[0].tolist() == [127, 0, 0, 2, -2, 2] and scale[0] == 3


def test_only_x_without_naming_a_norm(cuda):
    from naivediffusion_b200 import ops
    x, b, v, _, _ = _inputs(40, 1280, F16, 1, 5)
    keep = x.clone()
    new, none = ops.residual_norm(x, b, x_out=torch.empty_like(x), gate=v[0, 0], out_dtype=None)
    ops.sync()
    xn, dx, _, _ = residual_norm64(x, b, gate=v[0, 0])
    check(new, xn, dx)
    assert none is None and torch.equal(x, keep)


@pytest.mark.parametrize("rows,cols,group,start", [(5000, 1, 1, 0), (7001, 3, 3, 1), (3000, 8, 4, 0), (1001, 15, 15, 5), (513, 33, 33, 1),
                                                   (400, 129, 43, 3), (1000, 1155, 1155, 3), (301, 768, 256, 3), (77, 510, 255, 1),
                                                   (9, 771, 257, 7), (3, 40000, 8, 0), (2, 5000, 2500, 1)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_values_of_any_rows_and_groups(cuda, rows, cols, group, start, dtype):
    """Narrow rows, short groups, and long ones off a 16-byte address, bit for bit; nothing past the last value."""
    from naivediffusion_b200 import _lib, ops
    g = _gen(rows + cols)
    q = torch.randint(-127, 128, (rows * cols + start,), generator=g, device="cuda", dtype=torch.int32).to(I8)[start:].view(rows, cols)
    scale = _randn(g, rows, cols // group).abs()
    want = (q.float().view(rows, -1, group) * scale[:, :, None]).to(dtype).flatten()
    out = torch.full((rows * cols + 40,), 7, device="cuda", dtype=dtype)
    _lib.check(_lib.lib().nd_op_dequantize(q.data_ptr(), scale.data_ptr(), _lib.ND_F32, group, rows, cols, out.data_ptr(),
                                           ops._DT[dtype], torch.cuda.current_stream().cuda_stream))
    ops.sync()
    assert torch.equal(out[:rows * cols], want) and out[rows * cols:].eq(7).all()
    assert torch.equal(ops.dequantize(q, scale, group, dtype).flatten(), want)
