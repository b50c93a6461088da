"""Plain 64-bit forms of residual_norm, quantize_rows and linear_w8a8, with
bounds on what fp32 arithmetic may add.

U = 2^-24 is half a unit in fp32's last place: the largest relative error of
one rounded operation. A sum over a row adds at most C roundings to any one
term (16 values per thread, 5 shuffle steps, 32 warps, and the division by the
width): its error is at most C * U times the sum of absolute values.
"""
import math

import torch

U = 2.0 ** -24
C = 16 + 5 + 32 + 1


def norm64(z, dz, kind, eps):
    """kind over rows of z (64-bit) whose fp32 counterpart is off by at most dz: the result and its bound."""
    if kind == 0:
        return z, dz
    if kind == 2:
        mean = z.mean(1, keepdim=True)
        dm = dz.mean(1, keepdim=True) + C * U * z.abs().mean(1, keepdim=True)
        z = z - mean
        dz = dz + dm + U * (z.abs() + dm)
    ms = z.square().mean(1, keepdim=True)
    # |sum 2 z dz| <= 2 |z| |dz| (Cauchy-Schwarz), the squares' own sum, and the sum's roundings
    dms = 2 * (ms * dz.square().mean(1, keepdim=True)).sqrt() + dz.square().mean(1, keepdim=True) + C * U * ms
    r = (ms + eps).rsqrt()
    # d(x^-1/2) = x^-3/2 dx / 2; 10 % covers the second order; rsqrtf is 2 ulp (4 U), the sum ms + eps one rounding
    dr = r * (0.55 * dms / (ms + eps) + 5 * U)
    return z * r, dz * r + z.abs() * dr + U * (z * r).abs()


def residual_norm64(x, branch=None, post=0, post_weight=None, gate=None, residual_scale=1.0, pre=0, pre_weight=None,
                    scale=None, shift=None, rows_per_vec=0, plus_one=False, eps=1e-6):
    """x', its bound, y, its bound (before y's own rounding to the output type)."""
    x = x.double()
    rows = x.shape[0]

    def vec(t):
        if t is None:
            return None
        t = t.double().reshape(-1, x.shape[1])
        which = torch.arange(rows, device=x.device) // max(rows_per_vec, 1) if t.shape[0] > 1 else torch.zeros(rows, dtype=torch.long, device=x.device)
        return t[which.clamp(max=t.shape[0] - 1)]

    one = 1.0 if plus_one else 0.0
    xn, dx = x * residual_scale, U * (x * residual_scale).abs()
    if branch is not None:
        b, db = norm64(branch.double(), torch.zeros_like(x), post, eps)
        for factor in (None if post_weight is None else post_weight.double() + one, vec(gate)):
            if factor is not None:  # the factor's own sum with one, and the product: two roundings
                db = db * factor.abs() + 2 * U * (b * factor).abs()
                b = b * factor
        db = db + 2 * U * b.abs()  # rstd, weight and gate are multiplied together first: one order or the other
        xn = xn + b
        dx = dx + db + U * xn.abs()
    y, dy = norm64(xn, dx, pre, eps)
    if pre_weight is not None:
        w = pre_weight.double() + one
        dy = dy * w.abs() + 2 * U * (y * w).abs()
        y = y * w
    if scale is not None:
        s = 1 + vec(scale)
        dy = dy * s.abs() + U * (y.abs() * (1 + s.abs()) + (y * s).abs())
        y = y * s
    if shift is not None:
        y = y + vec(shift)
        dy = dy + U * y.abs()
    return xn, dx, y, dy


def half_step(y, dtype):
    """The most that rounding y to dtype moves it: half a step, relative, and in fp16 half of the smallest step."""
    return y.abs() * (torch.finfo(dtype).eps / 2) + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134)


def quantize64(x):
    """q and scale: the quotient is correctly rounded in 64 bits, and never falls onto a half that it is not."""
    x = x.double()
    peak = x.abs().amax(1)
    q = (x * 127 / peak[:, None]).round()
    q[peak == 0] = 0
    bad = ~torch.isfinite(peak)
    q[bad] = 0
    scale = (peak / 127).float()
    scale[bad] = math.nan
    return q.to(torch.int8), scale


def act64(v, dv, name):
    """An activation of v (off by at most dv) and its bound. Slopes are below 1.13; __expf is off by 2 + 1.16 |u| ulp."""
    if name == "silu":
        y = v * torch.sigmoid(v)
        return y, 1.13 * dv + y.abs() * 2 * U * (6 + 1.2 * v.abs())
    if name == "gelu_tanh":
        u = 2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)
        y = v * torch.sigmoid(u)
        return y, 1.13 * dv + y.abs() * 2 * U * (6 + 3.5 * u.abs())
    if name == "gelu_erf":
        y = 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))  # 1 + erf cancels: an absolute error of 4 U times x / 2
        return y, 1.13 * dv + v.abs() * 4 * U + 2 * U * y.abs()
    return v, dv


def linear64(x, x_scale, weight, w_scale, bias=None, act="store"):
    """The product and its bound (before the output's own rounding); x_scale, w_scale, bias per row / column."""
    acc = x.double() @ weight.double().t()
    v = acc * x_scale.double()[:, None] * w_scale.double()
    dv = 3 * U * v.abs() * 1.01
    if bias is not None:
        v = v + bias.double()
        dv = dv + U * (v.abs() + dv)
    if act in ("swiglu", "geglu"):
        f = v.shape[1] // 2
        first, second = (0, 1) if act == "swiglu" else (1, 0)
        halves = [(v[:, :f], dv[:, :f]), (v[:, f:], dv[:, f:])]
        a, da = act64(*halves[first], "silu" if act == "swiglu" else "gelu_erf")
        b, db = halves[second]
        return a * b, da * b.abs() + db * (a.abs() + da) + U * (a * b).abs()
    return act64(v, dv, act)


def check(got, want, bound, what=""):
    """got within bound of want everywhere; NaN where want has NaN."""
    got, want = got.double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    over = (got - want).abs() - bound
    over = over[~torch.isnan(over)]
    assert over.numel() == 0 or over.max().item() <= 0, f"{what}: {(over > 0).sum().item()} of {got.numel()} outside, by up to {over.max().item():.3g}"
