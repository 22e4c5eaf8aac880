"""float64 restatement of the batch-independent training layer (grid_gcn_amd/act8.py) on CPU tensors: the 8-bit form, group
normalisation with an activation, the linear layer with an 8-bit input -- and, beside every value, how far a float32
computation of it may be off, from the roundings it makes (U = 2^-24, half a step of float32).  Test infrastructure."""
import math

import torch

U = 2.0 ** -24
BLOCK, MIN_EXP = 32, -117


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """half the smallest positive number of the type: what rounding a value below it may cost"""
    return {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}[dtype]


def act8(x):
    """(values float64 [..., C], exponents int [..., blocks]) of the 8-bit form of x; non-finite -> NaN"""
    x = x.detach().double()
    C = x.shape[-1]
    p = torch.nn.functional.pad(x, (0, -C % BLOCK)).unflatten(-1, (-1, BLOCK))
    fin = torch.isfinite(p)
    amax = torch.where(fin, p.abs(), torch.zeros_like(p)).amax(-1)
    m, e = torch.frexp(amax)                                      # amax = m 2^e, m in [1/2, 1); 448 = 7/8 * 2^9
    E = torch.where(amax > 0, e - 9 + (m > 0.875).int(), torch.full_like(e, MIN_EXP)).clamp(min=MIN_EXP)
    v = p * torch.exp2(-E.double())[..., None]
    k = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6, max=448.0)))
    step = torch.exp2(k - 3)
    q = torch.round(v / step) * step                              # (torch.round: ties to even)
    q = torch.where(fin, q * torch.exp2(E.double())[..., None], torch.full_like(q, float("nan")))
    return q.flatten(-2)[..., :C], E


def act_fn(t, act):
    """act(t), act'(t), a bound of |act''|"""
    if act == "relu":
        return t.clamp(min=0), (t > 0).double(), 0.0
    if act == "silu":
        s = torch.sigmoid(t)
        return t * s, s * (1 + t * (1 - s)), 0.5
    if act == "gelu":
        c = 0.5 * (1 + torch.erf(t / math.sqrt(2)))
        return t * c, c + t * torch.exp(-t * t / 2) / math.sqrt(2 * math.pi), 0.8
    return t, torch.ones_like(t), 0.0


def group_norm_act(x, weight, bias, groups, eps, act, counts=None, dy=None, save8=False):
    """dict of float64 results y, dx, dw, db (the last three with dy) and their float32 bounds y_tol, ...

    Roundings of a float32 evaluation, in units of U relative to the term they act on: x - mean 2 (one subtraction of
    each half of the mean), rstd * weight 1, their product and sum with bias 1, so t is off by dt = 4 (|t - bias| + |t|) U; act and
    act' by their slope times dt, plus 8 (1 + |t|) U of their value for an exponential with a rounded argument (t * t / 2
    and t * log2(e) are off by U relative to themselves) or erf; then products and sums as they come."""
    B, C = x.shape[0], x.shape[-1]
    x3 = x.detach().double().reshape(B, -1, groups, C // groups)
    N = x3.shape[1]
    n = torch.full((B,), N) if counts is None else counts.reshape(B).cpu().long().clamp(0, N)
    valid = (torch.arange(N)[None] < n[:, None])[:, :, None, None]
    M = (n.clamp(min=1) * (C // groups)).double().reshape(B, 1, 1, 1)
    z = torch.where(valid, x3, torch.zeros_like(x3))
    mean = z.sum((1, 3), keepdim=True) / M
    d = torch.where(valid, z - mean, torch.zeros_like(z))
    rstd = ((d * d).sum((1, 3), keepdim=True) / M + eps).rsqrt()
    w = (torch.ones(C) if weight is None else weight.detach()).double().reshape(groups, -1)
    b = (torch.zeros(C) if bias is None else bias.detach()).double().reshape(groups, -1)

    def at(dev):
        xh = dev * rstd
        t = xh * w + b
        dt = 4 * U * ((xh * w).abs() + t.abs())
        return xh, t, dt

    keep = lambda v: torch.where(valid, v, torch.zeros_like(v))                         # noqa: E731
    xh, t, dt = at(d)
    f, _, _ = act_fn(t, act)
    soft = 0 if act in ("none", "relu") else 8
    out = dict(y=keep(f).reshape(x.shape), y_tol=keep(1.2 * dt + (soft * (1 + t.abs()) + 1) * U * f.abs()).reshape(x.shape),
               mean=mean.reshape(B, groups), rstd=rstd.reshape(B, groups))
    if dy is None:
        return out
    if save8:
        q, _ = act8(x)
        xh, t, dt = at(torch.where(valid, torch.nan_to_num(q.reshape(x3.shape)) - mean, torch.zeros_like(z)))
    _, f1, f2 = act_fn(t, act)
    gy = keep(dy.detach().double().reshape(x3.shape))
    g = gy * f1
    dg = gy.abs() * (f2 * dt + (soft * (1 + t.abs()) * U) * (f1.abs() + (1 if soft else 0)) + U * f1.abs())
    h, dh = g * w, (dg + 2 * U * g.abs()) * w.abs()
    s1, s2 = h.sum((1, 3), keepdim=True) / M, (h * xh).sum((1, 3), keepdim=True) / M
    # (sums: 4 terms in float32 before they are added in 64 bits)
    ds1 = (dh + 4 * U * h.abs()).sum((1, 3), keepdim=True) / M
    ds2 = ((dh + 8 * U * h.abs()) * xh.abs()).sum((1, 3), keepdim=True) / M
    dx = keep((h - s1 - xh * s2) * rstd)
    tol = keep((dh + ds1 + xh.abs() * ds2 + 6 * U * (h.abs() + s1.abs() + (xh * s2).abs())) * rstd)
    out.update(dx=dx.reshape(x.shape), dx_tol=tol.reshape(x.shape),
               db=g.sum((0, 1)).reshape(C), db_tol=(dg + 5 * U * g.abs()).sum((0, 1)).reshape(C),
               dw=(g * xh).sum((0, 1)).reshape(C), dw_tol=((dg + 8 * U * g.abs()) * xh.abs()).sum((0, 1)).reshape(C))
    return out


def linear_act8(x, weight, bias, dy=None):
    """dict y, dx, dw, db with bounds.  A float32 sum of n products: at most n + 16 roundings, each of a step (2 U: a matrix
    instruction may cut instead of rounding) of a partial sum, which is at most the sum of the magnitudes."""
    K, N = x.shape[-1], weight.shape[0]
    x2, w = x.detach().double().reshape(-1, K), weight.detach().double()
    R = x2.shape[0]
    b = 0.0 if bias is None else bias.detach().double()
    y = x2 @ w.t() + b
    mag = x2.abs() @ w.abs().t() + (0.0 if bias is None else b.abs())
    out = dict(y=y.reshape(x.shape[:-1] + (N,)), y_tol=(2 * U * (K + 16) * mag).reshape(x.shape[:-1] + (N,)))
    if dy is None:
        return out
    g = dy.detach().double().reshape(-1, N)
    q, _ = act8(x2)
    out.update(dx=(g @ w).reshape(x.shape), dx_tol=(2 * U * (N + 16) * (g.abs() @ w.abs())).reshape(x.shape),
               dw=g.t() @ q, dw_tol=2 * U * (R + 16) * (g.abs().t() @ q.abs()),
               db=g.sum(0), db_tol=2 * U * (R + 16) * g.abs().sum(0))
    return out


def check(got, want, tol, name=""):
    """got (its type's rounding on top of the float32 bound) against want"""
    assert tuple(got.shape) == tuple(want.shape), (name, got.shape, want.shape)
    g = got.detach().cpu().double()
    lim = tol * 1.0001 + half_step(got.dtype) * (want.abs() + tol) + tiny(got.dtype)
    off = (g - want).abs()
    bad = ~(off <= lim)
    assert not bool(bad.any()), "%s: %d of %d outside; worst off %.3g allowed %.3g at value %.6g" % (
        name, int(bad.sum()), bad.numel(), float(off[bad][0]), float(lim[bad][0]), float(want[bad][0]))


def check_norm(got, want, n, name=""):
    """the rounding errors of n-term sums of random signs: 2^-23 sqrt(n) of the result, in the 2-norm (a lost piece of
    an operand shows here, where the worst case above is too wide), plus the type's half step"""
    d = (got.detach().cpu().double() - want).norm() / want.norm().clamp(min=1e-300)
    lim = half_step(got.dtype) + 2.0 ** -23 * math.sqrt(n + 16)
    assert float(d) <= lim, "%s: %.3g of the norm off, %.3g allowed" % (name, float(d), lim)
