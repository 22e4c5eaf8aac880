"""Measured cases of the batch-independent training layer: group normalisation with an activation on channels-last rows,
activation checkpoints in 8 bits, and the linear layer whose weight gradient is formed from such a checkpoint.

A case is a dict of plain values: `op` (act8 | group_norm | linear), `dtype`, sizes, and the options of the call.
`run` computes it in elementary torch operations, or through grid_gcn_amd.ops where `own` is true."""
import math

import torch

own = False

ACTS = ("none", "relu", "silu", "gelu")
BLOCK = 32                # channels that share one scale of the 8-bit form
MIN_EXP = -117            # smallest exponent of a scale: every value of the 8-bit form is a normal float32 / bfloat16
MAX_ROW_ELEMS = 81920 * 8 * 128


def listed():
    return [
        # the pooled descriptors in front of the classifier's fully connected layers: latency
        dict(name="act8 cls head", op="act8", dtype="float32", rows=32, c=512, pad=0),
        # gathered source rows of the last up layer: 8 clouds of 81920 points, 128 features + 3 coordinates
        dict(name="act8 seg points", op="act8", dtype="float32", rows=655360, c=131, pad=0),
        # one descriptor per cloud (as the fully connected layers see it): each sample is a single row
        dict(name="gn cls head", op="group_norm", dtype="float32", batch=32, rows=1, c=512, groups=32, act="relu", ragged=False,
             save8=False, grad=True, pad=0),
        # centres of the second down layer, counts as the index operator leaves them, the input kept in 8 bits
        dict(name="gn ragged centres", op="group_norm", dtype="float32", batch=16, rows=1024, c=128, groups=32, act="relu",
             ragged=True, save8=True, grad=True, pad=0),
        # per-point features of a segmentation step: the largest
        dict(name="gn seg points", op="group_norm", dtype="float32", batch=8, rows=81920, c=128, groups=32, act="silu", ragged=False,
             save8=False, grad=True, pad=0),
        # edges of the first down layer (1024 centres x 64 neighbours), half precision, the input kept in 8 bits
        dict(name="gn edges 8 bit", op="group_norm", dtype="bfloat16", batch=16, rows=65536, c=64, groups=8, act="gelu", ragged=False,
             save8=True, grad=True, pad=0),
        # evaluation of one small batch: forward alone
        dict(name="gn serve", op="group_norm", dtype="float16", batch=2, rows=1024, c=256, groups=16, act="relu", ragged=True,
             save8=False, grad=False, pad=0),
        # fully connected layer of the classifier: 32 rows
        dict(name="linear cls head", op="linear", dtype="float32", rows=32, k=512, n=256, bias=True, grad=True, pad=0),
        # centre MLP of an up layer on rows with coordinates in front (131 columns)
        dict(name="linear odd", op="linear", dtype="bfloat16", rows=81920, k=131, n=128, bias=True, grad=True, pad=0),
        # update MLP of the last up layer of a segmentation step: the largest
        dict(name="linear seg points", op="linear", dtype="float32", rows=655360, k=256, n=128, bias=True, grad=True, pad=0),
        # widest edge layer of the classifier: 128 centres x 64 neighbours of 32 clouds
        dict(name="linear cls edges", op="linear", dtype="bfloat16", rows=262144, k=256, n=512, bias=False, grad=True, pad=0),
        # class scores of a small served batch: forward alone
        dict(name="linear serve", op="linear", dtype="float16", rows=24, k=256, n=40, bias=True, grad=False, pad=0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("act8", "group_norm", "linear", "linear", "group_norm"))
    dtype = rng.choice(("float32", "bfloat16", "float16"))
    pad = rng.choice((0, 0, 0, 1, 8))           # columns of a wider buffer behind the row
    if op == "act8":
        c = _log_int(rng, 1, 1027)
        return dict(op=op, dtype=dtype, rows=_log_int(rng, 1, max(2, min(655360, MAX_ROW_ELEMS // (c + pad)))), c=c, pad=pad)
    if op == "group_norm":
        groups = rng.choice((1, 2, 3, 4, 8, 16, 32))
        c = groups * _log_int(rng, 1, 512 // groups)
        # (a group of one or two values has no gradient but rounding: at least four)
        rows = _log_int(rng, -(-4 * groups // c), 81920)
        batch = _log_int(rng, 1, max(1, min(32, MAX_ROW_ELEMS // (rows * (c + pad)))))
        return dict(op=op, dtype=dtype, batch=batch, rows=rows, c=c, groups=groups, act=rng.choice(ACTS),
                    ragged=rng.random() < 0.4, save8=rng.random() < 0.5, grad=rng.random() < 0.8, pad=pad)
    k, n = _log_int(rng, 3, 1027), _log_int(rng, 1, 512)
    most = 655360 * 256 * 128
    rows = _log_int(rng, 1, max(2, min(655360, most // (k * n), MAX_ROW_ELEMS // (k + pad), MAX_ROW_ELEMS // n)))
    return dict(op=op, dtype=dtype, rows=rows, k=k, n=n, bias=rng.random() < 0.7, grad=rng.random() < 0.8, pad=pad)


def _rows(gen, lead, c, pad, dtype, kind):
    """[*lead, c] values in a buffer of c + pad columns.  kind: 'pre' = pre-activations with a mean of their own per
    channel, 'act' = ReLU outputs (half of them zero), 'grad' = gradients of a mean loss over many rows"""
    dev = gen.device
    x = torch.randn(*lead, c + pad, generator=gen, device=dev)
    if kind == "pre":
        x *= torch.rand(c + pad, generator=gen, device=dev) + 0.5
        x += torch.randn(c + pad, generator=gen, device=dev) * 0.5
    elif kind == "act":
        x = x.clamp_(min=0)
    else:
        x *= 2.0 ** -7
    return x.to(dtype)[..., :c]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dt = getattr(torch, case["dtype"])
    s = dict(case=dict(case))
    if case["op"] == "act8":
        s["x"] = _rows(gen, (case["rows"],), case["c"], case["pad"], dt, "pre")
        return s
    if case["op"] == "group_norm":
        B, N, C = case["batch"], case["rows"], case["c"]
        s["x"] = _rows(gen, (B, N), C, case["pad"], dt, "pre")
        s["dy"] = _rows(gen, (B, N), C, 0, dt, "grad")
        # (parameters of a normalisation stay in 32 bits whatever the rows' type)
        s["weight"] = torch.rand(C, generator=gen, device=dev) + 0.5
        s["bias"] = torch.randn(C, generator=gen, device=dev) * 0.2
        s["counts"] = None
        if case["ragged"]:
            n = torch.randint(0, N + 1, (B, 1), generator=gen, device=dev, dtype=torch.int32)
            n[0] = N
            s["counts"] = n
        leaves = ("x", "weight", "bias")
    else:
        R, K, N = case["rows"], case["k"], case["n"]
        s["x"] = _rows(gen, (R,), K, case["pad"], dt, "act")
        s["dy"] = _rows(gen, (R,), N, 0, dt, "grad")
        s["weight"] = (torch.randn(N, K, generator=gen, device=dev) * (2.0 / (N + K)) ** 0.5).to(dt)
        s["bias"] = (torch.randn(N, generator=gen, device=dev) * 0.1).to(dt) if case["bias"] else None
        leaves = ("x", "weight", "bias")
    if case["grad"]:
        for name in leaves:
            if s[name] is not None:
                s[name] = s[name].detach().requires_grad_()
    return s


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _plain_round_trip(x):
    """the values that the 8-bit form of x [..., c] stands for, in 32 bits"""
    x = x.float()
    lead, c = x.shape[:-1], x.shape[-1]
    cp = -(-c // BLOCK) * BLOCK
    p = torch.zeros(*lead, cp, dtype=torch.float32, device=x.device)
    p[..., :c] = x
    p = p.reshape(*lead, cp // BLOCK, BLOCK)
    amax = p.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(amax)                              # amax = m 2^e, m in [0.5, 1): 448 = 0.875 * 2^9
    e = (e - 9 + (m > 0.875).to(e.dtype)).clamp_(min=MIN_EXP)
    e = torch.where(amax > 0, e, torch.full_like(e, MIN_EXP))
    # |x| / 2^e <= 448; e4m3: 3 fraction bits above 2^-6, steps of 2^-9 below
    q = torch.ldexp(p, -e).to(torch.float8_e4m3fn).float()
    return torch.ldexp(q, e).reshape(*lead, cp)[..., :c]


def _act(t, act):
    if act == "relu":
        return t.clamp(min=0)
    if act == "silu":
        return t / (1 + torch.exp(-t))
    if act == "gelu":
        return 0.5 * t * (1 + torch.erf(t * (0.5 ** 0.5)))
    return t


def _act_grad(t, act):
    if act == "relu":
        return (t > 0).to(t.dtype)
    if act == "silu":
        s = 1 / (1 + torch.exp(-t))
        return s * (1 + t * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(t * (0.5 ** 0.5))) + t * torch.exp(-0.5 * t * t) * (1 / math.sqrt(2 * math.pi))
    return torch.ones_like(t)


def _plain_group_norm(s, case, eps=1e-5):
    x, dt = s["x"].detach(), s["x"].dtype
    B, N, C = x.shape
    G = case["groups"]
    x32 = x.float()
    w, b = s["weight"].detach(), s["bias"].detach()
    if s["counts"] is None:
        valid, m = None, torch.full((B, 1, 1, 1), float(N * (C // G)), dtype=torch.float64, device=x.device)
    else:
        cnt = s["counts"].reshape(B, 1, 1).clamp(0, N)
        valid = torch.arange(N, device=x.device).reshape(1, N, 1) < cnt
        x32 = torch.where(valid, x32, torch.zeros_like(x32))
        m = (cnt.double() * (C // G)).clamp(min=1).reshape(B, 1, 1, 1)

    def per_group(v):                                      # [B, N, C] -> [B, 1, G, 1], summed in 64 bits
        return v.sum(1, dtype=torch.float64).reshape(B, 1, G, C // G).sum(-1, keepdim=True)

    def spread(v):                                         # [B, 1, G, 1] -> [B, 1, C]
        return v.expand(B, 1, G, C // G).reshape(B, 1, C)

    mean = spread(per_group(x32) / m)
    d = x32.double() - mean                                # (the sign of t decides a ReLU's gradient: 64 bits up to t)
    if valid is not None:
        d = torch.where(valid, d, torch.zeros_like(d))
    rstd = spread((per_group(d * d) / m + eps).rsqrt())

    def affine(v):
        xh = (v.double() - mean) * rstd
        return xh.float(), xh * w.double() + b.double()

    _, t = affine(x32)
    y = _act(t.float(), case["act"])
    if valid is not None:
        y = torch.where(valid, y, torch.zeros_like(y))
    if not case["grad"]:
        return [y.to(dt)]
    if case["save8"]:
        xh, t = affine(_plain_round_trip(x))
    else:
        xh, t = affine(x32)
    gate = _act_grad(t, "relu").float() if case["act"] == "relu" else _act_grad(t.float(), case["act"])
    g = s["dy"].float() * gate
    if valid is not None:
        g = torch.where(valid, g, torch.zeros_like(g))
        xh = torch.where(valid, xh, torch.zeros_like(xh))
    dbeta = g.sum((0, 1), dtype=torch.float64)
    dgamma = (g * xh).sum((0, 1), dtype=torch.float64)
    h = g * w
    s1, s2 = spread(per_group(h) / m).float(), spread(per_group(h * xh) / m).float()
    dx = (h - s1 - xh * s2) * rstd.float()
    if valid is not None:
        dx = torch.where(valid, dx, torch.zeros_like(dx))
    return [y.to(dt), dx.to(dt), dgamma.float(), dbeta.float()]


def _plain_linear(s, case):
    x, dt = s["x"].detach(), s["x"].dtype
    w = s["weight"].detach().float()
    y = x.float() @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].detach().float()
    if not case["grad"]:
        return [y.to(dt)]
    dy = s["dy"].float()
    out = [y.to(dt), (dy @ w).to(dt), (dy.t() @ _plain_round_trip(x)).to(dt)]
    if s["bias"] is not None:
        out.append(dy.sum(0, dtype=torch.float64).to(dt))
    return out


def run(state):
    case = state["case"]
    if own:
        from grid_gcn_amd import ops
        if case["op"] == "act8":
            codes, scales = ops.act8_pack(state["x"])
            return [ops.act8_unpack(codes, scales, case["c"], dtype=state["x"].dtype)]
        if case["op"] == "group_norm":
            y = ops.group_norm_act(state["x"], state["weight"], state["bias"], case["groups"], eps=1e-5, act=case["act"],
                                   counts=state["counts"], save8=case["save8"])
            leaves = [state["x"], state["weight"], state["bias"]]
        else:
            y = ops.linear_act8(state["x"], state["weight"], state["bias"])
            leaves = [state["x"], state["weight"]] + ([state["bias"]] if state["bias"] is not None else [])
        if not case["grad"]:
            return [y]
        return [y.detach(), *torch.autograd.grad(y, leaves, state["dy"])]
    if case["op"] == "act8":
        return [_plain_round_trip(state["x"]).to(state["x"].dtype)]
    if case["op"] == "group_norm":
        return _plain_group_norm(state, case)
    return _plain_linear(state, case)


def work(case):
    t = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "act8":
        n = case["rows"] * case["c"]
        return dict(bytes=n * 2 * t, flops=4 * n)
    if case["op"] == "group_norm":
        # x in, y out; a training step also dy in and dx out
        n = case["batch"] * case["rows"] * case["c"]
        return dict(bytes=n * t * (4 if case["grad"] else 2) + case["c"] * (16 if case["grad"] else 8), flops=n * (24 if case["grad"] else 8))
    r, k, n = case["rows"], case["k"], case["n"]
    times = 2 if case["grad"] else 1
    return dict(bytes=times * t * (r * k + r * n + n * k), flops=(6 if case["grad"] else 2) * r * k * n)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def _exact_values8(x):
    """x [..., c] rounded to the 8-bit form, from its definition: the smallest power of two 2^e (e >= MIN_EXP) with
    max |x| <= 448 * 2^e per block, then the nearest multiple of 2^(max(exponent, -6) - 3), ties to even"""
    x = x.detach().double()
    c = x.shape[-1]
    x = torch.nn.functional.pad(x, (0, -c % BLOCK)).unflatten(-1, (-1, BLOCK))
    top = x.abs().amax(-1, keepdim=True) / 448
    e = torch.where(top > 0, torch.ceil(torch.log2(top.clamp(min=2.0 ** -300))), torch.full_like(top, float(MIN_EXP)))
    e = torch.where(torch.exp2(e - 1) >= top, e - 1, e)          # (log2 may be off by one unit at a power of two)
    e = torch.where(torch.exp2(e) < top, e + 1, e).clamp(min=MIN_EXP)
    v = x / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))).clamp(min=-6) - 3)
    return (torch.round(v / step) * step * torch.exp2(e)).flatten(-2)[..., :c]


def _exact_group_norm(s, case, eps=1e-5):
    ys, dxs, dgs, dbs = [], [], [], []
    G, act = case["groups"], case["act"]
    w, b = s["weight"].detach().double(), s["bias"].detach().double()
    C = w.numel()
    for i in range(s["x"].shape[0]):
        N = s["x"].shape[1]
        n = N if s["counts"] is None else min(max(int(s["counts"][i]), 0), N)
        y = torch.zeros(N, C, dtype=torch.float64, device=w.device)
        dx = torch.zeros_like(y)
        dg, db = torch.zeros_like(w), torch.zeros_like(w)
        if n:
            x = s["x"][i, :n].detach().double()
            grp = x.reshape(n, G, C // G)
            mean = grp.mean((0, 2)).repeat_interleave(C // G)
            var = grp.var((0, 2), unbiased=False).repeat_interleave(C // G)
            sd = (var + eps).sqrt()
            y[:n] = _act(w * (x - mean) / sd + b, act)
            if case["grad"]:
                xh = ((_exact_values8(s["x"][i, :n]) if case["save8"] else x) - mean) / sd
                g = s["dy"][i, :n].double() * _act_grad(w * xh + b, act)
                dg, db = (g * xh).sum(0), g.sum(0)
                h = (g * w).reshape(n, G, C // G)
                m1 = h.mean((0, 2)).repeat_interleave(C // G)
                m2 = (h * xh.reshape(n, G, C // G)).mean((0, 2)).repeat_interleave(C // G)
                dx[:n] = (g * w - m1 - xh * m2) / sd
        ys.append(y), dxs.append(dx), dgs.append(dg), dbs.append(db)
    if not case["grad"]:
        return [torch.stack(ys)]
    return [torch.stack(ys), torch.stack(dxs), torch.stack(dgs).sum(0), torch.stack(dbs).sum(0)]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "act8":
        return [_exact_values8(s["x"])]
    if case["op"] == "group_norm":
        return _exact_group_norm(s, case)
    x, w = s["x"].detach().double(), s["weight"].detach().double()
    y = torch.matmul(x, w.t())
    if s["bias"] is not None:
        y += s["bias"].detach().double()
    if not case["grad"]:
        return [y]
    dy = s["dy"].double()
    out = [y, torch.matmul(dy, w), torch.matmul(dy.t(), _exact_values8(s["x"]))]
    return out + ([dy.sum(0)] if s["bias"] is not None else [])
