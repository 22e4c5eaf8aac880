"""CPU tier of the batch-independent training layer (grid_gcn_amd/act8.py): the product's kernels and host code under the
emulator (tests/simt) against float64 (oracle/act8_ref.py), the formulas against differences, and every refusal."""
import ctypes
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "simt"))

import act8_cases as cases  # noqa: E402
from oracle import act8_ref as ref  # noqa: E402
from simt import emu  # noqa: E402
from grid_gcn_amd import gridconv, ops  # noqa: E402


@pytest.fixture(autouse=True)
def _no_guesses():
    c0 = emu.counters()
    yield
    c1 = emu.counters()
    assert c1[2] == c0[2], "a cross-lane read took a lane outside the set executing the operation"
    assert c1[3] == c0[3], "a cross-lane operation was reached in divergent control flow"


def _same(got, want):
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


# ---- the 8-bit form --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("R,C,pad", cases.PACK)
def test_act8_round_trip(R, C, pad, dtype):
    x = cases.rows((R,), C, dtype, 1, pad)
    want, E = ref.act8(x)
    with emu.emulated_gpu():
        codes, scales = ops.act8_pack(x)
        back = ops.act8_unpack(codes, scales, C, dtype=dtype)
        wide = ops.act8_unpack(codes, scales, C)
    assert codes.shape == (R, -(-C // 32) * 32) and torch.equal(scales.int() - 127, E.int())
    assert torch.equal(codes[:, C:], torch.zeros_like(codes[:, C:]))
    _same(wide.double(), want)
    _same(back.double(), want)                        # (exact in the type that was packed)
    assert float(((want - x.double()).abs() - 2.0 ** -4 * x.double().abs()).max()) <= float((torch.exp2(E.double()) * 2.0 ** -10).max())


@pytest.mark.parametrize("dtype", cases.DTYPES)
def test_act8_special_values(dtype):
    x = cases.special_rows(dtype)
    want, E = ref.act8(x)
    with emu.emulated_gpu():
        codes, scales = ops.act8_pack(x)
        back = ops.act8_unpack(codes, scales, 32)
    assert torch.equal(scales.int() - 127, E.int())
    _same(back.double(), want.float().double())       # (what rounds to 2^128 is infinite as a float32)
    assert int(scales.min()) >= 10


def test_act8_keeps_leading_dimensions_and_empty():
    x = cases.rows((2, 3), 40, torch.float32, 2)
    with emu.emulated_gpu():
        codes, scales = ops.act8_pack(x)
        assert codes.shape == (2, 3, 64) and scales.shape == (2, 3, 2)
        assert ops.act8_unpack(codes, scales, 40).shape == (2, 3, 40)
        c, s = ops.act8_pack(x[:0])
        assert c.shape == (0, 3, 64) and ops.act8_unpack(c, s, 40, torch.float16).shape == (0, 3, 40)


# ---- group normalisation ---------------------------------------------------------------------------------------------
def run_gn(case, dtype, dev="cpu", ptype=torch.float32, seed=5):
    B, N, C, G, act, ragged, save8, pad = case
    x = cases.rows((B, N), C, dtype, seed, pad)
    dy = cases.rows((B, N), C, dtype, seed + 1, 0, "grad")
    w = (torch.rand(C, generator=torch.Generator().manual_seed(seed)) + 0.5).to(ptype)
    b = (torch.randn(C, generator=torch.Generator().manual_seed(seed + 7)) * 0.3).to(ptype)
    counts = None
    if ragged:
        counts = torch.tensor([[(0, N, max(1, N // 2), N + 3, -2)[i % 5]] for i in range(B)], dtype=torch.int32)
    want = ref.group_norm_act(x, w, b, G, 1e-5, act, counts, dy, save8)
    buf = x.as_strided((B, N, C + pad), (N * (C + pad), C + pad, 1)) if pad else x
    xd = buf.to(dev)[..., :C].detach().requires_grad_()
    wd, bd = w.to(dev).requires_grad_(), b.to(dev).requires_grad_()
    if ragged:         # what stands behind the last row is nobody's business
        n = counts.reshape(B).long().clamp(0, N)
        with torch.no_grad():
            for i in range(B):
                xd[i, int(n[i]):] = float("nan")
                dy[i, int(n[i]):] = float("nan")
    y = ops.group_norm_act(xd, wd, bd, G, act=act, counts=counts.to(dev) if ragged else None, save8=save8)
    dx, dw, db = torch.autograd.grad(y, (xd, wd, bd), dy.to(dev))
    return dict(y=y, dx=dx, dw=dw, db=db), want


def check_gn(got, want):
    for k in ("y", "dx", "dw", "db"):
        ref.check(got[k], want[k], want[k + "_tol"], k)


@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("case", cases.GN)
def test_group_norm_act(case, dtype):
    with emu.emulated_gpu():
        got, want = run_gn(case, dtype)
    check_gn(got, want)


def test_group_norm_act_parameters_of_the_rows_type():
    for dtype in (torch.bfloat16, torch.float16):
        with emu.emulated_gpu():
            got, want = run_gn(cases.GN[4], dtype, ptype=dtype)
        assert got["dw"].dtype == dtype
        check_gn(got, want)


def test_group_norm_act_without_parameters_2d_and_4d():
    x = cases.rows((6,), 40, torch.float32, 3)
    x4 = cases.rows((2, 3, 5), 12, torch.float32, 4)
    with emu.emulated_gpu():
        y = ops.group_norm_act(x, None, None, 4, act="none")
        y4 = ops.group_norm_act(x4, None, None, 3, act="relu")
    want = ref.group_norm_act(x[:, None], None, None, 4, 1e-5, "none")
    ref.check(y, want["y"][:, 0], want["y_tol"][:, 0])
    want = ref.group_norm_act(x4, None, None, 3, 1e-5, "relu")
    ref.check(y4, want["y"], want["y_tol"])


def test_group_norm_act_large_mean():
    """a mean of 1000 standard deviations: the variance and x - mean keep their digits"""
    x = cases.rows((2, 50), 16, torch.float32, 9) * 0.01 + 10.0
    with emu.emulated_gpu():
        y = ops.group_norm_act(x, None, None, 2, eps=0.0, act="none")
    want = ref.group_norm_act(x, None, None, 2, 0.0, "none")
    ref.check(y, want["y"], want["y_tol"])


def test_group_norm_relu_gate_at_the_border():
    """values that put t within the rounding of float32 on either side of 0: the gate is that of 64 bits"""
    B, N, C = 1, 64, 4
    x = cases.rows((B, N), C, torch.float32, 11)
    dy = torch.ones(B, N, C)
    st = ref.group_norm_act(x, None, None, 1, 1e-5, "none")
    w = torch.ones(C)
    # beta cancels one row's t to the last bit of float32, for every channel another row
    b = -torch.stack([st["y"][0, 5 * c + 1, c] for c in range(C)]).float()
    want = ref.group_norm_act(x, w, b, 1, 1e-5, "relu", None, dy)
    with emu.emulated_gpu():
        xr = x.clone().requires_grad_()
        wr, br = w.clone().requires_grad_(), b.clone().requires_grad_()
        y = ops.group_norm_act(xr, wr, br, 1, act="relu")
        dx, dw, db = torch.autograd.grad(y, (xr, wr, br), dy)
    assert torch.equal(db.double(), want["db"])       # (a count of open gates)
    ref.check(dx, want["dx"], want["dx_tol"])


def run_gate_of_any_gain(dtype, N, save8, dev="cpu"):
    """gains of either sign, none, tiny and huge; shifts that put the border among the values, at them, and beyond them"""
    C = 32
    x = cases.rows((2, N), C, dtype, 12)
    dy = cases.rows((2, N), C, dtype, 13, kind="grad")
    w = torch.tensor([1.0, -1.0, 0.0, 0.0, 1e-30, -1e-30, 1e30, -1e30] * 4)
    b = torch.tensor([0.3, 0.3, 0.5, -0.5, 1e-30, 1e-30, 0.0, 0.0] * 2 + [0.0] * 8 + [1e30, 1e30, 0.0, 1e-40, 1.0, -1.0, 1e30, -1e30])
    want = ref.group_norm_act(x, w, b, 4, 1e-5, "relu", None, dy, save8)
    t = [v.to(dev).requires_grad_() for v in (x, w, b)]
    dx, dw, db = torch.autograd.grad(ops.group_norm_act(*t, 4, act="relu", save8=save8), t, dy.to(dev))
    ref.check(db, want["db"], want["db_tol"], "db")
    ref.check(dw, want["dw"], want["dw_tol"], "dw")
    # what lies past the type's largest number by more than its bound and a step is infinite in it (float16 and a gain of 1e30)
    lim = torch.finfo(dtype).max * (1 + torch.finfo(dtype).eps)
    past = want["dx"].abs() - want["dx_tol"] > lim
    got = dx.detach().cpu()
    assert torch.equal(got[past].double(), want["dx"][past].sign() * float("inf"))
    # (and may be where only its bound reaches past that)
    keep = ~past & ~(got.isinf() & (want["dx"].abs() + want["dx_tol"] > lim))
    ref.check(got[keep], want["dx"][keep], (want["dx_tol"] + torch.zeros_like(want["dx"]))[keep], "dx")


@pytest.mark.parametrize("save8", [False, True])
@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("N", [40, 600])
def test_group_norm_relu_gate_of_any_gain(N, dtype, save8):
    with emu.emulated_gpu():
        run_gate_of_any_gain(dtype, N, save8)


@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
def test_group_norm_formula_against_differences(act):
    """the oracle's gradients are the derivatives of its forward"""
    torch.manual_seed(0)
    x, dy = torch.randn(2, 6, 8, dtype=torch.float64), torch.randn(2, 6, 8, dtype=torch.float64)
    w, b = torch.rand(8, dtype=torch.float64) + 0.5, torch.randn(8, dtype=torch.float64)
    counts = torch.tensor([[4], [6]], dtype=torch.int32)
    f = lambda x, w, b: (ref.group_norm_act(x, w, b, 2, 1e-3, act, counts)["y"] * dy).sum()      # noqa: E731
    g = ref.group_norm_act(x, w, b, 2, 1e-3, act, counts, dy)
    h = 1e-6
    for name, t, put in (("dx", x, lambda v: f(v, w, b)), ("dw", w, lambda v: f(x, v, b)), ("db", b, lambda v: f(x, w, v))):
        for _ in range(3):
            u = torch.randn_like(t)
            num = float((put(t + h * u) - put(t - h * u)) / (2 * h))
            # (central differences of h = 1e-6: truncation h^2, rounding 2^-53 * |f| / h ~ 1e-9)
            assert abs(num - float((g[name] * u).sum())) < 1e-6 * (1 + abs(num))


def test_group_norm_only_some_gradients():
    x, dy = cases.rows((2, 50), 32, torch.float32, 3), cases.rows((2, 50), 32, torch.float32, 4)
    full = ref.group_norm_act(x, torch.ones(32), torch.zeros(32), 4, 1e-5, "silu", None, dy)
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1)):
        with emu.emulated_gpu():
            t = [x.clone(), torch.ones(32), torch.zeros(32)]
            for v, n in zip(t, need):
                v.requires_grad_(bool(n))
            ops.group_norm_act(*t, 4, act="silu").backward(dy)
        for v, n, k in zip(t, need, ("dx", "dw", "db")):
            assert (v.grad is not None) == bool(n)
            if n:
                ref.check(v.grad, full[k], full[k + "_tol"], k)


# ---- linear ----------------------------------------------------------------------------------------------------------
def run_linear(case, dtype, dev="cpu", seed=6, strided_dy=False):
    R, K, N, bias, pad = case
    x = cases.rows((R,), K, dtype, seed, pad, "act")
    dy = cases.rows((R,), N, dtype, seed + 1, 3 if strided_dy else 0, "grad")
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(N, K, generator=g) * (2.0 / (N + K)) ** 0.5).to(dtype)
    b = (torch.randn(N, generator=g) * 0.1).to(dtype) if bias else None
    want = ref.linear_act8(x, w, b, dy)
    buf = x.as_strided((R, K + pad), (K + pad, 1)) if pad else x
    xd = buf.to(dev)[..., :K].detach().requires_grad_()
    leaves = [xd, w.to(dev).requires_grad_()] + ([b.to(dev).requires_grad_()] if bias else [])
    y = ops.linear_act8(*leaves)
    dyd = dy.as_strided((R, N + 3), (N + 3, 1)).to(dev)[:, :N] if strided_dy else dy.to(dev)
    grads = torch.autograd.grad(y, leaves, dyd)
    return dict(zip(("y", "dx", "dw", "db"), (y,) + grads)), want


def check_linear(got, want, case):
    R, K, N = case[:3]
    for k, n in (("y", K), ("dx", N), ("dw", R), ("db", R)):
        if k in got:
            ref.check(got[k], want[k], want[k + "_tol"], k)
            if k != "db" and got[k].numel() >= 1024:
                ref.check_norm(got[k], want[k], n, k)


@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("case", cases.LINEAR)
def test_linear_act8(case, dtype):
    with emu.emulated_gpu():
        got, want = run_linear(case, dtype, strided_dy=case[0] % 2 == 1)
    check_linear(got, want, case)


def check_codes(R, K, dtype, dev="cpu"):
    """the 8-bit form that the linear layer writes is act8_pack's, special values among the rows"""
    from grid_gcn_amd import act8
    sp = cases.special_rows(dtype)
    x = cases.rows((R,), K, dtype, 3)
    rep = sp.repeat(1, -(-K // 32))[:, :K]
    x[::max(1, R // len(rep))][:len(rep)] = rep[:len(x[::max(1, R // len(rep))])]
    x = x.to(dev)
    w = torch.zeros(3, K, dtype=dtype, device=dev)
    _, codes, scales = act8._linear_forward(x, w, None, True)
    c, s = ops.act8_pack(x)
    assert torch.equal(scales, s)
    assert torch.equal(codes & 0x7f, c & 0x7f)                    # (a NaN has no sign)
    ok = (c & 0x7f) != 0x7f
    assert torch.equal(codes[ok], c[ok])


@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("R,K", [(40, 70), (90, 128)])
def test_linear_act8_writes_the_same_codes(R, K, dtype):
    with emu.emulated_gpu():
        check_codes(R, K, dtype)


def growing_rows(R, K, seed):
    """rows whose magnitude grows along them by 2^40, starts with zeros, falls off, or is far from 1 as a whole"""
    x = cases.rows((R,), K, torch.float32, seed)
    k = torch.arange(K) / K
    x[0::5] *= torch.exp2(40 * k)
    x[1::5, :K // 2] = 0
    x[2::5] *= torch.exp2(-40 * k)
    x[3::5] *= 2.0 ** -90
    return x


def run_scales(dev="cpu"):
    x, w, dy = growing_rows(260, 72, 3), cases.rows((5600,), 72, torch.float32, 4), growing_rows(260, 5600, 5)
    w[::3] *= 2.0 ** 20
    w[1::3] *= 2.0 ** -30
    xd, wd = x.to(dev).requires_grad_(), w.to(dev)
    y = ops.linear_act8(xd, wd)
    dx, = torch.autograd.grad(y, xd, dy.to(dev))
    want = ref.linear_act8(x, w, None, dy)
    # on top of the float32 bound: what an fp16 pair drops below 2^-33 of the largest value of its row (of x, dy; 448 2^e) or column
    # (of W), against the largest of the other operand
    def dropped(a, b):
        return 2.0 ** -32 * (a.double().abs().amax(1, keepdim=True) * b.double().abs().sum(0) + a.double().abs().sum(1, keepdim=True) * b.double().abs().amax(0))
    ref.check(y, want["y"], want["y_tol"] + dropped(x, w.t()), "y")
    ref.check(dx, want["dx"], want["dx_tol"] + dropped(dy, w), "dx")


def test_linear_act8_rows_and_columns_of_every_scale():
    with emu.emulated_gpu():
        run_scales()


def test_linear_act8_only_some_gradients_and_expanded_dy():
    x, w, b = cases.rows((20,), 40, torch.float32, 3), cases.rows((9,), 40, torch.float32, 4), torch.zeros(9)
    dy = torch.ones(20, 9)
    full = ref.linear_act8(x, w, b, dy)
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1)):
        with emu.emulated_gpu():
            t = [x.clone(), w.clone(), b.clone()]
            for v, n in zip(t, need):
                v.requires_grad_(bool(n))
            ops.linear_act8(*t).sum().backward()          # (the gradient of a sum: one value, expanded)
        for v, n, k in zip(t, need, ("dx", "dw", "db")):
            assert (v.grad is not None) == bool(n)
            if n:
                ref.check(v.grad, full[k], full[k + "_tol"], k)


def test_linear_act8_non_finite_rows_stay_rows():
    x, w = cases.rows((40,), 64, torch.float32, 3), cases.rows((32,), 64, torch.float32, 4)
    x[7, 3] = float("nan")
    with emu.emulated_gpu():
        y = ops.linear_act8(x, w)
    assert bool(torch.isnan(y[7]).all()) and bool(torch.isfinite(y[:7]).all()) and bool(torch.isfinite(y[8:]).all())


def test_empty_inputs():
    with emu.emulated_gpu():
        x = torch.zeros(0, 5, 8).requires_grad_()
        w = torch.ones(8).requires_grad_()
        ops.group_norm_act(x, w, w, 2).sum().backward()
        assert x.grad.shape == (0, 5, 8) and float(w.grad.abs().sum()) == 0
        x = torch.zeros(0, 8).requires_grad_()
        w = torch.ones(3, 8).requires_grad_()
        y = ops.linear_act8(x, w)
        assert y.shape == (0, 3)
        y.sum().backward()
        assert float(w.grad.abs().sum()) == 0


# ---- together --------------------------------------------------------------------------------------------------------
def run_layers(net, x, dy, dev="cpu"):
    """the ConvGNAct layers of `net` as calls of the operators; every tensor between them with its gradient, checked layer by
    layer against float64 on the very values and upstream gradients that the kernels saw"""
    y = x.to(dev).requires_grad_()
    seen = []
    for l in net:
        z = ops.linear_act8(y, l.lin.weight, l.lin.bias)
        o = ops.group_norm_act(z, l.norm.weight, l.norm.bias, l.norm.num_groups, eps=l.norm.eps, act=l.act, save8=True)
        for t in (y, z, o):
            t.retain_grad()
        seen.append((l, y, z, o))
        y = o
    params = list(net.parameters())
    for p in params:
        p.grad = None
    y.backward(dy.to(dev))
    c = lambda t: t.detach().cpu()                               # noqa: E731
    for l, y_in, z, o in seen:
        w = ref.group_norm_act(c(z), c(l.norm.weight), c(l.norm.bias), l.norm.num_groups, l.norm.eps, l.act, None, c(o.grad), True)
        check_gn(dict(y=o, dx=z.grad, dw=l.norm.weight.grad, db=l.norm.bias.grad), w)
        w = ref.linear_act8(c(y_in), c(l.lin.weight), c(l.lin.bias), c(z.grad))
        got = dict(y=z, dx=y_in.grad, dw=l.lin.weight.grad, db=l.lin.bias.grad)
        for k in got:
            ref.check(got[k], w[k], w[k + "_tol"], k)
    return y.detach(), [p.grad.clone() for p in params]


def test_layers_in_a_row_train():
    torch.manual_seed(1)
    net = gridconv.mlp(13, [32, 48, 16], norm="group")
    x, dy = torch.randn(2, 70, 13), torch.randn(2, 70, 16)
    with emu.emulated_gpu():
        y, grads = run_layers(net, x, dy)
        y2 = gridconv.run_mlp(list(net), x)
        grads2 = torch.autograd.grad(y2, list(net.parameters()), dy)
    assert torch.equal(y, y2)                                     # (the same calls: the same bits)
    assert all(torch.equal(a, b) for a, b in zip(grads, grads2))
    # forward: nothing is in 8 bits, the stock module differs by float32 roundings alone (a dozen per value and layer, each
    # worth at most 2^-20 of the norm)
    with torch.no_grad():
        want = net(x)
    assert float((y - want).norm() / want.norm()) < 36 * 2.0 ** -20


def test_conv_gn_act_counts_on_the_cpu_and_the_kernels():
    torch.manual_seed(2)
    l = gridconv.ConvGNAct(6, 24, act="silu")
    x = torch.randn(3, 11, 6)
    counts = torch.tensor([[11], [0], [5]], dtype=torch.int32)
    x[2, 5:] = float("nan")
    want = l(x, counts)
    with emu.emulated_gpu():
        got = l(x, counts)
    assert float((got - want).abs().max()) < 1e-5 and float(got[2, 5:].abs().max()) == 0 and float(got[1].abs().max()) == 0


def test_segmentation_net_with_group_norm():
    """GGCNSeg with cfg['norm'] = 'group' steps through its own host code; gradients reach every parameter"""
    from grid_gcn_amd import model, synth
    import copy
    cfg = copy.deepcopy(model.SEG_8192)
    cfg["norm"] = "group"
    for lv, (P, O) in zip(cfg["grid"]["down"], ((8, 24), (4, 12), (4, 6))):
        lv["max_p_grid"], lv["max_o_grid"] = P, O
    for lv, O in zip(cfg["grid"]["up"], (12, 24, 64)):
        lv["max_o_grid"] = O
    cfg.update(pt_ele_dim=[[16, 32]] + [[32, 32]] * 2, inputDim=[0, 32, 32], up_inputDim=[32] * 3, up_center_dim=[[32]] * 3,
               up_pt_ele_dim=[[32]] * 3, up_gcn_outDim=[[32]] * 3)
    torch.manual_seed(0)
    net = model.GGCNSeg(cfg).train()
    data, npn = synth.make_batch(1, 64, "planes")
    with emu.emulated_gpu():
        out = net(torch.from_numpy(data[..., :3].copy()), torch.from_numpy(npn))
        loss = model.seg_loss(out, torch.randint(1, 21, (1, 64)))
        loss.backward()
        assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in net.parameters())
        net.eval()
        with torch.no_grad():
            assert net(torch.from_numpy(data[..., :3].copy()), torch.from_numpy(npn)).shape == out.shape


# ---- refusals --------------------------------------------------------------------------------------------------------
def test_refusals():
    x, w, b = torch.zeros(2, 3, 8), torch.ones(8), torch.zeros(8)
    gn, lin = ops.group_norm_act, ops.linear_act8
    for call in (lambda: gn(x, w, b, 2), lambda: lin(x, torch.zeros(4, 8)), lambda: ops.act8_pack(x),
                 lambda: ops.act8_unpack(torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(2, 1, dtype=torch.uint8), 8)):
        with pytest.raises(RuntimeError):                       # CPU tensors: there is no CPU path
            call()
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)          # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)         # noqa: E731
    bad = [
        lambda: gn(x.double(), w, b, 2), lambda: gn(x, w, b, 3), lambda: gn(x, w, b, 0), lambda: gn(x, w, b, 16),
        lambda: gn(x, w, b, 2, act="tanh"), lambda: gn(x, w, b, 2, eps=-1.0), lambda: gn(x, w, b, 2, eps=float("nan")),
        lambda: gn(x, w[:7], b, 2), lambda: gn(x, w, b.double(), 2), lambda: gn(x, w.half(), b, 2),
        lambda: gn(x.half(), w.bfloat16(), b.bfloat16(), 2), lambda: gn(torch.zeros(8), w, b, 2),
        lambda: gn(x, w, b, 2, counts=i32(3)), lambda: gn(x, w, b, 2, counts=torch.zeros(2)),
        lambda: gn(x[:, None], w, b, 2, counts=i32(2)), lambda: gn(x, w, b, 2, counts=i32(2, 2)[:, 0]),
        lambda: gn(torch.zeros(1, 1, 8200), None, None, 1), lambda: gn(torch.zeros(65536, 1, 2), None, None, 1),
        lambda: lin(x, torch.zeros(4, 7)), lambda: lin(x, torch.zeros(8)), lambda: lin(x, torch.zeros(4, 8).half()),
        lambda: lin(x, torch.zeros(4, 8), torch.zeros(5)), lambda: lin(x, torch.zeros(4, 8), torch.zeros(4).half()),
        lambda: lin(x.int(), torch.zeros(4, 8).int()), lambda: lin(x, torch.zeros(0, 8)),
        lambda: ops.act8_pack(x.double()), lambda: ops.act8_pack(torch.zeros(1, 70000)),
        lambda: ops.act8_unpack(u8(2, 32), u8(2, 2), 8), lambda: ops.act8_unpack(u8(2, 64), u8(2, 2), 8),
        lambda: ops.act8_unpack(u8(2, 32), u8(3, 1), 8), lambda: ops.act8_unpack(u8(2, 33)[:, :32], u8(2, 1), 8),
        lambda: ops.act8_unpack(u8(2, 32), u8(2, 1), 8, dtype=torch.float64), lambda: ops.act8_unpack(u8(2, 32).int(), u8(2, 1), 8),
        lambda: ops.act8_unpack(u8(2, 32), u8(2, 1), 0), lambda: ops.act8_unpack(u8(40)[8:40].view(1, 32), u8(1, 1), 8),
    ]
    for i, call in enumerate(bad):
        with emu.emulated_gpu(poison=False):
            with pytest.raises(RuntimeError):
                call()
                print("accepted:", i)


def test_c_entries_refuse_without_a_launch():
    from grid_gcn_amd import _lib, build
    build.build()
    lib = _lib.load()
    a = ctypes.cast((ctypes.c_float * 256)(), ctypes.c_void_p).value
    a = (a + 15) & ~15
    n = ctypes.c_size_t(0)
    EINVAL, EWS = 1, 2
    assert lib.gridgcn_act8_pack(None, 0, 1, 8, 8, a, a, None) == EINVAL
    assert lib.gridgcn_act8_pack(a, 3, 1, 8, 8, a, a, None) == EINVAL
    assert lib.gridgcn_act8_pack(a, 0, 1, 8, 7, a, a, None) == EINVAL
    assert lib.gridgcn_act8_pack(a, 0, 1, 8, 8, a + 4, a, None) == EINVAL
    assert lib.gridgcn_act8_unpack(a, a, 0, 8, 0, a, 8, None) == EINVAL
    assert lib.gridgcn_group_norm_act_workspace_bytes(2, 10, 9, 2, 0, 0, 0, 0, ctypes.byref(n)) == EINVAL
    size = lambda N, back: (lib.gridgcn_group_norm_act_workspace_bytes(2, N, 8, 2, 0, 1, 0, back, ctypes.byref(n)), n.value)[1]   # noqa: E731
    assert size(10, 0) == 0 and size(100000, 0) > 0 and size(10, 1) > 0 and size(100000, 1) > 0
    fwd = lambda **k: lib.gridgcn_group_norm_act_fwd(                                        # noqa: E731
        k.get("x", a), k.get("dt", 0), 2, 100000, 8, 800000, k.get("ldn", 8), k.get("G", 2), a, a, 0, None, k.get("eps", 1e-5),
        k.get("act", 1), a, None, k.get("codes"), k.get("scales"), k.get("ws", a), k.get("nb", 0), None)
    assert fwd() == EWS and fwd(ws=None, nb=1 << 20) == EWS
    for kw in (dict(x=None), dict(dt=7), dict(ldn=7), dict(G=3), dict(eps=-1.0), dict(act=4), dict(codes=a)):
        assert fwd(**kw) == EINVAL, kw
    bwd = lambda **k: lib.gridgcn_group_norm_act_bwd(                                        # noqa: E731
        a, 80, k.get("ldgn", 8), k.get("x", a), 80, 8, k.get("codes"), None, 0, 2, 10, 8, 2, k.get("st", a), a, a, 0, None, 1,
        a, a, a, a, 0, None)
    assert bwd() == EWS
    for kw in (dict(x=None), dict(codes=a), dict(st=None), dict(ldgn=3)):
        assert bwd(**kw) == EINVAL, kw
    assert lib.gridgcn_linear_act8_fwd(a, 0, 4, 8, 8, None, None, 4, a, None, None, None, 0, None) == EINVAL
    assert lib.gridgcn_linear_act8_fwd(a, 0, 4, 8, 8, a, None, 4, a, a, None, None, 0, None) == EINVAL
    assert lib.gridgcn_linear_act8_fwd(a, 0, 4, 8, 4, a, None, 4, a, None, None, None, 0, None) == EINVAL
    assert lib.gridgcn_linear_act8_fwd(a, 0, 1 << 20, 8, 8, a, None, 4, a, None, None, None, 0, None) == EWS
    assert lib.gridgcn_linear_act8_workspace_bytes(0, 8, 4, 0, 0, ctypes.byref(n)) == EINVAL
    assert lib.gridgcn_linear_act8_workspace_bytes(1, 8, 4, 5, 0, ctypes.byref(n)) == EINVAL
    assert lib.gridgcn_linear_act8_bwd(a, 0, 4, 4, 4, None, 8, a, a, a, a, a, a, 256, None) == EINVAL
    assert lib.gridgcn_linear_act8_bwd(a, 0, 4, 4, 4, a, 8, None, None, a, a, a, a, 256, None) == EINVAL
    assert lib.gridgcn_linear_act8_bwd(a, 0, 1 << 20, 4, 4, a, 8, a, a, None, a, None, a, 256, None) == EWS
    assert lib.gridgcn_linear_act8_fwd(a, 0, 4, 8, (1 << 24) + 1, a, None, 4, a, None, None, None, 0, None) == EINVAL


def test_torch_ops_trace_on_fake_tensors():
    import grid_gcn_amd  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty((2, 100, 33), device="cuda", dtype=torch.bfloat16)
        w = torch.empty(33, device="cuda")
        y, st, codes, scales = torch.ops.gridgcn.group_norm_act(x, w, w, 3, act="silu", save8=True)
        assert y.shape == x.shape and st.shape == (2, 3, 2) and codes.shape == (200, 64) and scales.shape == (200, 2)
        y, codes, scales = torch.ops.gridgcn.linear_act8(x, torch.empty((7, 33), device="cuda", dtype=torch.bfloat16))
        assert y.shape == (2, 100, 7) and codes.shape == (200, 64)
        codes, scales = torch.ops.gridgcn.act8_pack(x)
        assert codes.shape == (2, 100, 64) and scales.shape == (2, 100, 2)
        assert torch.ops.gridgcn.act8_unpack(codes, scales, 33, torch.float16).shape == (2, 100, 33)
