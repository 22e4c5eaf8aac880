"""CPU tier: values of extreme magnitude, and calls off the usual path, of the batch-independent training layer
(grid_gcn_amd/act8.py).  The functions that tests/test_gpu_act8_range.py runs on an MI355X take the device as `dev`."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "simt"))

import act8_cases as cases  # noqa: E402
import test_act8 as base  # noqa: E402
from oracle import act8_ref as ref  # noqa: E402
from simt import emu  # noqa: E402
from grid_gcn_amd import gridconv, model, ops, synth  # noqa: E402


# ---- float32 products: the bound is that of a float32 sum of |x| |w|, whatever the range of a row or a column -----------
def wide(R):
    """columns: enough workgroups for the kernel of many rows where R goes there"""
    return 5600 if R > 128 else 40


def run_wide_rows(R, dev="cpu"):
    """a value of each row far above the others, against a weight of zero: what is left is the sum of the others"""
    K, N = 64, wide(R)
    x, w = cases.rows((R,), K, torch.float32, 3), cases.rows((N,), K, torch.float32, 4)
    x[:, 0] = torch.exp2(torch.arange(R) % 100 - 20.0)
    w[:, 0] = 0
    dy = cases.rows((R,), N, torch.float32, 5, kind="grad")
    dy[:, 7] = torch.exp2(torch.arange(R) % 100 - 20.0)
    w[7] = 0
    xd, wd = x.to(dev).requires_grad_(), w.to(dev)
    y = ops.linear_act8(xd, wd)
    dx, = torch.autograd.grad(y, xd, dy.to(dev))
    want = ref.linear_act8(x, w, None, dy)
    ref.check(y, want["y"], want["y_tol"], "y")
    ref.check(dx, want["dx"], want["dx_tol"], "dx")
    dy[:, 7] = 0
    ref.check_norm(y, want["y"], K, "y")
    ref.check_norm(dx, want["dx"], N, "dx")


def run_every_scale(R, dev="cpu"):
    """rows that grow by 2^40, fall off, start with zeros or lie far from 1; columns of three scales"""
    x, w, dy = base.growing_rows(R, 72, 3), cases.rows((wide(R),), 72, torch.float32, 4), base.growing_rows(R, wide(R), 5)
    w[::3] *= 2.0 ** 20
    w[1::3] *= 2.0 ** -30
    w[:, ::5] *= 2.0 ** -25
    xd, wd = x.to(dev).requires_grad_(), w.to(dev)
    y = ops.linear_act8(xd, wd)
    dx, = torch.autograd.grad(y, xd, dy.to(dev))
    want = ref.linear_act8(x, w, None, dy)
    ref.check(y, want["y"], want["y_tol"], "y")
    ref.check(dx, want["dx"], want["dx_tol"], "dx")


@pytest.mark.parametrize("R", [100, 260])                 # the kernel of few rows, and that of many
def test_linear_act8_wide_rows(R):
    with emu.emulated_gpu():
        run_wide_rows(R)


@pytest.mark.parametrize("R", [100, 260])
def test_linear_act8_rows_of_every_scale(R):
    with emu.emulated_gpu():
        run_every_scale(R)


def run_tiny(R, dev="cpu"):
    """values whose lower pieces are subnormal bf16 numbers, against weights that bring the products back: what lies below
    2^-134 (half of the smallest bf16 number) of a value may be gone"""
    x, w = cases.rows((R,), 72, torch.float32, 3), cases.rows((wide(R),), 72, torch.float32, 4)
    x[0::3] *= 2.0 ** -112
    x[1::3] *= 2.0 ** -121
    w = w * 2.0 ** 100
    with torch.no_grad():
        y = ops.linear_act8(x.to(dev), w.to(dev))
    want = ref.linear_act8(x, w, None)
    ref.check(y, want["y"], want["y_tol"] + 2.0 ** -134 * w.double().abs().sum(1), "y")


@pytest.mark.parametrize("R", [100, 260])
def test_linear_act8_tiny_values(R):
    with emu.emulated_gpu():
        run_tiny(R)


def run_same_row_in_any_company(dev="cpu"):
    """a row's result does not tell how many rows the call had, beyond the rounding of its sum"""
    x, w = base.growing_rows(260, 72, 3), cases.rows((5600,), 72, torch.float32, 4)
    with torch.no_grad():
        many = ops.linear_act8(x.to(dev), w.to(dev)).cpu()[:40].double()
        few = ops.linear_act8(x[:40].to(dev), w.to(dev)).cpu().double()
    tol = ref.linear_act8(x[:40], w, None)["y_tol"]
    assert bool(((many - few).abs() <= 2 * tol).all())


def test_linear_act8_same_row_in_any_company():
    with emu.emulated_gpu():
        run_same_row_in_any_company()


# ---- the top of float16: a magnitude of 63488 or more becomes 65536 in the 8-bit form -----------------------------------
def run_float16_top(dev="cpu"):
    """one large activation, alone in its column: dW is dy times its 8-bit value, a finite number"""
    x = torch.zeros(40, 40, dtype=torch.float16)
    x[3, 5] = 65000.0
    dy = cases.rows((40,), 4, torch.float16, 8, kind="grad")
    dy[3] = torch.tensor([2.0 ** -10, 0.0, 0.0, 0.0])
    w = torch.zeros(4, 40, dtype=torch.float16, device=dev, requires_grad=True)
    dw, = torch.autograd.grad(ops.linear_act8(x.to(dev), w), w, dy.to(dev))
    want = torch.zeros(4, 40)
    want[0, 5] = 64.0
    assert torch.equal(dw.cpu().float(), want)


def run_float16_magnitudes(dev="cpu"):
    """rows of every magnitude that float16 has, next to one another: row n of dW is the 8-bit value of row n of x times a power of two"""
    k = torch.arange(-24, 16)
    x = torch.exp2(k.double())[:, None] * torch.cat([torch.linspace(-1.99, 1.99, 47, dtype=torch.float64), torch.ones(1, dtype=torch.float64)])
    top = torch.finfo(torch.float16).max
    x = torch.cat([x, x.flip(0), torch.linspace(-top, top, 48, dtype=torch.float64)[None], torch.full((1, 48), -top, dtype=torch.float64)])
    x = x.clamp(-top, top).half()
    R = x.shape[0]
    gain = torch.where(x.float().abs().amax(1) > 1000, 2.0 ** -4, 1.0)
    dy = torch.diag(gain).half()
    w = torch.zeros(R, 48, dtype=torch.float16, device=dev, requires_grad=True)
    dw, = torch.autograd.grad(ops.linear_act8(x.to(dev), w), w, dy.to(dev))
    want = ref.act8(x)[0] * gain.double()[:, None]
    assert float(want.abs().max()) == 4096.0
    # (the value times the gain is within float16 but for what it has below 2^-24)
    ref.check(dw, want, torch.zeros_like(want), "dw")


def test_linear_act8_float16_top():
    with emu.emulated_gpu():
        run_float16_top()


def test_linear_act8_float16_magnitudes():
    with emu.emulated_gpu():
        run_float16_magnitudes()


# ---- group normalisation: standard deviations far from 1 ---------------------------------------------------------------
GN_SCALES = [(2.0 ** 77, 0.0), (2.0 ** 115, 1e-5), (2.0 ** -80, 0.0), (2.0 ** -100, 0.0)]


def run_gn_scale(scale, eps, N, act, dtype, save8, dev="cpu", dy_scale=1.0):
    C, G = 32, 4
    x = (cases.rows((2, N), C, torch.float32, 21) * scale).to(dtype)
    dy = (cases.rows((2, N), C, torch.float32, 22, kind="grad") * dy_scale).to(dtype)
    w = torch.rand(C, generator=torch.Generator().manual_seed(3)) + 0.5
    b = torch.randn(C, generator=torch.Generator().manual_seed(4)) * 0.3
    want = ref.group_norm_act(x, w, b, G, eps, act, None, dy, save8)
    t = [v.to(dev).requires_grad_() for v in (x, w, b)]
    y = ops.group_norm_act(*t, G, eps=eps, act=act, save8=save8)
    dx, dw, db = torch.autograd.grad(y, t, dy.to(dev))
    base.check_gn(dict(y=y, dx=dx, dw=dw, db=db), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,act,save8", [(40, "relu", False), (40, "silu", True), (2300, "gelu", False), (2300, "relu", True)])
@pytest.mark.parametrize("scale,eps", GN_SCALES)
def test_group_norm_act_far_from_one(scale, eps, N, act, save8, dtype):
    with emu.emulated_gpu():
        run_gn_scale(scale, eps, N, act, dtype, save8)


@pytest.mark.parametrize("N", [40, 2300])
def test_group_norm_act_small_values_and_gradients(N):
    with emu.emulated_gpu():
        run_gn_scale(2.0 ** -70, 0.0, N, "silu", torch.float32, False, dy_scale=2.0 ** -70)


# ---- counts through the framework's own layers ---------------------------------------------------------------------------
def run_padded_layers(dev="cpu"):
    """what pads a cloud changes nothing of its own results: rows of centres, and edges of centres"""
    torch.manual_seed(4)
    net = gridconv.mlp(10, [24, 32], norm="group").to(dev)
    for shape in ((1, 100, 10), (1, 30, 5, 10)):
        x = torch.randn(shape)
        pad = torch.cat([x, torch.zeros((1, 50) + shape[2:])], 1)
        both = torch.cat([pad, torch.randn(pad.shape)]).to(dev)
        n = torch.tensor([[shape[1]], [both.shape[1]]], dtype=torch.int32, device=dev)
        alone = gridconv.run_mlp(list(net), x.to(dev), counts=n[:1])
        g1 = torch.autograd.grad(alone.square().sum(), list(net.parameters()))
        got = gridconv.run_mlp(list(net), both, counts=n)
        g2 = torch.autograd.grad(got[:1, :shape[1]].square().sum(), list(net.parameters()))
        # (the same values on the same weights: float32 sums in another order at most, each worth 2^-20 of the norm)
        assert float((got[:1, :shape[1]] - alone).norm() / alone.norm()) < 2.0 ** -18
        assert float(got[0, shape[1]:].abs().max()) == 0.0
        assert all(float((a - b).norm()) <= 2.0 ** -8 * float(a.norm()) + 1e-4 for a, b in zip(g1, g2))


def test_padded_layers():
    run_padded_layers()                                    # stock operations
    with emu.emulated_gpu():
        run_padded_layers()


def _small_group_net():
    import copy
    cfg = copy.deepcopy(model.SEG_8192)
    cfg["norm"] = "group"
    for lv, (P, O) in zip(cfg["grid"]["down"], ((8, 24), (4, 12), (4, 6))):
        lv["max_p_grid"], lv["max_o_grid"] = P, O
    for lv, O in zip(cfg["grid"]["up"], (12, 24, 64)):
        lv["max_o_grid"] = O
    cfg.update(pt_ele_dim=[[16, 32]] + [[32, 32]] * 2, inputDim=[0, 32, 32], up_inputDim=[32] * 3, up_center_dim=[[32]] * 3,
               up_pt_ele_dim=[[32]] * 3, up_gcn_outDim=[[32]] * 3, dropout=0.0)
    return cfg


def run_cloud_in_any_company(index_ops, dev="cpu"):
    """a cloud of 40 points: its logits and the gradients of its loss, alone and in front of a cloud of 64"""
    torch.manual_seed(0)
    net = model.GGCNSeg(_small_group_net(), index_ops=index_ops, fixed_seed=True).to(dev).train()
    data, npn = synth.make_batch(2, 64, "planes")
    x = torch.from_numpy(data[..., :3].copy())
    n = torch.tensor([[40], [64]], dtype=torch.int32)
    lab = torch.randint(1, 21, (2, 64))
    lab[0, 40:] = 0
    lab[1] = 0                                             # (the ignored label)
    res = []
    for clouds, length in ((1, 40), (2, 64)):
        net.zero_grad()
        out = net(x[:clouds, :length].contiguous().to(dev), n[:clouds].to(dev))
        model.seg_loss(out, lab[:clouds, :length].contiguous().to(dev)).backward()
        res.append((out[0, :40].detach().cpu(), {k: p.grad.cpu().clone() for k, p in net.named_parameters()}))
    (a, ga), (b, gb) = res
    assert float((a - b).norm() / a.norm()) < 2.0 ** -16
    va, vb = (torch.cat([g[k].reshape(-1) for k in ga]) for g in (ga, gb))
    assert float((va - vb).norm() / va.norm()) < 2.0 ** -8, float((va - vb).norm() / va.norm())


def test_cloud_in_any_company_stock_operations():
    from oracle.torch_index_ops import OracleIndexOps
    run_cloud_in_any_company(OracleIndexOps)


def test_cloud_in_any_company_kernels():
    with emu.emulated_gpu():
        run_cloud_in_any_company(model.HipIndexOps)


# ---- forward-mode differentiation: refused, not dropped ------------------------------------------------------------------
def run_tangents_refused(dev="cpu"):
    import torch.autograd.forward_ad as fwd
    x, w, v = torch.randn(2, 6, 8, device=dev), torch.randn(4, 8, device=dev), torch.ones(8, device=dev)
    gn = lambda x, v: ops.group_norm_act(x, v, v, 2)                      # noqa: E731
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))             # noqa: E731
        for call in (lambda: gn(dual(x), v), lambda: gn(x, dual(v)), lambda: ops.linear_act8(dual(x), w),
                     lambda: ops.linear_act8(x, dual(w)), lambda: ops.linear_act8(x, w, dual(v[:4].clone())),
                     lambda: ops.linear_act8(dual(x[:0]), w), lambda: gn(dual(x[:0]), v)):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError):
                    call()
        assert ops.linear_act8(x, w).shape == (2, 6, 4) and gn(x, v).shape == x.shape       # (a level without tangents)
    for f, t in ((lambda x: gn(x, v), x), (lambda x: ops.linear_act8(x, w), x)):
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (t,), (torch.ones_like(t),))


def test_tangents_refused():
    with emu.emulated_gpu():
        run_tangents_refused()


# ---- the registered operators on fake tensors: what a compiled graph plans with --------------------------------------------
def _layouts(ts):
    return [(tuple(t.shape), t.stride(), t.dtype) for t in ts]


def test_fake_backwards_have_the_layouts_of_the_kernels():
    from torch._subclasses.fake_tensor import FakeTensorMode
    import grid_gcn_amd  # noqa: F401
    bf, g = torch.bfloat16, torch.ops.gridgcn
    with FakeTensorMode():
        w = torch.empty((33, 7), device="cuda", dtype=bf).t()                     # a transposed weight
        dy = torch.empty((7, 100, 2), device="cuda", dtype=bf).permute(2, 1, 0)
        codes, scales = torch.empty((200, 64), device="cuda", dtype=torch.uint8), torch.empty((200, 2), device="cuda", dtype=torch.uint8)
        assert _layouts(g.linear_act8_backward(dy, w, codes, scales)) == [
            ((2, 100, 33), (3300, 33, 1), bf), ((7, 33), (33, 1), bf), ((7,), (1,), bf)]
        gamma = torch.empty(66, device="cuda")[::2]
        beta = torch.empty(1, device="cuda").expand(33)
        dy = torch.empty((33, 100, 2), device="cuda", dtype=bf).permute(2, 1, 0)
        st = torch.empty((2, 3, 2), device="cuda", dtype=torch.float64)
        assert _layouts(g.group_norm_act_backward(dy, None, codes, scales, st, gamma, beta, 3, "silu")) == [
            ((2, 100, 33), (3300, 33, 1), bf), ((33,), (1,), torch.float32), ((33,), (1,), torch.float32)]


def test_statistics_of_the_registered_operator_are_not_differentiable():
    from torch._subclasses.fake_tensor import FakeTensorMode
    import grid_gcn_amd  # noqa: F401
    with FakeTensorMode():
        x = torch.empty((2, 100, 33), device="cuda", requires_grad=True)
        for save8 in (False, True):
            y, st, codes, scales = torch.ops.gridgcn.group_norm_act(x, None, None, 3, save8=save8)
            assert y.requires_grad and not st.requires_grad and not codes.requires_grad and not scales.requires_grad


def test_registered_backwards_leave_out_what_is_not_needed():
    from types import SimpleNamespace
    from torch._subclasses.fake_tensor import FakeTensorMode
    from grid_gcn_amd import torch_ops
    with FakeTensorMode():
        e = lambda *s: torch.empty(s, device="cuda")                      # noqa: E731
        codes, scales = (torch.empty(s, device="cuda", dtype=torch.uint8) for s in ((18, 32), (18, 1)))
        w, v, st = e(5, 32), e(32), torch.empty((2, 4, 2), device="cuda", dtype=torch.float64)
        for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 1)):
            sizes = lambda shapes: [s if n else (0,) for s, n in zip(shapes, need)]       # noqa: E731
            need = tuple(bool(n) for n in need)
            got = torch.ops.gridgcn.linear_act8_backward(e(2, 9, 5), w, codes, scales, *need)
            assert [tuple(t.shape) for t in got] == sizes(((2, 9, 32), (5, 32), (5,)))
            got = torch_ops._lin8_bwd(SimpleNamespace(saved_tensors=(w, codes, scales), needs_input_grad=need), e(2, 9, 5), None, None)
            assert [t is not None for t in got] == list(need)
            got = torch.ops.gridgcn.group_norm_act_backward(e(2, 9, 32), None, codes, scales, st, v, v, 4, "relu", None, *need)
            assert [tuple(t.shape) for t in got] == sizes(((2, 9, 32), (32,), (32,)))
            ctx = SimpleNamespace(saved_tensors=(None, codes, scales, st, v, v, None), needs_input_grad=need + (False,) * 5, gn=(4, "relu"))
            got = torch_ops._gn_bwd(ctx, e(2, 9, 32), None, None, None)
            assert len(got) == 8 and [t is not None for t in got[:3]] == list(need)


# ---- GELU: as many digits as float32's own 0.5 t (1 + erf), and where Phi is small -----------------------------------------
def run_gelu_digits(dev="cpu"):
    """Norms of the error, in units of U = 2^-24.  A rounding is uniform within half a step: 0.42 U of a value, root mean square.  t has four
    (x - mean, rstd, rstd weight, the product), which t f'/f <= 1.3 carries into f = t Phi(t): 1.1 U; Phi: 1 U (an erf good to a
    step), the last product 0.42 U: 1.6 U together.  Between -1.5 and -0.5 |t f'/f| <= 1.2 and 1 + erf is a difference of up to three
    times its size: 1 U, 2 U, 0.42 U: 2.3 U."""
    import math
    x = torch.randn(8, 4096, 16, generator=torch.Generator().manual_seed(5))
    with torch.no_grad():
        y = ops.group_norm_act(x.to(dev), None, None, 2, act="gelu").cpu().double()
        wide = ops.group_norm_act(x.to(dev), torch.full((16,), 2.0, device=dev), None, 2, act="gelu").cpu().double()
    t = ref.group_norm_act(x, None, None, 2, 1e-5, "none")["y"]
    f = lambda t: t * 0.5 * torch.special.erfc(-t / math.sqrt(2))          # noqa: E731
    for lo, hi, lim in ((-9.0, 9.0, 1.6), (-1.5, -0.5, 2.3)):
        at = (t > lo) & (t < hi)
        off = float((y - f(t))[at].norm() / f(t)[at].norm())
        assert off <= lim * ref.U, (lo, hi, off / ref.U)
    # value by value: t is off by 4 U of itself, f' / f is |t| + 1 / |t| at most; exponential and product as in the oracle's bound
    t = 2 * t
    off = ((wide - f(t)) / f(t)).abs()
    at = (t < -0.1) & (t > -8.0)
    assert int((t[at] < -6).sum()) > 20
    assert bool((off <= ref.U * (4 * t * t + 4 + 8 * (1 + t.abs()) + 2))[at].all())


def run_gelu_tail_of_16_bits(dtype, dev="cpu"):
    """half a step of the type, and what the coarser fit may add (1e-7 exp(1.5 |t|), at most 2e-4)"""
    import math
    x = torch.randn(8, 4096, 16, generator=torch.Generator().manual_seed(6)).to(dtype)
    with torch.no_grad():
        y = ops.group_norm_act(x.to(dev), torch.full((16,), 2.0, device=dev), None, 2, act="gelu").cpu().double()
    t = 2 * ref.group_norm_act(x, None, None, 2, 1e-5, "none")["y"]
    want = t * 0.5 * torch.special.erfc(-t / math.sqrt(2))
    at = (t < -0.1) & (want.abs() > torch.finfo(dtype).tiny)
    assert int((t[at] < -3.5).sum()) > 100
    fit = torch.clamp(1e-7 * torch.exp(1.5 * t.abs()), max=2e-4)
    u = ref.U * (4 * t * t + 4 + 8 * (1 + t.abs()) + 2)
    assert bool((((y - want) / want).abs() <= ref.half_step(dtype) * (1 + fit + u) + fit + u)[at].all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gelu_tail_of_16_bits(dtype):
    with emu.emulated_gpu():
        run_gelu_tail_of_16_bits(dtype)


def test_gelu_digits():
    with emu.emulated_gpu():
        run_gelu_digits()


def test_c_entries_refuse_a_workspace_off_its_alignment():
    import ctypes
    from grid_gcn_amd import _lib, build
    build.build()
    lib = _lib.load()
    a = (ctypes.cast((ctypes.c_float * 256)(), ctypes.c_void_p).value + 15) & ~15
    EWORKSPACE = 2
    for ws in (a + 4, a + 8):
        assert lib.gridgcn_group_norm_act_fwd(a, 0, 2, 100000, 8, 800000, 8, 2, a, a, 0, None, 1e-5, 1, a, None, None, None, ws, 1 << 30,
                                              None) == EWORKSPACE
        assert lib.gridgcn_group_norm_act_bwd(a, 800000, 8, a, 800000, 8, None, None, 0, 2, 100000, 8, 2, a, a, a, 0, None, 1, a, a, a,
                                              ws, 1 << 30, None) == EWORKSPACE


# ---- ConvBNReLU on the CPU: statistics that do not depend on the number of threads -------------------------------------------
def test_batch_statistics_on_the_cpu_keep_their_digits():
    """y, dx, dgamma, dbeta of 300000 rows against float64, on one thread and on all.  A dozen roundings per value, U = 2^-24 each at
    most, of terms up to twice the result: 24 U of the norm -- of dgamma and dbeta, whose terms
    cancel (3e5 of magnitude 0.8 leave 1e4), of the norm of the sums of their terms' magnitudes.  (A float32 sum over the rows of a thread: 70 U and more.  The
    linear layer's own weight gradient is a float32 product over the rows, not looked at here.)"""
    g = torch.Generator().manual_seed(7)
    x, dy = torch.randn(300000, 4, generator=g), torch.randn(300000, 6, generator=g) + 1
    torch.manual_seed(0)
    layer = gridconv.ConvBNReLU(4, 6).train()
    with torch.no_grad():
        layer.lin.bias.uniform_(-2, 2)
        layer.bn.bias.uniform_(2, 3)                       # (mostly open gates: a gate that flips is no rounding)
    xd, w = x.double().requires_grad_(), {k: v.detach().double().requires_grad_() for k, v in layer.named_parameters()}
    z = xd @ w["lin.weight"].t() + w["lin.bias"]
    t = (z - z.mean(0)) / torch.sqrt(z.var(0, unbiased=False) + layer.bn.eps) * w["bn.weight"] + w["bn.bias"]
    keep = (t.detach().abs() > 1e-4).double()
    want = torch.autograd.grad((torch.relu(t) * keep * dy).sum(), [xd, w["bn.weight"], w["bn.bias"]])
    g = (keep * (t > 0) * dy).detach()
    xh = ((t - w["bn.bias"]) / w["bn.weight"]).detach()
    size = [torch.relu(t), want[0], (g * xh).abs().sum(0), g.abs().sum(0)]
    threads = torch.get_num_threads()
    try:
        for n in {1, threads}:
            torch.set_num_threads(n)
            xr = x.clone().requires_grad_()
            y = layer(xr)
            got = torch.autograd.grad((y * keep.float() * dy).sum(), [xr, layer.bn.weight, layer.bn.bias])
            for a, b, s in zip((y,) + got, (torch.relu(t),) + want, size):
                assert float((a.double() - b).norm() / s.norm()) <= 24 * ref.U, n
    finally:
        torch.set_num_threads(threads)


# ---- what an edge block with 8-bit checkpoints holds between forward and backward -------------------------------------------
def run_edge_block_holds(dev="cpu"):
    B, O, P, C = 1, 40, 8, 64
    torch.manual_seed(3)
    layer = gridconv.SubGUpdate(16, [32, C], localfdim=3, norm="group").to(dev).train()
    src = torch.randn(B, 50, 4 + 16).to(dev).requires_grad_()
    cent = torch.randn(B, O, 4).to(dev)
    idx = torch.randint(0, 50, (B, O, P), dtype=torch.int32).to(dev)
    held = {}

    def pack(t):
        held[t.untyped_storage().data_ptr()] = (t.untyped_storage().nbytes(), t.dtype)
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        out = layer.forward_src(cent, src, idx)
    # the widest edge tensors as codes (of both products' inputs and both norms'), none of them in float32
    assert not [h for h in held.values() if h[0] >= B * O * P * C * 4 and h[1] == torch.float32], held
    edges = [c for l in (layer.att1, layer.att2, layer.pt_mlp) for c in l]
    codes = sum(-(-c // 32) * 33 for l in edges for c in (l.lin.in_features, l.lin.out_features))
    assert sum(h[0] for h in held.values()) <= B * O * P * codes + 4 * B * O * C * 8 + 100000
    dy = torch.randn(out.shape).to(dev)
    got = torch.autograd.grad(out, [src] + list(layer.parameters()), dy)
    # against the stock product and maximum on the same layers
    nf, att = ops.edge_inputs(src, idx, cent, has_feats=True, localfdim=3)
    pair = gridconv.run_mlp([layer.att1[0], layer.att2[0]], att) * gridconv.run_mlp(list(layer.pt_mlp), nf)
    want = layer.finish(pair.max(dim=2).values, None, None)
    assert torch.equal(out, want)
    for a, b in zip(got, torch.autograd.grad(want, [src] + list(layer.parameters()), dy)):
        # (the same values; the gather's gradient sums may come in another order)
        assert float((a - b).norm()) <= 2.0 ** -20 * float(b.norm())


def test_edge_block_holds_no_float32_edges():
    with emu.emulated_gpu():
        run_edge_block_holds()
