"""MI355X tier of tests/test_act8_range.py: extreme magnitudes and calls off the usual path, on the kernels themselves."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

import test_act8_range as cpu  # noqa: E402
from grid_gcn_amd import model  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("R", [100, 260, 4000])
def test_linear_act8_wide_rows(R):
    cpu.run_wide_rows(R, DEV)


@pytest.mark.parametrize("R", [100, 260])
def test_linear_act8_rows_of_every_scale(R):
    cpu.run_every_scale(R, DEV)


@pytest.mark.parametrize("R", [100, 260])
def test_linear_act8_tiny_values(R):
    cpu.run_tiny(R, DEV)


def test_linear_act8_same_row_in_any_company():
    cpu.run_same_row_in_any_company(DEV)


def test_linear_act8_float16_top():
    cpu.run_float16_top(DEV)


def test_linear_act8_float16_magnitudes():
    cpu.run_float16_magnitudes(DEV)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,act,save8", [(40, "relu", False), (40, "silu", True), (2300, "gelu", False), (2300, "relu", True)])
@pytest.mark.parametrize("scale,eps", cpu.GN_SCALES)
def test_group_norm_act_far_from_one(scale, eps, N, act, save8, dtype):
    cpu.run_gn_scale(scale, eps, N, act, dtype, save8, DEV)


@pytest.mark.parametrize("N", [40, 2300])
def test_group_norm_act_small_values_and_gradients(N):
    cpu.run_gn_scale(2.0 ** -70, 0.0, N, "silu", torch.float32, False, DEV, dy_scale=2.0 ** -70)


def test_padded_layers():
    cpu.run_padded_layers(DEV)


def test_cloud_in_any_company():
    cpu.run_cloud_in_any_company(model.HipIndexOps, DEV)


def test_tangents_refused():
    cpu.run_tangents_refused(DEV)


@pytest.mark.parametrize("need", [False, True])
def test_tangents_refused_by_the_registered_operators(need):
    import torch.autograd.forward_ad as fwd
    x, w, v = torch.randn(2, 6, 8, device=DEV, requires_grad=need), torch.randn(4, 8, device=DEV), torch.ones(8, device=DEV)
    g = torch.ops.gridgcn
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))             # noqa: E731
        for call in (lambda: g.group_norm_act(dual(x), v, v, 2), lambda: g.group_norm_act(x, dual(v), v, 2),
                     lambda: g.linear_act8(dual(x), w), lambda: g.linear_act8(x, dual(w))):
            with pytest.raises(RuntimeError):
                call()


def test_captured_step_of_the_group_norm_net_follows_the_counts():
    """replays of one captured training step, with other clouds, counts and eager work in between, against eager steps"""
    import copy
    from grid_gcn_amd import graph, synth
    torch.manual_seed(0)
    net = model.GGCNSeg(cpu._small_group_net(), fixed_seed=True).to(DEV).train()
    twin = copy.deepcopy(net)
    data, _ = synth.make_batch(4, 64, "planes")
    clouds = torch.from_numpy(data[..., :3].copy()).to(DEV)
    x, n = clouds[:2].clone(), torch.tensor([[64], [40]], dtype=torch.int32, device=DEV)
    lab = torch.randint(1, 21, (2, 64), device=DEV)
    adam = lambda m: torch.optim.Adam(m.parameters(), lr=1e-3, fused=True, capturable=True)          # noqa: E731
    opt, opt2 = adam(net), adam(twin)
    step = graph.GraphedTrainStep(net, opt, model.seg_loss, (x, n), lab, warmup=1)

    def eager():
        opt2.zero_grad(set_to_none=True)
        loss = model.seg_loss(twin(x, n), lab)
        loss.backward()
        opt2.step()
        return float(loss)

    eager()                                               # (the warm-up step)
    for i, counts in enumerate(((64, 40), (17, 64), (64, 64), (33, 50))):
        x.copy_(clouds[[i, (i + 1) % 4]])
        n.copy_(torch.tensor(counts, dtype=torch.int32)[:, None])
        got, want = float(step()), eager()
        torch.cuda.synchronize()
        # (the same kernels on the same values; only the gathers' gradient sums may come in another order)
        assert abs(got - want) < 1e-4 * abs(want), (i, got, want)


def test_registered_backwards_leave_out_what_is_not_needed():
    g = torch.ops.gridgcn
    x, w, b, v = (torch.randn(s, device=DEV) for s in ((40, 32), (5, 32), (5,), (32,)))
    _, codes, scales = g.linear_act8(x, w, b)
    y, st, c8, s8 = g.group_norm_act(x, v, v, 4, save8=True)
    dy = torch.randn(40, 5, device=DEV)
    full = g.linear_act8_backward(dy, w, codes, scales), g.group_norm_act_backward(x, None, c8, s8, st, v, v, 4, "relu")
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1)):
        need = tuple(bool(n) for n in need)
        part = g.linear_act8_backward(dy, w, codes, scales, *need), g.group_norm_act_backward(x, None, c8, s8, st, v, v, 4, "relu", None, *need)
        for f, p in zip(full, part):
            assert all(torch.equal(a, q) if n else q.numel() == 0 for a, q, n in zip(f, p, need))
        leaves = [t.clone().requires_grad_(n) for t, n in zip((x, w, b), need)]
        y = g.linear_act8(*leaves)[0]
        y.backward(dy)
        assert all((t.grad is not None) == n and (not n or torch.equal(t.grad, a)) for t, n, a in zip(leaves, need, full[0]))


def test_gelu_digits():
    cpu.run_gelu_digits(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gelu_tail_of_16_bits(dtype):
    cpu.run_gelu_tail_of_16_bits(dtype, DEV)


@pytest.mark.parametrize("R,N,K", [(65536, 2048, 2048), (1048576, 64, 3)])
def test_linear_act8_db_of_many_rows(R, N, K):
    """The sums run in float32 over eight rows, then in 64 bits.  The roundings of the first are independent and, over R / 8 sums, 0.02
    U of the result; what is left is the last rounding, half a step: 1 U = 2^-24 (a chain of float32 sums: 2 U and more)."""
    g = torch.Generator().manual_seed(3)
    dy = 1 + torch.rand(R, N, generator=g)
    x = torch.randn(64, K, generator=g).to(DEV).repeat(R // 64, 1)
    w, b = torch.zeros(N, K, device=DEV), torch.zeros(N, device=DEV, requires_grad=True)
    db, = torch.autograd.grad(cpu.ops.linear_act8(x, w.requires_grad_(), b), b, dy.to(DEV))
    want = dy.double().sum(0)
    assert float(((db.cpu().double() - want) / want).abs().max()) <= 1.05 * 2.0 ** -24
    # ... in the call that forms dW too
    db = torch.autograd.grad(cpu.ops.linear_act8(x, w, b), (w, b), dy.to(DEV))[1]
    assert float(((db.cpu().double() - want) / want).abs().max()) <= 1.05 * 2.0 ** -24


def test_edge_block_holds_no_float32_edges():
    cpu.run_edge_block_holds(DEV)
