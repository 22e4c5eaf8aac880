"""MI355X tier of the batch-independent training layer (grid_gcn_amd/act8.py): the cases of the CPU tier and larger ones against
float64, streams, captured graphs, offsets beyond 32 bits."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

import act8_cases as cases  # noqa: E402
import test_act8 as cpu  # noqa: E402
from oracle import act8_ref as ref  # noqa: E402
from grid_gcn_amd import gridconv, ops  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("R,C,pad", cases.PACK + [(20000, 131, 1), (3000, 512, 0)])
def test_act8_round_trip(R, C, pad, dtype):
    x = cases.rows((R,), C, dtype, 1, pad)
    want, E = ref.act8(x)
    xd = x.as_strided((R, C + pad), (C + pad, 1)).to(DEV)[:, :C]
    codes, scales = ops.act8_pack(xd)
    assert torch.equal(scales.cpu().int() - 127, E.int())
    assert int(codes[:, C:].max()) == 0 if C % 32 else True
    for t in {dtype, torch.float32}:
        cpu._same(ops.act8_unpack(codes, scales, C, dtype=t).cpu().double(), want)


@pytest.mark.parametrize("dtype", cases.DTYPES)
def test_act8_special_values(dtype):
    x = cases.special_rows(dtype)
    want, E = ref.act8(x)
    codes, scales = ops.act8_pack(x.to(DEV))
    assert torch.equal(scales.cpu().int() - 127, E.int())
    cpu._same(ops.act8_unpack(codes, scales, 32).cpu().double(), want.float().double())


def test_act8_every_code_and_scale():
    """all 256 codes under every scale that the packer writes, into the three types"""
    codes = torch.arange(256, dtype=torch.uint8, device=DEV).view(1, 256).repeat(238, 1)
    scales = torch.arange(10, 248, dtype=torch.uint8, device=DEV).view(238, 1).repeat(1, 8)
    want = codes.cpu().view(torch.float8_e4m3fn).double() * torch.exp2(scales.cpu().double() - 127).repeat_interleave(32, 1)
    for t in cases.DTYPES:
        cpu._same(ops.act8_unpack(codes, scales, 256, dtype=t).cpu().double(), want.float().to(t).double())


@pytest.mark.parametrize("dtype", cases.DTYPES)
def test_linear_act8_every_code_and_scale(dtype):
    """dW of unit rows of dy: row n of dW is the value of row n of the codes, whatever its scale"""
    from grid_gcn_amd import act8
    scale = torch.arange(10, 248) if dtype != torch.float16 else torch.arange(127 - 15, 127 + 8)     # (fp16: what packing fp16 gives)
    R = len(scale)
    codes = torch.arange(256, dtype=torch.uint8).view(1, 256).repeat(R, 1)
    codes[(codes & 0x7f) == 0x7f] = 0                    # (NaN would reach every result of its column)
    scales = scale.to(torch.uint8).view(R, 1).repeat(1, 8)
    if dtype != torch.float16:
        codes[scales.repeat_interleave(32, 1) > 246] &= 0xf7          # (2^128 and beyond)
    values = codes.view(torch.float8_e4m3fn).double() * torch.exp2(scales.double() - 127).repeat_interleave(32, 1)
    if dtype == torch.float16:
        values = values.half().double()                  # (below 2^-24: not what packing gives)
    dy = torch.eye(R, dtype=dtype, device=DEV)
    w = torch.zeros(R, 256, dtype=dtype, device=DEV)
    _, dw, _ = act8._linear_backward(dy, w, codes.to(DEV), scales.to(DEV), (R, 256), (False, True, False))
    assert bool(torch.isfinite(values).all())
    assert torch.equal(dw.cpu().double(), values.to(dtype).double())


@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("case", cases.GN + [
    (4, 20000, 128, 32, "silu", False, False, 0), (3, 9000, 200, 8, "relu", True, True, 1), (32, 700, 64, 8, "gelu", True, True, 0),
    (1, 50000, 24, 3, "relu", False, False, 0), (300, 1, 512, 32, "relu", False, False, 0), (2, 300, 2048, 1, "none", False, True, 0)])
def test_group_norm_act(case, dtype):
    got, want = cpu.run_gn(case, dtype, DEV)
    cpu.check_gn(got, want)


@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("case", cases.LINEAR + [
    (40000, 131, 128, True, 1), (33000, 256, 300, True, 0), (34000, 40, 24, False, 8), (66000, 64, 512, False, 0), (5000, 1027, 512, True, 0),
    (140000, 3, 32, True, 0)])
def test_linear_act8(case, dtype):
    got, want = cpu.run_linear(case, dtype, DEV, strided_dy=case[0] % 2 == 1)
    cpu.check_linear(got, want, case)


@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("R,K", [(40, 70), (90, 128), (17000, 131), (20000, 512)])
def test_linear_act8_writes_the_same_codes(R, K, dtype):
    cpu.check_codes(R, K, dtype, DEV)


def test_linear_act8_rows_and_columns_of_every_scale():
    cpu.run_scales(DEV)


def test_group_norm_relu_gate_at_the_border():
    """as on the CPU, at many rows: the gate is that of 64 bits"""
    x = cases.rows((1, 4000), 4, torch.float32, 11)
    st = ref.group_norm_act(x, None, None, 1, 1e-5, "none")
    w, b = torch.ones(4), -torch.stack([st["y"][0, 50 * c + 1, c] for c in range(4)]).float()
    dy = torch.ones(1, 4000, 4)
    want = ref.group_norm_act(x, w, b, 1, 1e-5, "relu", None, dy)
    t = [v.to(DEV).requires_grad_() for v in (x, w, b)]
    dx, dw, db = torch.autograd.grad(ops.group_norm_act(*t, 1, act="relu"), t, dy.to(DEV))
    assert torch.equal(db.cpu().double(), want["db"])
    ref.check(dx, want["dx"], want["dx_tol"])


@pytest.mark.parametrize("save8", [False, True])
@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("N", [40, 5000])
def test_group_norm_relu_gate_of_any_gain(N, dtype, save8):
    cpu.run_gate_of_any_gain(dtype, N, save8, DEV)


@pytest.mark.parametrize("dtype", cases.DTYPES)
@pytest.mark.parametrize("case", [
    # few rows against many columns, and the other way round: row blocks, splits and tiles that are no multiple of 8
    (1, 96, 20000, True, 0), (3, 9000, 40, False, 0), (130, 64, 17000, True, 0), (300, 72, 5000, False, 0), (700, 1100, 1000, True, 0),
    (2100, 900, 260, True, 0), (1300, 2000, 1900, False, 0), (9000, 130, 260, True, 0)])
def test_linear_act8_wide(case, dtype):
    got, want = cpu.run_linear(case, dtype, DEV)
    cpu.check_linear(got, want, case)


@pytest.mark.parametrize("dtype", cases.DTYPES)
def test_results_larger_than_the_caches(dtype):
    """more than 192 MB of output: every value as in a call on a part of the rows"""
    R, C = (220 << 20) // (4 if dtype == torch.float32 else 2) // 99, 99
    x = cases.rows((4096,), C, dtype, 7).to(DEV).repeat(R // 4096 + 1, 1)[:R]
    codes, scales = ops.act8_pack(x)
    back, part = ops.act8_unpack(codes, scales, C, dtype), ops.act8_unpack(codes[:4096], scales[:4096], C, dtype)
    assert torch.equal(back, part.repeat(R // 4096 + 1, 1)[:R])
    w = (torch.randn(C, C, generator=torch.Generator().manual_seed(2)) * 0.1).to(dtype).to(DEV)
    with torch.no_grad():
        y = ops.linear_act8(x, w)
        assert torch.equal(y, ops.linear_act8(x[:4096 * 8], w)[:4096].repeat(R // 4096 + 1, 1)[:R])
    B = R // 4096
    x3, dy = x[:B * 4096].view(B, 4096, C).requires_grad_(), y[:B * 4096].view(B, 4096, C)
    z = ops.group_norm_act(x3, None, None, 3, act="silu")
    xs = x3[:1].detach().requires_grad_()
    zs = ops.group_norm_act(xs, None, None, 3, act="silu")
    n = x.new_zeros(1).float()
    for a, b in ((z, zs), (torch.autograd.grad(z, x3, dy)[0], torch.autograd.grad(zs, xs, dy[:1])[0])):
        # (the partial sums of a cloud are cut by the number of clouds: last bits of the statistics in 64 bits, a rounding of the result)
        far = (a.detach().float() - b.detach().float()).abs() - torch.finfo(dtype).eps * 2 * b.detach().float().abs()
        n = torch.maximum(n, far.max())
    assert float(n) < 1e-5


def _step(x, w, g, b, dy, counts, save8=True):
    z = ops.linear_act8(x, w)
    y = ops.group_norm_act(z, g, b, 8, act="relu", counts=counts, save8=save8)
    return (y.detach(),) + torch.autograd.grad(y, (x, w, g, b), dy)


def _step_inputs(seed, N=1500, K=72, C=64, dtype=torch.float32):
    x = cases.rows((4, N), K, dtype, seed, kind="act").to(DEV).requires_grad_()
    w = (cases.rows((C,), K, torch.float32, seed + 1, kind="grad") * 0.1).to(dtype).to(DEV).requires_grad_()
    g = torch.ones(C, device=DEV).requires_grad_()
    b = torch.full((C,), 0.1, device=DEV).requires_grad_()
    dy = cases.rows((4, N), C, dtype, seed + 2, kind="grad").to(DEV)
    return x, w, g, b, dy, torch.tensor([[N], [N // 3], [0], [N - 1]], dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype", cases.DTYPES)
def test_same_bits_again(dtype):
    a = _step_inputs(3, dtype=dtype)
    r0 = _step(*a)
    for _ in range(3):
        assert all(torch.equal(u, v) for u, v in zip(r0, _step(*a)))


def test_two_streams_at_once():
    ins = [_step_inputs(s) for s in (3, 13)]
    want = [_step(*i) for i in ins]
    streams = [torch.cuda.Stream() for _ in ins]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(_step(*ins[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for r in got[k]:
            assert all(torch.equal(u, v) for u, v in zip(want[k], r))


def test_captured_step_replays():
    """two graphs of a step, replayed in turn on new inputs with eager steps and synchronisations in between"""
    ins = [_step_inputs(s) for s in (3, 13)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in ins:
            _step(*i)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_step(*i))
        graphs.append(g)
    for r in range(4):
        for k in range(2):
            with torch.no_grad():
                for dst, src in zip(ins[k], _step_inputs(30 + 10 * r + k)):
                    dst.copy_(src)
            graphs[k].replay()
            torch.cuda.synchronize()
            seen = [t.clone() for t in outs[k]]
            want = _step(*[t.detach().clone().requires_grad_(t.requires_grad) for t in ins[k]])
            torch.cuda.synchronize()
            assert all(torch.equal(u, v) for u, v in zip(seen, want)), (r, k)


def test_offsets_beyond_32_bits():
    """more than 2^32 bytes and 2^31 elements in one tensor: the last rows are right"""
    R, C = (1 << 31) // 64 + 70000, 64
    x = torch.zeros(R, C, dtype=torch.bfloat16, device=DEV)
    tail = cases.rows((512,), C, torch.bfloat16, 3)
    x[-512:] = tail.to(DEV)
    codes, scales = ops.act8_pack(x)
    want, _ = ref.act8(tail)
    back = ops.act8_unpack(codes[-600:], scales[-600:], C)
    cpu._same(back[-512:].cpu().double(), want)
    assert float(back[:-512].abs().max()) == 0
    x.requires_grad_()
    w = torch.randn(48, C, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    wd = w.to(DEV).requires_grad_()
    y = ops.linear_act8(x, wd)
    dy = torch.zeros_like(y)
    dyt = cases.rows((512,), 48, torch.bfloat16, 4)
    dy[-512:] = dyt.to(DEV)
    full = ref.linear_act8(tail, w, None, dyt)
    ref.check(y[-512:], full["y"], full["y_tol"])
    dx, dw = torch.autograd.grad(y, (x, wd), dy)
    ref.check(dx[-512:], full["dx"], full["dx_tol"])
    assert float(dx[:-512].abs().max()) == 0
    ref.check(dw, full["dw"], full["dw_tol"])
    del y, dy, dx, codes, scales, back
    n = R // 2
    x3 = x.detach()[:2 * n].view(2, n, C)
    counts = torch.tensor([[5], [n]], dtype=torch.int32, device=DEV)
    y = ops.group_norm_act(x3, None, None, 4, act="none", counts=counts)
    t = tail.double().reshape(512, 4, 16)[-(512 - R % 2):] if R % 2 else tail.double().reshape(512, 4, 16)
    mean = t.sum((0, 2), keepdim=True) / (n * 16)
    var = ((t - mean) ** 2).sum((0, 2), keepdim=True) / (n * 16) + (n - t.shape[0]) / n * mean ** 2
    want = ((t - mean) / (var + 1e-5).sqrt()).reshape(-1, 64)
    # (bf16 results: half a step, and float32 roundings far below it)
    assert float(((y[1, -want.shape[0]:].cpu().double() - want).abs() - 2.0 ** -8 * want.abs()).max()) < 1e-5
    assert float(y[0].abs().max()) == 0 or float(y[0, 5:].abs().max()) == 0


def test_layers_in_a_row_train():
    torch.manual_seed(1)
    net = gridconv.mlp(131, [128, 128, 64], norm="group").to(DEV)
    x, dy = torch.randn(3, 2000, 131), torch.randn(3, 2000, 64)
    y, grads = cpu.run_layers(net, x, dy, DEV)
    y2 = gridconv.run_mlp(list(net), x.to(DEV))
    grads2 = torch.autograd.grad(y2, list(net.parameters()), dy.to(DEV))
    assert torch.equal(y, y2.detach()) and all(torch.equal(a, b) for a, b in zip(grads, grads2))


def test_torch_ops_are_the_same_calls():
    x, w, g, b, dy, counts = _step_inputs(5)
    want = _step(x, w, g, b, dy, counts)
    z = torch.ops.gridgcn.linear_act8(x, w)[0]
    y = torch.ops.gridgcn.group_norm_act(z, g, b, 8, act="relu", counts=counts, save8=True)[0]
    got = (y.detach(),) + torch.autograd.grad(y, (x, w, g, b), dy)
    assert all(torch.equal(u, v) for u, v in zip(want, got))
    codes, scales = torch.ops.gridgcn.act8_pack(x.detach())
    c2, s2 = ops.act8_pack(x.detach())
    assert torch.equal(codes, c2) and torch.equal(scales, s2)
    assert torch.equal(torch.ops.gridgcn.act8_unpack(codes, scales, 72, torch.float32), ops.act8_unpack(c2, s2, 72))


def test_segmentation_net_with_group_norm_trains():
    import copy
    from grid_gcn_amd import model, synth
    cfg = dict(copy.deepcopy(model.SEG_8192), norm="group")
    torch.manual_seed(0)
    net = model.GGCNSeg(cfg).to(DEV).train()
    data, npn = synth.make_batch(2, 2048, "planes")
    x, n = torch.from_numpy(data[..., :3].copy()).to(DEV), torch.from_numpy(npn).to(DEV)
    model.seg_loss(net(x, n), torch.randint(1, 21, (2, 2048), device=DEV)).backward()
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in net.parameters())
    net.eval()
    with torch.no_grad():
        out = net(x, n)
    assert out.shape == (2, 2048, 21) and bool(torch.isfinite(out).all())
