"""Batch-independent training layers on channels-last rows, and the 8-bit form of activations that they keep between
forward and backward (csrc/gridgcn_act8.h, gridgcn_gnorm.hip, gridgcn_lin8.hip).  Reached through grid_gcn_amd.ops
(this module's functions are its members), torch.ops.gridgcn.* and gridconv.ConvGNAct.

    act8_pack(x) -> codes, scales          act8_unpack(codes, scales, C, dtype) -> x
    group_norm_act(x, weight, bias, groups, eps, act, counts, save8) -> y        differentiable
    linear_act8(x, weight, bias) -> y                                            differentiable

Rows are float32, bfloat16 or float16 GPU tensors; the last axis (channels) must be contiguous, rows may be strided
(columns of a wider buffer) -- anything else is copied first.  Errors raise RuntimeError, as in ops.py."""
import contextlib
import ctypes
import functools

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}     # GRIDGCN_F32 / _BF16 / _F16
ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}                   # GRIDGCN_ACT_*
ACT8_BLOCK = 32
ACT8_MAX_C = 65536
GN_MAX_C = 8192
MAX_LD = 1 << 24                  # row strides above it are copied together first (32-bit offsets inside a tile of rows)


def _require(cond, msg):
    if not cond:
        raise RuntimeError(msg)


# The host's share of a small call is most of it (a training step of 32 rows: 160 us, of which 20 on the GPU): no context
# manager where the device is the current one, no stream object, no query of a size that was asked before.
def _p(t):
    return t.data_ptr() if t is not None else None


def _st(t):
    i = t.device.index
    return torch._C._cuda_getCurrentRawStream(i) if i is not None else torch.cuda.current_stream(t.device).cuda_stream


_HERE = contextlib.nullcontext()


def _on(dev):
    return _HERE if dev.index is None or dev.index == torch.cuda.current_device() else torch.cuda.device(dev)


def _packed(t):
    """a parameter as the kernels read it: contiguous (its pointer is all they get)"""
    return t if t is None or t.is_contiguous() else t.detach().contiguous()


def _check_rows(t, name, min_dim=1):
    _require(isinstance(t, torch.Tensor), "%s must be a torch.Tensor" % name)
    _require(t.is_cuda, "%s must live on the GPU (there is no CPU path)" % name)
    _require(t.dtype in _DTYPES, "%s must be float32, bfloat16 or float16" % name)
    _require(t.dim() >= min_dim, "%s should have at least %d dimensions" % (name, min_dim))


def _no_tangents(name, *ts):
    if forward_ad._current_level >= 0:
        for t in ts:
            _require(t is None or forward_ad.unpack_dual(t).tangent is None, "%s has no forward-mode derivative" % name)


def _rows2(t):
    """[..., C] -> ([R, C] with contiguous channels and rows that do not overlap, row stride in elements)"""
    C = t.shape[-1]
    if t.dim() != 2:
        t = t.reshape(-1, C)
    if (C > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and not C <= t.stride(0) <= MAX_LD):
        t = t.contiguous()
    return t, (t.stride(0) if t.shape[0] > 1 else C)


def _rows3(t, B):
    """[B, ..., C] -> ([B, N, C], cloud stride, row stride), channels contiguous"""
    C = t.shape[-1]
    if t.dim() != 3:
        t = t.reshape(B, -1, C)
    N = t.shape[1]
    if (C > 1 and t.stride(2) != 1) or (N > 1 and not C <= t.stride(1) <= MAX_LD):
        t = t.contiguous()
    return t, (t.stride(0) if B > 1 else 0), (t.stride(1) if N > 1 else C)


def act8_shapes(rows, C):
    """shapes of (codes, scales) for `rows` rows of C channels"""
    Cp = -(-C // ACT8_BLOCK) * ACT8_BLOCK
    return (rows, Cp), (rows, Cp // ACT8_BLOCK)


def _new_act8(rows, C, dev):
    c, s = act8_shapes(rows, C)
    return torch.empty(c, dtype=torch.uint8, device=dev), torch.empty(s, dtype=torch.uint8, device=dev)


@torch.no_grad()
def act8_pack(x):
    """x [..., C] -> (codes uint8 [..., Cp], scales uint8 [..., Cp / 32]), Cp = C rounded up to 32: 32 consecutive channels
    share the smallest power of two 2^(scale - 127) >= max |x| / 448 (scale >= 10), a channel is the nearest e4m3 number of
    x / 2^(scale - 127); infinities and NaN become NaN (and a magnitude above 3.29e38 rounds to 2^128, infinite; a float16 one
    of 63488 or more to 65536, infinite as a float16).  Off by at most 2^-4 of the value, or 2^-10 of 2^(scale - 127)."""
    _check_rows(x, "x")
    C = x.shape[-1]
    _require(1 <= C <= ACT8_MAX_C, "x must have 1..%d channels" % ACT8_MAX_C)
    lead = tuple(x.shape[:-1])
    x2, ld = _rows2(x)
    R = x2.shape[0]
    codes, scales = _new_act8(R, C, x.device)
    if R:
        with _on(x.device):
            rc = _lib.load().gridgcn_act8_pack(_p(x2), _DTYPES[x.dtype], R, C, ld, _p(codes), _p(scales), _st(x))
        _lib.check(rc, "gridgcn_act8_pack")
    return codes.view(lead + (codes.shape[1],)), scales.view(lead + (scales.shape[1],))


@torch.no_grad()
def act8_unpack(codes, scales, C, dtype=torch.float32):
    """The values [..., C] that (codes, scales) of act8_pack stand for (exact in float32 and bfloat16; in float16 if
    they were packed from float16, but for 65536: infinite)."""
    C = int(C)
    _require(1 <= C <= ACT8_MAX_C, "C must be 1..%d" % ACT8_MAX_C)
    _check_codes(codes, scales, None, C)
    _require(dtype in _DTYPES, "dtype must be float32, bfloat16 or float16")
    lead = tuple(codes.shape[:-1])
    x = torch.empty(lead + (C,), dtype=dtype, device=codes.device)
    R = x.numel() // C
    if R:
        with _on(codes.device):
            rc = _lib.load().gridgcn_act8_unpack(_p(codes), _p(scales), R, C, _DTYPES[dtype], _p(x), C, _st(codes))
        _lib.check(rc, "gridgcn_act8_unpack")
    return x


def _check_codes(codes, scales, rows, C):
    c, s = act8_shapes(1, C)
    for t, name, w in ((codes, "codes", c[1]), (scales, "scales", s[1])):
        _require(isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == torch.uint8 and t.is_contiguous() and t.dim() >= 1,
                 "%s must be a contiguous uint8 GPU tensor" % name)
        _require(t.shape[-1] == w, "last dim of %s should be %d for %d channels" % (name, w, C))
        _require(rows is None or t.numel() == rows * w, "%s should have %s rows" % (name, rows))
    _require(codes.shape[:-1] == scales.shape[:-1] and codes.device == scales.device, "codes and scales do not belong together")
    _require(codes.data_ptr() % 16 == 0, "codes must be 16-byte aligned")


# ---- group normalisation + activation -------------------------------------------------------------------------------
def _check_param(t, name, x, C):
    _require(isinstance(t, torch.Tensor) and t.device == x.device and t.dim() == 1 and t.shape[0] == C,
             "%s should be a [%d] tensor on the device of x" % (name, C))
    _require(t.dtype == torch.float32 or t.dtype == x.dtype, "%s must be float32 or of x's type" % name)
    return t.dtype


def _check_gn(x, weight, bias, groups, eps, act, counts):
    _check_rows(x, "x", 2)
    C = x.shape[-1]
    groups = int(groups)
    _require(1 <= C <= GN_MAX_C, "x must have 1..%d channels" % GN_MAX_C)
    _require(x.shape[0] <= 65535, "x may have at most 65535 samples")
    _require(groups >= 1 and C % groups == 0, "%d channels cannot be cut into %d groups" % (C, groups))
    _require(act in ACTS, "act must be one of none, relu, silu, gelu")
    _require(0.0 <= eps < float("inf"), "eps must be finite and >= 0")
    ptype = torch.float32
    if weight is not None:
        ptype = _check_param(weight, "weight", x, C)
    if bias is not None:
        t = _check_param(bias, "bias", x, C)
        _require(weight is None or t == ptype, "weight and bias must have one type")
        ptype = t
    if counts is not None:
        _require(isinstance(counts, torch.Tensor) and counts.device == x.device and counts.dtype == torch.int32,
                 "counts must be an int32 tensor on the device of x")
        _require(x.dim() == 3, "counts need x as [B, N, C]")
        _require(counts.numel() == x.shape[0] and counts.is_contiguous(), "counts should be a [B,1] tensor")
    return C, groups, _DTYPES[ptype]


@functools.lru_cache(maxsize=1024)
def _gn_workspace_bytes(B, N, C, groups, dt, save8, stats, backward):
    nb = ctypes.c_size_t(0)
    _lib.check(_lib.load().gridgcn_group_norm_act_workspace_bytes(B, N, C, groups, dt, save8, stats, backward, ctypes.byref(nb)),
               "gridgcn_group_norm_act_workspace_bytes")
    return nb.value


def _gn_forward(x, weight, bias, groups, ptype, eps, act, counts, save8, stats):
    """-> (y, x as [B, N, C] rows, stats or None, codes, scales)"""
    lib, dev = _lib.load(), x.device
    B, C = x.shape[0], x.shape[-1]
    x3, sb, sn = _rows3(x, B)
    N, dt = x3.shape[1], _DTYPES[x.dtype]
    nb = _gn_workspace_bytes(B, N, C, groups, dt, int(save8), int(stats), 0)
    with _on(dev):
        y = torch.empty(x.shape, dtype=x.dtype, device=dev)
        st = torch.empty((B, groups, 2), dtype=torch.float64, device=dev) if stats else None
        codes, scales = _new_act8(B * N, C, dev) if save8 else (None, None)
        ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
        w, b = _packed(weight), _packed(bias)
        rc = lib.gridgcn_group_norm_act_fwd(x3.data_ptr(), dt, B, N, C, sb, sn, groups, _p(w), _p(b), ptype, _p(counts), eps,
                                            ACTS[act], y.data_ptr(), _p(st), _p(codes), _p(scales), _p(ws), nb, _st(x))
    _lib.check(rc, "gridgcn_group_norm_act_fwd")
    return y, x3, st, codes, scales


def _gn_backward(dy, x3, codes, scales, stats, weight, bias, shape, groups, ptype, act, counts, need):
    """gradients of x (shape `shape`), weight and bias; need: which of the three"""
    lib, dev = _lib.load(), dy.device
    B, C = shape[0], shape[-1]
    g3, gb, gn = _rows3(dy, B)
    N, dt = g3.shape[1], _DTYPES[dy.dtype]
    xb = xn = 0
    if codes is None:
        xb, xn = (x3.stride(0) if B > 1 else 0), (x3.stride(1) if N > 1 else C)
    nb = _gn_workspace_bytes(B, N, C, groups, dt, 0, 1, 1)
    with _on(dev):
        dx = torch.empty(shape, dtype=dy.dtype, device=dev) if need[0] else None
        dw = torch.empty(C, dtype=weight.dtype, device=dev) if need[1] else None
        db = torch.empty(C, dtype=bias.dtype, device=dev) if need[2] else None
        ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
        w, b = _packed(weight), _packed(bias)
        rc = lib.gridgcn_group_norm_act_bwd(g3.data_ptr(), gb, gn, _p(x3), xb, xn, _p(codes), _p(scales), dt, B, N, C, groups,
                                            stats.data_ptr(), _p(w), _p(b), ptype, _p(counts), ACTS[act], _p(dx), _p(dw),
                                            _p(db), _p(ws), nb, _st(dy))
    _lib.check(rc, "gridgcn_group_norm_act_bwd")
    return dx, dw, db


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, counts, groups, ptype, eps, act, save8):
        ctx.meta = (tuple(x.shape), groups, ptype, act)
        y, x3, st, codes, scales = _gn_forward(x, weight, bias, groups, ptype, eps, act, counts, save8, True)
        ctx.save_for_backward(None if save8 else x3, codes, scales, st, weight, bias, counts)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x3, codes, scales, st, weight, bias, counts = ctx.saved_tensors
        shape, groups, ptype, act = ctx.meta
        dx, dw, db = _gn_backward(dy, x3, codes, scales, st, weight, bias, shape, groups, ptype, act, counts,
                                  ctx.needs_input_grad[:3])
        return dx, dw, db, None, None, None, None, None, None


def group_norm_act(x, weight, bias, groups, eps=1e-5, act="relu", counts=None, save8=False):
    """y = act(group_norm(x) * weight + bias) on channels-last x [B, ..., C]; C in `groups` groups of consecutive channels,
    statistics per (sample, group) over all positions in between ([B, C]: over the group's channels alone).  At most
    65535 samples and 8192 channels.

    weight, bias: [C] or None, float32 or x's type.  act: 'none' | 'relu' | 'silu' | 'gelu'.
    counts: int32 [B] or [B, 1] with x [B, N, C]: rows n >= counts[b] (an index operator's unused centres) are in no
    statistics; their output and gradient are 0 and what they hold is never read.
    save8: keep x for the backward in 8 bits (act8_pack) instead of x itself: 1.03 bytes a value.  The gradients are then those of
    the formulas at the 8-bit values of x, with the statistics of x.
    Not differentiable twice, nor in forward mode."""
    eps = float(eps)
    C, groups, ptype = _check_gn(x, weight, bias, groups, eps, act, counts)
    _no_tangents("group_norm_act", x, weight, bias)
    if x.numel() == 0:
        y = x * 0
        for t in (weight, bias):
            y = y if t is None else y + (t.sum() * 0).to(x.dtype)
        return y
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or
                                    (bias is not None and bias.requires_grad)):
        return _GroupNormAct.apply(x, weight, bias, counts, groups, ptype, eps, act, bool(save8))
    return _gn_forward(x, weight, bias, groups, ptype, eps, act, counts, False, False)[0]


# ---- linear layer with an 8-bit checkpoint --------------------------------------------------------------------------
def _check_linear(x, weight, bias):
    _check_rows(x, "x")
    K = x.shape[-1]
    _require(isinstance(weight, torch.Tensor) and weight.dim() == 2 and weight.device == x.device and weight.dtype == x.dtype,
             "weight should be a 2D tensor of x's type on the device of x")
    N = weight.shape[0]
    _require(weight.shape[1] == K, "weight should be [N, %d]" % K)
    _require(1 <= K <= ACT8_MAX_C and 1 <= N <= ACT8_MAX_C, "1..%d channels" % ACT8_MAX_C)
    if bias is not None:
        _require(isinstance(bias, torch.Tensor) and bias.device == x.device and bias.dtype == x.dtype and
                 tuple(bias.shape) == (N,), "bias should be a [%d] tensor of x's type on the device of x" % N)
    return K, N


@functools.lru_cache(maxsize=1024)
def _linear_workspace_bytes(R, K, N, dt, backward):
    nb = ctypes.c_size_t(0)
    _lib.check(_lib.load().gridgcn_linear_act8_workspace_bytes(R, K, N, dt, backward, ctypes.byref(nb)),
               "gridgcn_linear_act8_workspace_bytes")
    return nb.value


def _linear_forward(x, weight, bias, save8):
    lib, dev = _lib.load(), x.device
    N, K = weight.shape
    x2, ld = _rows2(x)
    R, dt = x2.shape[0], _DTYPES[x.dtype]
    nb = _linear_workspace_bytes(R, K, N, dt, 0)
    with _on(dev):
        y = torch.empty(x.shape[:-1] + (N,), dtype=x.dtype, device=dev)
        codes, scales = _new_act8(R, K, dev) if save8 else (None, None)
        ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
        w, b = _packed(weight), _packed(bias)
        rc = lib.gridgcn_linear_act8_fwd(x2.data_ptr(), dt, R, K, ld, w.data_ptr(), _p(b), N, y.data_ptr(), _p(codes),
                                         _p(scales), _p(ws), nb, _st(x))
    _lib.check(rc, "gridgcn_linear_act8_fwd")
    return y, codes, scales


def _linear_backward(dy, weight, codes, scales, x_shape, need):
    """gradients of x, weight and bias; need: which of the three"""
    lib, dev = _lib.load(), dy.device
    N, K = weight.shape
    g2, ld = _rows2(dy)
    R, dt = g2.shape[0], _DTYPES[dy.dtype]
    nb = _linear_workspace_bytes(R, K, N, dt, 1)
    with _on(dev):
        dx = torch.empty(x_shape, dtype=dy.dtype, device=dev) if need[0] else None
        dw = torch.empty((N, K), dtype=dy.dtype, device=dev) if need[1] else None
        db = torch.empty(N, dtype=dy.dtype, device=dev) if need[2] else None
        ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
        w = _packed(weight) if need[0] else None
        rc = lib.gridgcn_linear_act8_bwd(g2.data_ptr(), dt, R, N, ld, _p(w), K, _p(codes), _p(scales), _p(dx),
                                         _p(dw), _p(db), _p(ws), nb, _st(dy))
    _lib.check(rc, "gridgcn_linear_act8_bwd")
    return dx, dw, db


class _LinearAct8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        ctx.x_shape = tuple(x.shape)
        y, codes, scales = _linear_forward(x, weight, bias, ctx.needs_input_grad[1])
        ctx.save_for_backward(codes, scales, weight)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        codes, scales, weight = ctx.saved_tensors
        need = ctx.needs_input_grad
        return _linear_backward(dy, weight, codes, scales, ctx.x_shape, need)


def linear_act8(x, weight, bias=None):
    """y = x W^T + bias on x [..., K], weight [N, K], bias [N] (all of one type: float32, bfloat16 or float16), keeping for the
    backward the 8-bit form of x (act8_pack) instead of x: 1.03 bytes a value, written in the forward's pass over x.

    Sums are in float32.  A float32 operand enters the matrix instructions as a sum of three bfloat16 numbers, whatever stands
    beside it in its row and however many rows there are; the error of a product is that of a float32 product, but an operand that is
    infinite or beyond 3.39e38 gives NaN, and what of an operand lies below 2^-134 is dropped.
    Backward: dx = dy W and dbias as ever; dW = dy^T x^ with x^ the 8-bit values of x.  Not differentiable twice, nor in forward mode."""
    K, N = _check_linear(x, weight, bias)
    _no_tangents("linear_act8", x, weight, bias)
    if x.numel() == 0:
        return torch.nn.functional.linear(x, weight, bias)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        return _LinearAct8.apply(x, weight, bias)
    return _linear_forward(x, weight, bias, False)[0]
