"""Shared cases of tests/test_act8.py (CPU: the kernels under the emulator) and tests/test_gpu_act8.py (MI355X)."""
import torch

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DTYPES = [F32, BF16, F16]


def rows(lead, C, dtype, seed, pad=0, kind="pre"):
    """CPU values [*lead, C], columns of a buffer of C + pad"""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*lead, C + pad, generator=g)
    if kind == "pre":
        x = x * (torch.rand(C + pad, generator=g) + 0.5) + torch.randn(C + pad, generator=g)
    elif kind == "act":
        x = x.clamp(min=0)
    return x.to(dtype)[..., :C]


def special_rows(dtype):
    """rows of one block each, where the 8-bit form can go wrong"""
    f = torch.finfo(dtype)
    r = [torch.zeros(32)]
    for top in (448.0, 449.0, 447.9, 1.75, 1.7501, 1.0, f.max, f.tiny, f.smallest_normal * f.eps, 2.0 ** -14):
        v = torch.linspace(-1, 1, 32) * min(top, f.max)
        v[5] = top
        r.append(v)
    ties = torch.tensor([1.0625 + 0.125 * i for i in range(16)] + [2.0 ** -10 * (2 * i + 1) for i in range(15)] + [448.0])
    r += [ties, -ties]
    v = torch.arange(32.0)
    for bad in (float("inf"), float("-inf"), float("nan")):
        w = v.clone()
        w[7] = bad
        r.append(w)
    r.append(torch.full((32,), float("inf")))
    r.append(torch.full((32,), 2.0 ** -140))
    return torch.stack(r).to(dtype)


PACK = [(1, 1, 0), (3, 31, 0), (5, 32, 8), (7, 33, 1), (2, 1027, 0), (70, 131, 3), (9, 64, 5), (33, 512, 0)]

# B, N, C, groups, act, ragged, save8, pad
GN = [
    (1, 1, 4, 1, "none", False, False, 0),
    (3, 1, 96, 3, "relu", False, True, 0),
    (2, 7, 5, 5, "silu", False, False, 1),          # groups of one channel
    (2, 9, 6, 2, "gelu", True, True, 3),
    (4, 33, 64, 8, "relu", True, True, 0),
    (3, 40, 66, 2, "silu", True, False, 5),         # groups that end inside a 16-byte chunk
    (2, 17, 131, 1, "gelu", False, True, 0),        # one group of an odd width
    (1, 300, 256, 32, "relu", False, False, 8),
    (5, 3, 320, 16, "silu", True, True, 0),
    (2, 2500, 16, 2, "relu", True, True, 0),        # many rows: two passes
    (1, 2100, 21, 7, "gelu", False, False, 2),
    (2, 600, 96, 1, "silu", True, False, 0),        # one group of many values: two passes
    (2, 20, 1100, 4, "none", False, True, 0),       # more channels than a workgroup's columns
]

# R, K, N, bias, pad
LINEAR = [
    (1, 1, 1, True, 0),
    (1, 34, 5, False, 0),
    (31, 64, 32, True, 0),
    (33, 65, 33, True, 1),
    (5, 3, 130, False, 0),
    (70, 131, 128, True, 5),
    (64, 520, 40, True, 0),
    (300, 40, 129, False, 8),
    (17, 192, 260, True, 0),
    (260, 35, 5600, True, 0),          # enough workgroups for the kernel of many rows: forward ...
    (260, 5600, 35, False, 1),         # ... and dx
]
