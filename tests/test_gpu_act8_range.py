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
