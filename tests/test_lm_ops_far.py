"""Token log probabilities and distillation of rows far from 0 and of masks of the type's lowest value, on the CPU and the GPU."""
import math

import pytest
import torch
from test_lm_ops_cpu import check_distill, check_tokens

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _rows(dtype):
    torch.manual_seed(0)
    x = 2 * torch.randn(6, 40)
    x[0] = torch.finfo(dtype).min               # nothing but the mask: all equal
    x[1, torch.rand(40) < 0.5] = torch.finfo(dtype).min
    x[2] = 2e6 + torch.floor(x[2])
    x[3] = -2e6 + torch.floor(x[3])
    x[4, 1:] = -math.inf
    x[5] = -3e38
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [1.0, 0.5, 2.0 ** -10, 2.0])
@pytest.mark.parametrize("device", DEVICES)
def test_log_probabilities_of_rows_far_from_zero(device, dtype, temperature):
    x = _rows(dtype).to(device)
    tok = x.float().argmax(1)
    g = torch.randn(6, device=device)
    check_tokens(x, tok, 0, temperature, g, g)
    check_tokens(x, tok, 1, temperature)


@pytest.mark.parametrize("temperature", [1.0, 0.5, 2.0])
@pytest.mark.parametrize("device", DEVICES)
def test_distillation_of_rows_far_from_zero(device, temperature):
    x = _rows(torch.float32)[[0, 1, 2, 3, 5]]
    ids = x.argsort(1, descending=True)[:, :3]
    t = torch.randn(5, 3)
    t[0] = torch.finfo(torch.float32).min       # a teacher of nothing but the mask: all equal
    t[1, 2] = torch.finfo(torch.float32).min
    t[2] += 2.0 ** 20
    check_distill(x.to(device), t.to(device), ids.to(device), None, temperature)
