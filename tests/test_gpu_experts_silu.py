"""SiLU(gate) * up in the experts' layer at gates whose exponential is near the end of fp32's range."""
import math

import pytest
import torch

import vq_gemm_b200 as V
from vq_gemm_b200 import quantize

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [8, 40, 400])
@pytest.mark.parametrize("gate", [-60.0, -87.0, -87.5, -88.0, -88.5, -90.0, -91.0, 88.0])
def test_silu_near_the_end_of_the_exponentials_range(t, gate):
    # one expert, one input of 1, weights of one code step: gate and up are exact, so the only errors are those of the exponential
    # (half a step of an argument below 2^8: 2^-16), a few of 2^-22, and the roundings of h and y, half a step of bf16 each
    up_size = 2.0 ** 100 if gate < 0 else 1.0
    one = quantize.int4_pack(torch.full((1, 64, 32), 9, dtype=torch.uint8)).cuda()
    scales = torch.tensor([gate, up_size]).repeat(32).to(torch.bfloat16).reshape(1, 1, 64).cuda()
    down = quantize.int4_pack(torch.full((1, 32, 32), 9, dtype=torch.uint8)).cuda()
    x = torch.zeros(t, 32, dtype=torch.bfloat16, device="cuda")
    x[:, 3] = 1
    ids, w = torch.zeros(t, 1, dtype=torch.int32, device="cuda"), torch.ones(t, 1, device="cuda")
    y = V.int4_experts(x, ids, w, (one, scales, None), (down, torch.ones(1, 1, 32, dtype=torch.bfloat16, device="cuda"), None))
    gate = float(torch.tensor(gate).bfloat16())
    want = 32 * gate / (1 + math.exp(-gate)) * up_size
    assert bool(((y.double() / want - 1).abs() <= 2 * 2.0 ** -8 + 2.0 ** -14).all()), (float(y[0, 0]), want)
