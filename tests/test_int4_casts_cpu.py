"""What a cast of a model does to the 4-bit layers' buffers, without a GPU."""
import copy

import pytest
import torch

from tests.test_int4_cpu import _packed
from vq_gemm_b200.linear import Int4Experts, Int4Linear

TYPES = [torch.float16, torch.bfloat16, torch.float32, torch.float64]


def experts(dtype=torch.float16, bias=True):
    up, down = _packed(64, 96, 32, dtype, lead=(4,))[1:], _packed(96, 32, 32, dtype, True, lead=(4,), seed=1)[1:]
    return Int4Experts(torch.nn.Linear(96, 4), up, down, top_k=2, in_features=96,
                       bias=torch.randn(4, generator=torch.Generator().manual_seed(3)) * 0.05 if bias else None)


@pytest.mark.parametrize("to", TYPES)
def test_the_balance_bias_keeps_its_bits(to):
    layer = experts()
    was = layer.bias.clone()
    for cast in (layer.to(to), copy.deepcopy(layer).to("cpu", to), torch.nn.Sequential(layer).to(to)[0]):
        assert cast.bias.dtype == torch.float32 and torch.equal(cast.bias, was) and cast.router.weight.dtype == to
    assert experts(bias=False).to(to).bias is None


def test_the_balance_bias_follows_to_another_device():
    layer = experts().half().to("meta")
    assert layer.bias.device.type == "meta" and layer.bias.dtype == torch.float32
    assert experts().to("meta", torch.bfloat16).bias.dtype == torch.float32
    other = experts().half()
    other.load_state_dict({k: v + 1 if k == "bias" else v for k, v in other.state_dict().items()})
    assert other.bias.dtype == torch.float32


@pytest.mark.parametrize("own", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("to", TYPES)
def test_the_weights_keep_their_bits(own, to):
    _, packed, scales, zeros = _packed(20, 96, 32, own, True)
    layer = Int4Linear(packed, scales, zeros, torch.randn(20), in_features=96)
    was = {k: v.clone() for k, v in layer.state_dict().items()}
    assert layer.result_type is None and layer.cpu().result_type is None and layer.share_memory().result_type is None
    assert layer.to("cpu", non_blocking=True).result_type is None
    for cast in (copy.deepcopy(layer).to(to), copy.deepcopy(layer).half().to(to), torch.nn.Sequential(copy.deepcopy(layer)).to("cpu", to)[0]):
        assert cast.result_type == to
        assert all(v.dtype == was[k].dtype and torch.equal(v, was[k]) for k, v in cast.state_dict().items())
    assert copy.deepcopy(layer).half().float().half().result_type == torch.float16
    up = experts(own)
    was = {k: v.clone() for k, v in up.state_dict().items()}
    assert all(v.dtype == was[k].dtype and torch.equal(v, was[k]) for k, v in up.to(to).state_dict().items() if "router" not in k)
    assert up.result_type == to and up.to("meta").gate_up_scales.dtype == own and up.down_scales.device.type == "meta"
    empty = Int4Linear(packed, scales, zeros, in_features=96).to("meta").to_empty(device="cpu")
    assert empty.scales.dtype == own and empty.scales.device.type == "cpu" and empty.result_type is None
