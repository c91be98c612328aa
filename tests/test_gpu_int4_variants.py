"""Products and experts' layers at sizes of large models: long rows of X, which the few-rows kernels read from memory instead of shared
memory, wide hidden and inner dimensions, and either side of the choice between the kernels."""
import pytest
import torch

import vq_gemm_b200 as V
from oracle import int4_oracle as O
from tests.test_gpu_experts import choices
from tests.test_gpu_int4 import BF16, F16, acts, check, make
from vq_gemm_b200.linear import Int4Experts, Int4Linear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,zeros,group", [(F16, True, 64), (BF16, False, 32)])
@pytest.mark.parametrize("m,n,k", [(8, 100, 8192), (5, 33, 20032), (9, 77, 9024), (12, 130, 7232), (16, 50, 4224), (16, 300, 8192), (24, 40, 8192)])
def test_products_of_few_long_rows(m, n, k, dtype, zeros, group):
    w, x = make(n, k, group, dtype, zeros, seed=m + n), acts(m, k, dtype, seed=m)
    y = V.int4_gemm(x, *w)
    check(y, O.gemm(x, *w))
    assert torch.equal(V.int4_gemm(x, *w), y)


# tokens, choices, experts, hidden, inner: over 32 slots, under 11 per expert; chunks of 8 rows up to 5 per expert, else of 16
@pytest.mark.parametrize("dtype,zeros,group", [(F16, False, 128), (BF16, True, 32)])
@pytest.mark.parametrize("t,k,e,hidden,inner", [(12, 4, 16, 4096, 128), (30, 4, 16, 4096, 128), (16, 8, 32, 2304, 160), (40, 4, 16, 2304, 160),
                                                (12, 4, 16, 128, 4096), (30, 4, 16, 128, 4096)])
def test_planned_experts_of_few_long_rows(t, k, e, hidden, inner, dtype, zeros, group):
    group = 32 if inner % group else group
    up, down = make(2 * inner, hidden, group, dtype, zeros, (e,), seed=t), make(hidden, inner, group, dtype, zeros, (e,), seed=t + 1)
    x = acts(t, hidden, dtype, seed=t)
    ids, w = choices(t, k, e, seed=t, drop=0.1)
    y = V.int4_experts(x, ids, w, up, down)
    check(y, O.experts(x, ids, w, up, down))
    assert torch.equal(V.int4_experts(x, ids, w, up, down), y)


@pytest.mark.parametrize("t", [1, 16, 17, 60])
@pytest.mark.parametrize("hidden,inner,e", [(7168, 640, 8), (256, 14336, 4), (4096, 1536, 8)])
def test_experts_of_large_models(t, hidden, inner, e):
    up, down = make(2 * inner, hidden, 128, BF16, False, (e,), seed=t), make(hidden, inner, 128, BF16, False, (e,), seed=t + 1)
    x = acts(t, hidden, BF16, seed=t)
    ids, w = choices(t, 2, e, seed=t)
    check(V.int4_experts(x, ids, w, up, down), O.experts(x, ids, w, up, down))
    assert V.device_status() == 0


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_cast_layer_routes_with_the_balance_bias_it_was_given(dtype):
    # biases whose order neither 16-bit type holds: logits are all equal, so the largest biases choose
    e = 32
    up, down = make(64, 128, 64, dtype, False, (e,)), make(128, 32, 32, dtype, False, (e,))
    bias = 0.05 + torch.randperm(e, generator=torch.Generator().manual_seed(4)).float() * 1e-6
    router = torch.nn.Linear(128, e, bias=False).requires_grad_(False)
    router.weight.zero_()
    layer = Int4Experts(router, up, down, top_k=2, in_features=128, scoring="sigmoid", bias=bias).cuda().to(dtype)
    x = acts(5, 128, dtype)
    w, ids = V.route_experts(layer.router(x), 2, scoring="sigmoid", bias=bias.cuda(), renormalize=True)
    assert torch.equal(ids[0].cpu(), bias.topk(2).indices.int())
    assert torch.equal(layer(x), V.int4_experts(x, ids, w, up, down))


@pytest.mark.parametrize("own", [F16, BF16])
@pytest.mark.parametrize("to", [F16, BF16, torch.float32])
def test_cast_layers_multiply_the_same_weights_and_answer_in_the_models_type(own, to):
    packed, scales, zeros = make(40, 128, 32, own, True)
    bias = torch.linspace(-1, 1, 40)
    layer = Int4Linear(packed, scales, zeros, bias.cuda(), 128)
    model = torch.nn.Sequential(layer, torch.nn.Linear(40, 8).requires_grad_(False)).cuda().to(to)
    x = acts(6, 128, torch.float32).to(to)
    y = layer(x)
    assert y.dtype == to and torch.equal(y, (V.int4_gemm(x.to(own), packed, scales, zeros) + bias.to(own).cuda()).to(to))
    assert model(x).dtype == to
    assert torch.equal(torch.compile(layer, backend="eager", fullgraph=True)(x), y)
    up, down = make(64, 128, 64, own, False, (8,)), make(128, 32, 32, own, False, (8,))
    moe = Int4Experts(torch.nn.Linear(128, 8, bias=False).requires_grad_(False), up, down, top_k=2, in_features=128).cuda().to(to)
    w, ids = V.route_experts(moe.router(x), 2, renormalize=True)
    y = moe(x)
    assert y.dtype == to and torch.equal(y, V.int4_experts(x.to(own), ids, w, up, down).to(to))


@pytest.mark.parametrize("dtype,zeros", [(F16, True), (BF16, False)])
@pytest.mark.parametrize("t,k,e,hidden,inner", [(3, 2, 2, 96, 64), (8, 2, 8, 1024, 512), (12, 2, 8, 1024, 512), (3, 8, 64, 512, 256), (4, 8, 64, 2048, 96),
                                                (2, 4, 2, 64, 32), (32, 1, 1, 128, 128), (5, 6, 3, 2080, 1024), (4, 2, 2, 4096, 4256)])
def test_few_slots_either_side_of_the_plan(t, k, e, hidden, inner, dtype, zeros):
    up, down = make(2 * inner, hidden, 32, dtype, zeros, (e,), seed=t), make(hidden, inner, 32, dtype, zeros, (e,), seed=t + 1)
    x = acts(t, hidden, dtype, seed=t)
    ids = torch.randint(-1, e, (t, k), dtype=torch.int32, generator=torch.Generator().manual_seed(t)).cuda()      # repeats and dropped ones
    w = torch.rand(t, k, generator=torch.Generator().manual_seed(k)).cuda()
    y = V.int4_experts(x, ids, w, up, down)
    check(y, O.experts(x, ids, w, up, down))
    assert torch.equal(V.int4_experts(x, ids, w, up, down), y) and V.device_status() == 0
