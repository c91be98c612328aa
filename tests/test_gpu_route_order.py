"""The router's order where 32 bits do not show it: what it answers is the definition's order in 64 bits."""
import numpy as np
import pytest
import torch

import vq_gemm_b200 as V
from oracle import int4_oracle as O

pytestmark = pytest.mark.gpu


def check(x, k, **kw):
    w, i = V.route_experts(x, k, **kw)
    want, ids = O.route(x, k, **kw)
    wrong = (i.cpu() != ids).any(-1)
    assert not wrong.any(), (int(wrong.sum()), len(wrong), x[wrong.to(x.device)][:2], i.cpu()[wrong][:2], ids[wrong][:2])
    # p = exp(d) / sum, d >= -104 where p is not zero in fp32: half a step of d (2^-24 of it), the exponential 2^-22, a sum of at
    # most 21 roundings and the divisions, below (104 + 40) 2^-24 of p in all; below the normal numbers p has fewer bits
    assert bool(((w.cpu().double() - want).abs() <= want.abs() * 2.0 ** -16 + 1e-37).all())


def logit_of(p):
    return np.log(p / (1 - p))


def groups_of_equal_sums(rows, groups, apart, seed):
    """p [rows, groups, 2]: pairs whose sums differ by about `apart`"""
    g = np.random.default_rng(seed)
    total = g.uniform(0.8, 1.2, (rows, 1)) + g.normal(0, apart, (rows, groups))
    first = g.uniform(0.25, 0.55, (rows, groups))
    return np.stack((first, total - first), -1)


def test_groups_whose_large_biases_cancel_one_row():
    x = torch.tensor([[1.75845480, 0.46500289, 1.75849342, 0.46500289]]).cuda()
    bias = torch.tensor([64.0, -64.0, 80.0, -80.0]).cuda()
    check(x, 2, scoring="sigmoid", bias=bias, groups=2, top_groups=1)


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("size", [1.0, 64.0, 1000.0])
def test_groups_whose_large_biases_cancel(scoring, size):
    p = groups_of_equal_sums(1500, 4, 2e-6 if size < 100 else 2e-5, 7).reshape(1500, 8)
    x = torch.from_numpy(logit_of(p) if scoring == "sigmoid" else np.log(p)).float().cuda()
    b = torch.tensor([size, 1.125 * size, 1.25 * size, 1.5 * size])
    bias = torch.stack((b, -b), -1).flatten().cuda()
    check(x, 4, scoring=scoring, bias=bias, groups=4, top_groups=2)


def test_softmax_with_a_bias_that_takes_a_large_p_back():
    # two experts of small p whose choices are a few steps of fp32 apart, and one whose large p its negative bias takes back: its choice
    # is only known to some 1e-7
    g = np.random.default_rng(5)
    for e, k in ((4, 1), (4, 2), (40, 1), (70, 3)):
        for _ in range(60):
            x = np.full(e, -60.0)
            big, small, other, middle = g.permutation(e)[:4]
            x[big] = g.uniform(0, 3)
            x[small], x[other] = x[big] - 11 + g.normal(0, 0.5, 2)
            x[middle] = x[big] - g.uniform(0.1, 4)
            x = torch.from_numpy(x).float()[None]
            p = torch.softmax(x.double(), -1)[0]
            bias = torch.full((e,), -2.0)
            bias[small], bias[other] = 0.01, 0.01 + float(p[small] - p[other] + g.uniform(-1e-8, 1e-8))
            bias[big] = float(0.01 + p[small] + g.uniform(-1e-7, 1e-7) - p[big])
            check(x.cuda(), k, bias=bias.cuda())


@pytest.mark.parametrize("low,high", [(40, 63), (63, 87), (87, 104)])
@pytest.mark.parametrize("group_score", ["top2", "max"])
def test_softmax_groups_far_below_the_largest_logit(low, high, group_score):
    g = np.random.default_rng(int(low))
    rows, apart = 4000, 1e-5
    x = np.empty((rows, 3, 2))
    x[:, 0] = 16.75, -30.0
    depth = 16.75 - g.uniform(low, high, (rows, 1, 1))
    if group_score == "top2":
        x[:, 1:] = depth + np.log(groups_of_equal_sums(rows, 2, apart, low))
    else:
        x[:, 1:, :1] = depth + g.normal(0, apart, (rows, 2, 1))
        x[:, 1:, 1:] = x[:, 1:, :1] - 1
    order = torch.from_numpy(x.reshape(rows, 6)).float().cuda()
    check(order, 4, groups=3, top_groups=2, group_score=group_score)


def test_ties_of_64_bits_between_logits_that_differ():
    x = torch.full((4, 64), -1.0)
    x[0, 5], x[0, 6], x[0, 0] = 40.0, 40.0, 39.875          # sigmoid: p = 1 in 64 bits
    x[1, 9:] = 40.0
    x[1, 3] = 38.0
    x[2] = 0.0                                              # softmax: exp(-1e-20) = 1
    x[2, 40:50] = 1e-20
    x[3, 60] = 800.0                                        # softmax: the others' p is zero
    x[3, 20:30] = -0.5
    for k in (1, 2, 12):
        for scoring in ("softmax", "sigmoid"):
            check(x.cuda(), k, scoring=scoring)
            check(x[:, :8].contiguous().cuda(), min(k, 8), scoring=scoring)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (8, 3)])
def test_biases_of_every_size_and_sign(scoring, groups, top_groups):
    g = torch.Generator().manual_seed(8)
    x = torch.randn(200, 64, generator=g) * 1.5
    for size in (1e-6, 1.0, 64.0, 1e6, 1e30):
        bias = torch.randint(-2, 3, (64,), generator=g).float() * size            # many experts share one
        bias[5], bias[40] = -float("inf"), torch.finfo(torch.float32).min
        check(x.cuda(), 8, scoring=scoring, bias=bias.cuda(), groups=groups, top_groups=top_groups)
