"""Routing to experts and the experts' products against the 64-bit restatement."""
import pytest
import torch

import vq_gemm_b200 as V
from oracle import int4_oracle as O
from tests.test_gpu_int4 import BF16, F16, acts, check, make
from vq_gemm_b200.linear import Int4Experts, Int4Linear

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def logits(t, e, dtype=torch.float32, seed=0):
    return (torch.randn(t, e, generator=torch.Generator().manual_seed(seed)) * 1.5).to(dtype).cuda()


def check_route(x, k, **kw):
    w, i = V.route_experts(x, k, **kw)
    want, ids = O.route(x, k, **{n: v for n, v in kw.items()})
    assert w.dtype == torch.float32 and i.dtype == torch.int32 and w.shape == i.shape == (x.shape[0], k)
    assert torch.equal(i.cpu(), ids), (i.cpu() != ids).nonzero()[:5]
    # fp32: exponential and division off by a few steps, the exponent's argument by half a step of at most 2^6, sums of
    # at most 512 terms in trees
    assert bool(((w.cpu().double() - want).abs() <= want.abs() * 2.0 ** -17 + 1e-37).all()), float((w.cpu().double() - want).abs().max())
    return w, i


@pytest.mark.parametrize("e,k", [(1, 1), (2, 1), (8, 2), (33, 5), (64, 8), (65, 3), (128, 6), (160, 10), (256, 8), (384, 32), (512, 8)])
@pytest.mark.parametrize("scoring,bias", [("softmax", False), ("sigmoid", False), ("sigmoid", True), ("softmax", True)])
def test_route(e, k, scoring, bias):
    b = torch.randn(e, generator=torch.Generator().manual_seed(e)).cuda() * 0.1 if bias else None
    for t, dtype in ((1, torch.float32), (5, BF16), (67, F16)):
        check_route(logits(t, e, dtype, e + t), k, scoring=scoring, bias=b, renormalize=t != 5, scale=2.5 if t == 67 else 1.0)


@pytest.mark.parametrize("e,groups,top_groups,k", [(8, 2, 1, 3), (64, 8, 3, 6), (160, 8, 3, 6), (256, 8, 4, 8), (32, 32, 5, 5), (96, 3, 2, 8),
                                                   (512, 16, 16, 8), (256, 32, 1, 8)])
@pytest.mark.parametrize("group_score", ["top2", "max"])
def test_route_with_groups(e, groups, top_groups, k, group_score):
    b = torch.randn(e, generator=torch.Generator().manual_seed(e)).cuda() * 0.1
    for scoring, bias in (("sigmoid", b), ("softmax", None)):
        check_route(logits(50, e, seed=e), k, scoring=scoring, bias=bias, groups=groups, top_groups=top_groups,
                    group_score=group_score, renormalize=True)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (4, 2)])
def test_route_of_masked_and_special_rows(scoring, groups, top_groups):
    x = logits(12, 16, seed=3)
    x[0] = -INF                       # nothing to choose
    x[1, 3:] = -INF                   # fewer than top_k
    x[2] = NAN
    x[3, ::2] = NAN
    x[4] = torch.finfo(torch.float32).min
    x[5, 4:8] = INF                   # takes all of the softmax
    x[6] = 0.0                        # all equal: the lowest indices
    x[7] = 1e4 * x[7]                 # softmax of one expert, the others underflow
    x[8] = -1e4 * x[8].abs()          # sigmoid underflows
    x[9, 1:] = torch.finfo(torch.float32).min
    w, i = check_route(x, 6, scoring=scoring, groups=groups, top_groups=top_groups, renormalize=True)
    assert (i[0] == -1).all() and (w[0] == 0).all() and (i[2] == -1).all()
    check_route(x, 6, scoring=scoring, groups=groups, top_groups=top_groups)


def test_route_ties_in_coarse_logits_go_to_the_lower_index():
    x = (logits(300, 64, seed=5) * 2).round().div(2).to(BF16)          # many equal values
    for kw in (dict(), dict(scoring="sigmoid"), dict(scoring="sigmoid", groups=8, top_groups=3),
               dict(groups=8, top_groups=3, group_score="max")):
        check_route(x, 8, **kw)


def test_route_of_nearly_equal_choices():
    # values one fp32 step apart, and sums with a bias that differ only beyond fp32: the order is that of exact arithmetic
    e = 64
    base = torch.full((e,), 0.3)
    x = base.clone().view(torch.int32).add_(torch.randperm(e, generator=torch.Generator().manual_seed(1)).int()).view(torch.float32)
    rows = torch.stack([x, x.flip(0), x * 4, torch.full((e,), 0.3)]).cuda()
    bias = torch.randn(e, generator=torch.Generator().manual_seed(2)).cuda()
    for scoring in ("softmax", "sigmoid"):
        check_route(rows, 8, scoring=scoring)
        check_route(rows, 8, scoring=scoring, bias=bias * 1e-9)
        check_route(rows, 8, scoring=scoring, bias=bias * 1e-7, groups=8, top_groups=3)
        # choices that the bias makes equal up to rounding
        p = torch.sigmoid(rows[:1].double()) if scoring == "sigmoid" else torch.softmax(rows[:1].double(), -1)
        check_route(rows[:1].contiguous(), 8, scoring=scoring, bias=(0.7 - p[0]).float())


def test_route_refusals_and_empty_batch():
    x = logits(4, 16)
    w, i = V.route_experts(logits(0, 16), 2)
    assert w.shape == i.shape == (0, 2)
    for kw in (dict(top_k=0), dict(top_k=17), dict(top_k=2, scoring="linear"), dict(top_k=2, groups=3), dict(top_k=2, groups=4, top_groups=5),
               dict(top_k=2, bias=torch.zeros(15, device="cuda")), dict(top_k=2, bias=torch.zeros(16, device="cuda", dtype=F16)),
               dict(top_k=2, group_score="mean")):
        with pytest.raises(RuntimeError):
            V.route_experts(x, **kw)
    with pytest.raises(RuntimeError):
        V.route_experts(x.double(), 2)
    with pytest.raises(RuntimeError):
        V.route_experts(logits(4, 513), 2)
    with pytest.raises(RuntimeError):
        V.route_experts(x.t(), 2)


@pytest.mark.parametrize("scoring,bias,groups,top_groups", [("sigmoid", True, 8, 4), ("sigmoid", True, 1, 1), ("softmax", False, 8, 4), ("sigmoid", False, 1, 1)])
def test_rows_with_few_experts_left_and_with_none(scoring, bias, groups, top_groups):
    x = logits(40, 256, seed=11)
    g = torch.Generator(device=x.device).manual_seed(12)
    for row in range(20):                      # 0 ... 19 experts left
        left = torch.randperm(256, generator=g, device=x.device)[:row]
        kept = x[row, left].clone()
        x[row] = -INF
        x[row, left] = kept
    b = torch.randn(256, generator=g, device=x.device) * 0.05 if bias else None
    check_route(x, 8, scoring=scoring, bias=b, groups=groups, top_groups=top_groups, renormalize=True)
    w, ids = V.route_experts(x, 8, scoring=scoring, bias=b, groups=groups, top_groups=top_groups, renormalize=True)
    assert bool((ids[0] == -1).all()) and not bool(w[0].any())


def moe(e, hidden, inner, group, dtype, zeros, seed=0):
    return make(2 * inner, hidden, group, dtype, zeros, (e,), seed), make(hidden, inner, 32 if group > inner else group, dtype, zeros, (e,), seed + 1)


def choices(t, k, e, seed=0, drop=0.0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(e, generator=g)[:k] for _ in range(t)]).int()
    ids[torch.rand(t, k, generator=g) < drop] = -1
    w = torch.rand(t, k, generator=g) + 0.1
    return ids.cuda(), (w / w.sum(-1, keepdim=True)).cuda()


@pytest.mark.parametrize("dtype,zeros", [(F16, True), (BF16, False)])
@pytest.mark.parametrize("t,k,e,hidden,inner,group", [(1, 1, 1, 32, 32, 32), (1, 2, 4, 96, 32, 32), (1, 8, 16, 256, 160, 32), (4, 8, 64, 128, 64, 64),
                                                      (5, 3, 8, 192, 128, 64), (33, 1, 5, 64, 96, 32), (50, 8, 16, 256, 128, 128),
                                                      (200, 4, 6, 160, 224, 32), (300, 2, 3, 512, 256, 128), (700, 6, 8, 128, 64, 64)])
def test_experts(t, k, e, hidden, inner, group, dtype, zeros):
    up, down = moe(e, hidden, inner, group, dtype, zeros, seed=t)
    x = acts(t, hidden, dtype, seed=t) * 2
    ids, w = choices(t, k, e, seed=t, drop=0.1 if t > 4 else 0.0)
    y = V.int4_experts(x, ids, w, up, down)
    check(y, O.experts(x, ids, w, up, down))
    assert torch.equal(V.int4_experts(x, ids, w, up, down), y)          # the same bits every time
    assert V.device_status() == 0


@pytest.mark.parametrize("t", [3, 40, 300])
def test_experts_with_dropped_repeated_and_lopsided_choices(t):
    e, hidden, inner = 12, 128, 96
    up, down = moe(e, hidden, inner, 32, F16, False)
    x = acts(t, hidden, F16) * 2
    ids, w = choices(t, 4, e)
    ids[0] = -1                                             # a token with no expert at all
    ids[1] = torch.tensor([e, 2, 1 << 30, -5])              # outside the range: dropped
    ids[2] = 7                                              # the same expert four times
    ids[3:, 0] = 0                                          # one busy expert; others stay empty
    y = V.int4_experts(x, ids, w, up, down)
    assert torch.equal(y[0], torch.zeros_like(y[0]))
    check(y, O.experts(x, ids, w, up, down))
    everything = torch.full_like(ids, -1)
    assert torch.equal(V.int4_experts(x, everything, w, up, down), torch.zeros_like(x))
    one = torch.full_like(ids, 3)
    check(V.int4_experts(x, one, w, up, down), O.experts(x, one, w, up, down))


@pytest.mark.parametrize("t", [2, 60])
def test_a_token_with_nan_does_not_reach_its_neighbours(t):
    up, down = moe(4, 64, 64, 32, BF16, False)
    x = acts(t, 64, BF16)
    ids, w = choices(t, 2, 4)
    clean = V.int4_experts(x, ids, w, up, down)
    x[1, 3] = NAN
    y = V.int4_experts(x, ids, w, up, down)
    assert torch.isnan(y[1]).all() and torch.equal(torch.cat([y[:1], y[2:]]), torch.cat([clean[:1], clean[2:]]))


def test_a_dropped_slot_ignores_its_weight_and_a_far_scratch_is_not_needed_clean():
    up, down = moe(4, 64, 64, 32, BF16, False)
    for t in (2, 60):
        x = acts(t, 64, BF16)
        ids, w = choices(t, 2, 4)
        ids[:, 1] = -1
        w[:, 1] = NAN
        junk = torch.full((1 << 22,), NAN, device="cuda")   # memory that the call's scratch may be cut from
        del junk
        y = V.int4_experts(x, ids, w, up, down)
        check(y, O.experts(x, ids, torch.where(ids < 0, 0.0, w), up, down))


@pytest.mark.parametrize("t", [4, 30, 200])
def test_graphs_captured_on_one_stream_and_replayed_on_two(t):
    # each call's scratch is its own
    side, jobs = torch.cuda.Stream(), []
    for seed in (1, 2):
        up, down = moe(8, 256, 128, 64, F16, False, seed=seed)
        x, (ids, w) = acts(t, 256, F16, seed=seed), choices(t, 2, 8, seed=seed)
        jobs.append((x, ids, w, up, down))
    want = [V.int4_experts(*j) for j in jobs]
    torch.cuda.synchronize()
    graphs, got = [], []
    for j in jobs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            got.append([V.int4_experts(*j) for _ in range(6)])
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for y, ys in zip(want, got):
        assert all(torch.equal(v, y) for v in ys)


@pytest.mark.parametrize("t", [15, 17, 40, 380, 390])
def test_large_experts_either_side_of_the_kernels_limits(t):
    up, down = moe(8, 2080, 2048, 32, BF16, False, seed=t)       # more than 2^25 places; 4 and 96 rows each are limits
    x = acts(t, 2080, BF16, seed=t)
    ids, w = choices(t, 2, 8, seed=t)
    check(V.int4_experts(x, ids, w, up, down), O.experts(x, ids, w, up, down))


def test_rows_of_experts_past_32_bits():
    # 2.2e9 values of all rows' second products; the last and middle tokens against 64 bits
    t, k, e, hidden, inner = 140_000, 4, 6, 4096, 32
    up, down = moe(e, hidden, inner, 32, F16, False)
    x = acts(t, hidden, F16)
    ids, w = choices(40, k, e, seed=1)
    ids, w = ids.repeat(t // 40, 1), w.repeat(t // 40, 1)
    y = V.int4_experts(x, ids, w, up, down)
    for at in (0, 69_980, t - 20):
        part = slice(at, at + 20)
        check(y[part], O.experts(x[part], ids[part], w[part], up, down))
    assert V.device_status() == 0


def test_experts_refusals_and_empty_batch():
    up, down = moe(4, 64, 96, 32, F16, False)
    ids, w = choices(3, 2, 4)
    x = acts(3, 64, F16)
    assert V.int4_experts(acts(0, 64, F16), ids[:0], w[:0], up, down).shape == (0, 64)
    for bad in (lambda: V.int4_experts(x.bfloat16(), ids, w, up, down), lambda: V.int4_experts(x, ids.long(), w, up, down),
                lambda: V.int4_experts(x, ids, w.half(), up, down), lambda: V.int4_experts(x, ids[:2], w, up, down),
                lambda: V.int4_experts(x, ids, w[:, :1].contiguous(), up, down), lambda: V.int4_experts(x, ids, w, down, up),
                lambda: V.int4_experts(x, ids, w, up, tuple(None if v is None else v[:3] for v in down)),
                lambda: V.int4_experts(x[:, :32].contiguous(), ids, w, up, down), lambda: V.int4_experts(x, ids.cpu(), w, up, down)):
        with pytest.raises(RuntimeError):
            bad()


@pytest.mark.parametrize("t", [1, 20, 260])
def test_the_layer_router_choice_and_experts_together(t):
    hidden, inner, e, k = 256, 128, 16, 4
    g = torch.Generator().manual_seed(9)
    rand = lambda *s: (torch.randn(*s, generator=g) * 0.05).to(BF16).cuda()
    router = Int4Linear.from_weight(rand(e, hidden) * 4, group=64)
    layer = Int4Experts.from_weights(router, rand(e, inner, hidden), rand(e, inner, hidden), rand(e, hidden, inner), group=64,
                                     symmetric=False, top_k=k, scoring="sigmoid", bias=torch.randn(e, generator=g) * 0.01,
                                     groups=4, top_groups=2, scale=1.5).cuda()
    x = acts(t, hidden, BF16, seed=t)
    y = layer(x.reshape(1, t, hidden))
    assert y.shape == (1, t, hidden)
    # step by step: each operator on what the one before it gave
    raw = V.int4_gemm(x, router.packed, router.scales)
    check(raw, O.gemm(x, router.packed, router.scales))
    w, ids = check_route(raw, k, scoring="sigmoid", bias=layer.bias, groups=4, top_groups=2, renormalize=True, scale=1.5)
    up = (layer.gate_up_packed, layer.gate_up_scales, layer.gate_up_zeros)
    down = (layer.down_packed, layer.down_scales, layer.down_zeros)
    check(y[0], O.experts(x, ids, w, up, down))
    # captured as one graph, replayed on new inputs
    static = x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(static)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = layer(static)
    torch.cuda.current_stream().wait_stream(side)
    for seed in (21, 22):
        static.copy_(acts(t, hidden, BF16, seed=seed))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, layer(static.clone()))
    torch.library.opcheck(torch.ops.vq_gemm_b200.int4_experts.default, (x, ids, w, *up, *down), test_utils=("test_schema", "test_faketensor"))
    compiled = torch.compile(layer, backend="eager", fullgraph=True)
    assert torch.equal(compiled(x), layer(x))
    assert V.device_status() == 0


def test_a_layer_over_another_model_part():
    # a compressed (VQ) gate projection routes, the 4-bit experts answer
    from oracle import vq_oracle as Q
    from vq_gemm_b200.linear import VQLinear
    x, idx, cb = Q.make_bl_inputs(24, 256, 32, 8, 256, 0, seed=3)
    up, down = moe(32, 256, 64, 64, F16, False)
    layer = Int4Experts(VQLinear(idx, cb, 0).cuda(), up, down, top_k=2, in_features=256).cuda()
    y = layer(x.cuda())
    w, ids = check_route(layer.router(x.cuda()), 2, renormalize=True)
    check(y, O.experts(x.cuda(), ids, w, up, down))


def test_a_layer_cast_with_its_model():
    up, down = moe(8, 128, 64, 64, F16, False)
    router = torch.nn.Linear(128, 8, bias=False).requires_grad_(False)
    layer = Int4Experts(router, up, down, top_k=2, in_features=128, scoring="sigmoid", bias=torch.arange(8.0) / 16).cuda().half()
    x = acts(5, 128, F16)
    w, ids = check_route(layer.router(x), 2, scoring="sigmoid", bias=torch.arange(8.0).cuda() / 16, renormalize=True)
    assert torch.equal(layer(x), V.int4_experts(x, ids, w, up, down))
