"""4-bit weights on the GPU against the 64-bit restatement: quantiser and dequantisation bit for bit, products within the
bound that follows from their sums."""
import threading

import pytest
import torch

import vq_gemm_b200 as V
from oracle import int4_oracle as O
from vq_gemm_b200 import quantize
from vq_gemm_b200.linear import Int4Linear

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def make(n, k, group, dtype=F16, zeros=False, lead=(), seed=0):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (*lead, n, k), dtype=torch.uint8, generator=g)
    scales = (torch.rand(*lead, k // group, n, generator=g) * 0.02 + 0.005).to(dtype)
    z = torch.randint(0, 16, (*lead, k // group, n), dtype=torch.uint8, generator=g) if zeros else None
    return quantize.int4_pack(codes).cuda(), scales.cuda(), None if z is None else z.cuda()


def acts(m, k, dtype, seed=1):
    return torch.randn(m, k, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def check(y, ref, what=""):
    want, bound = ref
    got = y.cpu().double()
    assert got.shape == want.shape
    over = (got - want).abs() - bound
    assert not torch.isnan(over).any() and float(over.max()) <= 0, (what, float(over.max()), int((over > 0).sum()))


def same(a, b):
    return torch.equal(a.cpu().contiguous().view(torch.int16), b.cpu().contiguous().view(torch.int16))


WEIGHTS = [(1, 32, 32), (15, 64, 64), (16, 96, 32), (33, 96, 96), (130, 160, 160), (77, 192, 64), (256, 256, 128), (31, 1024, 512),
           (129, 2080, 32), (48, 4096, 4096)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("n,k,group", WEIGHTS)
def test_dequantisation_is_exact(n, k, group, zeros, dtype):
    w = make(n, k, group, dtype, zeros, seed=n + k)
    assert same(V.int4_dequant(*w, in_features=k), O.weights(*w, k).to(dtype))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("n,k,group", WEIGHTS)
def test_quantiser_is_exact(n, k, group, symmetric, dtype):
    g = torch.Generator().manual_seed(n * k)
    w = (torch.randn(n, k, generator=g) * 0.05).to(dtype)
    w[0, :32] = 0                                                        # a group of zeros (or part of one)
    if n > 2:
        w[1] = w[1].abs()                                                # no negative values
        w[2, :32] = torch.arange(32).to(dtype) * 2.0 ** -24              # fp16: subnormal numbers; halves
    packed, scales, zeros = quantize.int4_quantize(w.cuda(), group=group, symmetric=symmetric)
    codes, s, z = O.quantize(w, group, symmetric)
    assert same(scales, s)
    assert (zeros is None) == symmetric and (symmetric or torch.equal(zeros.cpu(), z))
    assert torch.equal(quantize.int4_unpack(packed.cpu(), n, k), codes)


def test_quantiser_rounds_halves_to_even_codes():
    # scale is exactly one: every multiple of a half from -7 to 7 is a tie or a whole number
    w = torch.zeros(16, 64, dtype=F16)
    w[:, :29] = torch.arange(-14, 15).half() / 2
    packed, scales, _ = quantize.int4_quantize(w.cuda(), group=64)
    assert torch.equal(scales.cpu(), torch.ones(1, 16, dtype=F16))
    assert torch.equal(quantize.int4_unpack(packed.cpu(), 16, 64)[0, :29].double(), torch.round(w[0, :29].double()) + 8)


def test_quantiser_and_dequantisation_of_experts():
    w = (torch.randn(3, 40, 96, generator=torch.Generator().manual_seed(4)) * 0.05).to(BF16)
    packed, scales, zeros = quantize.int4_quantize(w.cuda(), group=32, symmetric=False)
    back = V.int4_dequant(packed, scales, zeros, in_features=96)
    assert back.shape == w.shape
    for e in range(3):
        codes, s, z = O.quantize(w[e], 32, False)
        assert torch.equal(quantize.int4_unpack(packed[e].cpu(), 40, 96), codes) and torch.equal(zeros[e].cpu(), z)
        assert same(back[e], O.weights(packed[e], scales[e], zeros[e], 96).to(BF16))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 16, 17, 31, 33, 40])
@pytest.mark.parametrize("n,k,group,zeros", [(1, 32, 32, True), (33, 96, 96, False), (100, 1024, 128, True), (77, 2080, 32, False)])
def test_product(m, n, k, group, zeros, dtype):
    w = make(n, k, group, dtype, zeros, seed=m + n)
    x = acts(m, k, dtype, seed=m)
    check(V.int4_gemm(x, *w), O.gemm(x, *w))


@pytest.mark.parametrize("dtype,zeros", [(F16, False), (BF16, True)])
@pytest.mark.parametrize("m,n,k,group", [(64, 128, 128, 64), (65, 130, 192, 64), (100, 300, 96, 32), (128, 256, 2048, 128), (129, 257, 1056, 32),
                                         (255, 128, 512, 512), (257, 511, 640, 128), (300, 1000, 64, 32), (1000, 768, 256, 128),
                                         (600, 5003, 160, 160), (1, 4096, 8192, 128), (3, 1000, 14336, 128), (40, 300, 8224, 32)])
def test_product_of_many_rows_and_long_columns(m, n, k, group, dtype, zeros):
    w = make(n, k, group, dtype, zeros, seed=m + n)
    x = acts(m, k, dtype, seed=m)
    check(V.int4_gemm(x, *w), O.gemm(x, *w))
    assert V.device_status() == 0


@pytest.mark.parametrize("m", [1, 12, 70, 300])
def test_product_leaves_what_lies_behind_it_and_repeats_bit_for_bit(m):
    w = make(45, 320, 64, zeros=True)
    x = acts(m, 320, F16)
    room = torch.full((m + 3, 45), 7.0, dtype=F16, device="cuda")
    y = V.int4_gemm(x, *w, out=room[:m])
    assert torch.equal(room[m:], torch.full_like(room[m:], 7.0))
    for _ in range(3):
        assert torch.equal(V.int4_gemm(x, *w), y)


@pytest.mark.parametrize("m", [3, 80])
def test_nan_and_infinity_stay_in_their_row_and_column(m):
    packed, scales, _ = make(50, 96, 32)
    x = acts(m, 96, F16)
    clean = V.int4_gemm(x, packed, scales)
    x2, s2 = x.clone(), scales.clone()
    x2[1, 5] = float("nan")
    s2[1, 20] = float("nan")
    y = V.int4_gemm(x2, packed, s2)
    bad = torch.isnan(y)
    assert bad[1].all() and bad[:, 20].all() and int(bad.sum()) == 50 + m - 1
    assert torch.equal(y[~bad], clean[~bad])


@pytest.mark.parametrize("m", [2, 70])
def test_extreme_codes_and_scales(m):
    # all codes 0 with zero point 15 and all 15 with zero point 0, at the largest finite products
    for code, zero in ((0, 15), (15, 0)):
        packed = quantize.int4_pack(torch.full((32, 64), code, dtype=torch.uint8)).cuda()
        scales = torch.full((2, 32), 64.0, dtype=F16, device="cuda")
        zeros = torch.full((2, 32), zero, dtype=torch.uint8, device="cuda")
        x = torch.full((m, 64), 0.25, dtype=F16, device="cuda")
        want = (code - zero) * 64.0 * 0.25 * 64
        assert torch.equal(V.int4_gemm(x, packed, scales, zeros), torch.full((m, 32), want, dtype=F16, device="cuda"))


def test_empty_batch_and_refusals():
    w = make(45, 320, 64)
    assert V.int4_gemm(acts(0, 320, F16), *w).shape == (0, 45)
    x = acts(2, 320, F16)
    for bad in (lambda: V.int4_gemm(x.bfloat16(), *w), lambda: V.int4_gemm(x[:, :256].contiguous(), *w), lambda: V.int4_gemm(x[0], *w),
                lambda: V.int4_gemm(x.t(), *w), lambda: V.int4_gemm(x.cpu(), *w),
                lambda: V.int4_gemm(x, *w, out=torch.empty(2, 44, dtype=F16, device="cuda")),
                lambda: V.int4_gemm(torch.empty(2 * 320 + 1, dtype=F16, device="cuda")[1:].view(2, 320), *w),
                lambda: V.int4_dequant(w[0], w[1], in_features=352), lambda: quantize.int4_quantize(x, group=48),
                lambda: quantize.int4_quantize(x.float())):
        with pytest.raises(RuntimeError):
            bad()
    assert V.device_status() == 0


@pytest.mark.parametrize("m", [1, 40, 200])
def test_on_a_side_stream_and_in_two_graphs(m):
    # two captured graphs on streams of their own, replayed against each other, and the eager call beside them
    w1, w2 = make(700, 1024, 128, seed=1), make(300, 512, 64, BF16, True, seed=2)
    x1, x2 = acts(m, 1024, F16), acts(m, 512, BF16)
    want1, want2 = V.int4_gemm(x1, *w1), V.int4_gemm(x2, *w2)
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for st, x, w in ((streams[0], x1, w1), (streams[1], x2, w2)):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            V.int4_gemm(x, *w)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                outs.append(V.int4_gemm(x, *w))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(10):
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        eager = V.int4_gemm(x1, *w1)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want1) and torch.equal(outs[1], want2) and torch.equal(eager, want1)
    assert V.device_status() == 0


def test_graphs_captured_on_one_stream_and_replayed_on_two_keep_their_scratch_apart():
    side = torch.cuda.Stream()
    jobs = [(acts(77, 4096, F16, seed=1), make(1024, 4096, 128, F16, seed=2)), (acts(70, 4096, F16, seed=3), make(1280, 4096, 64, F16, seed=4))]
    want = [V.int4_gemm(x, *w) for x, w in jobs]
    torch.cuda.synchronize()
    graphs, got = [], []
    for x, w in jobs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            got.append([V.int4_gemm(x, *w) for _ in range(8)])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for w, ys in zip(want, got):
        assert all(torch.equal(y, w) for y in ys)


@pytest.mark.parametrize("m", [1, 7, 16, 24, 40, 300])
def test_tensors_that_start_inside_others(m):
    # scales 2 bytes, zero points 1 byte, everything else 16 bytes behind a wide boundary
    n, k = 150, 320
    packed, scales, zeros = make(n, k, 64, F16, True, seed=m)
    x = acts(m, k, F16, seed=m)
    shift = lambda t, by: torch.cat([t.new_zeros(by), t.reshape(-1)])[by:].view(t.shape)
    w = (shift(packed, 16), shift(scales, 1), shift(zeros, 1))
    out = torch.full((m * n + 16,), 9.0, dtype=F16, device="cuda")
    y = V.int4_gemm(shift(x, 8), *w, out=out[8:8 + m * n].view(m, n))
    assert torch.equal(y, V.int4_gemm(x, packed, scales, zeros))
    assert bool((out[:8] == 9).all()) and bool((out[8 + m * n:] == 9).all())
    dense = V.int4_dequant(packed, scales, zeros)
    assert torch.equal(V.int4_dequant(*w, out=shift(torch.empty_like(dense), 8)), dense)
    for symmetric in (True, False):
        a, b = quantize.int4_quantize(dense, group=64, symmetric=symmetric), quantize.int4_quantize(shift(dense, 8), group=64, symmetric=symmetric)
        assert all((u is None and v is None) or torch.equal(u, v) for u, v in zip(a, b))


@pytest.mark.parametrize("m", [1, 20, 40])
def test_the_longest_rows(m):
    k = 1 << 19
    w, x = make(16, k, 64, F16, seed=3), acts(m, k, F16) * 0.25
    check(V.int4_gemm(x, *w), O.gemm(x, *w))
    with pytest.raises(RuntimeError):
        V.int4_gemm(torch.zeros(m, k + 64, dtype=F16, device="cuda"), torch.zeros(1, k // 64 + 1, 512, dtype=torch.uint8, device="cuda"),
                    torch.zeros(k // 64 + 1, 16, dtype=F16, device="cuda"))


def test_outputs_and_weights_past_32_bits():
    # 2.2e9 results: the last rows are those of the same rows alone (the K loop of a tile is summed in one piece either way)
    m, n, k = 270_000, 8192, 64
    w, x = make(n, k, 64, F16, seed=5), acts(m, k, F16)
    y = V.int4_gemm(x, *w)
    check(y[-40:], O.gemm(x[-40:], *w))
    check(y[130_000:130_040], O.gemm(x[130_000:130_040], *w))
    del x, y
    # 2.2e9 weights of 18 experts, quantised and read back
    e, n, k = 18, 15_000, 8192
    dense = torch.zeros(e, n, k, dtype=BF16, device="cuda")
    dense[-1, -300:] = acts(300, k, BF16, seed=6) * 0.05
    q = quantize.int4_quantize(dense, group=128)
    back = V.int4_dequant(*q)
    alone = V.int4_dequant(*quantize.int4_quantize(dense[-1, -300:].contiguous(), group=128))
    assert torch.equal(back[-1, -300:], alone) and not bool(back[:-1].any()) and not bool(back[-1, :-300].any())


@pytest.mark.parametrize("m", [8, 9, 16, 17, 32, 33, 128, 129])
def test_either_side_of_the_kernels_limits(m):
    w, x = make(8200, 6176, 32, BF16, True, seed=m), acts(m, 6176, BF16, seed=m)       # more than 3 * 2^24 places
    check(V.int4_gemm(x, *w), O.gemm(x, *w))


def test_two_threads_on_streams_of_their_own():
    jobs = [(acts(m, 512, F16, seed=m), make(400, 512, 128, F16, seed=m)) for m in (2, 60)]
    want = [V.int4_gemm(x, *w) for x, w in jobs]
    torch.cuda.synchronize()
    wrong = []

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            ys = [V.int4_gemm(jobs[i][0], *jobs[i][1]) for _ in range(200)]
            torch.cuda.current_stream().synchronize()
            wrong.extend(1 for y in ys if not torch.equal(y, want[i]))

    threads = [threading.Thread(target=run, args=(i % 2,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and V.device_status() == 0


def test_quantised_just_before_the_product():
    for seed in range(8):      # the product reads weights that the kernel in front of it has just written
        w = (torch.randn(512, 1024, generator=torch.Generator().manual_seed(seed)) * 0.05).half().cuda()
        x = acts(2, 1024, F16, seed)
        q = quantize.int4_quantize(w)
        y = V.int4_gemm(x, *q)
        check(y, O.gemm(x, *q))


def test_module():
    w = (torch.randn(200, 416, generator=torch.Generator().manual_seed(1)) * 0.05).to(BF16)
    layer = Int4Linear.from_weight(w.cuda(), group=32, symmetric=False, bias=torch.arange(200.0).cuda())
    x = acts(12, 416, BF16)
    y = layer(x.reshape(3, 4, 416))
    assert y.shape == (3, 4, 200)
    plain = V.int4_gemm(x, layer.packed, layer.scales, layer.zeros)
    assert torch.equal(y.reshape(12, 200), plain + layer.bias)
    check(plain, O.gemm(x, layer.packed, layer.scales, layer.zeros))
    # every weight is at most half a step from the dense one; the ends of the range may be off by the scale's rounding too
    step = layer.scales.float().t().repeat_interleave(32, 1).cpu()
    off = (layer.dequantized_weight().float().cpu() - w.float()).abs()
    assert float((off / step).max()) <= 0.5 + 15 * 2.0 ** -8 + 2.0 ** -4
    clone = Int4Linear(torch.zeros_like(layer.packed), torch.zeros_like(layer.scales), torch.zeros_like(layer.zeros), layer.bias, 416)
    clone.load_state_dict(layer.state_dict())
    assert torch.equal(clone(x), layer(x))
    torch.library.opcheck(torch.ops.vq_gemm_b200.int4_linear.default, (x, layer.packed, layer.scales, layer.zeros),
                          test_utils=("test_schema", "test_faketensor"))
    compiled = torch.compile(layer, backend="eager", fullgraph=True)
    assert torch.equal(compiled(x), layer(x))


def test_quantiser_at_the_smallest_scales():
    # bf16 scales down to the smallest subnormal number, whose reciprocal 32 bits do not hold
    for power in (-100, -118, -124, -130, -133):
        w = ((torch.arange(16 * 64).reshape(16, 64) % 23 - 11).float() * 2.0 ** power).to(BF16)
        for symmetric in (True, False):
            packed, scales, zeros = quantize.int4_quantize(w.cuda(), group=64, symmetric=symmetric)
            codes, s, z = O.quantize(w, 64, symmetric)
            assert same(scales, s) and torch.equal(quantize.int4_unpack(packed.cpu(), 16, 64), codes)
            assert symmetric or torch.equal(zeros.cpu(), z)


def test_quantiser_and_dequantisation_of_tensors_that_start_on_16_bytes_only():
    w = (torch.randn(32 * 64 + 8, generator=torch.Generator().manual_seed(2)) * 0.05).half().cuda()[8:].view(32, 64)
    assert w.data_ptr() % 32 == 16
    packed, scales, _ = quantize.int4_quantize(w, group=64)
    codes, s, _ = O.quantize(w.cpu(), 64, True)
    assert same(scales, s) and torch.equal(quantize.int4_unpack(packed.cpu(), 32, 64), codes)
    out = torch.zeros(32 * 64 + 8, dtype=F16, device="cuda")[8:].view(32, 64)
    V.int4_dequant(packed, scales, out=out)
    assert same(out, O.weights(packed, scales, None, 64).half())
