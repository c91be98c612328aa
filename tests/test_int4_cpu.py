"""4-bit weights, the expert router and the experts' layer without a GPU: the layout, the shape rules, the refusals."""
import ctypes

import pytest
import torch

import vq_gemm_b200 as V
from oracle import int4_oracle as O
from vq_gemm_b200 import _lib, ops, quantize
from vq_gemm_b200.linear import Int4Experts, Int4Linear


@pytest.fixture(scope="module")
def lib():
    from vq_gemm_b200.build import build
    build()
    return _lib.load()


def _packed(n, k, group, dtype=torch.float16, zeros=False, lead=(), seed=0):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (*lead, n, k), dtype=torch.uint8, generator=g)
    scales = (torch.rand(*lead, k // group, n, generator=g) * 0.02 + 0.005).to(dtype)
    z = torch.randint(0, 16, (*lead, k // group, n), dtype=torch.uint8, generator=g) if zeros else None
    return codes, quantize.int4_pack(codes), scales, z


@pytest.mark.parametrize("n,k", [(1, 32), (16, 64), (17, 96), (5003, 64), (40, 4064)])
def test_layout_round_trip_and_the_written_byte_order(n, k):
    codes, packed, _, _ = _packed(n, k, 32, seed=n)
    assert packed.shape == (-(-n // 16), -(-k // 64), 512)
    assert torch.equal(quantize.int4_unpack(packed, n, k), codes)
    assert torch.equal(O.unpack(packed, n, k), codes)


def test_layout_with_experts():
    codes, packed, _, _ = _packed(18, 96, 32, lead=(3,))
    assert packed.shape == (3, 2, 2, 512)
    assert torch.equal(quantize.int4_unpack(packed, 18, 96), codes)
    assert torch.equal(quantize.int4_unpack(packed[1], 18, 96), codes[1])
    with pytest.raises(RuntimeError):
        quantize.int4_unpack(packed, 33, 96)
    with pytest.raises(RuntimeError):
        quantize.int4_pack(codes.int())


def test_bad_arguments_are_rejected_without_cuda(lib):
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4096 + 8)
    gemm = lambda x=p, w=p, s=p, z=None, y=p, m=1, n=16, k=64, g=32, t=0: lib.vqg_int4_gemm(x, w, s, z, y, m, n, k, g, t, None, 0, None)
    assert gemm(m=-1) == gemm(n=-1) == gemm(k=-1) == gemm(t=2) == gemm(t=-1) == _lib.ERR_BAD_ARG
    assert gemm(x=None) == gemm(w=None) == gemm(s=None) == gemm(y=None) == _lib.ERR_BAD_ARG
    assert gemm(x=odd) == gemm(w=odd) == gemm(y=odd) == _lib.ERR_BAD_ARG
    for k, g in ((48, 48), (64, 0), (64, -32), (96, 64), (192, 96), (64, 16), (33, 33)):
        assert gemm(k=k, g=g) == _lib.ERR_UNSUPPORTED, (k, g)
    assert gemm(m=0) == gemm(n=0) == _lib.OK
    assert lib.vqg_int4_dequant(p, p, None, None, 1, 16, 64, 32, 0, None) == _lib.ERR_BAD_ARG
    assert lib.vqg_int4_dequant(p, p, None, p, 0, 16, 64, 32, 0, None) == _lib.OK
    assert lib.vqg_int4_dequant(p, p, None, odd, 1, 16, 64, 32, 0, None) == _lib.ERR_BAD_ARG
    assert lib.vqg_int4_quantize(None, p, p, None, 1, 16, 64, 32, 0, None) == _lib.ERR_BAD_ARG
    assert lib.vqg_int4_quantize(p, p, p, None, 1, 16, 64, 48, 0, None) == _lib.ERR_UNSUPPORTED
    assert lib.vqg_int4_quantize(p, p, p, None, 70000, 16, 64, 32, 0, None) == _lib.ERR_UNSUPPORTED
    route = lambda x=p, w=p, i=p, t=4, e=8, k=2, sc=0, g=1, tg=1, gs=0, ty=2: lib.vqg_route_experts(x, None, w, i, t, e, k, sc, g, tg, gs, 0, 1.0, ty, None)
    assert route(x=None) == route(w=None) == route(i=None) == route(t=-1) == _lib.ERR_BAD_ARG
    assert route(k=0) == route(k=9) == route(sc=2) == route(g=3) == route(tg=2) == route(tg=0) == route(gs=2) == route(ty=3) == _lib.ERR_BAD_ARG
    assert route(e=513) == route(e=64, k=33) == route(e=66, g=33) == _lib.ERR_UNSUPPORTED
    assert route(t=0) == _lib.OK
    need = lib.vqg_int4_experts_workspace_bytes(4, 2, 8, 64, 32)
    assert need > 4 * 2 * 32 * 2
    ex = lambda x=p, w=p, y=p, t=4, k=2, e=8, h=64, i=32, ws=p, nb=need, ty=0: lib.vqg_int4_experts(
        x, p, p, w, p, None, p, p, None, y, t, k, e, h, i, h, i, ty, ws, nb, None)
    assert ex(x=None) == ex(w=None) == ex(y=None) == ex(y=odd) == ex(t=-1) == ex(k=0) == ex(e=0) == ex(h=0) == ex(ty=5) == _lib.ERR_BAD_ARG
    assert ex(h=48) == ex(i=40) == ex(e=513) == ex(t=1 << 30) == _lib.ERR_UNSUPPORTED
    assert ex(ws=None) == ex(nb=need - 1) == ex(ws=odd) == _lib.ERR_WORKSPACE
    assert ex(t=0) == _lib.OK


def test_scratch_is_asked_for_where_pieces_are_summed(lib):
    """Above 32 rows, above 16 for weights of 2^24 places or more, above 8 for more than 3 * 2^24."""
    need = lib.vqg_int4_workspace_bytes
    assert need(8, 8192, 8192) == need(16, 4096, 4096) == need(32, 4096, 4064) == need(33, 0, 64) == need(0, 4096, 4096) == 0
    assert need(9, 8192, 8192) == need(17, 4096, 4096) == need(33, 64, 64) > 0


def test_python_layer_refuses_cpu_tensors():
    _, packed, scales, _ = _packed(16, 64, 32)
    x = torch.zeros(1, 64, dtype=torch.float16)
    for call in (lambda: V.int4_gemm(x, packed, scales), lambda: V.int4_dequant(packed, scales),
                 lambda: V.route_experts(torch.zeros(2, 8), 2), lambda: quantize.int4_quantize(x),
                 lambda: V.int4_experts(x, torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, 1), (packed[None], scales[None], None),
                                        (packed[None], scales[None], None))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_weight_checks():
    codes, packed, scales, zeros = _packed(20, 128, 64, zeros=True)
    ok = ops._int4_weight(packed, scales, zeros, 128, False)
    assert ok == (20, 64)
    for bad in (lambda: ops._int4_weight(packed.int(), scales, zeros, 128, False),
                lambda: ops._int4_weight(packed, scales.float(), zeros, 128, False),
                lambda: ops._int4_weight(packed, scales, zeros[:1], 128, False),
                lambda: ops._int4_weight(packed, scales, zeros.int(), 128, False),
                lambda: ops._int4_weight(packed, scales, zeros, 192, False),
                lambda: ops._int4_weight(packed[:1], scales, zeros, 128, False),
                lambda: ops._int4_weight(packed[..., :256], scales, zeros, 128, False),
                lambda: ops._int4_weight(packed, scales, zeros, 128, True),
                lambda: ops._int4_weight(packed[None], scales[None].expand(2, -1, -1), None, 128, True),
                lambda: ops._int4_weight(packed, scales[:, :16].contiguous().t().contiguous()[:8].contiguous(), None, 128, False)):
        with pytest.raises(RuntimeError):
            bad()


def test_fake_tensor_rules():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        e = lambda *s, t=torch.uint8: torch.empty(*s, dtype=t, device="cuda")
        x, packed, scales = e(5, 96, t=torch.bfloat16), e(3, 2, 512), e(3, 33, t=torch.bfloat16)
        y = torch.ops.vq_gemm_b200.int4_linear(x, packed, scales, None)
        assert y.shape == (5, 33) and y.dtype == torch.bfloat16
        with pytest.raises(RuntimeError):
            torch.ops.vq_gemm_b200.int4_linear(e(5, 64, t=torch.bfloat16), packed, scales, None)
        w, i = torch.ops.vq_gemm_b200.route_experts(e(5, 8, t=torch.float32), 2, "softmax", None, 1, 1, "top2", True, 1.0)
        assert w.shape == i.shape == (5, 2) and w.dtype == torch.float32 and i.dtype == torch.int32
        y = torch.ops.vq_gemm_b200.int4_experts(x, i, w, e(8, 8, 2, 512), e(8, 3, 128, t=torch.bfloat16), None,
                                                e(8, 6, 1, 512), e(8, 2, 96, t=torch.bfloat16), None)
        assert y.shape == (5, 96)


def test_modules_keep_their_books():
    _, packed, scales, zeros = _packed(20, 96, 32, zeros=True)
    layer = Int4Linear(packed, scales, zeros, torch.zeros(20), in_features=96)
    assert (layer.in_features, layer.out_features, layer.group) == (96, 20, 32)
    assert set(layer.state_dict()) == {"packed", "scales", "zeros", "bias"}
    assert set(Int4Linear(packed, scales, in_features=96).state_dict()) == {"packed", "scales"}
    for bad in (lambda: Int4Linear(packed, scales, zeros), lambda: Int4Linear(packed, scales, in_features=96, bias=torch.zeros(3))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        layer(torch.zeros(1, 64))
    up = _packed(64, 96, 32, lead=(4,))[1:]
    down = _packed(96, 32, 32, lead=(4,))[1:]
    moe = Int4Experts(torch.nn.Linear(96, 4), up, down, top_k=2, in_features=96, bias=torch.zeros(4))
    assert (moe.experts, moe.inner, moe.in_features) == (4, 32, 96) and "experts=4" in repr(moe)
    for bad in (dict(top_k=5), dict(top_k=0)):
        with pytest.raises(ValueError):
            Int4Experts(torch.nn.Linear(96, 4), up, down, in_features=96, **bad)
    with pytest.raises(ValueError):
        Int4Experts(torch.nn.Linear(96, 4), up, _packed(96, 64, 32, lead=(4,))[1:], top_k=1, in_features=96)


def test_oracle_quantiser_and_router_on_cases_worked_by_hand():
    w = torch.tensor([[7.0, -7.0, 0.5, 1.5, 2.5] + [0.0] * 27]).half()
    codes, scale, _ = O.quantize(w, 32, True)
    assert scale.item() == 1.0 and codes[0, :5].tolist() == [15, 1, 8, 10, 10]     # halves to the even number
    w = torch.tensor([[-3.0, 12.0] + [0.0] * 30]).half()
    codes, scale, zero = O.quantize(w, 32, False)
    assert scale.item() == 1.0 and zero.item() == 3 and codes[0, :3].tolist() == [0, 15, 3]
    weights, ids = O.route(torch.tensor([[0.0, 0.0, -float("inf"), float("nan")]]), 3, renormalize=True)
    assert ids.tolist() == [[0, 1, -1]] and weights.tolist() == [[0.5, 0.5, 0.0]]
    _, ids = O.route(torch.tensor([[3.0, 0.0, 2.0, 2.0]]), 2, scoring="sigmoid", groups=2, top_groups=1)
    assert ids.tolist() == [[2, 3]]                                                  # the better pair wins over the best expert
    _, ids = O.route(torch.tensor([[3.0, 0.0, 2.0, 2.0]]), 2, scoring="sigmoid", groups=2, top_groups=1, group_score="max")
    assert ids.tolist() == [[0, 1]]
