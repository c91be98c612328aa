"""Performance cases of the 4-bit product, its quantiser, the expert router and the experts' products.

``listed()`` and ``draw()`` give cases, ``prepare()`` the tensors that a program holds before the call, ``run()`` one pass:
with ``own`` set the calls that a user of ``vq_gemm_b200`` makes, otherwise the same operators written out in elementary
torch operations.  ``exact()`` evaluates the definitions in 64 bits.

The 4-bit format.  A weight W [N, K] has 4-bit codes, one scale (fp16 or bf16, the model's type T) and optionally one
zero point (0 ... 15, otherwise 8) per row and group of consecutive K values:

    W[n, k] = round_T((code[n, k] - zero[k // group, n]) * scale[k // group, n])

``scales`` and ``zeros`` are [K / group, N].  ``packed`` is [ceil(N / 16), ceil(K / 64), 512] bytes: tiles of 16 rows
and 64 columns, in which the byte at (((t * 8 + g) * 4 + s) * 2 + e) * 2 + q holds column 16 t + 4 s + 2 q + e of row g
(low four bits) and of row g + 8 (high four bits).  Experts add a leading dimension to all three.
"""
import math

import torch

own = False

_T = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---- cases ---------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token through a square projection: the smallest product, where latency counts
        _gemm("gemm 1x4096x4096", 1, 4096, 4096, 128, "fp16", False),
        # one token through the widest layer: the weight stream
        _gemm("gemm 1x28672x8192 bf16", 1, 28672, 8192, 128, "bf16", False),
        # sixteen sequences decoded together, zero points, groups of 64
        _gemm("gemm 16x11008x4096 zeros", 16, 11008, 4096, 64, "fp16", True),
        # a ragged batch on a weight whose rows and columns fill no tile
        _gemm("gemm 77x5003x4064 bf16 g32", 77, 5003, 4064, 32, "bf16", True),
        # a prompt
        _gemm("gemm 4096x14336x4096", 4096, 14336, 4096, 128, "fp16", False),
        # routing of a decode step: few rows, plain softmax scores
        _route("route 8 of 64, 16 tokens", 16, 64, 8, "softmax", False, 1, 1, True, "bf16", False),
        # routing of a prompt: sigmoid scores, balance bias, groups, a few experts out of service and padded rows
        _route("route 8 of 256, 16384 tokens", 16384, 256, 8, "sigmoid", True, 8, 4, True, "fp32", True),
        # one token through its eight experts
        _experts("experts 1 token", 1, 64, 8, 2048, 1024, 128, "bf16", False, False),
        # a decode batch that reaches almost every expert with a few rows each, some slots dropped, zero points
        _experts("experts 50 tokens zeros", 50, 64, 8, 2048, 1024, 64, "fp16", True, True),
        # a prompt: hundreds of rows per expert, unevenly spread
        _experts("experts 4096 tokens", 4096, 64, 8, 2048, 1024, 128, "bf16", False, False),
        # quantising a layer, and reading its weights back: symmetric
        _quantize("quantise 11008x4096", 11008, 4096, 128, "fp16", False),
        # with zero points, small groups and an odd number of rows
        _quantize("quantise 1001x2080 zeros bf16", 1001, 2080, 32, "bf16", True),
    ]


def _gemm(name, m, n, k, group, dtype, zeros):
    return dict(name=name, op="gemm", m=m, n=n, k=k, group=group, dtype=dtype, zeros=zeros)


def _route(name, t, e, top_k, scoring, bias, groups, top_groups, renormalize, dtype, masked):
    return dict(name=name, op="route", t=t, e=e, top_k=top_k, scoring=scoring, bias=bias, groups=groups,
                top_groups=top_groups, renormalize=renormalize, dtype=dtype, masked=masked)


def _experts(name, t, e, top_k, hidden, inner, group, dtype, zeros, dropped):
    return dict(name=name, op="experts", t=t, e=e, top_k=top_k, hidden=hidden, inner=inner, group=group, dtype=dtype,
                zeros=zeros, dropped=dropped)


def _quantize(name, n, k, group, dtype, zeros):
    return dict(name=name, op="quantize", n=n, k=k, group=group, dtype=dtype, zeros=zeros)


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("gemm", "gemm", "route", "experts", "experts", "quantize"))
    dtype = rng.choice(("fp16", "bf16"))
    zeros = rng.random() < 0.5
    group = rng.choice((32, 64, 128))
    if op == "gemm":
        k = group * max(1, _log(rng, 128, 8192) // group)
        m, n = _log(rng, 1, 4096), _log(rng, 64, 28672)
        while m * n > 4096 * 14336 * 4096 // k:
            m = max(1, m // 2)
        case = _gemm("", m, n, k, group if rng.random() < 0.85 else k, dtype, zeros)
    elif op == "route":
        groups = rng.choice((1, 1, 2, 4, 8))
        e = groups * rng.randint(2, max(2, 384 // groups))
        top_groups = rng.randint(1, groups)
        top_k = rng.randint(1, min(10, top_groups * (e // groups)))
        case = _route("", _log(rng, 1, 16384), e, top_k, rng.choice(("softmax", "sigmoid")), rng.random() < 0.5, groups,
                      top_groups, rng.random() < 0.7, rng.choice(("fp32", "bf16", "fp16")), rng.random() < 0.4)
    elif op == "experts":
        e = _log(rng, 4, 64)
        hidden, inner = group * max(1, _log(rng, 256, 2048) // group), group * max(1, _log(rng, 128, 1024) // group)
        case = _experts("", _log(rng, 1, 4096), e, rng.randint(1, min(8, e)), hidden, inner, group, dtype, zeros,
                        rng.random() < 0.4)
    else:
        case = _quantize("", _log(rng, 16, 11008), group * max(1, _log(rng, 256, 8192) // group), group, dtype, zeros)
    del case["name"]
    return case


# ---- inputs --------------------------------------------------------------------------------------------------------
def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _activations(gen, rows, cols, dtype):
    """Normalised activations: unit variance, with a few channels that are ten times as large as the others."""
    gain = torch.where(torch.rand(cols, generator=gen, device="cuda") < 0.005, 10.0, 1.0)
    return (_normal(gen, rows, cols) * gain).to(dtype)


def _pack(codes):
    """Codes [..., N, K] of 0 ... 15 into the tile order of the format."""
    *lead, n, k = codes.shape
    codes = torch.nn.functional.pad(codes, (0, -k % 64, 0, -n % 16))
    n16, k64 = codes.shape[-2] // 16, codes.shape[-1] // 64
    c = codes.reshape(-1, n16, 2, 8, k64, 4, 4, 2, 2)                   # row half h, row g, tile, t, s, q, e
    c = c.permute(2, 0, 1, 4, 5, 3, 6, 8, 7)                            # h first, then tile and byte order
    return (c[0] | (c[1] << 4)).reshape(*lead, n16, k64, 512).contiguous()


def _weights(gen, lead, n, k, group, dtype, zeros):
    """A trained layer's weights: normal, coded by group with the largest value on the last code (or with the range on all
    sixteen when there are zero points)."""
    packed, scales, zero = [], [], []
    for _ in range(lead or 1):
        w = (_normal(gen, n, k) * 0.02).view(n, k // group, group)
        if zeros:
            low, high = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
            s = ((high - low) / 15).clamp(min=1e-5).to(dtype).float()
            z = (-low / s).round().clamp(0, 15)
        else:
            s = (w.abs().amax(-1) / 7).clamp(min=1e-5).to(dtype).float()
            z = torch.full_like(s, 8.0)
        code = ((w / s[..., None]).round() + z[..., None]).clamp(0, 15).to(torch.uint8).view(n, k)
        packed.append(_pack(code))
        scales.append(s.t().to(dtype).contiguous())
        zero.append(z.t().to(torch.uint8).contiguous())
    if lead is None:
        return packed[0], scales[0], zero[0] if zeros else None
    return torch.stack(packed), torch.stack(scales), torch.stack(zero) if zeros else None


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(case)
    if case["op"] == "gemm":
        st["x"] = _activations(gen, case["m"], case["k"], _T[case["dtype"]])
        st["w"] = _weights(gen, None, case["n"], case["k"], case["group"], _T[case["dtype"]], case["zeros"])
    elif case["op"] == "route":
        t, e = case["t"], case["e"]
        logits = _normal(gen, t, e) * 1.5 + 0.5 * _normal(gen, 1, e)
        if case["masked"]:
            off = torch.rand(e, generator=gen, device="cuda") < 0.05
            logits = logits.masked_fill(off, -math.inf)                 # experts out of service
            logits[t - t // 16:] = -math.inf                            # rows behind the last sequence
        st["logits"] = logits.to({"fp32": torch.float32, **_T}[case["dtype"]])
        st["bias_values"] = 0.05 * _normal(gen, e) if case["bias"] else None
    elif case["op"] == "experts":
        t, e, k = case["t"], case["e"], case["top_k"]
        dtype = _T[case["dtype"]]
        st["x"] = _activations(gen, t, case["hidden"], dtype)
        st["gate_up"] = _weights(gen, e, 2 * case["inner"], case["hidden"], case["group"], dtype, case["zeros"])
        st["down"] = _weights(gen, e, case["hidden"], case["inner"], case["group"], dtype, case["zeros"])
        score = torch.softmax(_normal(gen, t, e) + 0.5 * _normal(gen, 1, e), -1)   # some experts are more popular
        weights, ids = score.topk(k, -1)
        ids = ids.to(torch.int32)
        if case["dropped"]:
            ids = ids.masked_fill(torch.rand(t, k, generator=gen, device="cuda") < 0.03, -1)
        st["weights"], st["ids"] = (weights / weights.sum(-1, keepdim=True)).contiguous(), ids.contiguous()
        st["most"] = max(1, int(torch.bincount(ids.clamp(min=0).flatten(), minlength=e).max()))   # rows of the busiest expert
    else:
        st["w"] = (_normal(gen, case["n"], case["k"]) * 0.02).to(_T[case["dtype"]])
    return st


# ---- one pass ------------------------------------------------------------------------------------------------------
def run(st):
    if own:
        return _run_own(st)
    return {"gemm": _plain_gemm, "route": _plain_route, "experts": _plain_experts, "quantize": _plain_quantize}[st["op"]](st)


def _run_own(st):
    import vq_gemm_b200 as V
    if st["op"] == "gemm":
        return V.int4_gemm(st["x"], *st["w"])
    if st["op"] == "route":
        return V.route_experts(st["logits"], st["top_k"], scoring=st["scoring"], bias=st["bias_values"], groups=st["groups"],
                               top_groups=st["top_groups"], renormalize=st["renormalize"])
    if st["op"] == "experts":
        return V.int4_experts(st["x"], st["ids"], st["weights"], st["gate_up"], st["down"])
    packed, scales, zeros = V.quantize.int4_quantize(st["w"], group=st["group"], symmetric=not st["zeros"])
    return V.int4_dequant(packed, scales, zeros, in_features=st["k"]), scales


def _codes(packed, n, k):
    """The codes [..., n, k] of a packed weight, as fp32."""
    *lead, n16, k64, _ = packed.shape
    b = packed.reshape(-1, n16, k64, 4, 8, 4, 2, 2)                      # t, g, s, e, q
    c = torch.stack((b & 15, b >> 4))                                   # row half first
    c = c.permute(1, 2, 0, 5, 3, 4, 6, 8, 7)                            # tile row, h, g, tile column, t, s, q, e
    return c.reshape(*lead, n16 * 16, k64 * 64)[..., :n, :k].float()


def _values(weight, n, k):
    """W in fp32, rounded to the scales' type as the format says."""
    packed, scales, zeros = weight
    s = scales.transpose(-1, -2).float().unsqueeze(-1)
    z = 8.0 if zeros is None else zeros.transpose(-1, -2).float().unsqueeze(-1)
    c = _codes(packed, n, k)
    w = (c.unflatten(-1, (s.shape[-2], -1)) - z) * s
    return w.flatten(-2).to(scales.dtype).float()


def _plain_gemm(st):
    w = _values(st["w"], st["n"], st["k"])
    return (st["x"].float() @ w.t()).to(st["x"].dtype)


def _plain_route(st):
    # scores in 64 bits: which of two close scores is the larger must not depend on their rounding
    x = st["logits"].double()
    usable = x > -math.inf
    x = x.masked_fill(~usable, -math.inf)
    if st["scoring"] == "softmax":
        top = x.amax(-1, keepdim=True)
        p = torch.exp(x - torch.where(top > -math.inf, top, 0.0))
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total > 0, total, 1.0)
    else:
        p = 1 / (1 + torch.exp(-x))
    choice = p if st["bias_values"] is None else p + st["bias_values"].double()
    choice = choice.masked_fill(~usable, -math.inf)
    if st["groups"] > 1:
        g = choice.unflatten(-1, (st["groups"], -1))
        best = g.sort(dim=-1, descending=True).values[..., :2]
        best = torch.where(torch.isinf(best).any(-1) & (best[..., 0] > -math.inf), best[..., 0], best.sum(-1))
        kept = best.sort(dim=-1, descending=True, stable=True).indices[..., :st["top_groups"]]
        mask = torch.zeros_like(best, dtype=torch.bool).scatter(-1, kept, True)
        choice = torch.where(mask.unsqueeze(-1), g, -math.inf).flatten(-2)
    values, ids = choice.sort(dim=-1, descending=True, stable=True)
    values, ids = values[:, :st["top_k"]], ids[:, :st["top_k"]]
    w = torch.where(values > -math.inf, p.gather(-1, ids), 0.0)
    ids = torch.where(values > -math.inf, ids, -1)
    if st["renormalize"]:
        total = w.sum(-1, keepdim=True)
        w = w / torch.where(total > 0, total, 1.0)
    return w.float(), ids.to(torch.int32)


def _plain_experts(st):
    t, e, k, hidden, inner = st["t"], st["e"], st["top_k"], st["hidden"], st["inner"]
    flat = st["ids"].flatten().long()
    there = flat >= 0
    x = st["x"].float()
    if t * k <= e:      # fewer rows than experts: the chosen experts' weights row by row
        pick = flat.clamp(min=0)
        gu = _values([None if v is None else v[pick] for v in st["gate_up"]], 2 * inner, hidden)
        dn = _values([None if v is None else v[pick] for v in st["down"]], hidden, inner)
        h = torch.bmm(gu, x.repeat_interleave(k, 0).unsqueeze(-1)).squeeze(-1)
        h = h[:, 0::2] / (1 + torch.exp(-h[:, 0::2])) * h[:, 1::2]
        y = torch.bmm(dn, h.unsqueeze(-1)).squeeze(-1)
    else:               # the rows of each expert next to each other, as many as the busiest one has
        key = torch.where(there, flat, e)
        order = key.sort(stable=True).indices
        first = torch.searchsorted(key[order], torch.arange(e + 1, device=key.device))
        place = torch.empty_like(key)
        place[order] = torch.arange(t * k, device=key.device) - first[key[order]]
        place = place % st["most"]                                      # dropped slots share places of a row of their own
        rows = torch.zeros(e + 1, st["most"], hidden, device=x.device)
        rows[key, place] = x.repeat_interleave(k, 0)
        h = torch.bmm(rows[:e], _values(st["gate_up"], 2 * inner, hidden).transpose(-1, -2))
        h = h[..., 0::2] / (1 + torch.exp(-h[..., 0::2])) * h[..., 1::2]
        y = torch.bmm(h, _values(st["down"], hidden, inner).transpose(-1, -2))
        y = y[key.clamp(max=e - 1), place]
    y = torch.where(there.unsqueeze(-1), y * st["weights"].flatten().unsqueeze(-1), 0.0)
    return y.view(t, k, hidden).sum(1).to(st["x"].dtype)


def _plain_quantize(st):
    n, k, group = st["n"], st["k"], st["group"]
    w = st["w"].float().view(n, k // group, group)
    if st["zeros"]:
        low, high = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
        s = ((high - low) / 15).to(st["w"].dtype)
    else:
        s = (w.abs().amax(-1) / 7).to(st["w"].dtype)
    d = torch.where(s > 0, s.float(), 1.0)
    z = (-low / d).round().clamp(0, 15) if st["zeros"] else torch.full_like(d, 8.0)
    c = ((w / d[..., None]).round() + z[..., None]).clamp(0, 15)
    packed = _pack(c.to(torch.uint8).view(n, k))
    scales = s.t().contiguous()
    zeros = z.t().to(torch.uint8).contiguous() if st["zeros"] else None
    return _values((packed, scales, zeros), n, k).to(st["w"].dtype), scales


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def _weight_bytes(n, k, group, zeros):
    return n * k / 2 + n * (k // group) * (3 if zeros else 2)


def work(case):
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": _weight_bytes(n, k, case["group"], case["zeros"]) + 2 * m * (n + k), "flops": 2 * m * n * k}
    if case["op"] == "route":
        t, e = case["t"], case["e"]
        return {"bytes": t * e * (4 if case["dtype"] == "fp32" else 2) + t * case["top_k"] * 8 + (4 * e if case["bias"] else 0),
                "flops": 4 * t * e}
    if case["op"] == "experts":
        t, e, k, hidden, inner = case["t"], case["e"], case["top_k"], case["hidden"], case["inner"]
        reached = e * (1 - (1 - k / e) ** t)                            # experts that an even routing reaches
        one = _weight_bytes(2 * inner, hidden, case["group"], case["zeros"]) + _weight_bytes(hidden, inner, case["group"], case["zeros"])
        return {"bytes": reached * one + 4 * t * hidden + 8 * t * k, "flops": 6 * t * k * hidden * inner}
    n, k = case["n"], case["k"]
    return {"bytes": 4 * n * k + 2 * n * (k // case["group"]), "flops": 4 * n * k}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------
def _exact_weight(packed, scales, zeros, n, k):
    """W from the byte and nibble address of every (row, column), in 64 bits, rounded to the scales' type."""
    dev = packed.device
    r, c = torch.arange(n, device=dev)[:, None], torch.arange(k, device=dev)[None, :]
    col = c % 64
    t, s, q, e = col // 16, col // 4 % 4, col // 2 % 2, col % 2
    address = ((r // 16) * packed.shape[-2] + c // 64) * 512 + t * 128 + (r % 8) * 16 + s * 4 + e * 2 + q
    code = (packed.reshape(-1)[address].long() >> (4 * (r // 8 % 2))) & 15
    g = (c // (k // scales.shape[0])).expand(n, k)
    r = r.expand(n, k)
    z = zeros[g, r].double() if zeros is not None else 8.0
    return ((code.double() - z) * scales[g, r].double()).to(scales.dtype).double()


def _exact_route(st):
    x, p = st["logits"].double().cpu(), None
    if st["scoring"] == "softmax":
        p = torch.softmax(x, -1).nan_to_num(0.0)
    else:
        p = torch.special.expit(x)
    key = p + (st["bias_values"].double().cpu() if st["bias_values"] is not None else 0.0)
    key = torch.where(torch.isneginf(x), -math.inf, key)
    if st["groups"] > 1:
        size = st["e"] // st["groups"]
        per = key.reshape(-1, st["groups"], size)
        two = torch.topk(per, 2, -1).values if size > 1 else per
        two = two.clamp(min=-1e300)
        group = torch.where(two[..., 0] <= -1e300, -math.inf, torch.where(two[..., -1] <= -1e300, two[..., 0], two.sum(-1)))
        rank = torch.argsort(torch.argsort(-group, dim=-1, stable=True), dim=-1)
        key = torch.where((rank < st["top_groups"]).repeat_interleave(size, -1), key, -math.inf)
    ids = torch.argsort(-key, dim=-1, stable=True)[:, :st["top_k"]]
    good = torch.isfinite(torch.take_along_dim(key, ids, -1))
    w = torch.take_along_dim(p, ids, -1) * good
    if st["renormalize"]:
        w = (w / w.sum(-1, keepdim=True)).nan_to_num(0.0)
    return w, torch.where(good, ids, -1).to(torch.int32)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "gemm":
        return st["x"].double() @ _exact_weight(*st["w"], case["n"], case["k"]).t()
    if case["op"] == "route":
        return _exact_route(st)
    if case["op"] == "experts":
        y = torch.zeros(case["t"], case["hidden"], dtype=torch.float64, device="cuda")
        for i in range(case["e"]):
            token, slot = torch.where(st["ids"] == i)
            if not len(token):
                continue
            one = [[None if v is None else v[i] for v in st[name]] for name in ("gate_up", "down")]
            h = st["x"][token].double() @ _exact_weight(*one[0], 2 * case["inner"], case["hidden"]).t()
            h = torch.nn.functional.silu(h[:, ::2]) * h[:, 1::2]
            y.index_add_(0, token, h @ _exact_weight(*one[1], case["hidden"], case["inner"]).t() * st["weights"][token, slot].double()[:, None])
        return y
    n, k, group, w = case["n"], case["k"], case["group"], st["w"].double()
    blocks = w.reshape(n, -1, group)
    if case["zeros"]:
        bottom, top = blocks.min(-1).values.clamp(max=0), blocks.max(-1).values.clamp(min=0)
        scale = ((top - bottom) / 15).to(st["w"].dtype).double()
        zero = torch.round(-bottom / scale).clamp(0, 15)
    else:
        scale, zero = (blocks.abs().max(-1).values / 7).to(st["w"].dtype).double(), 8.0
    zero = zero[..., None] if case["zeros"] else zero
    code = (torch.round(blocks / scale[..., None]) + zero).clamp(0, 15)
    value = ((code - zero) * scale[..., None]).nan_to_num(0.0).reshape(n, k)
    return value.to(st["w"].dtype).double(), scale.t()
