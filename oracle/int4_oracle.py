"""CPU restatement in 64 bits of the 4-bit weights, the expert router and the experts' products (test infrastructure).

The bounds that come with the products follow from the formulas: u is half a step of the result's type relative to its
value, and a sum of K products in fp32 over matrix instructions of sixteen is off by at most (K / 16 + 32) steps of 2^-23 of
the sum of the products' magnitudes, whatever its order."""
import numpy as np
import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def unpack(packed, n, k):
    """Codes [n, k] from the byte and nibble address of every (row, column)."""
    p = packed.cpu().numpy().reshape(-1)
    tiles = packed.shape[-2]
    r, c = np.arange(n)[:, None], np.arange(k)[None, :]
    col = c % 64
    t, s, q, e = col // 16, col // 4 % 4, col // 2 % 2, col % 2
    byte = p[((r // 16) * tiles + c // 64) * 512 + ((((t * 8 + r % 8) * 4 + s) * 2 + e) * 2 + q)]
    return torch.from_numpy((byte >> (4 * (r // 8 % 2))) & 15)


def weights(packed, scales, zeros, k):
    """W [n, k] as float64: (code - zero) * scale rounded to the type of the scales."""
    n = scales.shape[1]
    group = torch.arange(k) // (k // scales.shape[0])
    s = scales.cpu().double()[group].t()
    z = 8.0 if zeros is None else zeros.cpu().double()[group].t()
    return ((unpack(packed, n, k).double() - z) * s).to(scales.dtype).double()


def quantize(w, group, symmetric):
    """(codes [n, k], scales [k/group, n], zeros or None) by the quantiser's rule; numpy fp32 arithmetic."""
    n, k = w.shape
    v = w.cpu().float().numpy().reshape(n, k // group, group)
    if symmetric:
        raw, low = np.abs(v).max(-1) / np.float32(7), None
    else:
        low, high = np.minimum(v.min(-1), np.float32(0)), np.maximum(v.max(-1), np.float32(0))
        raw = (high - low) / np.float32(15)
    scale = torch.from_numpy(raw).to(w.dtype)
    d = scale.float().numpy()
    d = np.where(d > 0, d, np.float32(1))
    zero = np.full_like(d, 8) if symmetric else np.clip(np.rint(-low / d), 0, 15)
    code = np.clip(np.rint(v / d[..., None]) + zero[..., None], 0, 15)
    return (torch.from_numpy(code.astype(np.uint8)).reshape(n, k), scale.t().contiguous(),
            None if symmetric else torch.from_numpy(zero.astype(np.uint8)).t().contiguous())


def sum_error(k):
    return (k / 16 + 32) * 2.0 ** -23


def gemm(x, packed, scales, zeros=None):
    """(Y, bound) as float64."""
    w = weights(packed, scales, zeros, x.shape[1])
    xd = x.cpu().double()
    y = xd @ w.t()
    return y, HALF_STEP[x.dtype] * y.abs() + sum_error(x.shape[1]) * (xd.abs() @ w.abs().t()) + TINY[x.dtype]


def route(logits, top_k, scoring="softmax", bias=None, groups=1, top_groups=None, group_score="top2", renormalize=False, scale=1.0):
    """(weights float64, ids int32), row by row."""
    out_w, out_i = [], []
    top_groups = groups if top_groups is None else top_groups
    for row in logits.cpu().double().numpy():
        usable = row > -np.inf                              # False for NaN too
        p = np.zeros_like(row)
        if usable.any():
            top = row[usable].max()
            if scoring == "softmax":
                if np.isinf(top):
                    p[row == np.inf] = 1.0
                else:
                    p[usable] = np.exp(row[usable] - top)
                p = p / p.sum()
            else:
                p[usable] = 1.0 / (1.0 + np.exp(-row[usable]))
        choice = p + (0.0 if bias is None else bias.cpu().double().numpy())
        choice = np.where(usable, choice, -np.inf)
        if groups > 1:
            per = choice.reshape(groups, -1)
            score = []
            for g in per:
                best = sorted((c for c in g if c > -np.inf), reverse=True)
                score.append(-np.inf if not best else best[0] if group_score == "max" else sum(best[:2]))
            keep = sorted(range(groups), key=lambda i: (-score[i], i))[:top_groups]
            for i in range(groups):
                if i not in keep:
                    per[i] = -np.inf
            choice = per.reshape(-1)
        ids = [e for e in sorted(range(len(row)), key=lambda e: (-choice[e], e))[:top_k] if choice[e] > -np.inf]
        w = p[ids]
        if renormalize:
            w = w / w.sum() if w.sum() > 0 else np.zeros_like(w)
        pad = top_k - len(ids)
        out_w.append(np.concatenate([w * scale, np.zeros(pad)]))
        out_i.append(ids + [-1] * pad)
    return torch.from_numpy(np.array(out_w).reshape(-1, top_k)), torch.tensor(out_i, dtype=torch.int32).reshape(-1, top_k)


def experts(x, ids, weights_, gate_up, down):
    """(Y, bound) as float64.  The bound carries the gated product's rounding to x's type through the second product."""
    t, hidden = x.shape
    u, xd = HALF_STEP[x.dtype], x.cpu().double()
    inner = gate_up[1].shape[2] // 2
    y, size, off = torch.zeros(t, hidden, dtype=torch.float64), torch.zeros(t, hidden, dtype=torch.float64), 0.0
    off = torch.zeros_like(y)
    for e in range(gate_up[0].shape[0]):
        token, slot = torch.where(ids.cpu() == e)
        if not len(token):
            continue
        one = [[None if v is None else v[e] for v in wt] for wt in (gate_up, down)]
        wu, wd = weights(*one[0], hidden), weights(*one[1], inner)
        a, s = xd[token] @ wu.t(), sum_error(hidden) * (xd[token].abs() @ wu.abs().t())
        g, up, sg, su = a[:, 0::2], a[:, 1::2], s[:, 0::2], s[:, 1::2]
        silu = g / (1 + torch.exp(-g))
        h = silu * up
        # |d silu| <= 1.1; the exponential, its division and the product in fp32 are off by a few steps
        dh = 1.1 * sg * (up.abs() + su) + silu.abs() * su + (u + 2.0 ** -18) * h.abs() + TINY[x.dtype]
        c = weights_.cpu().double()[token, slot][:, None]
        y.index_add_(0, token, c * (h @ wd.t()))
        off.index_add_(0, token, c.abs() * (dh @ wd.abs().t()))
        size.index_add_(0, token, c.abs() * ((h.abs() + dh) @ wd.abs().t()))
    return y, u * y.abs() + off + (sum_error(inner) + ids.shape[1] * 2.0 ** -23) * size + TINY[x.dtype]
