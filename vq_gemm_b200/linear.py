"""Caller side of the boundary: the VQ-GEMM as a registered torch operator and an ``nn.Module``.

The reference stops at ``bench.py`` calling ``e2e_gemm`` on raw tensors (bench.py:66-80); a model
needs the product as a layer.  ``vq_gemm_b200::vq_linear`` is registered with ``torch.library`` so
that it can be traced (a fake-tensor rule gives shapes and dtypes without running anything), used
under ``torch.compile`` as an opaque call, and captured in CUDA graphs: the launch allocates nothing
but its output, and the scratch it uses is cached per (device, stream) and left as it found it.

Inference only: no autograd formula is registered.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import nn

from . import ops


@torch.library.custom_op("vq_gemm_b200::vq_linear", mutates_args=(), device_types="cuda")
def vq_linear(x: torch.Tensor, indices: torch.Tensor, codebook: torch.Tensor, rows_per_codebook: int) -> torch.Tensor:
    """x [M, K] fp16, indices [N, K/v] uint8/int16, codebook [G, C, v] fp16 -> [M, N] fp16."""
    return ops.vq_gemm(x, indices, codebook, rows_per_codebook=rows_per_codebook, layout="bl")


@vq_linear.register_fake
def _(x, indices, codebook, rows_per_codebook):
    if x.dim() != 2 or indices.dim() != 2 or codebook.dim() != 3:
        raise RuntimeError("vq_linear expects x [M, K], indices [N, K/v], codebook [G, C, v]")
    if indices.shape[1] * codebook.shape[2] != x.shape[1]:
        raise RuntimeError("indices [N, K/v] and codebook [G, C, v] do not match x [M, K]")
    return x.new_empty((x.shape[0], indices.shape[0]))


@torch.library.custom_op("vq_gemm_b200::vq_linear_residual", mutates_args=(), device_types="cuda")
def vq_linear_residual(x: torch.Tensor, indices: torch.Tensor, codebook: torch.Tensor, rows_per_codebook: int) -> torch.Tensor:
    """Residual weights: x [M, K] fp16, indices [S, N, K/v], codebook [S, G, C, v] fp16 -> [M, N] fp16."""
    return ops.vq_gemm_residual(x, indices, codebook, rows_per_codebook=rows_per_codebook)


@vq_linear_residual.register_fake
def _(x, indices, codebook, rows_per_codebook):
    if x.dim() != 2 or indices.dim() != 3 or codebook.dim() != 4 or indices.shape[0] != codebook.shape[0]:
        raise RuntimeError("vq_linear_residual expects x [M, K], indices [S, N, K/v], codebook [S, G, C, v]")
    if indices.shape[2] * codebook.shape[3] != x.shape[1]:
        raise RuntimeError("indices [S, N, K/v] and codebook [S, G, C, v] do not match x [M, K]")
    return x.new_empty((x.shape[0], indices.shape[1]))


@torch.library.custom_op("vq_gemm_b200::vq_linear_packed12", mutates_args=(), device_types="cuda")
def vq_linear_packed12(x: torch.Tensor, packed: torch.Tensor, codebook: torch.Tensor, rows_per_codebook: int) -> torch.Tensor:
    """12-bit indices packed two to three bytes: x [M, K] fp16, packed [N, K/v * 3/2] uint8, codebook [G, C, v]."""
    return ops.vq_gemm(x, packed, codebook, rows_per_codebook=rows_per_codebook, layout="bl", index_bits=12)


@vq_linear_packed12.register_fake
def _(x, packed, codebook, rows_per_codebook):
    if x.dim() != 2 or packed.dim() != 2 or codebook.dim() != 3 or packed.shape[1] % 3:
        raise RuntimeError("vq_linear_packed12 expects x [M, K], packed [N, K/v * 3/2], codebook [G, C, v]")
    if packed.shape[1] * 2 // 3 * codebook.shape[2] != x.shape[1]:
        raise RuntimeError("packed [N, K/v * 3/2] and codebook [G, C, v] do not match x [M, K]")
    return x.new_empty((x.shape[0], packed.shape[0]))


@torch.library.custom_op("vq_gemm_b200::vq_swiglu", mutates_args=(), device_types="cuda")
def vq_swiglu(x: torch.Tensor, indices: torch.Tensor, codebook: torch.Tensor, rows_per_codebook: int) -> torch.Tensor:
    """x [M, K]; indices [2*N_out, K/v] with (gate, up) row pairs -> SiLU(x g^T) * (x u^T), [M, N_out] fp16."""
    return ops.vq_gemm_swiglu(x, indices, codebook, rows_per_codebook=rows_per_codebook)


@vq_swiglu.register_fake
def _(x, indices, codebook, rows_per_codebook):
    if x.dim() != 2 or indices.dim() != 2 or codebook.dim() != 3 or indices.shape[0] % 2:
        raise RuntimeError("vq_swiglu expects x [M, K], indices [2*N_out, K/v], codebook [G, C, v]")
    if indices.shape[1] * codebook.shape[2] != x.shape[1]:
        raise RuntimeError("indices [2*N_out, K/v] and codebook [G, C, v] do not match x [M, K]")
    return x.new_empty((x.shape[0], indices.shape[0] // 2))


@torch.library.custom_op("vq_gemm_b200::int4_linear", mutates_args=(), device_types="cuda")
def int4_linear(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor]) -> torch.Tensor:
    """x [M, K], packed [ceil(N/16), ceil(K/64), 512] uint8, scales [K/group, N] (and zeros, uint8) -> [M, N] of x's type."""
    return ops.int4_gemm(x, packed, scales, zeros)


@int4_linear.register_fake
def _(x, packed, scales, zeros):
    if x.dim() != 2:
        raise RuntimeError("int4_linear expects x [M, K]")
    N, _ = ops._int4_weight(packed, scales, zeros, x.shape[1], False)
    return x.new_empty((x.shape[0], N))


@torch.library.custom_op("vq_gemm_b200::route_experts", mutates_args=(), device_types="cuda")
def route_experts(logits: torch.Tensor, top_k: int, scoring: str, bias: Optional[torch.Tensor], groups: int, top_groups: int,
                  group_score: str, renormalize: bool, scale: float) -> Tuple[torch.Tensor, torch.Tensor]:
    """logits [T, E] -> (weights [T, top_k] float32, experts [T, top_k] int32); see ``ops.route_experts``."""
    return ops.route_experts(logits, top_k, scoring=scoring, bias=bias, groups=groups, top_groups=top_groups,
                             group_score=group_score, renormalize=renormalize, scale=scale)


@route_experts.register_fake
def _(logits, top_k, scoring, bias, groups, top_groups, group_score, renormalize, scale):
    if logits.dim() != 2:
        raise RuntimeError("route_experts expects logits [T, E]")
    shape = (logits.shape[0], top_k)
    return logits.new_empty(shape, dtype=torch.float32), logits.new_empty(shape, dtype=torch.int32)


@torch.library.custom_op("vq_gemm_b200::int4_experts", mutates_args=(), device_types="cuda")
def int4_experts(x: torch.Tensor, experts: torch.Tensor, weights: torch.Tensor, up_packed: torch.Tensor,
                 up_scales: torch.Tensor, up_zeros: Optional[torch.Tensor], down_packed: torch.Tensor,
                 down_scales: torch.Tensor, down_zeros: Optional[torch.Tensor]) -> torch.Tensor:
    """x [T, hidden] through its chosen experts; see ``ops.int4_experts``."""
    return ops.int4_experts(x, experts, weights, (up_packed, up_scales, up_zeros), (down_packed, down_scales, down_zeros))


@int4_experts.register_fake
def _(x, experts, weights, up_packed, up_scales, up_zeros, down_packed, down_scales, down_zeros):
    if x.dim() != 2 or experts.dim() != 2 or experts.shape[0] != x.shape[0]:
        raise RuntimeError("int4_experts expects x [T, hidden], experts and weights [T, top_k]")
    rows, _ = ops._int4_weight(up_packed, up_scales, up_zeros, x.shape[1], True)
    ops._int4_weight(down_packed, down_scales, down_zeros, rows // 2, True)
    return torch.empty_like(x)


class VQLinear(nn.Module):
    """``y = x @ dequant(indices, codebook)^T (+ bias)`` with the weight kept in compressed form.

    ``indices`` [out_features, in_features / v] (uint8, or int16 for codebooks of more than 256
    entries), ``codebook`` [groups, C, v] fp16 with one codebook per ``rows_per_codebook``
    consecutive output features (0: a single codebook).  Both are buffers, so ``state_dict`` /
    ``load_state_dict`` / ``.to(device)`` carry them.  Accepts inputs of any leading shape.

    Residual (multi-codebook) weights: ``indices`` [S, out_features, in_features / v] and ``codebook``
    [S, groups, C, v]; the weight is the running fp16 sum of the S stages' entries (``from_weight(stages=2)``).

    ``index_bits=12``: ``indices`` is the uint8 [out_features, in_features / v * 3/2] tensor ``quantize.pack12``
    makes of 12-bit indices (codebooks of up to 4096 entries at 1.5 bytes per index); ``pack()`` converts a layer
    that holds them in int16.
    """

    def __init__(self, indices: torch.Tensor, codebook: torch.Tensor, rows_per_codebook: int = 0,
                 bias: Optional[torch.Tensor] = None, index_bits: Optional[int] = None):
        super().__init__()
        self.packed = index_bits == 12
        if index_bits not in (None, 8, 16, 12):
            raise ValueError("index_bits must be 8, 16 or 12 (packed)")
        if self.packed and (indices.dim() != 2 or indices.dtype != torch.uint8 or indices.shape[1] % 3):
            raise ValueError("packed indices must be a uint8 [N, K/v * 3/2] tensor")
        self.residual = indices.dim() == 3
        if self.residual:
            if codebook.dim() != 4 or codebook.shape[0] != indices.shape[0]:
                raise ValueError("residual weights need indices [S, N, K/v] and codebook [S, G, C, v]")
        elif indices.dim() != 2 or codebook.dim() not in (2, 3):
            raise ValueError("indices must be [N, K/v] and codebook [G, C, v] (or [C, v])")
        if indices.dtype not in (torch.uint8, torch.int16, torch.uint16):
            raise ValueError("indices must be uint8 or (u)int16")
        cb = codebook if codebook.dim() >= 3 else codebook.unsqueeze(0)
        N = indices.shape[-2]
        groups = 1 if rows_per_codebook <= 0 else -(-N // rows_per_codebook)
        if cb.shape[-3] < groups or (self.residual and cb.shape[-3] != groups):
            raise ValueError(f"{cb.shape[-3]} codebooks given, {groups} needed")
        self.out_features = N
        self.v = cb.shape[-1]
        self.in_features = (indices.shape[-1] * 2 // 3 if self.packed else indices.shape[-1]) * self.v
        self.rows_per_codebook = int(rows_per_codebook)
        self.register_buffer("indices", indices.contiguous())
        self.register_buffer("codebook", cb.to(torch.float16).contiguous())
        if bias is not None:
            if bias.shape != (N,):
                raise ValueError("bias must be [out_features]")
            self.register_buffer("bias", bias.to(torch.float16).contiguous())
        else:
            self.bias = None

    @classmethod
    def from_weight(cls, weight: torch.Tensor, *, v: int = 8, entries: int = 256, rows_per_codebook: int = 128,
                    iters: int = 10, seed: int = 0, bias: Optional[torch.Tensor] = None, stages: int = 1) -> "VQLinear":
        """Quantises a dense [out_features, in_features] weight (on its CUDA device) with k-means; ``stages`` > 1
        gives residual weights (every further stage quantises what the stages before it left over)."""
        from .quantize import kmeans_quantize, kmeans_quantize_residual
        if stages > 1:
            idx, cb = kmeans_quantize_residual(weight, stages=stages, v=v, entries=entries, rows_per_codebook=rows_per_codebook,
                                               iters=iters, seed=seed)
        else:
            idx, cb = kmeans_quantize(weight, v=v, entries=entries, rows_per_codebook=rows_per_codebook, iters=iters, seed=seed)
        return cls(idx, cb, rows_per_codebook, bias)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.in_features:
            raise RuntimeError(f"last dimension {x.shape[-1]} != in_features {self.in_features}")
        lead = x.shape[:-1]
        x2 = x.reshape(-1, self.in_features)
        if x2.dtype != torch.float16:
            x2 = x2.to(torch.float16)
        op = (torch.ops.vq_gemm_b200.vq_linear_residual if self.residual else
              torch.ops.vq_gemm_b200.vq_linear_packed12 if self.packed else torch.ops.vq_gemm_b200.vq_linear)
        y = op(x2.contiguous(), self.indices, self.codebook, self.rows_per_codebook)
        if self.bias is not None:
            y = y + self.bias
        return y.reshape(*lead, self.out_features)

    def dequantized_weight(self) -> torch.Tensor:
        """The dense fp16 [out_features, in_features] weight this layer stands for (bit-exact gather)."""
        if self.residual:
            return ops.dequant_residual(self.indices, self.codebook, rows_per_codebook=self.rows_per_codebook)
        return ops.dequant(self.indices, self.codebook, rows_per_codebook=self.rows_per_codebook,
                           index_bits=12 if self.packed else None)

    def pack(self) -> "VQLinear":
        """The same layer with its 12-bit indices (held in int16, at most 4096 entries) packed two to three bytes."""
        from .quantize import pack12
        if self.packed:
            return self
        if self.residual or self.indices.dtype == torch.uint8 or self.codebook.shape[-2] > 4096:
            raise RuntimeError("pack() is for plain weights with int16 indices and at most 4096 entries")
        return VQLinear(pack12(self.indices), self.codebook, self.rows_per_codebook, self.bias, index_bits=12)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, v={self.v}, "
                f"entries={self.codebook.shape[-2]}, rows_per_codebook={self.rows_per_codebook}, "
                f"stages={self.indices.shape[0] if self.residual else 1}, packed12={self.packed}, bias={self.bias is not None}")


class VQGatedUp(nn.Module):
    """First half of a gated MLP with compressed weights: ``SiLU(x W_gate^T) * (x W_up^T)``.

    ``indices`` [2 * intermediate, in_features / v] holds the two projections row-interleaved
    (row 2i = gate row i, row 2i+1 = up row i; ``ops.interleave_gate_up`` builds that order), one
    codebook per ``rows_per_codebook`` of those interleaved rows.  For more than 128 input rows the
    combination happens in the GEMM kernel's epilogue and the two products never reach memory."""

    def __init__(self, indices: torch.Tensor, codebook: torch.Tensor, rows_per_codebook: int = 0):
        super().__init__()
        if indices.dim() != 2 or indices.shape[0] % 2 or codebook.dim() not in (2, 3):
            raise ValueError("indices must be [2*N_out, K/v] and codebook [G, C, v] (or [C, v])")
        cb = codebook if codebook.dim() == 3 else codebook.unsqueeze(0)
        self.v = cb.shape[2]
        self.in_features = indices.shape[1] * self.v
        self.out_features = indices.shape[0] // 2
        self.rows_per_codebook = int(rows_per_codebook)
        self.register_buffer("indices", indices.contiguous())
        self.register_buffer("codebook", cb.to(torch.float16).contiguous())

    @classmethod
    def from_weights(cls, gate: torch.Tensor, up: torch.Tensor, *, v: int = 8, entries: int = 256,
                     rows_per_codebook: int = 128, iters: int = 10, seed: int = 0) -> "VQGatedUp":
        """Quantises two dense [intermediate, in_features] fp16 CUDA weights, interleaved, with k-means."""
        from .quantize import kmeans_quantize
        w = ops.interleave_gate_up(gate, up)
        idx, cb = kmeans_quantize(w, v=v, entries=entries, rows_per_codebook=rows_per_codebook, iters=iters, seed=seed)
        return cls(idx, cb, rows_per_codebook)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.in_features:
            raise RuntimeError(f"last dimension {x.shape[-1]} != in_features {self.in_features}")
        lead = x.shape[:-1]
        x2 = x.reshape(-1, self.in_features)
        if x2.dtype != torch.float16:
            x2 = x2.to(torch.float16)
        y = torch.ops.vq_gemm_b200.vq_swiglu(x2.contiguous(), self.indices, self.codebook, self.rows_per_codebook)
        return y.reshape(*lead, self.out_features)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, v={self.v}, "
                f"entries={self.codebook.shape[1]}, rows_per_codebook={self.rows_per_codebook}")


class _KeptTypes(nn.Module):
    """A module with floating buffers (``_kept``) whose bits matter: casting a model (``.half()``, ``.to(dtype)``) moves them with it and
    leaves their type; what the model is cast to becomes the type of the module's results (``result_type``, None before: the
    module's own)."""

    _kept: Tuple[str, ...] = ()
    result_type: Optional[torch.dtype] = None

    def _apply(self, fn, recurse=True):
        # what fn makes of two types tells a cast from a move
        to = {fn(torch.empty(0, dtype=t)).dtype for t in (torch.float64, torch.float32)}
        if len(to) == 1:
            self.result_type = to.pop()
        before = {name: self._buffers[name] for name in self._kept if self._buffers.get(name) is not None}
        super()._apply(fn, recurse)
        for name, t in before.items():
            if self._buffers[name].dtype != t.dtype:
                self._buffers[name] = t.to(self._buffers[name].device)
        return self


class Int4Linear(_KeptTypes):
    """``y = x @ W^T (+ bias)`` with 4-bit weights and group scales, for the layers that one or two bits do not serve.

    ``packed`` [ceil(out/16), ceil(in/64), 512] uint8, ``scales`` [in/group, out] float16 or bfloat16 -- the layer's type --
    and optionally ``zeros`` [in/group, out] uint8, as ``quantize.int4_quantize`` makes them; ``in_features`` where it is
    not a multiple of 64.  All are buffers.  Accepts inputs of any leading shape and casts them to the layer's type.  Casting a
    model leaves the layer's type and weights as they are and has the result in the model's type."""

    _kept = ("scales", "bias")

    def __init__(self, packed: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None,
                 bias: Optional[torch.Tensor] = None, in_features: Optional[int] = None):
        super().__init__()
        self.in_features = packed.shape[-2] * 64 if in_features is None else int(in_features)
        try:
            self.out_features, self.group = ops._int4_weight(packed, scales, zeros, self.in_features, False)
        except RuntimeError as e:
            raise ValueError(str(e)) from None
        self.register_buffer("packed", packed.contiguous())
        self.register_buffer("scales", scales.contiguous())
        self.register_buffer("zeros", None if zeros is None else zeros.contiguous())
        if bias is not None and bias.shape != (self.out_features,):
            raise ValueError("bias must be [out_features]")
        self.register_buffer("bias", None if bias is None else bias.to(scales.dtype).contiguous())

    @classmethod
    def from_weight(cls, weight: torch.Tensor, *, group: int = 128, symmetric: bool = True,
                    bias: Optional[torch.Tensor] = None) -> "Int4Linear":
        """Quantises a dense [out_features, in_features] fp16 or bf16 weight on its CUDA device."""
        from .quantize import int4_quantize
        return cls(*int4_quantize(weight, group=group, symmetric=symmetric), bias, weight.shape[1])

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.in_features:
            raise RuntimeError(f"last dimension {x.shape[-1]} != in_features {self.in_features}")
        x2 = x.reshape(-1, self.in_features).to(self.scales.dtype)
        y = torch.ops.vq_gemm_b200.int4_linear(x2.contiguous(), self.packed, self.scales, self.zeros)
        if self.bias is not None:
            y = y + self.bias
        return (y if self.result_type is None else y.to(self.result_type)).reshape(*x.shape[:-1], self.out_features)

    def dequantized_weight(self) -> torch.Tensor:
        """The dense [out_features, in_features] weight this layer stands for, bit for bit."""
        return ops.int4_dequant(self.packed, self.scales, self.zeros, in_features=self.in_features)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, group={self.group}, "
                f"zeros={self.zeros is not None}, bias={self.bias is not None}")


class Int4Experts(_KeptTypes):
    """Mixture-of-experts MLP with 4-bit experts: ``router`` (a module that gives logits [..., E], e.g. an ``Int4Linear``, a
    ``VQLinear`` or an ``nn.Linear``), then ``route_experts``, then the gated products of the chosen experts.

    ``gate_up`` and ``down`` are (packed, scales, zeros or None) of [E, 2 * inner, hidden] and [E, hidden, inner] weights;
    ``in_features`` is hidden.  ``bias`` [E] float32 is the router's balance bias.  Casting a
    model casts the router (an ``nn.Linear``, say), leaves the experts' weights and the balance bias as they are and has the result
    in the model's type."""

    _kept = ("gate_up_scales", "down_scales", "bias")

    def __init__(self, router: nn.Module, gate_up, down, *, top_k: int, in_features: int, scoring: str = "softmax",
                 bias: Optional[torch.Tensor] = None, groups: int = 1, top_groups: Optional[int] = None,
                 group_score: str = "top2", renormalize: bool = True, scale: float = 1.0):
        super().__init__()
        try:
            rows, _ = ops._int4_weight(*gate_up, in_features, True)
            hidden, _ = ops._int4_weight(*down, rows // 2, True)
        except RuntimeError as e:
            raise ValueError(str(e)) from None
        if rows % 2 or hidden != in_features or down[0].shape[0] != gate_up[0].shape[0]:
            raise ValueError("gate_up must be [E, 2 * inner, hidden] and down [E, hidden, inner]")
        self.router = router
        self.in_features, self.inner, self.experts = in_features, rows // 2, gate_up[0].shape[0]
        if not 1 <= top_k <= self.experts:
            raise ValueError(f"cannot choose {top_k} of {self.experts} experts")
        self.top_k, self.scoring, self.groups = top_k, scoring, groups
        self.top_groups = groups if top_groups is None else top_groups
        self.group_score, self.renormalize, self.scale = group_score, renormalize, scale
        for name, weight in (("gate_up", gate_up), ("down", down)):
            for part, t in zip(("packed", "scales", "zeros"), weight):
                self.register_buffer(f"{name}_{part}", None if t is None else t.contiguous())
        self.register_buffer("bias", None if bias is None else bias.to(torch.float32).contiguous())

    @classmethod
    def from_weights(cls, router: nn.Module, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor, *, group: int = 128,
                     symmetric: bool = True, **routing) -> "Int4Experts":
        """Quantises dense gate, up [E, inner, hidden] and down [E, hidden, inner] weights on their CUDA device."""
        from .quantize import int4_quantize
        pairs = torch.stack((gate, up), dim=2).flatten(1, 2).contiguous()      # row pairs: gate row i, up row i
        return cls(router, int4_quantize(pairs, group=group, symmetric=symmetric),
                   int4_quantize(down, group=group, symmetric=symmetric), in_features=gate.shape[2], **routing)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.in_features:
            raise RuntimeError(f"last dimension {x.shape[-1]} != in_features {self.in_features}")
        x2 = x.reshape(-1, self.in_features)
        logits = self.router(x2).contiguous()
        bias = None if self.bias is None else self.bias.float()       # (a checkpoint that was assigned may hold another type)
        weights, chosen = torch.ops.vq_gemm_b200.route_experts(
            logits, self.top_k, self.scoring, bias, self.groups, self.top_groups, self.group_score, self.renormalize,
            self.scale)
        y = torch.ops.vq_gemm_b200.int4_experts(
            x2.to(self.gate_up_scales.dtype).contiguous(), chosen, weights, self.gate_up_packed, self.gate_up_scales,
            self.gate_up_zeros, self.down_packed, self.down_scales, self.down_zeros)
        return (y if self.result_type is None else y.to(self.result_type)).reshape(x.shape)

    def extra_repr(self) -> str:
        return (f"hidden={self.in_features}, inner={self.inner}, experts={self.experts}, top_k={self.top_k}, "
                f"scoring={self.scoring}, groups={self.groups}, top_groups={self.top_groups}")
