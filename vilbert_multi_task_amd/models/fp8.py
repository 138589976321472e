"""Optional FP8 (OCP e4m3) serving mode with producer-fused quantization.

MI355X runs fp8 MFMA at ~2x the bf16 rate (~5 PF dense; gfx950 is OCP
e4m3fn, NOT MI300X's fnuz — cdna_hip_programming.md §4). The first
implementation (standalone per-GEMM quantization) measured SLOWER than bf16
— each GEMM paid an amax pass + a cast pass over its activations. This
version makes quantization ~free:

- DELAYED SCALING: every quantization site has a persistent (scale, amax)
  slot (Fp8Context). Producers emit e4m3 using the PREVIOUS step's scale
  while atomically accumulating this step's amax; one tiny kernel refreshes
  all scales at the end of the forward. Fully hipGraph-capturable.
- PRODUCER FUSION: the residual+LayerNorm and GELU kernels emit the e4m3
  copy as a side output (ops/csrc/elementwise.hip FP8OUT variants) — the
  data is already in registers, so the only cost is the 1-byte/elem write.
  The e4m3 tensor + its scale ride on the bf16 output as the `_fp8`
  attribute; consumers (Fp8Linear / the fused-QKV paths) use the pack when
  present and fall back to dynamic quantization otherwise (e.g. the text
  embeddings after task-token insertion).

Attention math, LayerNorm statistics and ALL task heads stay bf16. This is
an OPT-IN serving mode (GraphRunner(fp8=True) / bench.py --fp8); the judged
benchmark keeps the reference-grade bf16 path.

A second mode, ``convert_encoder_to_fp8_block`` (GraphRunner(fp8="block") /
bench.py --fp8-block), has one scale per 128 values, taken from the values
themselves (ops.functional's ``*_fp8_block``): no state between calls, no
warm-up steps, an outlier costs only its own block, and the same batch gives
the same bits whenever it is repeated. (A request in a batch of another size may
meet another kernel, which adds in another order; the last bit of a sum can move
an 8-bit value by a step.) LayerNorm emits its 8-bit form beside the bf16 one
(``_fp8b`` on the result), and a feed-forward's intermediate leaves the first
product in 8 bits, GELU applied, and never exists otherwise. Convert where the
model is served: the fused projections' weights stay on the device that they
were made on.
"""

from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

E4M3_MAX = 448.0


class Fp8Context:
    """Per-model registry of (scale, amax) slots for delayed scaling."""

    def __init__(self, nsites: int, device):
        self.scales = torch.ones(nsites, dtype=torch.float32, device=device)
        self.inv_scales = torch.ones(nsites, dtype=torch.float32, device=device)
        self.amaxes = torch.zeros(nsites, dtype=torch.float32, device=device)
        self.nsites = nsites

    def update(self) -> None:
        torch.ops.vilbert_amd.update_fp8_scales(
            self.scales, self.inv_scales, self.amaxes
        )


class _SiteAllocator:
    def __init__(self):
        self.n = 0

    def take(self) -> int:
        s = self.n
        self.n += 1
        return s


def quantize_weight(w: torch.Tensor):
    """Per-tensor symmetric quantization -> (w_fp8 [N,K], scale scalar)."""
    scale = (w.abs().amax().float() / E4M3_MAX).clamp(min=1e-12)
    w8 = (w.float() / scale).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return w8, scale.to(w.device)


def _dynamic_quant(x2: torch.Tensor):
    x_scale = (x2.abs().amax().float() / E4M3_MAX).clamp(min=1e-12)
    x8 = (x2.float() / x_scale).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return x8, x_scale


def fp8_mm(
    x: torch.Tensor,
    w8: torch.Tensor,
    w_scale: torch.Tensor,
    bias: Optional[torch.Tensor],
) -> torch.Tensor:
    """y = x @ w8.T * scales + bias, out bf16. Uses the producer-emitted
    e4m3 pack riding on x when present; dynamic quantization otherwise."""
    if w_scale.dim() == 2:  # a scale per block of 128 x 128
        return fp8_block_mm(x, w8, w_scale, bias).to(x.dtype)
    shape = x.shape
    pack = getattr(x, "_fp8", None)
    if pack is not None:
        x8, x_scale = pack
        x8 = x8.reshape(-1, shape[-1])
    else:
        x8, x_scale = _dynamic_quant(x.reshape(-1, shape[-1]))
    if bias is not None:
        try:
            y = torch.ops.vilbert_amd.fp8_linear(x8, w8, bias, w_scale, x_scale)
            return y.reshape(*shape[:-1], y.shape[-1])
        except RuntimeError:
            pass  # no hipBLASLt algo: _scaled_mm fallback
    y = torch._scaled_mm(
        x8, w8.t(), scale_a=x_scale, scale_b=w_scale, bias=bias,
        out_dtype=torch.bfloat16,
    )
    return y.reshape(*shape[:-1], y.shape[-1])


# backwards-compat alias used by the attention modules
def fp8_linear(x, w8, w_scale, bias):
    return fp8_mm(x, w8, w_scale, bias)


class Fp8Linear(nn.Module):
    """Inference-only drop-in for nn.Linear (weights pre-quantized)."""

    def __init__(self, linear: nn.Linear):
        super().__init__()
        w8, scale = quantize_weight(linear.weight.detach())
        self.register_buffer("w8", w8)
        self.register_buffer("w_scale", scale)
        self.bias = linear.bias
        self.in_features = linear.in_features
        self.out_features = linear.out_features

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return fp8_mm(x, self.w8, self.w_scale, self.bias)


class Fp8LayerNorm(nn.Module):
    """FusedLayerNorm replacement that emits the e4m3 pack as a side output
    (kernel-fused; the pack rides on the bf16 result as `_fp8`)."""

    def __init__(self, ln, ctx: Fp8Context, site: int):
        super().__init__()
        self.weight = ln.weight
        self.bias = ln.bias
        self.eps = ln.eps
        self.ctx = ctx
        self.site = site

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        if x.is_cuda and not torch.is_grad_enabled():
            y, y8 = torch.ops.vilbert_amd.residual_layer_norm_fp8(
                x.contiguous(),
                residual.contiguous() if residual is not None else None,
                self.weight, self.bias, self.eps,
                self.ctx.scales, self.ctx.amaxes, self.site,
            )
            y._fp8 = (y8, self.ctx.scales[self.site])
            return y
        from ..ops import functional as F_ops

        return F_ops.layer_norm(x, self.weight, self.bias, self.eps, residual)


def attach_quant_pack(x: torch.Tensor, ctx: Fp8Context, site: int) -> torch.Tensor:
    """Standalone quantize (single fused amax+cast pass) for producers that
    do not have an FP8OUT kernel variant (attention context, embeddings)."""
    x8 = torch.ops.vilbert_amd.quantize_fp8(
        x.contiguous(), ctx.scales, ctx.amaxes, site
    )
    x._fp8 = (x8, ctx.scales[site])
    return x


def _refuse_converted(bert) -> None:
    """A conversion is of the whole encoder or of nothing."""
    for m in bert.modules():
        if isinstance(m, (Fp8Linear, BlockFp8Linear)):
            raise RuntimeError("the encoder's products are in 8 bits already")


def convert_encoder_to_fp8(model) -> int:
    """Swap the two-stream encoder onto the fp8 path. Returns #GEMM sites.
    One that is in 8 bits already, in either way, is refused."""
    from .vilbert import (
        CrossAttention,
        FeedForward,
        FusedLayerNorm,
        ImageEmbeddings,
        MultiHeadSelfAttention,
    )

    bert = model.bert if hasattr(model, "bert") else model
    _refuse_converted(bert)
    device = next(bert.parameters()).device

    # pass 1: count quantization sites
    alloc = _SiteAllocator()
    plan = []
    for m in bert.modules():
        if isinstance(m, MultiHeadSelfAttention):
            plan.append(("mha", m, alloc.take()))   # ctx quant site
        elif isinstance(m, CrossAttention):
            plan.append(("xattn", m, alloc.take()))
        elif isinstance(m, FeedForward):
            plan.append(("ffn", m, alloc.take()))   # gelu site
    ln_plan = []
    for m in bert.modules():
        if isinstance(m, (MultiHeadSelfAttention, CrossAttention, FeedForward, ImageEmbeddings)):
            if isinstance(m.layer_norm, FusedLayerNorm):
                ln_plan.append((m, alloc.take()))

    ctx = Fp8Context(alloc.n, device)
    n_gemms = 0
    for kind, m, site in plan:
        if kind == "mha":
            w = torch.cat([m.query.weight, m.key.weight, m.value.weight], dim=0)
            m._wqkv8, m._wqkv_scale = quantize_weight(w.detach())
            m._bqkv = torch.cat([m.query.bias, m.key.bias, m.value.bias]).detach()
            m._wqkv = None
            m.out = Fp8Linear(m.out)
            m._fp8_ctx_site = site
            m._fp8_ctx_obj = ctx
            n_gemms += 4
        elif kind == "xattn":
            w = torch.cat([m.key.weight, m.value.weight], dim=0)
            m._wkv8, m._wkv_scale = quantize_weight(w.detach())
            m._bkv = torch.cat([m.key.bias, m.value.bias]).detach()
            m._wkv = None
            m.query = Fp8Linear(m.query)
            m.out = Fp8Linear(m.out)
            m._fp8_ctx_site = site
            m._fp8_ctx_obj = ctx
            n_gemms += 4
        elif kind == "ffn":
            m.intermediate = Fp8Linear(m.intermediate)
            m.output = Fp8Linear(m.output)
            m._fp8_gelu_site = site
            m._fp8_ctx_obj = ctx
            n_gemms += 2
    for m, site in ln_plan:
        m.layer_norm = Fp8LayerNorm(m.layer_norm, ctx, site)
    model._fp8_ctx = ctx
    return n_gemms


# --------------------------------------------------------------------------
# one scale per block of 128
# --------------------------------------------------------------------------


def _block_pack(x):
    """x in 8 bits: as it is where it is (values, scales) already, what its
    producer emitted where x has not been written since, or quantised here."""
    if isinstance(x, tuple):
        return x
    pack = getattr(x, "_fp8b", None)
    if pack is not None and pack[2] == x._version:
        return pack[:2]
    from ..ops import functional as F_ops

    return F_ops.quantize_fp8_block(x)


def fp8_block_mm(
    x,
    w8: torch.Tensor,
    w_scales: torch.Tensor,
    bias: Optional[torch.Tensor],
) -> torch.Tensor:
    """y = x @ w.T + bias, out bf16, with scales per block of 128."""
    from ..ops import functional as F_ops

    return F_ops.fp8_block_linear(*_block_pack(x), w8, w_scales, bias)


class BlockFp8Linear(nn.Module):
    """Inference-only drop-in for nn.Linear, weights in blocks of 128 x 128."""

    def __init__(self, linear: nn.Linear):
        super().__init__()
        from ..ops import functional as F_ops

        w8, scales = F_ops.quantize_fp8_block_weight(linear.weight.detach())
        self.register_buffer("w8", w8)
        self.register_buffer("w_scales", scales)
        self.register_buffer(
            "bias", None if linear.bias is None else linear.bias.detach())
        self.in_features = linear.in_features
        self.out_features = linear.out_features
        # of no size: what type the module's results have, also after a cast
        self.register_buffer("_like", linear.weight.detach().new_empty(0), persistent=False)

    @property
    def dtype(self) -> torch.dtype:
        return self._like.dtype

    def _apply(self, fn, recurse=True):
        """Moves the 8-bit weight and its scales with the rest, and casts neither:
        what moves them sees whole numbers."""
        held = {}
        for name, as_int in (("w8", torch.uint8), ("w_scales", torch.int16)):
            t = self._buffers[name]
            moved = fn(t.view(as_int))
            if moved.dtype != as_int:  # Module.type() casts whatever there is
                moved = t.view(as_int).to(moved.device)
            held[name] = moved.view(t.dtype)
        for name in held:
            del self._buffers[name]
        try:
            return super()._apply(fn, recurse)
        finally:
            self._buffers.update(held)

    def forward(self, x) -> torch.Tensor:
        return fp8_block_mm(x, self.w8, self.w_scales, self.bias).to(self.dtype)

    def gelu8(self, x):
        """gelu(forward(x)) in 8 bits alone, (values, scales): another
        BlockFp8Linear's input."""
        from ..ops import functional as F_ops

        return F_ops.fp8_block_linear_fp8(
            *_block_pack(x), self.w8, self.w_scales, self.bias, gelu=True)


class BlockFp8LayerNorm(nn.Module):
    """FusedLayerNorm replacement that emits the 8-bit form as well (`_fp8b`: values,
    scales and the version of the result that they belong to)."""

    def __init__(self, ln):
        super().__init__()
        self.weight = ln.weight
        self.bias = ln.bias
        self.eps = ln.eps

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        from ..ops import functional as F_ops

        if torch.is_grad_enabled():
            return F_ops.layer_norm(x, self.weight, self.bias, self.eps, residual)
        y, y8, scales = F_ops.layer_norm_fp8_block(
            x, self.weight, self.bias, self.eps, residual=residual)
        if not y.is_inference():  # those do not count their writes
            y._fp8b = (y8, scales, y._version)
        return y


def convert_encoder_to_fp8_block(model) -> int:
    """Swap the two-stream encoder's products onto e4m3 with a scale per block
    of 128. For inference (no gradient). Returns #GEMM sites. One that is in 8 bits
    already, in either way, is refused."""
    from ..ops import functional as F_ops
    from .vilbert import (
        CrossAttention,
        FeedForward,
        FusedLayerNorm,
        ImageEmbeddings,
        MultiHeadSelfAttention,
    )

    bert = model.bert if hasattr(model, "bert") else model
    _refuse_converted(bert)
    n_gemms = 0
    with torch.no_grad():
        for m in list(bert.modules()):
            if isinstance(m, MultiHeadSelfAttention):
                w = torch.cat([m.query.weight, m.key.weight, m.value.weight], dim=0)
                m._wqkv8, m._wqkv_scale = F_ops.quantize_fp8_block_weight(w)
                m._bqkv = torch.cat([m.query.bias, m.key.bias, m.value.bias]).detach()
                m._wqkv = None
                m.out = BlockFp8Linear(m.out)
                n_gemms += 4
            elif isinstance(m, CrossAttention):
                w = torch.cat([m.key.weight, m.value.weight], dim=0)
                m._wkv8, m._wkv_scale = F_ops.quantize_fp8_block_weight(w)
                m._bkv = torch.cat([m.key.bias, m.value.bias]).detach()
                m._wkv = None
                m.query = BlockFp8Linear(m.query)
                m.out = BlockFp8Linear(m.out)
                n_gemms += 4
            elif isinstance(m, FeedForward):
                m.intermediate = BlockFp8Linear(m.intermediate)
                m.output = BlockFp8Linear(m.output)
                n_gemms += 2
            if isinstance(
                m, (MultiHeadSelfAttention, CrossAttention, FeedForward, ImageEmbeddings)
            ) and isinstance(m.layer_norm, FusedLayerNorm):
                m.layer_norm = BlockFp8LayerNorm(m.layer_norm)
    return n_gemms
