"""Attention and gated feed-forward whose weights are kept in 8 or 4 bits, and the block around them.

``weight_format`` "q8": weights in e4m3 with a scale an output channel, and every product takes its rows in e4m3 with a scale a row. The
norms write such rows themselves (``ops.add_rmsnorm_q8``), so does the gated activation (``ops.swiglu_q8``); the heads' results take a launch of
their own (``ops.quantize_q8``). "w4": weights in 4 bits with a scale and a zero point a group of 128 input channels, rows in bfloat16. In both the
residual stream is fp32 and queries, keys, values and what the products return are bfloat16, as without a format; embedding, norms and LM head
keep their own.

The matrices come from the checkpoint in bfloat16 and are quantised when they are loaded (``quantize``): 8 bits by the largest entry of a row; 4
bits between the smallest and the largest entry of a group, zero always among them.

The kinds are "quantized_attention" and "quantized_gated_mlp"; ``quantized_layer`` turns a layer's spec into one of them. Attention in its general form
and other mixers and feed-forwards have no such form.
"""
from __future__ import annotations

from dataclasses import dataclass, replace
from typing import Optional

import torch

from ..csrc import ops
from .attention import Attention
from .base import register_feed_forward, register_mixer
from .block import register_arrangement
from .mlp import GatedMLP
from .norm import RMSNorm

FORMATS = ("q8", "w4")
W4_GROUP = 128


@dataclass
class Q8Weight:
    """[N, K] as ``codes`` (e4m3) times ``scale`` (fp32 [N])."""
    codes: torch.Tensor
    scale: torch.Tensor

    @property
    def stored(self) -> torch.Tensor:
        return self.codes

    def dense(self) -> torch.Tensor:
        """The values it stands for, fp32 (tests and tools)."""
        return self.codes.float() * self.scale.unsqueeze(1)


@dataclass
class W4Weight:
    """[N, K] as int32 ``words`` of eight entries (``ops.pack_w4``), ``scales`` bf16 and ``zeros`` uint8 [N, ceil(K / group)]."""
    words: torch.Tensor
    scales: torch.Tensor
    zeros: Optional[torch.Tensor]
    group: int

    @property
    def stored(self) -> torch.Tensor:
        return self.words

    def dense(self) -> torch.Tensor:
        q = ops.unpack_w4(self.words)
        K = q.shape[1]
        spread = lambda t: t.float().repeat_interleave(self.group, 1)[:, :K]
        return (q.float() - (8.0 if self.zeros is None else spread(self.zeros))) * spread(self.scales)


def quantize_w4(w: torch.Tensor, group: int = W4_GROUP) -> W4Weight:
    """A matrix [N, K] (K a multiple of 8) in 4 bits: in each group of ``group`` columns scale = (max - min) / 15 over its entries and zero, rounded
    to bfloat16, and the zero point is the entry that stands for zero. On the matrix's device, in plain tensor operations."""
    N, K = w.shape
    G = -(-K // group)
    x = torch.nn.functional.pad(w.float(), (0, G * group - K)).view(N, G, group)
    lo, hi = x.amin(2).clamp_max(0.0), x.amax(2).clamp_min(0.0)
    scales = ((hi - lo) / 15.0).clamp_min(2.0 ** -100).to(torch.bfloat16)      # a group of zeros: any scale will do
    zeros = (-lo / scales.float()).round().clamp(0, 15)
    q = (x / scales.float().unsqueeze(2) + zeros.unsqueeze(2)).round().clamp(0, 15)
    return W4Weight(ops.pack_w4(q.view(N, -1)[:, :K]), scales, zeros.to(torch.uint8), group)


def quantize(w: torch.Tensor, weight_format: str):
    """A matrix of the checkpoint in the format's own form."""
    if weight_format == "w4":
        if w.shape[1] % 8:
            raise ValueError(f"weight format 'w4' takes matrices whose input size is a multiple of 8, found {tuple(w.shape)}")
        return quantize_w4(w)
    codes = torch.empty(w.shape, dtype=ops.E4M3, device=w.device)
    scale = torch.empty(w.shape[0], dtype=torch.float32, device=w.device)
    ops.quantize_q8(w, codes, scale)
    return Q8Weight(codes, scale)


@dataclass
class Q8Rows:
    """Rows [T, n] as ``codes`` (e4m3) times ``scale`` (fp32 [T]): what the norms and the gated activation hand to a product."""
    codes: torch.Tensor
    scale: torch.Tensor

    @classmethod
    def of(cls, ctx, key: str, T: int, n: int) -> "Q8Rows":
        return cls(ctx.buf(key, (T, n), ops.E4M3), ctx.buf(key + "_scale", (T,), torch.float32))

    @property
    def shape(self):
        return self.codes.shape


def product(x, w, out: torch.Tensor, ctx, key: str) -> torch.Tensor:
    """``out = x @ w^T`` for a quantised weight. Rows in bfloat16 become ``Q8Rows`` (in scratch under ``key``) where the weight is in 8 bits."""
    if isinstance(w, W4Weight):
        ops.gemm_w4(x, w.words, w.scales, w.zeros, w.group, out, ctx.status)
        return out
    if not isinstance(x, Q8Rows):
        rows = Q8Rows.of(ctx, key, *x.shape)
        ops.quantize_q8(x, rows.codes, rows.scale)
        x = rows
    ops.gemm_q8(x.codes, x.scale, w.codes, w.scale, out, ctx.status)
    return out


def _format_of(params, dtype) -> str:
    fmt = params.get("weight_format")
    if fmt not in FORMATS:
        raise ValueError(f"weight_format must be one of {list(FORMATS)}, found {fmt!r}")
    if dtype != torch.bfloat16:
        raise ValueError(f"weight format {fmt!r} goes with bfloat16 activations, found {dtype}")
    return fmt


# Rows up to which a product reads its weights once, as a stream: what the norm before it may fetch into L2 ahead.
STREAM_ROWS = 8


class QuantizedAttention(Attention):
    """``Attention`` (its plain form) with the stacked q/k/v projection and the output projection in ``weight_format``."""
    adds_into_residual = False

    def __init__(self, params, dtype, device, position=None):
        super().__init__(params, dtype, device, position)
        self.weight_format = _format_of(params, dtype)
        if self.general:
            raise ValueError("quantized_attention: the general form of attention has no weight formats")
        if position is None or position.rotary() is None:
            raise ValueError("quantized_attention: goes with a rotary position encoding")

    def load_weights(self, tensors):
        super().load_weights(tensors)
        self.qkv, self.o = quantize(self.qkv, self.weight_format), quantize(self.o, self.weight_format)

    def streams_first(self, rows):
        return self.qkv.stored if rows <= STREAM_ROWS else None

    def kernel_files(self, page_size):
        names = [n for n in super().kernel_files(page_size) if not n.startswith("gemm_")]
        return tuple(names + (["quant_rows", "gemm_q8"] if self.weight_format == "q8" else ["gemm_w4"]) + ["gemm_quant"])

    def forward(self, x, ctx, cache):
        T = x.shape[0]
        H, KV, hs = self.H, self.KV, self.hs
        qkv = product(x, self.qkv, ctx.buf("attn_qkv", (T, (H + 2 * KV) * hs), self.dtype), ctx, "block_x_q8")
        inv_freq, rot_dim = self.position.rotary()
        ops.rope_kv_write(qkv, ctx.positions, ctx.row_seq, inv_freq, rot_dim, cache.block_table, cache.k if cache.writes else None,
                          cache.v if cache.writes else None, cache.page_size, ctx.seq_slots, H, KV, hs, status=ctx.status)
        attn = ctx.buf("attn_out", (T, H * hs), self.dtype)
        self.attend(qkv[:, :H * hs], cache, ctx, attn)
        return product(attn, self.o, ctx.buf("delta", (T, self.hidden), self.dtype), ctx, "attn_out_q8")


register_mixer("quantized_attention", QuantizedAttention)


class QuantizedGatedMLP(GatedMLP):
    """``GatedMLP`` with its matrices in ``weight_format``."""
    adds_into_residual = False

    def __init__(self, params, dtype, device):
        super().__init__(params, dtype, device)
        self.weight_format = _format_of(params, dtype)

    def load_weights(self, tensors):
        super().load_weights(tensors)
        self.gate_up, self.down = quantize(self.gate_up, self.weight_format), quantize(self.down, self.weight_format)

    def streams_first(self, rows):
        return self.gate_up.stored if rows <= STREAM_ROWS else None

    def kernel_files(self, page_size):
        return ("quant_rows", "gemm_q8", "gemm_quant") if self.weight_format == "q8" else ("swiglu", "gemm_w4", "gemm_quant")

    def streamed(self, x):
        return None

    def forward(self, x, ctx):
        T = x.shape[0]
        gu = product(x, self.gate_up, ctx.buf("ffn_gate_up", (T, 2 * self.inter), self.dtype), ctx, "block_x_q8")
        if self.weight_format == "q8":
            act = Q8Rows.of(ctx, "ffn_act_q8", T, self.inter)
            ops.swiglu_q8(gu, act.codes, act.scale, self.group)
        else:
            act = ctx.buf("ffn_act", (T, self.inter), self.dtype)
            ops.swiglu(gu, act, self.group)
        return product(act, self.down, ctx.buf("delta", (T, self.hidden), self.dtype), ctx, "ffn_act_q8")


register_feed_forward("quantized_gated_mlp", QuantizedGatedMLP)


def norm_q8(norm: RMSNorm, resid, delta, out: Q8Rows, ahead=None) -> None:
    """``resid += delta`` and the norm of it as 8-bit rows; ``delta``: the result of the sublayer before, or None. (Blocks of "pre_norm" hand on nothing
    else, and a format's layers have no other arrangement.)"""
    ops.add_rmsnorm_q8(resid, delta, norm.weight, norm.eps, out.codes, out.scale, ahead=ahead)


def pre_norm_q8(block, resid, delta, ctx, cache):
    """"pre_norm" whose norms write 8-bit rows."""
    x = Q8Rows.of(ctx, "block_x_q8", *resid.shape)
    T = resid.shape[0]
    norm_q8(block.mixer_norm, resid, delta, x, block.mixer.streams_first(T))
    a = block.mixer.forward(x, ctx, cache)
    norm_q8(block.feed_forward_norm, resid, a, x, block.feed_forward.streams_first(T))
    return block.feed_forward.forward(x, ctx)


register_arrangement("pre_norm_q8", pre_norm_q8, capturable=True)


def quantized_layer(layer, weight_format: str):
    """The layer's spec with its parts in ``weight_format``; an error names what has no such form."""
    if weight_format not in FORMATS:
        raise ValueError(f"weight_format must be one of {list(FORMATS)}, found {weight_format!r}")
    if layer.mixer.kind != "attention":
        raise ValueError(f"weight format {weight_format!r}: mixer kind {layer.mixer.kind!r} has no form for it (only 'attention')")
    if layer.feed_forward is None or layer.feed_forward.kind != "gated_mlp":
        raise ValueError(f"weight format {weight_format!r}: feed-forward kind "
                         f"{None if layer.feed_forward is None else layer.feed_forward.kind!r} has no form for it (only 'gated_mlp')")
    norms = tuple(None if n is None else n.kind for n in (layer.mixer_norm, layer.feed_forward_norm))      # some arrangements have one norm for both
    if layer.arrangement != "pre_norm" or norms != ("rmsnorm", "rmsnorm") or layer.token_side_prefix is not None:
        raise ValueError(f"weight format {weight_format!r}: goes with the arrangement 'pre_norm' and RMS norms (found {layer.arrangement!r}, "
                         f"{norms[0]!r}, {norms[1]!r})")
    with_format = lambda spec, kind: replace(spec, kind=kind, params={**spec.params, "weight_format": weight_format})
    return replace(layer, mixer=with_format(layer.mixer, "quantized_attention"), feed_forward=with_format(layer.feed_forward, "quantized_gated_mlp"),
                   arrangement="pre_norm_q8" if weight_format == "q8" else "pre_norm")
