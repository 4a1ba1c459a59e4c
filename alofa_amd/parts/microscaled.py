"""Layers whose matrices are held in 4 bits: a "prenorm" layer of attention and a gated feed-forward (parts/block.py), its seven matrices as microscaled
rows of e2m1 (blocks of 32 along the inputs, a power of two each), made of the stored ones when the weights are loaded. What the products read is
microscaled rows of e4m3: the two norms leave them, the activated gate does, and attention's output is brought into them. Everything else is as
it was: the stream and all sums in float32, queries, keys and values in bfloat16, embedding, norms' weights, biases and head as stored.

a = stream; n0 = q8(norm0(a)); qkv = n0 Wqkv^T + b; o = q8(attention(qkv)); a += o Wo^T; n1 = q8(norm1(a)); a += q8(act(n1 Wg^T) * (n1 Wu^T)) Wd^T

The output product leaves the shares of its sum and the norm behind it adds them to the stream on its way. So does the product down, where its sum is
shared out, with the first norm of the next such layer (a launch less: 4.6 us of 106 a layer, 64 rows at 3,584 x 18,944).

Unlike the stored layer this one turns queries and keys and writes the cache by a launch of their own, does not say that it may be run by making another layer's launches again (its matrices
are no tensors), and has no decode step in one launch: at 0.5B sizes, where launches are what a step costs, it is the slower one."""
from __future__ import annotations

import dataclasses

import torch

from .. import ops
from ..config.base import ModelSpec, PartSpec
from ..errors import AlofaError
from .attention import paged_attend
from .base import register_part
from .block import PreNormBlock

KIND = "microscaled_prenorm"


def microscaled(spec: ModelSpec) -> ModelSpec:
    """The same model with the matrices of its layers held in 4 bits; refused for layers of other kinds."""
    layers = []
    for layer in spec.layers:
        kinds = {} if layer.block.kind != "prenorm" else {"mixer": layer.part("mixer").kind, "feed_forward": layer.part("feed_forward").kind, "norms": {n.kind for n in layer.part("norms")}}
        if kinds != {"mixer": "gqa_attention", "feed_forward": "swiglu", "norms": {"rmsnorm"}}:
            raise AlofaError("unsupported", "matrices in 4 bits are built for layers of attention and a gated feed-forward with a norm in front of each", f"prefix={layer.prefix} block={layer.block.kind}")
        layers.append(dataclasses.replace(layer, block=PartSpec(KIND, layer.block.params)))
    return dataclasses.replace(spec, layers=type(spec.layers)(layers))


class _MicroscaledNorm:
    """The norm that a layer starts with, as what it asks the layer before for: rows that no other block leaves."""

    def __init__(self, norm):
        self.norm = norm

    def as_rmsnorm(self):
        return None


class MicroscaledPreNorm(PreNormBlock):
    def wants_normed(self, rows):
        return _MicroscaledNorm(self.norms[0])

    def can_leave(self, norm):
        return isinstance(norm, _MicroscaledNorm)

    def normed_rows(self, ctx, hidden):
        return self._rows(ctx, "mx_normed", *hidden.shape)

    def __init__(self, layer, weights, rt):
        if rt.exact:
            raise AlofaError("unsupported", "matrices in 4 bits go with bfloat16; float32 is the exact path", f"prefix={layer.prefix}")
        super().__init__(layer, weights, rt)
        m, f = self.mixer, self.feed_forward
        self.w_qkv, self.w_o, self.w_gate, self.w_up, self.w_down = map(self._quantised, (m.w_qkv, m.w_o, f.w_gate, f.w_up, f.w_down))
        m.w_qkv = m.w_o = f.w_gate = f.w_up = f.w_down = None      # (the parts' own forms of the products are not run)

    @staticmethod
    def _quantised(w: torch.Tensor) -> ops.MXRows:
        with torch.cuda.device(w.device):
            q = ops.MXRows(*w.shape, "e2m1", w.device)
            ops.mx_quantize(q, w)
        return q

    @staticmethod
    def _rows(ctx, name: str, rows: int, k: int) -> ops.MXRows:
        return ops.MXRows(rows, k, "e4m3", buffer=ctx.scratch(name, (ops.MXRows.bytes(rows, k, "e4m3"),), torch.uint8))

    def forward(self, ctx, entry, hidden, normed=None, then=None):
        (T, h), m, f = hidden.shape, self.mixer, self.feed_forward
        if normed is None:
            normed = self.normed_rows(ctx, hidden)
            ops.rmsnorm_mx(normed, hidden, *self.norms[0].as_rmsnorm())
        qkv = ctx.scratch("qkv", (T, m.qkv_width), self.rt.dtype)
        ops.gemm_mx(qkv, normed, self.w_qkv, m.b_qkv, scratch=ctx.scratch)
        attn = ctx.scratch("attn", (T, m.heads * m.d), self.rt.dtype)
        paged_attend(ctx, entry, qkv, attn, m.heads, m.kv_heads, m.d, m.window, m.scale, m.position, self.rt)
        rows = self._rows(ctx, "mx_attn", T, m.heads * m.d)
        ops.mx_quantize(rows, attn)
        if m.b_o is not None:
            mixed = ctx.scratch("attn_proj", (T, h), torch.float32)
            ops.gemm_mx(mixed, rows, self.w_o, m.b_o, scratch=ctx.scratch)
        else:
            mixed = ctx.scratch("mx_shares", (ops.mx_shares(T, h, rows.k), T, h), torch.float32)
            ops.gemm_mx_shares(mixed, rows, self.w_o)
        ops.rmsnorm_mx(normed, hidden, *self.norms[1].as_rmsnorm(), add=mixed, total=hidden)
        act = self._rows(ctx, "mx_act", T, f.intermediate)
        ops.gemm_swiglu_mx(act, normed, self.w_gate, self.w_up, f.activation)
        shares = 1 if then is None else ops.mx_shares(T, h, f.intermediate)
        if shares == 1:      # (whole sums are added where they are formed: a norm that adds them would read and write the stream once more)
            ops.gemm_mx(hidden, act, self.w_down, add_to_out=True, scratch=ctx.scratch)
            return False
        down = ctx.scratch("mx_down", (shares, T, h), torch.float32)
        ops.gemm_mx_shares(down, act, self.w_down)
        norm, rows = then
        ops.rmsnorm_mx(rows, hidden, *norm.norm.as_rmsnorm(), add=down, total=hidden)
        return True


register_part("block", KIND, MicroscaledPreNorm)
