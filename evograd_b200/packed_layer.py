"""Decoder layer over a packed batch, forward and backward: the dense layer of
``pairs/llama3_decoder_layer.py`` for documents of different lengths in one token
axis, with the norms on both sides of each block and a gate and scale on what a block
adds to the residual stream.

    (h, y) -> y Wqkv -> rotary by position -> packed causal attention -> Wo
           -> h1 = h + alpha gate_attn norm(.) w_post_attn,  y1 = norm(h1) w_pre_mlp
           -> SwiGLU MLP of y1
           -> h2 = h1 + alpha gate_mlp norm(.) w_post_mlp,   y2 = norm(h2) w_pre_next
           -> (h2, y2)

A layer takes the residual stream h ``[T, C]`` together with its normalised form y, which
the boundary before it has written in the same pass, and hands both on; ``w_pre_next``
is the next layer's (or the final) norm weight. q, k and v stay the thirds of one
projection ``[T, (Hq + 2 Hkv) D]``: the rotation runs in place on them, the attention
reads them through their strides, and the backward writes their gradients into the
thirds of one gradient, so the projection is one product each way and nothing is copied.
The projections are plain library products through ``torch``; everything else are this
package's kernels. The plan and the positions belong to the batch: one of each serves
all layers. ``clip_grad_norm`` of :mod:`evograd_b200.ops` takes the gradients as they
come.

Saved state: y, the projection (rotated), the attention's output and log-sum-exp, both
blocks' outputs, both residual streams, y1, the four float32 rstd vectors and the MLP's
gate / up activations; the SwiGLU product is formed again in the backward, from the same
numbers. (y1 could not be: the forward normalises h1 before it is rounded, so a y1 formed
from the saved h1 differs in the last bits from the one that the projections multiplied.)
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import ops


class PackedLayerWeights(NamedTuple):
    """Parameters of one layer; :func:`packed_layer_backward` returns their gradients in the
    same form. ``gate_attn`` / ``gate_mlp`` (``[C]``) may be None."""

    qkv: torch.Tensor          # [(Hq + 2 Hkv) D, C]
    out: torch.Tensor          # [C, Hq D]
    mlp_gate: torch.Tensor     # [F, C]
    mlp_up: torch.Tensor       # [F, C]
    mlp_down: torch.Tensor     # [C, F]
    post_attn: torch.Tensor    # [C]
    pre_mlp: torch.Tensor      # [C]
    post_mlp: torch.Tensor     # [C]
    pre_next: torch.Tensor     # [C]
    gate_attn: torch.Tensor | None = None
    gate_mlp: torch.Tensor | None = None


class PackedBatch(NamedTuple):
    """What all layers share about a batch: the attention's work plan, the position of every
    token inside its document, and the rotary frequencies with their factor."""

    plan: ops.PackedPlan
    positions: torch.Tensor    # [T] int32 / int64
    inv_freq: torch.Tensor     # [rotary_dim / 2]
    mscale: float = 1.0
    interleaved: bool = False


def _thirds(qkv, heads, kv_heads, head_dim):
    a, b = heads * head_dim, (heads + kv_heads) * head_dim
    return (qkv[:, :a].unflatten(1, (heads, head_dim)), qkv[:, a:b].unflatten(1, (kv_heads, head_dim)),
            qkv[:, b:].unflatten(1, (kv_heads, head_dim)))


def packed_layer_forward(h, y, w: PackedLayerWeights, batch: PackedBatch, *, heads: int, kv_heads: int,
                         alpha: float = 1.0, eps: float = 1e-6):
    """Returns ``(h2, y2, saved)`` for the residual stream ``h`` and its norm ``y``."""
    head_dim, rest = divmod(w.qkv.shape[0], heads + 2 * kv_heads)
    if rest or w.out.shape[1] != heads * head_dim:
        raise ValueError(f"projections {tuple(w.qkv.shape)} and {tuple(w.out.shape)} do not fit "
                         f"{heads} + 2 x {kv_heads} heads")
    qkv = torch.mm(y, w.qkv.t())
    q, k, v = _thirds(qkv, heads, kv_heads, head_dim)
    ops.rope_positions_fwd(q, k, batch.positions, batch.inv_freq, interleaved=batch.interleaved,
                           mscale=batch.mscale, outs=(q, k))
    o, lse = ops.packed_attention_fwd(q, k, v, batch.plan)
    attn = torch.mm(o.flatten(1), w.out.t())
    h1, y1, ra, rb = ops.post_pre_norm_fwd(attn, h, w.post_attn, w.pre_mlp, w.gate_attn, alpha=alpha, eps=eps)
    g, u = torch.mm(y1, w.mlp_gate.t()), torch.mm(y1, w.mlp_up.t())
    mlp = torch.mm(ops.swiglu_fwd(g, u), w.mlp_down.t())
    h2, y2, rc, rd = ops.post_pre_norm_fwd(mlp, h1, w.post_mlp, w.pre_next, w.gate_mlp, alpha=alpha, eps=eps)
    return h2, y2, (y, qkv, o, lse, attn, h1, y1, mlp, h2, ra, rb, rc, rd, g, u)


def packed_layer_backward(dh2, dy2, saved, w: PackedLayerWeights, batch: PackedBatch, *, heads: int,
                          kv_heads: int, alpha: float = 1.0, eps: float = 1e-6):
    """From the gradients of ``h2`` and ``y2``: ``(dh, dy, dw)`` with ``dw`` a
    :class:`PackedLayerWeights` of gradients. Arguments as in the forward (whose rstd vectors
    are saved: ``eps`` enters no sum here)."""
    y, qkv, o, lse, attn, h1, y1, mlp, h2, ra, rb, rc, rd, g, u = saved
    q, k, v = _thirds(qkv, heads, kv_heads, o.shape[2])

    d_mlp, dh1, d_post_mlp, d_pre_next, d_gate_mlp = ops.post_pre_norm_bwd(
        dy2, dh2, mlp, h2, w.post_mlp, w.pre_next, w.gate_mlp, rc, rd, alpha=alpha)
    act = ops.swiglu_fwd(g, u)
    d_down = torch.mm(d_mlp.t(), act)
    dg, du = ops.swiglu_bwd(torch.mm(d_mlp, w.mlp_down), g, u)
    d_mlp_gate, d_mlp_up = torch.mm(dg.t(), y1), torch.mm(du.t(), y1)
    dy1 = torch.addmm(torch.mm(dg, w.mlp_gate), du, w.mlp_up)

    d_attn, dh, d_post_attn, d_pre_mlp, d_gate_attn = ops.post_pre_norm_bwd(
        dy1, dh1, attn, h1, w.post_attn, w.pre_mlp, w.gate_attn, ra, rb, alpha=alpha)
    d_out = torch.mm(d_attn.t(), o.flatten(1))
    do = torch.mm(d_attn, w.out).view_as(o)
    dqkv = torch.empty_like(qkv)
    dq, dk, dv = _thirds(dqkv, heads, kv_heads, o.shape[2])
    ops.packed_attention_bwd(do, q, k, v, o, lse, batch.plan, outs=(dq, dk, dv))
    ops.rope_positions_bwd(dq, dk, batch.positions, batch.inv_freq, interleaved=batch.interleaved,
                           mscale=batch.mscale, outs=(dq, dk))
    d_qkv = torch.mm(dqkv.t(), y)
    dy = torch.mm(dqkv, w.qkv)
    return dh, dy, PackedLayerWeights(d_qkv, d_out, d_mlp_gate, d_mlp_up, d_down, d_post_attn, d_pre_mlp,
                                      d_post_mlp, d_pre_next, d_gate_attn, d_gate_mlp)
