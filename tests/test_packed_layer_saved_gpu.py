"""What a packed layer's backward reads: the activations that its forward used, and a captured
step's gradient norm."""

import pytest
import torch

from tests.test_packed_layer_gpu import weights

pytestmark = pytest.mark.gpu


def test_the_mlp_gradients_belong_to_the_forwards_y1(monkeypatch):
    """d_mlp_gate and d_mlp_up are products with the y1 that the forward multiplied: the same
    product of the same operands, so the same bits."""
    from evograd_b200 import ops
    from evograd_b200.packed_layer import (PackedBatch, PackedLayerWeights, packed_layer_backward,
                                           packed_layer_forward)

    g = torch.Generator(device="cuda").manual_seed(9)
    heads, kv, hd, C, F, T = 4, 2, 64, 128, 192, 200
    cu = torch.tensor([0, 60, 200], device="cuda", dtype=torch.int32)
    pos = torch.cat([torch.arange(60), torch.arange(140)]).cuda()
    batch = PackedBatch(ops.packed_plan(cu, T), pos, ops.rope_inv_freq(hd, device="cuda")[0])
    w = PackedLayerWeights(*weights(g, C, F, heads, kv, hd, torch.bfloat16))
    h, dh, dy = (torch.randn(T, C, device="cuda", generator=g).bfloat16() for _ in range(3))
    y, _ = ops.rmsnorm_fwd(h, w.pre_mlp)
    seen = {}
    fwd, bwd = ops.post_pre_norm_fwd, ops.swiglu_bwd

    def norms(*a, **kw):
        out = fwd(*a, **kw)
        seen.setdefault("y1", out[1].clone())
        return out

    def swiglu(*a, **kw):
        seen["dg"], seen["du"] = (t.clone() for t in bwd(*a, **kw))
        return seen["dg"], seen["du"]

    monkeypatch.setattr(ops, "post_pre_norm_fwd", norms)
    monkeypatch.setattr(ops, "swiglu_bwd", swiglu)
    _, _, saved = packed_layer_forward(h, y, w, batch, heads=heads, kv_heads=kv, alpha=0.7)
    _, _, dw = packed_layer_backward(dh, dy, saved, w, batch, heads=heads, kv_heads=kv, alpha=0.7)
    assert torch.equal(dw.mlp_gate, torch.mm(seen["dg"].t(), seen["y1"]))
    assert torch.equal(dw.mlp_up, torch.mm(seen["du"].t(), seen["y1"]))


def test_a_captured_norm_follows_its_gradients():
    """Plan, attention and gradient norm in one graph: after each replay the norm is that of
    the replayed gradients, bit for bit the eager call's on them."""
    from evograd_b200 import ops

    T, hq, hk, d = 300, 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    q, do = (torch.randn(T, hq, d, device="cuda", generator=g).bfloat16() for _ in range(2))
    k, v = (torch.randn(T, hk, d, device="cuda", generator=g).bfloat16() for _ in range(2))
    cu = torch.tensor([0, 100, 300], device="cuda", dtype=torch.int32)

    def step():
        plan = ops.packed_plan(cu, T)
        o, lse = ops.packed_attention_fwd(q, k, v, plan)
        grads = ops.packed_attention_bwd(do, q, k, v, o, lse, plan)
        return grads, ops.grad_norm(grads)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads, norm = step()
    seen = set()
    for offsets, size in (([0, 100, 300], 1.0), ([0, 1, 200], 4.0), ([0, 0, 0], 1.0), ([0, 300, 300], 0.01)):
        cu.copy_(torch.tensor(offsets, dtype=torch.int32))
        do.normal_(generator=g).mul_(size)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, ops.grad_norm(grads))
        seen.add(float(norm))
    assert len(seen) == 4 and 0.0 in seen
