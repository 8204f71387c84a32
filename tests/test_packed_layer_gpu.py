"""The packed operators together, as a training step uses them: two decoder layers over a
packed batch, forward, backward, clipping, against autograd of the whole in float64 with
every document computed on its own.

Tolerances (relative 2-norm): between the input and an output lie about thirty roundings
to T along the longest path (projections, rotated q and k, P, o, block outputs, streams,
activations, their gradients), each at most u = finfo(T).eps / 2 relative and mostly
independent; sqrt(30) u = 5.5 u, and cancellation in the norms' and the softmax's backward
is allowed a factor of two more: 12 u. float32 products of length n <= 96 add n 2^-24 each:
30 of them 2e-4 at most, in the 2-norm far less: 2e-5.
"""

import pytest
import torch

DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-6


def weights(g, C, F, heads, kv, hd, dtype):
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    return [x.to(dtype) for x in (
        r((heads + 2 * kv) * hd, C) * C ** -0.5, r(C, heads * hd) * (heads * hd) ** -0.5, r(F, C) * C ** -0.5,
        r(F, C) * C ** -0.5, r(C, F) * F ** -0.5, 1 + 0.1 * r(C), 1 + 0.1 * r(C), 1 + 0.1 * r(C), 1 + 0.1 * r(C),
        0.5 + 0.1 * r(C), 0.5 + 0.1 * r(C))]


def norm64(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def layer64(h, y, w, lens, pos, f, heads, kv, hd, alpha):
    qkv, wo, wg, wu, wd, pa, pm, pp, pn, ga, gm = w
    T = h.shape[0]
    x = y @ qkv.T
    q, k, v = (t.unflatten(1, (-1, hd)) for t in x.split([heads * hd, kv * hd, kv * hd], 1))
    ang = pos.double()[:, None, None] * f
    n = f.numel()

    def rot(t):
        a, b = t[..., :n], t[..., n: 2 * n]
        return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin(), t[..., 2 * n:]], -1)

    q, k = rot(q), rot(k).repeat_interleave(heads // kv, 1)
    v = v.repeat_interleave(heads // kv, 1)
    outs, a = [], 0
    for m in lens:
        s = torch.einsum("ihd,jhd->hij", q[a:a + m], k[a:a + m]) / hd ** 0.5
        s = s.masked_fill(torch.ones(m, m, device=h.device, dtype=torch.bool).triu(1), float("-inf"))
        outs.append(torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v[a:a + m]))
        a += m
    outs.append(torch.zeros(T - a, heads, hd, device=h.device, dtype=torch.float64))
    h1 = h + alpha * ga * norm64(torch.cat(outs).flatten(1) @ wo.T, pa)
    y1 = norm64(h1, pm)
    h2 = h1 + alpha * gm * norm64((torch.nn.functional.silu(y1 @ wg.T) * (y1 @ wu.T)) @ wd.T, pp)
    return h2, norm64(h2, pn)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,heads,kv,hd,C,F", [("bf16", 4, 2, 64, 128, 192), ("bf16", 6, 6, 64, 96, 64),
                                                   ("fp32", 4, 1, 16, 96, 80)])
def test_two_layers_and_clipping(dtype, heads, kv, hd, C, F):
    from evograd_b200 import ops
    from evograd_b200.packed_layer import (PackedBatch, PackedLayerWeights, packed_layer_backward,
                                           packed_layer_forward)

    g = torch.Generator(device="cuda").manual_seed(3)
    dt, lens, alpha = DT[dtype], [70, 1, 133, 0, 40], 0.7
    T = sum(lens)
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), device="cuda", dtype=torch.int32)
    pos = torch.cat([torch.arange(n) for n in lens]).cuda()
    inv_freq, mscale = ops.rope_inv_freq(hd // 2, 10000.0, device="cuda")
    batch = PackedBatch(ops.packed_plan(cu, T), pos, inv_freq, mscale)
    batch.plan.check()
    ws = [weights(g, C, F, heads, kv, hd, dt) for _ in range(2)]
    w0 = (1 + 0.1 * torch.randn(C, device="cuda", generator=g)).to(dt)
    h0, dh, dy = (torch.randn(T, C, device="cuda", generator=g).to(dt) for _ in range(3))

    h, saved = h0, []
    y, rstd = ops.rmsnorm_fwd(h0, w0, EPS)
    for w in ws:
        h, y, s = packed_layer_forward(h, y, PackedLayerWeights(*w), batch, heads=heads, kv_heads=kv, alpha=alpha, eps=EPS)
        saved.append(s)
    gh, gy, grads = dh, dy, []
    for w, s in zip(reversed(ws), reversed(saved)):
        gh, gy, gw = packed_layer_backward(gh, gy, s, PackedLayerWeights(*w), batch, heads=heads, kv_heads=kv,
                                           alpha=alpha, eps=EPS)
        grads.insert(0, list(gw))
    dx, dw0 = ops.rmsnorm_bwd(gy, h0, w0, rstd)
    dx = dx + gh
    ops.device_status()

    ws64 = [[x.double().requires_grad_() for x in w] for w in ws]
    x64, w064 = h0.double().requires_grad_(), w0.double().requires_grad_()
    hh, yy = x64, norm64(x64, w064)
    for w in ws64:
        hh, yy = layer64(hh, yy, w, lens, pos, inv_freq, heads, kv, hd, alpha)
    leaves = [x64, w064] + [x for w in ws64 for x in w]
    want = torch.autograd.grad([hh, yy], leaves, [dh.double(), dy.double()])
    u = torch.finfo(dt).eps / 2
    bound = 2e-5 if dtype == "fp32" else 12 * u
    got = [dx, dw0] + [x for w in grads for x in w]
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    assert rel(h, hh.detach()) <= bound and rel(y, yy.detach()) <= bound
    for i, (a, b) in enumerate(zip(got, want)):
        assert rel(a, b) <= bound, (i, rel(a, b))

    before = [x.double().clone() for x in got]
    norm = float(ops.clip_grad_norm(got, 0.5))
    true = float(torch.stack([x.square().sum() for x in before]).sum().sqrt())
    assert abs(norm - true) <= 2e-6 * true
    for a, b in zip(got, before):
        assert bool(((a.double() - b * (0.5 / true)).abs() <= (u + 3e-6) * (b * (0.5 / true)).abs() + 1e-38).all())


@pytest.mark.gpu
def test_a_step_captured_and_replayed_with_other_lengths():
    """Plan, rotation, attention, norms and clipping in one captured graph; the offsets and
    inputs change under it and every replay equals the eager call bit by bit (dk, dv, o) or
    up to the order of float32 additions (dq)."""
    from evograd_b200 import ops

    T, hq, hk, d = 384, 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()  # noqa: E731
    q, k, v, do = r(T, hq, d), r(T, hk, d), r(T, hk, d), r(T, hq, d)
    cu = torch.tensor([0, 100, 384], device="cuda", dtype=torch.int32)
    f = ops.rope_inv_freq(d, device="cuda")[0]
    pos = torch.arange(T, device="cuda")

    def step():
        plan = ops.packed_plan(cu, T)
        qr, kr = ops.rope_positions_fwd(q, k, pos, f)
        o, lse = ops.packed_attention_fwd(qr, kr, v, plan)
        dq, dk, dv = ops.packed_attention_bwd(do, qr, kr, v, o, lse, plan)
        norm = ops.grad_norm([dk, dv])
        return o, lse, dk, dv, dq, norm

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for offsets in ([0, 100, 384], [0, 1, 1 + 128], [0, 0, 300], [0, 384, 384]):
        cu.copy_(torch.tensor(offsets, dtype=torch.int32))
        q.copy_(r(T, hq, d))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        for a, b in zip(out[:4], eager[:4]):
            assert torch.equal(a, b)
        # float32 sums of at most three key tiles in another order, rounded to bfloat16
        assert float((out[4].double() - eager[4].double()).norm()) <= 1e-3 * float(eager[4].double().norm())
