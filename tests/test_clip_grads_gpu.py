"""Global gradient norm and clipping against float64. The norm's float32 part is a
thread's at most 64 squares per chunk (64 2^-24 relative at worst, half of that in the
norm: 2e-6), the scaling one float32 product and one rounding to the tensor's type."""

import math

import pytest
import torch

TYPES = [torch.bfloat16, torch.float32, torch.float16]


def make(sizes, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(n, device="cuda", generator=g) * std).to(TYPES[i % 3]) for i, n in enumerate(sizes)]


def norm64(grads):
    return math.sqrt(math.fsum(float(g.double().square().sum()) for g in grads))


SIZES = [[1], [0, 5, 0], [7, 16384, 16385, 100003], [3] * 700 + [40000], [1 << 20, 1, 12345], [300000] * 49]


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("max_norm", [0.0, 0.5, 1e9])
def test_against_float64(sizes, max_norm):
    from evograd_b200 import ops

    grads = make(sizes)
    want = norm64(grads)
    before = [g.clone() for g in grads]
    assert abs(float(ops.grad_norm(grads)) - want) <= 2e-6 * want
    outs = [torch.full_like(g, 7.0) for g in grads]
    norm = ops.clip_grad_norm(grads, max_norm, outs=outs)
    assert norm.dtype == torch.float32 and norm.shape == () and abs(float(norm) - want) <= 2e-6 * want
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    coef = min(1.0, max_norm / (want + 1e-6))
    for o, g in zip(outs, grads):
        u = torch.finfo(g.dtype).eps / 2
        exact = g.double() * coef
        tiny = torch.finfo(g.dtype).smallest_normal * u * 2
        assert bool(((o.double() - exact).abs() <= (u + 3e-6) * exact.abs() + tiny).all())
    norm2 = ops.clip_grad_norm(grads, max_norm)  # in place
    assert torch.equal(norm, norm2) and all(torch.equal(a, b) for a, b in zip(grads, outs))


@pytest.mark.gpu
def test_alignment_order_and_repeats():
    from evograd_b200 import ops

    base = torch.randn(5001, device="cuda").bfloat16()
    odd, turned = base[1:], torch.randn(60, 70, device="cuda").t()
    assert not turned.is_contiguous()
    grads = [odd, turned]
    want, keep = norm64(grads), [g.double().clone() for g in grads]
    a = ops.grad_norm(grads)
    assert torch.equal(a, ops.grad_norm(grads)) and abs(float(a) - want) <= 2e-6 * want
    first = base[0].clone()
    ops.clip_grad_norm(grads, want / 2)
    assert torch.equal(base[0], first)
    for g, k in zip(grads, keep):
        u = torch.finfo(g.dtype).eps / 2
        assert bool(((g.double() - k * 0.5).abs() <= (u + 1e-5) * k.abs()).all())


@pytest.mark.gpu
def test_squares_beyond_float32():
    """Elements whose squares overflow float32 leave the norm finite and the scaling exact to
    the float32 rounding of the factor and one rounding of the result."""
    from evograd_b200 import ops

    g = [1e25 * torch.randn(40001, device="cuda"), (3e30 * torch.randn(5000, device="cuda")).bfloat16()[1:],
         torch.randn(70, device="cuda")]
    want, keep = norm64(g), [t.double().clone() for t in g]
    norm = ops.clip_grad_norm(g, 2.0)
    assert abs(float(norm) - want) <= 1e-6 * want
    for t, k in zip(g[:2], keep):
        u = torch.finfo(t.dtype).eps / 2
        assert bool(((t.double() - k * (2.0 / want)).abs() <= (u + 1e-6) * k.abs() * (2.0 / want) + 1e-44).all())


@pytest.mark.gpu
def test_norms_that_are_not_finite():
    from evograd_b200 import ops

    g = torch.ones(100, device="cuda")
    g[3] = float("inf")
    assert math.isinf(float(ops.clip_grad_norm([g], 1.0)))
    assert not g[:3].any() and torch.isnan(g[3])  # as max_norm / inf = 0 says
    g = torch.ones(100, device="cuda")
    g[5] = float("nan")
    assert math.isnan(float(ops.clip_grad_norm([g], 1.0))) and torch.isnan(g).all()


@pytest.mark.gpu
def test_captured_and_replayed():
    from evograd_b200 import ops

    grads = make([5000, 33, 70000])
    source = [g.clone() for g in grads]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.clip_grad_norm(grads, 1.0)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ops.clip_grad_norm(grads, 1.0)
    for scale in (1.0, 3.0):
        for g, s in zip(grads, source):
            g.copy_(s * scale)
        want = norm64(grads)
        graph.replay()
        torch.cuda.synchronize()
        assert abs(float(norm) - want) <= 2e-6 * want
        # bf16 elements round by 2^-8 of themselves at most, their norm by less
        assert abs(norm64(grads) - 1.0) <= 2.0 ** -8


@pytest.mark.gpu
def test_refusals():
    from evograd_b200 import ops

    g = torch.zeros(8, device="cuda")
    for bad in (lambda: ops.clip_grad_norm([], 1.0), lambda: ops.grad_norm([]),
                lambda: ops.clip_grad_norm([g], -1.0), lambda: ops.clip_grad_norm([g], float("nan")),
                lambda: ops.clip_grad_norm([g, g], 1.0),
                lambda: ops.clip_grad_norm([g[::2]], 1.0),
                lambda: ops.clip_grad_norm([g[:1].expand(8)], 1.0),
                lambda: ops.clip_grad_norm([g], 1.0, outs=[]),
                lambda: ops.clip_grad_norm([g], 1.0, outs=[g.half()]),
                lambda: ops.clip_grad_norm([g], 1.0, outs=[g[:4]])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        ops.grad_norm([g.double()])
    with pytest.raises(RuntimeError):
        ops.grad_norm([g, torch.zeros(2)])
