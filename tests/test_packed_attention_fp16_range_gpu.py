"""float16 packed attention where the gradients are not of size one: P and dS are rounded to
float16 as operands of the products, whose normal range is 6.1e-5 .. 65504 only.

Tolerance (relative 2-norm of a whole output, as for gradients of size one): the operands'
and the result's roundings, 4 u, and half a step of float16's subnormals, 2^-25, for every
element of the output."""

import math

import pytest
import torch

from tests.test_packed_attention_gpu import make, reference

pytestmark = pytest.mark.gpu
U = 2.0 ** -11


def grads(q, k, v, do, cu, scale=None):
    from evograd_b200 import ops

    plan = ops.packed_plan(cu, q.shape[0])
    o, lse = ops.packed_attention_fwd(q, k, v, plan, scale=scale)
    return ops.packed_attention_bwd(do, q, k, v, o, lse, plan, scale=scale)


def assert_close(got, want, names=("dq", "dk", "dv")):
    for name, a, (b, slack) in zip(names, got, want):
        assert bool(torch.isfinite(a).all()), name
        off = float((a.double() - b).norm())
        bound = 4 * U * float(b.norm()) + slack + 2.0 ** -25 * math.sqrt(b.numel())
        assert off <= bound, (name, off, bound)


@pytest.mark.parametrize("lens,hq,hkv,d", [([4100, 37], 2, 1, 96), ([2000, 1, 300], 2, 2, 64)])
@pytest.mark.parametrize("power", [-14, -10, -7, 0, 8])
def test_scaled_gradients(lens, hq, hkv, d, power):
    q, k, v, do, cu = make(lens, 3, hq, hkv, d, "fp16", seed=2)
    do = (do.float() * 2.0 ** power).half()
    assert_close(grads(q, k, v, do, cu), reference(q, k, v, lens, do)[2])


@pytest.mark.parametrize("power", [-10, 7])
def test_the_gradient_is_linear_in_do(power):
    """A power of two on do is one on the gradients: exact but for the results' rounding (dq
    also for the order of float32 sums)."""
    lens = [1500, 200]
    q, k, v, do, cu = make(lens, 0, 2, 1, 64, "fp16", seed=3)
    do = torch.where(do.abs() < 2.0 ** -3, torch.full_like(do, 0.125), do)  # exact when scaled down
    one = grads(q, k, v, do, cu)
    other = grads(q, k, v, (do.float() * 2.0 ** power).half(), cu)
    for a, b in zip(one, other):
        a, b = a.double() * 2.0 ** power, b.double()
        assert float((a - b).norm()) <= 2 * U * float(a.norm()) + 2.0 ** -24 * math.sqrt(a.numel()) * max(1.0, 2.0 ** power)


def test_large_gradients():
    """dS beyond 65504 with results inside: values of 64, do of 256, a small scale."""
    lens, d = [300, 40], 96
    q, k, v, do, cu = make(lens, 0, 2, 1, d, "fp16", seed=5)
    v, do, scale = v * 64, do * 256, 1.0 / 64
    got = grads(q, k, v, do, cu, scale=scale)
    # the reference's scale is 1 / sqrt(d): fold the rest into q and out of dq
    fold = scale * math.sqrt(d)
    dq, dk, dv = reference(q.double() * fold, k.double(), v.double(), lens, do.double())[2]
    largest = 0.0
    for a, n in ((0, 300), (300, 40)):
        s = scale * (q[a:a + n].double().transpose(0, 1) @ k[a:a + n].double().permute(1, 2, 0))
        p = s.masked_fill(torch.ones(n, n, device="cuda", dtype=torch.bool).triu(1), float("-inf")).softmax(-1)
        dp = do[a:a + n].double().transpose(0, 1) @ v[a:a + n].double().permute(1, 2, 0)
        largest = max(largest, float((p * (dp - (p * dp).sum(-1, keepdim=True))).abs().max()))
    assert largest > 65504.0
    assert_close(got, [(dq[0] * fold, dq[1] * fold), dk, dv])


def test_sequences_and_rows_of_different_size():
    """One factor serves a k/v head: documents whose gradients are 2^-8 of another's keep
    their accuracy, and a row of do that is not finite takes it from nobody."""
    lens = [300, 2000, 77]
    q, k, v, do, cu = make(lens, 3, 2, 1, 64, "fp16", seed=6)
    do[300:2300] = (do[300:2300].float() * 2.0 ** -8).half()
    got = grads(q, k, v, do, cu)
    for sl in (slice(0, 300), slice(300, 2300), slice(2300, 2377)):
        n = sl.stop - sl.start
        assert_close([t[sl] for t in got], reference(q[sl], k[sl], v[sl], [n], do[sl])[2])
    do[5, 0, 3], v[310, 0, 1] = float("inf"), float("nan")
    again = grads(q, k, v, do, cu)
    sl = slice(2300, 2377)
    for i, (a, b) in enumerate(zip(again, got)):
        assert bool(((a[sl].double() - b[sl].double()).abs() <= 2 * U * b[sl].double().abs() + 2.0 ** -24).all()), i


def test_gradients_of_zero():
    q, k, v, do, cu = make([200, 9], 3, 2, 1, 64, "fp16", seed=7)
    assert not any(bool(t.any()) for t in grads(q, k, v, torch.zeros_like(do), cu))
    dq, dk, dv = grads(q, k, torch.zeros_like(v), do, cu)
    assert not bool(dq.any()) and not bool(dk.any()) and bool(dv.any())


def test_captured_and_replayed_with_gradients_of_other_sizes():
    """The norms that set the scale are found again in every replay: small gradients after large ones
    have the bits of an eager call (dq up to the order of float32 sums)."""
    from evograd_b200 import ops

    q, k, v, do, cu = make([700, 130], 2, 4, 2, 64, "fp16", seed=8)
    base = do.clone()

    def step():
        plan = ops.packed_plan(cu, q.shape[0])
        o, lse = ops.packed_attention_fwd(q, k, v, plan)
        return ops.packed_attention_bwd(do, q, k, v, o, lse, plan)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for power in (0, 9, -12, -3):
        do.copy_((base.float() * 2.0 ** power).half())
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert torch.equal(out[1], eager[1]) and torch.equal(out[2], eager[2])
        # six key tiles' sums in another order: a few float32 roundings of numbers up to the
        # largest, and one of float16 on each side
        a, b = out[0].double(), eager[0].double()
        assert bool(((a - b).abs() <= 2 * U * b.abs() + 2.0 ** -24 + 2.0 ** -20 * b.abs().max()).all())
        assert_close(out, reference(q, k, v, [700, 130], do)[2])
