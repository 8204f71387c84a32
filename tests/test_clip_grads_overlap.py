"""Gradients or outputs that share memory: blocks scale all tensors at the same time, so an
overlap would make the result depend on their order. The entry point refuses it before
anything is enqueued (the addresses here are never read); neighbours are taken."""

import ctypes as C

import pytest
import torch

EBADSHAPE = -1


def clip(grads, outs, sizes, dtypes=None, clip=1):
    from evograd_b200 import _cabi

    n = len(grads)
    ptrs = lambda a: None if a is None else (C.c_void_p * n)(*a)  # noqa: E731
    ws = 1 << 20
    return _cabi.lib.evg_clip_grads(ptrs(grads), ptrs(outs), (C.c_int64 * n)(*sizes), (C.c_int * n)(*(dtypes or [0] * n)),
                                    n, 1.0, clip, ws, ws, 1 << 40, None)


A = 1 << 24
MANY = [A + 4000 * i for i in range(60)]


@pytest.mark.parametrize("grads,outs,sizes,dtypes", [
    ([A, A + 36], None, [10, 10], None),                     # the last element of one is the first of the other
    ([A + 36, A], None, [10, 10], None),
    ([A, A + 8], None, [100, 1], None),                      # one inside the other
    ([A, A + 18], None, [10, 10], [2, 2]),                   # 2-byte elements
    ([A, A + 400], [A + 400, A], [10, 10], None),            # outputs exchanged
    ([A, A + 400], [A + 800, A + 836], [10, 10], None),      # outputs that overlap
    ([A, A + 400], [A + 4, A + 800], [10, 10], None),        # an output shifted against its gradient
    ([A, A], [A + 800, A], [10, 10], None),                  # a gradient read twice and written
    (MANY, [p + 4 for p in MANY], [10] * 60, None),
    (MANY, [p + 4000 for p in MANY], [10] * 60, None),
])
def test_refused(grads, outs, sizes, dtypes):
    from evograd_b200 import _cabi

    assert clip(grads, outs, sizes, dtypes) == EBADSHAPE
    assert b"overlaps" in _cabi.lib.evg_last_error()


@pytest.mark.gpu
def test_neighbours_and_shared_inputs():
    from evograd_b200 import ops

    base = torch.arange(1.0, 101.0, device="cuda")
    want = base.clone()
    parts = [base[60:], base[:30], base[30:60], base[30:30]]
    norm = float(want.norm())
    ops.clip_grad_norm(parts, norm / 2)
    assert torch.allclose(base, want / 2, rtol=1e-6)
    # the same gradient read twice, its results in places of their own; one in place beside them
    g, out, other = torch.ones(50, device="cuda"), torch.empty(100, device="cuda"), torch.ones(7, device="cuda")
    n = ops.clip_grad_norm([g, g, other], 1.0, outs=[out[:50], out[50:], other])
    assert abs(float(n) - 107 ** 0.5) <= 1e-5
    for t in (out, other):
        assert torch.allclose(t, torch.full_like(t, 107 ** -0.5), rtol=1e-5)
    assert bool((g == 1).all())
    with pytest.raises(ops.EvgError, match="overlaps"):
        ops.clip_grad_norm([base[:40], base[39:]], 1.0)
    with pytest.raises(ops.EvgError, match="overlaps"):
        ops.clip_grad_norm([base[:50], base[50:]], 1.0, outs=[base[50:], base[:50]])
    ops.grad_norm([base[:40], base[39:]])  # reads only
