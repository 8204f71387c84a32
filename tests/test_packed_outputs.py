"""Outputs that are another tensor of the call: blocks read inputs while others write, so the
entry points refuse them before anything is enqueued (the addresses here are never read)."""

import pytest
import torch

EBADSHAPE = -1
A, B, X, Y, Z = (i << 24 for i in range(1, 6))


def rope(rows, T=64, D=64):
    from evograd_b200._cabi import RopePositionsTensor, lib

    n = len(rows)
    return lib.evg_rope_positions((RopePositionsTensor * n)(*rows), n, X, 4, Y, 4, T, D, D, 0, 1.0, 2, 0, None)


@pytest.mark.parametrize("rows", [
    [(A, B, 2, 128, 64, 128, 64), (B, A, 2, 128, 64, 128, 64)],     # exchanged
    [(A, Z, 2, 128, 64, 128, 64), (B, Z, 2, 128, 64, 128, 64)],     # one output for both
    [(A, B, 2, 128, 64, 128, 64), (B, Z, 2, 128, 64, 128, 64)],     # over the other input
    [(A, A, 64, 4096, 64, 64, 4096)],                               # over itself, tokens and heads exchanged
    [(A, A, 1, 128, 64, 64, 64)],                                   # over itself, rows closer together
])
def test_rope_refuses(rows):
    assert rope(rows) == EBADSHAPE


def view(p):
    from evograd_b200._cabi import PackedView

    return PackedView(p, 128, 64)


def test_attention_refuses():
    from evograd_b200._cabi import lib

    q, k, v, o, do = (view(p) for p in (A, B, X, Y, Z))
    plan = lse = ws = 1 << 28

    def fwd(out):
        return lib.evg_packed_attention_fwd(q, k, v, out, lse, plan, 128, 1, 2, 2, 64, 0.125, 2, None)

    def bwd(dq, dk, dv):
        return lib.evg_packed_attention_bwd(do, q, k, v, o, lse, view(dq), view(dk), view(dv), ws, 1 << 40, plan,
                                            128, 1, 2, 2, 64, 0.125, 2, None)

    for p in (A, B, X):
        assert fwd(view(p)) == EBADSHAPE
    free = [7 << 24, 8 << 24, 9 << 24]
    for i in range(3):
        for p in (A, B, X, Y, Z, free[i - 1]):
            outs = list(free)
            outs[i] = p
            assert bwd(*outs) == EBADSHAPE


@pytest.mark.gpu
def test_in_place_and_thirds_are_taken():
    """Rotation in place on the thirds of one projection; one token and one head, whose strides
    mean nothing; no heads."""
    from evograd_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(0)
    buf = torch.randn(30, 6 * 64, device="cuda", generator=g)
    q, k = buf[:, :256].unflatten(1, (4, 64)), buf[:, 256:].unflatten(1, (2, 64))
    pos, f = torch.arange(30, device="cuda"), ops.rope_inv_freq(64, device="cuda")[0]
    want = ops.rope_positions_fwd(q, k, pos, f)
    got = ops.rope_positions_fwd(q, k, pos, f, outs=(q, k))
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[0].data_ptr() == buf.data_ptr()
    one = buf[:1, :64].view(1, 1, 64)
    same = one.as_strided((1, 1, 64), (7 * 64, 3 * 64, 1))
    (want,) = ops.rope_positions_fwd(one, None, pos[5:6], f)
    ops.rope_positions_fwd(one, None, pos[5:6], f, outs=(same,))
    assert torch.equal(one, want)
    with pytest.raises(ops.EvgError):
        ops.rope_positions_fwd(q[:, :2], k, pos, f, outs=(k, q[:, :2]))
    x = torch.zeros(8, 2, 64, device="cuda", dtype=torch.bfloat16)
    plan = ops.packed_plan(torch.tensor([0, 8], device="cuda", dtype=torch.int32), 8)
    with pytest.raises(ops.EvgError):
        ops.packed_attention_fwd(x, x, x, plan, out=x)
