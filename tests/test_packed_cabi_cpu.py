"""Refusals of the packed-sequence operators that need no GPU: bad arguments are turned
down before anything is enqueued, and CPU tensors before the library is called."""

import ctypes as C

import pytest
import torch

EBADSHAPE, EALIGN, EDTYPE, ENULL, EWORKSPACE, EUNSUPPORTED = -1, -2, -3, -6, -7, -8


@pytest.fixture(scope="module")
def lib():
    from evograd_b200 import _cabi

    return _cabi.lib


def aligned(nbytes=256):
    buf = (C.c_char * (nbytes + 16))()
    addr = C.addressof(buf)
    return buf, (addr + 15) & ~15


def view(addr, st=64, sh=64):
    from evograd_b200._cabi import PackedView

    return PackedView(addr, st, sh)


def test_plan_sizes_and_refusals(lib):
    buf, p = aligned()
    assert lib.evg_packed_plan_bytes(-1, 1) == 0 and lib.evg_packed_plan_bytes(1, -1) == 0
    assert lib.evg_packed_plan_bytes((1 << 27) + 1, 1) == 0
    # every sequence and the tokens behind the last one round up to whole tiles
    small, more = lib.evg_packed_plan_bytes(1000, 1), lib.evg_packed_plan_bytes(1000, 200)
    assert 0 < small < more
    assert lib.evg_packed_plan(None, 1, 128, p, 1 << 20, None) == ENULL
    assert lib.evg_packed_plan(p, 1, -1, p, 1 << 20, None) == EBADSHAPE
    assert lib.evg_packed_plan(p, 1, 128, p + 4, 1 << 20, None) == EALIGN
    assert lib.evg_packed_plan(p, 1, 128, p, 16, None) == EWORKSPACE


def test_attention_refusals(lib):
    buf, p = aligned()
    v = view(p)

    def fwd(q=v, k=v, vv=v, o=v, lse=p, plan=p, T=128, n=1, hq=2, hkv=1, d=64, scale=0.125, dtype=2):
        return lib.evg_packed_attention_fwd(q, k, vv, o, lse, plan, T, n, hq, hkv, d, scale, dtype, None)

    def bwd(ws=p, nbytes=1 << 40, T=128, n=1, hq=2, hkv=1, d=64, scale=0.125, dtype=2, plan=p, lse=p, dq=v):
        return lib.evg_packed_attention_bwd(v, v, v, v, v, lse, dq, v, v, ws, nbytes, plan, T, n, hq, hkv, d,
                                            scale, dtype, None)

    for call in (fwd, bwd):
        assert call(plan=None) == ENULL and call(plan=p + 4) == EALIGN
        for bad in (0.0, -1.0, float("inf"), float("nan")):
            assert call(scale=bad) == EUNSUPPORTED
        assert call(T=-1) == EBADSHAPE and call(n=-1) == EBADSHAPE and call(T=(1 << 27) + 1) == EBADSHAPE
        assert call(hq=0) == EBADSHAPE and call(d=0) == EBADSHAPE and call(hq=3, hkv=2) == EBADSHAPE
        assert call(dtype=3) == EDTYPE and call(d=257) == EUNSUPPORTED and call(hq=65536) == EUNSUPPORTED
        assert call(lse=None) == ENULL
        assert call(T=0) == 0  # nothing to do
    assert fwd(q=None) == ENULL and fwd(k=view(None)) == ENULL
    assert bwd(dq=view(None)) == ENULL
    assert bwd(ws=None) == EWORKSPACE and bwd(nbytes=16) == EWORKSPACE and bwd(ws=p + 4) == EALIGN
    need = lib.evg_packed_attention_bwd_workspace_bytes
    assert need(0, 1, 1, 64) == 0 and 0 < need(128, 1, 1, 64) < need(128, 1, 1, 128) < need(128, 50, 1, 128)


def test_rope_norm_and_clip_refusals(lib):
    from evograd_b200._cabi import RopePositionsTensor

    buf, p = aligned()
    one = (RopePositionsTensor * 1)((p, p, 1, 64, 64, 64, 64))

    def rope(t=one, count=1, pos=p, pb=4, freq=p, fb=4, T=1, d=64, rd=64, dtype=2):
        return lib.evg_rope_positions(t, count, pos, pb, freq, fb, T, d, rd, 0, 1.0, dtype, 0, None)

    assert rope(t=None) == ENULL and rope(count=0) == EBADSHAPE and rope(count=3) == EBADSHAPE
    assert rope(rd=63) == EBADSHAPE and rope(rd=0) == EBADSHAPE and rope(rd=66) == EBADSHAPE
    assert rope(d=0) == EBADSHAPE and rope(d=5000, rd=2) == EBADSHAPE and rope(T=-1) == EBADSHAPE
    assert rope(pb=2) == EDTYPE and rope(fb=2) == EDTYPE and rope(pos=None) == ENULL and rope(freq=None) == ENULL
    assert rope(pos=p + 2) == EALIGN and rope(freq=p + 4, fb=8) == EALIGN and rope(dtype=7) == EDTYPE
    assert rope(t=(RopePositionsTensor * 1)((None, p, 1, 64, 64, 64, 64))) == ENULL
    assert rope(t=(RopePositionsTensor * 1)((p, p, -1, 64, 64, 64, 64))) == EBADSHAPE
    assert rope(T=0, pos=None) == 0

    def fwd(x=p, kind=0, gate=None, rows=1, c=8, dtype=0):
        return lib.evg_post_pre_norm_fwd(x, p, p, p, gate, kind, p, p, p, p, rows, c, 1.0, 1e-6, dtype, None)

    def bwd(x=p, kind=0, gate=None, dgate=None, ws=p, nbytes=1 << 40, rows=1, c=8, dtype=0):
        return lib.evg_post_pre_norm_bwd(p, p, x, p, p, p, gate, kind, p, p, p, p, p, p, dgate, ws, nbytes,
                                         rows, c, 1.0, dtype, None)

    for call in (fwd, bwd):
        assert call(x=None) == ENULL and call(kind=1) == ENULL and call(kind=4) == EBADSHAPE
        assert call(kind=-1) == EBADSHAPE and call(rows=-1) == EBADSHAPE and call(c=0) == EBADSHAPE
        assert call(dtype=3) == EDTYPE
    assert fwd(rows=0) == 0 and bwd(rows=0) == EBADSHAPE
    assert bwd(kind=1, gate=p) == ENULL  # a gate without a place for its gradient
    assert bwd(ws=None) == EWORKSPACE and bwd(nbytes=8) == EWORKSPACE and bwd(ws=p + 4) == EALIGN

    ptr, size, kind = (C.c_void_p * 1)(p), (C.c_int64 * 1)(4), (C.c_int * 1)(0)

    def clip(g=ptr, n=size, k=kind, count=1, mx=1.0, norm=p, ws=p, nbytes=1 << 40, outs=None):
        return lib.evg_clip_grads(g, outs, n, k, count, mx, 1, norm, ws, nbytes, None)

    assert clip(norm=None) == ENULL and clip(g=None) == ENULL and clip(count=-1) == EBADSHAPE
    assert clip(mx=-1.0) == EBADSHAPE and clip(mx=float("nan")) == EBADSHAPE
    assert clip(n=(C.c_int64 * 1)(-1)) == EBADSHAPE and clip(k=(C.c_int * 1)(5)) == EDTYPE
    assert clip(g=(C.c_void_p * 1)(None)) == ENULL and clip(outs=(C.c_void_p * 1)(None)) == ENULL
    assert clip(ws=None) == EWORKSPACE and clip(nbytes=8) == EWORKSPACE and clip(ws=p + 4) == EALIGN


def test_cpu_tensors_are_refused():
    from evograd_b200 import ops

    x = torch.zeros(4, 2, 64)
    plan = ops.PackedPlan(torch.zeros(64, dtype=torch.int32), 4, 1)
    for call in (lambda: ops.packed_plan(torch.zeros(2, dtype=torch.int32), 4),
                 lambda: ops.packed_attention_fwd(x, x, x, plan),
                 lambda: ops.packed_attention_bwd(x, x, x, x, x, torch.zeros(2, 4), plan),
                 lambda: ops.rope_positions_fwd(x, x, torch.arange(4), torch.ones(32)),
                 lambda: ops.post_pre_norm_fwd(x[0], x[0], torch.ones(64), torch.ones(64)),
                 lambda: ops.clip_grad_norm([x], 1.0), lambda: ops.grad_norm([x])):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(TypeError):
        ops.packed_plan([0, 4], 4)


def test_backward_workspace_follows_the_tokens(lib):
    """One-token sequences pad their statistics to whole tiles, not the float32 copy of dq."""
    need = lib.evg_packed_attention_bwd_workspace_bytes
    tokens, heads = 16384, 32
    copy = tokens * heads * 128 * 4
    assert need(tokens, 1, heads, 128) <= copy + (tokens + 256) * heads * 8
    assert need(tokens, tokens, heads, 128) <= copy + (tokens + tokens // 128 + 1) * 128 * heads * 8
