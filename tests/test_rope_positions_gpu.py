"""Rotary embedding from position numbers against the definition in float64.

Tolerance: the angle is exact to float64 before one float32 sincospi (its argument
rounds by 2^-25 of at most one half turn, so the angle is off by at most 2^-25 pi <
1e-7, and sine and cosine by that plus two ulp: under 4e-7), products and sums are
float32 and the result rounds once to T: |y - exact| <= u |exact| + 1e-6 m (|x1| + |x2|).
"""

import math

import pytest
import torch

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def rotate64(x, pos, f, interleaved, mscale, inverse):
    rd = 2 * f.numel()
    ang = pos.double()[:, None, None] * f.double()
    c, s = ang.cos() * mscale, ang.sin() * mscale * (-1 if inverse else 1)
    y = x.double().clone()
    if interleaved:
        a, b = x[..., 0:rd:2].double(), x[..., 1:rd:2].double()
        y[..., 0:rd:2], y[..., 1:rd:2] = a * c - b * s, b * c + a * s
        mag = (a.abs() + b.abs()).repeat_interleave(2, -1)
    else:
        a, b = x[..., : rd // 2].double(), x[..., rd // 2: rd].double()
        y[..., : rd // 2], y[..., rd // 2: rd] = a * c - b * s, b * c + a * s
        mag = torch.cat([a.abs() + b.abs()] * 2, -1)
    slack = torch.zeros_like(y)
    slack[..., :rd] = 1e-6 * mscale * mag
    return y, slack


def near(got, want, slack, dtype):
    u = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * u * 2  # half a step of the subnormals
    off = (got.double() - want).abs()
    assert bool((off <= u * want.abs() + slack + tiny).all()), float((off - u * want.abs() - slack).max())


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype,T,hq,hk,d,rd", [
    ("bf16", 1, 32, 8, 128, 128), ("fp16", 3, 24, 6, 80, 20), ("fp32", 7, 3, 1, 64, 64),
    ("bf16", 300, 4, 4, 96, 50), ("fp32", 33, 2, 1, 10, 6), ("fp16", 1000, 5, 3, 256, 2),
    ("bf16", 2, 700, 1, 64, 32), ("bf16", 5, 1, 0, 7, 2), ("bf16", 4100, 1, 1, 512, 512),
])
def test_against_float64(dtype, T, hq, hk, d, rd, interleaved):
    from evograd_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(T)
    q, k = (torch.randn(T, h, d, device="cuda", generator=g).to(DT[dtype]) for h in (hq, hk))
    pos = torch.randint(-50, 1_000_000, (T,), device="cuda", generator=g)
    f, _ = ops.rope_inv_freq(rd, 500000.0, scaling="wavelength", factor=8.0, device="cuda")
    for inverse, fn in ((False, ops.rope_positions_fwd), (True, ops.rope_positions_bwd)):
        got = fn(q, k, pos, f, interleaved=interleaved, mscale=1.25)
        for x, y in zip((q, k), got):
            want, slack = rotate64(x, pos, f, interleaved, 1.25, inverse)
            near(y, want, slack, DT[dtype])
            assert torch.equal(y[..., rd:], x[..., rd:])


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_views_positions_and_in_place(interleaved, offset):
    """Thirds of one projection, any alignment, int32 positions, float32 frequencies, in place."""
    from evograd_b200 import ops

    T, hq, hk, d = 65, 6, 2, 64
    buf = torch.randn(T, (hq + 2 * hk) * d + 8, device="cuda").to(torch.bfloat16)
    q = buf[:, offset: offset + hq * d].unflatten(1, (hq, d))
    k = buf[:, offset + hq * d: offset + (hq + hk) * d].unflatten(1, (hk, d))
    pos = torch.arange(T, device="cuda", dtype=torch.int32) * 37
    f = ops.rope_inv_freq(d, device="cuda")[0].float()
    want = [rotate64(x, pos, f, interleaved, 1.0, False) for x in (q, k)]
    rest = buf.clone()
    out = ops.rope_positions_fwd(q, k, pos, f, interleaved=interleaved)
    assert torch.equal(buf, rest)
    res = ops.rope_positions_fwd(q, k, pos, f, interleaved=interleaved, outs=(q, k))
    for r, x, o, (w, slack) in zip(res, (q, k), out, want):
        assert r.data_ptr() == x.data_ptr() and torch.equal(r, o)
        near(r, w, slack, torch.bfloat16)
    end = offset + (hq + hk) * d
    assert torch.equal(buf[:, :offset], rest[:, :offset]) and torch.equal(buf[:, end:], rest[:, end:])


@pytest.mark.gpu
def test_transpose_and_one_tensor():
    """<rotate(x), y> = <x, rotate_bwd(y)>, and one tensor alone gives the same bits."""
    from evograd_b200 import ops

    x, y = torch.randn(2, 40, 3, 32, device="cuda").unbind(0)
    pos = torch.arange(40, device="cuda") * 1001
    f, m = ops.rope_inv_freq(32, scaling="ramp", factor=4.0, slow=1.0, fast=32.0, device="cuda")
    (rx,) = ops.rope_positions_fwd(x, None, pos, f, mscale=m)
    (ry,) = ops.rope_positions_bwd(y, None, pos, f, mscale=m)
    a, b = float((rx.double() * y.double()).sum()), float((x.double() * ry.double()).sum())
    # 3840 products of size about 1, each off by at most a few float32 roundings
    assert abs(a - b) <= 3840 * 4 * 2.0 ** -24 * 8
    assert torch.equal(ops.rope_positions_fwd(x, y, pos, f, mscale=m)[0], rx)
    assert ops.rope_positions_fwd(x[:0], None, pos[:0], f)[0].shape == (0, 3, 32)


@pytest.mark.gpu
def test_nan_beside_the_rotated_columns_stays_there():
    from evograd_b200 import ops

    for interleaved in (False, True):
        x = torch.ones(3, 2, 24, device="cuda", dtype=torch.bfloat16)
        x[..., 12:] = float("nan")
        f, _ = ops.rope_inv_freq(12, device="cuda")
        (y,) = ops.rope_positions_fwd(x, None, torch.arange(3, device="cuda"), f, interleaved=interleaved)
        assert torch.isfinite(y[..., :12]).all() and torch.isnan(y[..., 12:]).all()


@pytest.mark.gpu
def test_refusals():
    from evograd_b200 import ops

    x = torch.zeros(4, 2, 16, device="cuda")
    pos, f = torch.arange(4, device="cuda"), ops.rope_inv_freq(16, device="cuda")[0]
    for bad in (lambda: ops.rope_positions_fwd(x[0], None, pos, f),
                lambda: ops.rope_positions_fwd(x, x[:3], pos, f),
                lambda: ops.rope_positions_fwd(x, x.half(), pos, f),
                lambda: ops.rope_positions_fwd(x, None, pos[:3], f),
                lambda: ops.rope_positions_fwd(x, None, pos.float(), f),
                lambda: ops.rope_positions_fwd(x, None, pos, torch.ones(9, device="cuda")),
                lambda: ops.rope_positions_fwd(x, None, pos, f[:0]),
                lambda: ops.rope_positions_fwd(x, None, pos, f.half()),
                lambda: ops.rope_positions_fwd(x, None, pos, f, outs=(x, x)),
                lambda: ops.rope_positions_fwd(x, None, pos, f, outs=(x[:, :1].expand(4, 2, 16),))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        ops.rope_positions_fwd(x.double(), None, pos, f)


def test_frequencies():
    from evograd_b200 import ops

    f, m = ops.rope_inv_freq(8, 10000.0)
    assert m == 1.0 and f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14)
    assert torch.allclose(ops.rope_inv_freq(8, scaling="linear", factor=4.0)[0], f / 4, rtol=1e-15)
    g = ops.rope_inv_freq(8, scaling="base", factor=4.0)[0]
    assert g[0] == 1.0 and math.isclose(float(g[-1]), 0.001 / 4, rel_tol=1e-12)
    w = ops.rope_inv_freq(8, scaling="wavelength", factor=8.0, original_context=1000)[0]
    # 159, 15.9, 1.59 and 0.159 turns over 1000 positions
    keep = (1000 * 0.01 / (2 * math.pi) - 1.0) / 3.0
    want = [1.0, 0.1, 0.01 * (keep + (1 - keep) / 8), 0.001 / 8]
    assert torch.allclose(w, torch.tensor(want, dtype=torch.float64), rtol=1e-12)
    r, m = ops.rope_inv_freq(64, scaling="ramp", factor=4.0, original_context=4096, slow=1.0, fast=32.0)
    base = ops.rope_inv_freq(64)[0]
    assert math.isclose(m, 0.1 * math.log(4.0) + 1.0)
    assert r[0] == base[0] and math.isclose(float(r[-1]), float(base[-1]) / 4, rel_tol=1e-12)
    assert bool(((r <= base) & (r >= base / 4)).all())
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, base=0.5),
                dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, slow=4.0, fast=4.0)):
        with pytest.raises(ValueError):
            ops.rope_inv_freq(**bad)
