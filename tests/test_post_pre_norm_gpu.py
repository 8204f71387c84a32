"""The norms after and before a block with gate and residual scale against autograd of
the definition in float64.

Tolerances (relative 2-norm of a whole output, u = finfo(T).eps / 2): the forward
rounds once, u, plus float32 sums of C terms (C 2^-24 at most, far less in practice:
1e-6 covers C = 16384). The backward reads h rounded to T (relative u, which enters every
term of the two norms' gradients once) and rounds once: 3u, plus 2e-6.
"""

import pytest
import torch

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def make(rows, cols, gate, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    shape = {"none": None, "channel": (cols,), "token": (rows, 1), "full": (rows, cols)}[gate]
    t = dict(x=r(rows, cols), h=2 * r(rows, cols), wp=1 + 0.1 * r(cols), wn=1 + 0.1 * r(cols),
             dy=r(rows, cols), dh=r(rows, cols), gate=None if shape is None else torch.sigmoid(r(*shape)))
    return {k: None if v is None else v.to(DT[dtype]) for k, v in t.items()}


def reference(t, alpha):
    x, h, wp, wn = (t[n].double().requires_grad_() for n in ("x", "h", "wp", "wn"))
    g = None if t["gate"] is None else t["gate"].double().requires_grad_()
    n = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * wp
    h2 = h + alpha * (n if g is None else g * n)
    y = h2 * torch.rsqrt(h2.square().mean(-1, keepdim=True) + EPS) * wn
    leaves = [x, h, wp, wn] + ([] if g is None else [g])
    return h2.detach(), y.detach(), torch.autograd.grad([y, h2], leaves, [t["dy"].double(), t["dh"].double()])


def rel(a, b):
    return float((a.double() - b).norm() / b.norm())


def check(t, alpha, dtype):
    from evograd_b200 import ops

    u = torch.finfo(DT[dtype]).eps / 2
    h, y, r1, r2 = ops.post_pre_norm_fwd(t["x"], t["h"], t["wp"], t["wn"], t["gate"], alpha=alpha, eps=EPS)
    grads = ops.post_pre_norm_bwd(t["dy"], t["dh"], t["x"], h, t["wp"], t["wn"], t["gate"], r1, r2, alpha=alpha)
    wh, wy, want = reference(t, alpha)
    assert rel(h, wh) <= u + 1e-6 and rel(y, wy) <= u + 1e-6
    assert (grads[4] is None) == (t["gate"] is None)
    for name, got, w in zip(("dx", "dres", "dpost", "dpre", "dgate"), grads, want):
        assert got.dtype == DT[dtype] and got.shape == w.shape
        assert rel(got, w) <= 3 * u + 2e-6, (name, rel(got, w))
    return h, y, grads


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,cols", [(1, 4096), (3, 16), (700, 256), (33, 500), (9, 17), (1000, 1536),
                                       (257, 5120), (40, 8192), (5, 16384), (2, 20000)])
def test_against_float64(rows, cols, gate, dtype):
    check(make(rows, cols, gate, dtype), 0.5, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("dtype,rows,cols", [
    ("bf16", 5000, 1), ("fp32", 9, 255), ("bf16", 2500, 201), ("fp16", 300, 257), ("fp32", 1200, 1001),
    ("bf16", 700, 1500), ("fp16", 400, 2047), ("bf16", 333, 2049), ("fp32", 150, 4095), ("bf16", 300, 4097),
    ("fp32", 64, 6001), ("fp16", 170, 6145), ("bf16", 151, 8191), ("bf16", 3, 8193)])
def test_rows_off_the_vector_boundary(dtype, rows, cols, gate):
    """Each shape of the element-wise kernels, below and above its limits."""
    check(make(rows, cols, gate, dtype), 0.5, dtype)


@pytest.mark.gpu
def test_bits_do_not_change_between_runs():
    t = make(3001, 2048, "channel", "bf16")
    a, b = check(t, 0.22, "bf16"), check(t, 0.22, "bf16")
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert all(torch.equal(p, q) for p, q in zip(a[2], b[2]))


@pytest.mark.gpu
def test_shapes_strides_and_empty():
    from evograd_b200 import ops

    t = make(24, 64, "token", "fp32")
    h, y, r1, r2 = ops.post_pre_norm_fwd(t["x"], t["h"], t["wp"], t["wn"], t["gate"])
    wide = torch.zeros(64, 24, device="cuda").t()  # another order in memory
    wide.copy_(t["x"])
    h3, y3, *_ = ops.post_pre_norm_fwd(wide.view(2, 12, 64), t["h"].view(2, 12, 64), t["wp"], t["wn"],
                                       t["gate"].view(2, 12, 1))
    assert h3.shape == (2, 12, 64) and torch.equal(h3.view(24, 64), h) and torch.equal(y3.view(24, 64), y)
    # a gate broadcast over rows by its strides is one of full width
    gate = t["wp"].expand(24, 64)
    hf, yf, *_ = ops.post_pre_norm_fwd(t["x"], t["h"], t["wp"], t["wn"], gate)
    hc, yc, _, rc = ops.post_pre_norm_fwd(t["x"], t["h"], t["wp"], t["wn"], t["wp"])
    # n = x (w g) rstd or (x w) g rstd: at most five float32 roundings each way, relative to
    # n and not to the sum h + n, which can cancel; the sum rounds once more. y is off by
    # that times rstd w, and by its own roundings and the rstd's (a sum of 64 squares).
    n = hc - t["h"]
    off = 10 * 2.0 ** -24 * n.abs() + 2 * 2.0 ** -24 * hc.abs()
    assert bool(((hf - hc).abs() <= off).all())
    assert bool(((yf - yc).abs() <= off * (rc[:, None] * t["wn"]).abs() + 1e-5 * yc.abs()).all())
    # tensors that start off a 16-byte boundary take the kernels without vectors
    buf = torch.zeros(24 * 64 + 1, device="cuda")
    off = buf[1:].view(24, 64)
    off.copy_(t["x"])
    ho, yo, *_ = ops.post_pre_norm_fwd(off, t["h"], t["wp"], t["wn"], t["gate"])
    assert torch.allclose(ho, h, rtol=1e-5, atol=1e-6) and torch.allclose(yo, y, rtol=1e-5, atol=1e-6)
    e = t["x"][:0]
    h, y, r1, r2 = ops.post_pre_norm_fwd(e, e, t["wp"], t["wn"], t["gate"][:0])
    assert h.shape == (0, 64) and r1.numel() == 0
    dx, dres, dwp, dwn, dg = ops.post_pre_norm_bwd(e, e, e, e, t["wp"], t["wn"], t["gate"][:0], r1, r2)
    assert dx.shape == (0, 64) and not dwp.any() and not dwn.any() and dg.shape == (0, 1)


@pytest.mark.gpu
def test_gradient_against_differences():
    """Directional derivative of sum(dy y + dh h) by central differences, float32: the step
    1e-2 leaves a relative truncation of about 1e-4 and the float32 sums of 7 x 96 terms
    of size one an error of 1e-5 / 1e-2."""
    from evograd_b200 import ops

    t = make(7, 96, "full", "fp32")
    def value(x):
        h, y, *_ = ops.post_pre_norm_fwd(x, t["h"], t["wp"], t["wn"], t["gate"], alpha=0.7)
        return float((t["dy"].double() * y.double()).sum() + (t["dh"].double() * h.double()).sum())
    h, y, r1, r2 = ops.post_pre_norm_fwd(t["x"], t["h"], t["wp"], t["wn"], t["gate"], alpha=0.7)
    dx = ops.post_pre_norm_bwd(t["dy"], t["dh"], t["x"], h, t["wp"], t["wn"], t["gate"], r1, r2, alpha=0.7)[0]
    d = torch.randn_like(t["x"])
    step = 1e-2
    num = (value(t["x"] + step * d) - value(t["x"] - step * d)) / (2 * step)
    ana = float((dx.double() * d.double()).sum())
    assert abs(num - ana) <= 1e-2 * float(dx.double().norm() * d.double().norm())


@pytest.mark.gpu
def test_refusals():
    from evograd_b200 import ops

    t = make(4, 32, "token", "bf16")
    a = (t["x"], t["h"], t["wp"], t["wn"])
    for bad in (lambda: ops.post_pre_norm_fwd(t["x"], t["h"][:3], t["wp"], t["wn"]),
                lambda: ops.post_pre_norm_fwd(t["x"], t["h"].float(), t["wp"], t["wn"]),
                lambda: ops.post_pre_norm_fwd(t["x"], t["h"], t["wp"][:31], t["wn"]),
                lambda: ops.post_pre_norm_fwd(t["x"], t["h"], t["wp"], t["wn"].float()),
                lambda: ops.post_pre_norm_fwd(*a, t["gate"].float()),
                lambda: ops.post_pre_norm_fwd(*a, t["gate"][:2]),
                lambda: ops.post_pre_norm_fwd(*a, t["gate"].view(4))):
        with pytest.raises(ValueError):
            bad()
    h, y, r1, r2 = ops.post_pre_norm_fwd(*a, t["gate"])
    with pytest.raises(ValueError):
        ops.post_pre_norm_bwd(t["dy"], t["dh"], t["x"], h, t["wp"], t["wn"], t["gate"], r1[:2], r2)
    with pytest.raises(ValueError):
        ops.post_pre_norm_bwd(t["dy"][:2], t["dh"], t["x"], h, t["wp"], t["wn"], t["gate"], r1, r2)
    with pytest.raises(RuntimeError):
        ops.post_pre_norm_fwd(t["x"].cpu(), t["h"], t["wp"], t["wn"])
