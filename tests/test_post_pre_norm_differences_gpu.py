"""Gradients of the two norms against central differences, float32, 7 rows of 96 columns.

Tolerance: the step 1e-2 leaves a truncation of step^2 = 1e-4 times third derivatives, which
for these normalised functions are a few times the first; y and h are off by a few 2^-24
each, 1e-5 over 672 terms of size one for both values, and five times that is allowed. Along the
gradient itself the quotient is the gradient's norm times the direction's: 2e-3 of it; along
a random direction, whose quotient is typically the direction's rms times the gradient's
norm, 5e-3 of that."""

import pytest
import torch

from tests.test_post_pre_norm_gpu import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
def test_directions(gate):
    from evograd_b200 import ops

    t = make(7, 96, gate, "fp32")
    names = ["x", "h", "wp", "wn"] + (["gate"] if gate != "none" else [])

    def forward(s):
        return ops.post_pre_norm_fwd(s["x"], s["h"], s["wp"], s["wn"], s["gate"], alpha=0.7)

    def value(s):
        h, y, *_ = forward(s)
        return float((t["dy"].double() * y.double()).sum() + (t["dh"].double() * h.double()).sum())

    h, y, r1, r2 = forward(t)
    grads = ops.post_pre_norm_bwd(t["dy"], t["dh"], t["x"], h, t["wp"], t["wn"], t["gate"], r1, r2, alpha=0.7)
    g, step = torch.Generator(device="cuda").manual_seed(1), 1e-2
    for name, grad in zip(names, grads):
        grad = grad.double().view(t[name].shape)
        along = grad / grad.square().mean().sqrt()
        other = torch.randn(t[name].shape, device="cuda", generator=g, dtype=torch.float64)
        for d, slack in ((along, 2e-3 * float(grad.norm() * along.norm())), (other, 5e-3 * float(grad.norm()))):
            up = dict(t, **{name: (t[name].double() + step * d).float()})
            down = dict(t, **{name: (t[name].double() - step * d).float()})
            moved = (up[name].double() - down[name].double())  # what the rounded inputs differ by
            assert abs(value(up) - value(down) - float((grad * moved).sum())) <= 2 * step * slack + 5e-5, name
