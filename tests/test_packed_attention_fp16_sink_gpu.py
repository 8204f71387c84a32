"""float16 packed attention whose rows rest on one key: the first token takes all but 2^-9 of every
row's weight and has the value zero, as trained models' first tokens do. The other keys'
probabilities, 2^-21, are the whole result, and lie below float16's normal range.

Tolerance (relative 2-norm), as for ordinary attention: o 2 u, gradients 4 u, with half a step
of float16's subnormals, 2^-25, for every element of the output."""

import math

import pytest
import torch

from tests.test_packed_attention_gpu import make, reference

pytestmark = pytest.mark.gpu
U = 2.0 ** -11


@pytest.mark.parametrize("d,hq,hkv", [(64, 2, 1), (128, 2, 2), (80, 3, 1)])
def test_weights_below_the_normal_range(d, hq, hkv):
    from evograd_b200 import ops

    L = 4100
    q, k, v, do, cu = make([L, 60], 4, hq, hkv, d, "fp16", seed=12)
    q, k = q * 0.1, k * 0.1
    score = 21 * math.log(2.0) * math.sqrt(d)  # of the first key, before the scale
    q[..., 0] = math.sqrt(score)
    k[..., 0] = 0
    k[0] = 0
    k[0, :, 0] = math.sqrt(score)
    v, do = v * 64, do * 128
    v[0] = 0
    plan = ops.packed_plan(cu, q.shape[0])
    o, lse = ops.packed_attention_fwd(q, k, v, plan)
    grads = ops.packed_attention_bwd(do, q, k, v, o, lse, plan)
    wo, wl, want = reference(q, k, v, [L, 60], do)
    rows = slice(1000, L)
    weight = torch.exp(q[2000].double().mul(k[0, 0].double()).sum(-1) / math.sqrt(d) - wl[:, 2000])
    assert bool((weight > 0.99).all())  # one key has the weight
    got, ref = o[rows].double(), wo[rows]
    assert float((got - ref).norm()) <= 2 * U * float(ref.norm()) + 2.0 ** -25 * math.sqrt(ref.numel())
    seen = wl > float("-inf")
    assert float((lse.double()[seen] - wl[seen]).abs().max()) <= 1e-4
    for name, a, (b, slack) in zip(("dq", "dk", "dv"), grads, want):
        a, b = a[rows].double(), b[rows]
        bound = 4 * U * float(b.norm()) + slack + 2.0 ** -25 * math.sqrt(b.numel())
        assert float((a - b).norm()) <= bound, (name, float((a - b).norm()) / float(b.norm()))
