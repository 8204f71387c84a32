"""Rows of packed attention's dq on their own: whole-tensor norms hide the few rows that see
only a handful of keys, where dS = P (dP - delta) is a small difference."""

import math

import pytest
import torch

from tests.test_packed_attention_gpu import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv,d,dtype", [(4, 2, 128, "bf16"), (6, 2, 80, "bf16"), (3, 1, 64, "fp16"),
                                            (8, 1, 64, "bf16"), (2, 2, 16, "fp32")])
def test_first_rows_of_a_sequence(hq, hkv, d, dtype):
    """dq of rows 0 .. 7 of sequences of 8, 9 and several hundred tokens, row by row. With
    u = finfo(T).eps / 2, the row's dq = scale sum_j dS_ij k_j has every dS rounded once (u), P
    off by the hardware's exp2 and the float32 scores (1e-5), and itself rounded once (u):
        |err| <= (u + 1e-5) scale sum_j |dS_ij| |k_j| + u |dq|   (2-norms along the head),
    and dP - delta carries the float32 roundings of sums of D products: independent ones
    add up as sqrt(D), four times that is allowed, relative to the products' magnitudes, for dP
    and delta and, through the score, for P's weight in delta."""
    from evograd_b200 import ops

    lens = [300, 9, 8, 300, 2, 131, 9, 640, 3, 8, 129]
    q, k, v, do, cu = make(lens, 5, hq, hkv, d, dtype, seed=11)
    plan = ops.packed_plan(cu, q.shape[0])
    o, lse = ops.packed_attention_fwd(q, k, v, plan)
    dq = ops.packed_attention_bwd(do, q, k, v, o, lse, plan)[0].double()
    u, scale = torch.finfo(q.dtype).eps / 2, 1.0 / math.sqrt(d)
    eta = 4 * math.sqrt(d) * 2.0 ** -24
    worst, a = 0.0, 0
    for n in lens:
        m = min(n, 8)
        qd, gd = (t[a:a + m].double().transpose(0, 1) for t in (q, do))
        kd, vd = (t[a:a + m].double().transpose(0, 1).repeat_interleave(hq // hkv, 0) for t in (k, v))
        a_rows = dq[a:a + m].transpose(0, 1)
        a += n
        s = (qd @ kd.transpose(1, 2)) * scale
        hidden = torch.ones(m, m, device="cuda", dtype=torch.bool).triu(1)
        p = s.masked_fill(hidden, float("-inf")).softmax(-1)
        dp = gd @ vd.transpose(1, 2)
        ds = p * (dp - (p * dp).sum(-1, keepdim=True))
        want = scale * ds @ kd
        knorm = kd.norm(dim=-1)
        size = (gd.abs() @ vd.abs().transpose(1, 2)).masked_fill(hidden, 0).amax(-1, keepdim=True)
        steep = 1 + scale * (qd.abs() @ kd.abs().transpose(1, 2)).masked_fill(hidden, 0).amax(-1, keepdim=True)
        slack = scale * ((p * 2 * eta * steep * size) * knorm[:, None]).sum(-1)
        bound = (u + 1e-5) * scale * (ds.abs() * knorm[:, None]).sum(-1) + u * want.norm(dim=-1) + slack
        worst = max(worst, float(((a_rows - want).norm(dim=-1) / bound).max()))
    assert worst <= 1.0, worst


def test_appending_tokens_keeps_the_first_rows_accurate():
    """Row 1 of a document has the same two terms whatever follows it: its dq agrees with the
    two-token document's to the roundings named above (dS and dq, once on each side)."""
    from evograd_b200 import ops

    hq, hkv, d = 32, 8, 128
    q, k, v, do, _ = make([300], 0, hq, hkv, d, "bf16", seed=4)

    def dq_of(n):
        t = [x[:n].contiguous() for x in (q, k, v, do)]
        plan = ops.packed_plan(torch.tensor([0, n], device="cuda", dtype=torch.int32), n)
        o, lse = ops.packed_attention_fwd(*t[:3], plan)
        return ops.packed_attention_bwd(t[3], *t[:3], o, lse, plan)[0][1].double()

    u, two = 2.0 ** -8, dq_of(2)
    for n in (9, 128, 300):
        off = (dq_of(n) - two).norm(dim=-1) / two.norm(dim=-1)
        # two terms of equal weight: sum |dS| |k| <= 2.9 |dq| for keys of 128 random numbers
        assert float(off.max()) <= 2 * (2.9 * u + u), (n, float(off.max()))
