"""Causal attention over packed sequences (``ops.packed_*``) against the definition
in float64, sequence by sequence, with gradients by autograd in float64.

Tolerances (relative 2-norm of a whole output). With u = finfo(T).eps / 2 the kernel
rounds P and dS to T as tensor-core operands (each term off by at most u, the sums
over many terms well below that in the 2-norm), o once on the way out (u), and the
backward takes delta from the rounded o (u again, on one of two terms of dS):
o 2u, gradients 4u. float32 runs in float32 throughout, sums of n terms: n * 2^-24
at most, 2e-6 for the n <= 300 here.

dS = P (do.v - do.o) is a difference that can vanish (it does for a sequence of one
token), so next to that relative part dq and dk have an absolute one: a float32 sum of
D products is off by at most D 2^-24 times the sum of their magnitudes, hence dS by
P D 2^-24 (|do|.|v| + |do|.|o|) and dq, dk by what that gives behind |k|, |q|.
"""

import math

import pytest
import torch

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def reference(q, k, v, lens, do=None):
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    group = Hq // Hkv
    o = torch.zeros(T, Hq, D, dtype=torch.float64, device=q.device)
    lse = torch.full((Hq, T), float("-inf"), dtype=torch.float64, device=q.device)
    grads = [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (q, k, v)]
    slack = [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (q, k, v)]
    a = 0
    for n in lens:
        if n == 0:
            continue
        sl = slice(a, a + n)
        a += n
        qq, kk, vv = (t[sl].double().transpose(0, 1).detach().requires_grad_() for t in (q, k, v))
        s = qq @ kk.repeat_interleave(group, 0).transpose(1, 2) / math.sqrt(D)
        s = s.masked_fill(torch.ones(n, n, device=q.device, dtype=torch.bool).triu(1), float("-inf"))
        oo = torch.softmax(s, -1) @ vv.repeat_interleave(group, 0)
        o[sl] = oo.detach().transpose(0, 1)
        lse[:, sl] = torch.logsumexp(s.detach(), -1)
        if do is not None:
            for g, x in zip(grads, torch.autograd.grad(oo, (qq, kk, vv), do[sl].double().transpose(0, 1))):
                g[sl] = x.transpose(0, 1)
            with torch.no_grad():
                gg = do[sl].double().transpose(0, 1).abs()
                parts = torch.softmax(s, -1) * (gg @ vv.abs().repeat_interleave(group, 0).transpose(1, 2)
                                                + (gg * oo.abs()).sum(-1, keepdim=True)) / math.sqrt(D)
                slack[0][sl] = (parts @ kk.abs().repeat_interleave(group, 0)).transpose(0, 1)
                slack[1][sl] = (parts.transpose(1, 2) @ qq.abs()).unflatten(0, (Hkv, group)).sum(1).transpose(0, 1)
    return o, lse, [(g, D * 2.0 ** -24 * float(x.norm())) for g, x in zip(grads, slack)]


def rel(x, y):
    d = (x.double() - y).norm()
    return float(d / y.norm()) if float(y.norm()) else float(d)


def make(lens, pad, hq, hkv, d, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = sum(lens) + pad
    mk = lambda h: torch.randn(T, h, d, device="cuda", generator=g).to(DT[dtype])  # noqa: E731
    cu = torch.tensor([0] + list(torch.tensor(lens, dtype=torch.int64).cumsum(0)), dtype=torch.int32,
                      device="cuda")
    return mk(hq), mk(hkv), mk(hkv), mk(hq), cu


def check(lens, pad, hq, hkv, d, dtype, seed=0):
    from evograd_b200 import ops

    q, k, v, do, cu = make(lens, pad, hq, hkv, d, dtype, seed)
    T, n = q.shape[0], sum(lens)
    plan = ops.packed_plan(cu, T)
    plan.check()
    o, lse = ops.packed_attention_fwd(q, k, v, plan)
    dq, dk, dv = ops.packed_attention_bwd(do, q, k, v, o, lse, plan)
    ops.device_status()
    ro, rlse, (rdq, rdk, rdv) = reference(q, k, v, lens, do)
    u = torch.finfo(DT[dtype]).eps / 2
    fwd, bwd = (2e-6, 4e-6) if dtype == "fp32" else (2 * u, 4 * u)
    assert o.dtype == q.dtype and lse.dtype == torch.float32
    assert rel(o, ro) <= fwd, rel(o, ro)
    if n:
        assert float((lse[:, :n].double() - rlse[:, :n]).abs().max()) <= 2e-5
    for name, got, (want, slack) in (("dq", dq, rdq), ("dk", dk, rdk), ("dv", dv, rdv)):
        assert torch.isfinite(got).all(), name
        off = float((got.double() - want).norm())
        assert off <= bwd * float(want.norm()) + slack, (name, off, float(want.norm()), slack)
    for t in (o, dq, dk, dv):
        assert not t[n:].any()
    assert bool((lse[:, n:] == float("-inf")).all())


LENGTHS = [
    ([1], 0), ([128], 0), ([129], 0), ([0, 0], 3), ([5, 0, 1, 127, 128, 129, 0], 0),
    ([64, 1, 100, 0, 37], 6), ([300, 17, 513, 260], 131), ([1] * 70, 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,pad", LENGTHS)
@pytest.mark.parametrize("hq,hkv,d,dtype", [(4, 2, 128, "bf16"), (3, 3, 64, "fp16"), (6, 2, 64, "bf16"),
                                            (8, 2, 80, "bf16"), (2, 1, 24, "fp16")])
def test_tensor_core_against_float64(lens, pad, hq, hkv, d, dtype):
    check(lens, pad, hq, hkv, d, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,pad", [([1], 0), ([33, 0, 130, 1], 5), ([0], 2)])
@pytest.mark.parametrize("hq,hkv,d,dtype", [(2, 1, 16, "fp32"), (2, 2, 200, "fp32"), (4, 2, 20, "bf16"),
                                            (1, 1, 256, "fp16")])
def test_plain_kernels_against_float64(lens, pad, hq, hkv, d, dtype):
    check(lens, pad, hq, hkv, d, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,pad,hq,hkv,d", [([2100, 700, 1300], 0, 8, 2, 128), ([1500, 40], 9, 5, 5, 64)])
def test_longer_sequences(lens, pad, hq, hkv, d):
    check(lens, pad, hq, hkv, d, "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("d", list(range(8, 129, 8)))
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_every_head_size_of_the_tensor_cores(d, dtype):
    check([140, 1, 260], 4, 4, 2, d, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,hq,hkv,d,dtype", [
    ([4200], 3, 1, 128, "bf16"),              # two neighbouring tiles of one head per block
    ([4100, 4300], 3, 1, 96, "fp16"),
    ([70] * 40, 6, 2, 128, "bf16"),           # one tile per block
    ([300, 301], 4, 2, 128, "fp16"),          # two heads' tiles per block
    ([385, 640, 1000], 2, 2, 64, "bf16"),
    ([300], 4, 1, 64, "fp32"), ([97, 64, 33], 2, 2, 130, "bf16")])
def test_every_shape_of_the_blocks(lens, hq, hkv, d, dtype):
    check(lens, 0, hq, hkv, d, dtype)
