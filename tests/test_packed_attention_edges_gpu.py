"""Packed attention where it can go wrong: content of other sequences and of unused rows,
strides, streams, invalid offsets, plans, tensors of more than 2^31 elements, refusals.
Comparisons are bit by bit unless a comment says why not."""

import pytest
import torch

from tests.test_packed_attention_gpu import make, reference, rel

pytestmark = pytest.mark.gpu


def run(q, k, v, do, cu, **kw):
    from evograd_b200 import ops

    plan = ops.packed_plan(cu, q.shape[0])
    o, lse = ops.packed_attention_fwd(q, k, v, plan, **kw)
    return (o, lse, *ops.packed_attention_bwd(do, q, k, v, o, lse, plan, **kw))


def same(a, b, rows=slice(None)):
    """o, lse, dk, dv bit by bit; dq is summed over key tiles in no fixed order: float32
    additions reordered, then rounded, so at most one step of the type apart."""
    for i, (x, y) in enumerate(zip(a, b)):
        x, y = (x[:, rows], y[:, rows]) if i == 1 else (x[rows], y[rows])
        if i == 2:
            step = torch.finfo(x.dtype).eps
            assert bool(((x.double() - y.double()).abs() <= step * y.double().abs() + 1e-5).all())
        else:
            assert torch.equal(x, y), i


@pytest.mark.parametrize("hq,hkv,d,dtype", [(4, 2, 128, "bf16"), (3, 1, 64, "fp16"), (2, 1, 16, "fp32")])
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_sequences_and_unused_rows_do_not_reach_one_another(hq, hkv, d, dtype, poison):
    lens, pad = [130, 77, 1, 200], 60
    q, k, v, do, cu = make(lens, pad, hq, hkv, d, dtype)
    clean = run(q, k, v, do, cu)
    for t in (q, k, v, do):
        t[130:207] = poison   # the second sequence
        t[408:] = poison      # behind the last one
    dirty = run(q, k, v, do, cu)
    same(dirty, clean, slice(0, 130))
    same(dirty, clean, slice(207, 408))
    for i, t in enumerate(dirty):
        tail = t[:, 408:] if i == 1 else t[408:]
        assert bool((tail == (float("-inf") if i == 1 else 0)).all())
    assert torch.isnan(dirty[0][130:207]).any()


@pytest.mark.parametrize("d,dtype", [(64, "bf16"), (80, "fp16"), (128, "bf16"), (20, "fp32")])
def test_views_of_one_projection_and_of_one_gradient(d, dtype):
    from evograd_b200 import ops

    hq, hkv, lens = 4, 2, [150, 33]
    q, k, v, do, cu = make(lens, 0, hq, hkv, d, dtype)
    want = run(q, k, v, do, cu)
    T = q.shape[0]
    buf = torch.full((T, (hq + 2 * hkv) * d + 8), 9.0, device="cuda", dtype=q.dtype)
    grad = torch.full_like(buf, 7.0)
    a, b, c = hq * d, (hq + hkv) * d, (hq + 2 * hkv) * d
    cut = lambda t: (t[:, :a].unflatten(1, (hq, d)), t[:, a:b].unflatten(1, (hkv, d)),  # noqa: E731
                     t[:, b:c].unflatten(1, (hkv, d)))
    for dst, src in zip(cut(buf), (q, k, v)):
        dst.copy_(src)
    head_major = do.transpose(0, 1).contiguous().transpose(0, 1)  # [T, H, D] over [H, T, D] memory
    plan = ops.packed_plan(cu, T)
    qv, kv, vv = cut(buf)
    ohm = torch.empty(hq, T, d, device="cuda", dtype=q.dtype).transpose(0, 1)
    o, lse = ops.packed_attention_fwd(qv, kv, vv, plan, out=ohm)
    assert o.data_ptr() == ohm.data_ptr()
    got = ops.packed_attention_bwd(head_major, qv, kv, vv, o, lse, plan, outs=cut(grad))
    same((o, lse, *got), want)
    assert bool((grad[:, c:] == 7.0).all()) and bool((buf[:, c:] == 9.0).all())
    # the last dimension strided, heads repeated by a stride of zero, an odd start
    wide = torch.zeros(T, hkv, 2 * d, device="cuda", dtype=q.dtype)
    wide[..., ::2] = v
    odd = torch.zeros(T * hkv * d + 1, device="cuda", dtype=q.dtype)[1:].view(T, hkv, d)
    odd.copy_(k)
    same(run(q, odd, wide[..., ::2], do, cu), want)
    one = k[:, :1].expand(T, hkv, d)
    same(run(q, one, one, do, cu), run(q, one.contiguous(), one.contiguous(), do, cu))


def test_bits_do_not_change_between_runs_but_for_dq():
    q, k, v, do, cu = make([700, 5, 300], 9, 8, 2, 128, "bf16")
    a = run(q, k, v, do, cu)
    for _ in range(3):
        same(run(q, k, v, do, cu), a)


def test_sequences_of_a_batch_equal_the_dense_kernels():
    """One sequence of a packed batch against the dense causal operators on that sequence:
    both round P and dS once as operands and differ in the order of sums, 4 u."""
    from evograd_b200 import ops

    q, k, v, do, cu = make([300, 256], 0, 4, 2, 128, "bf16")
    got = run(q, k, v, do, cu)
    sl = slice(300, 556)
    dense = [t[sl].transpose(0, 1)[None] for t in (q, k, v, do)]
    o, lse = ops.causal_gqa_attention_fwd(*dense[:3])
    dq, dk, dv = ops.causal_gqa_attention_bwd(dense[3], *dense[:3], o, lse)
    u = 2.0 ** -8
    for x, y in zip((got[0], *got[2:]), (o, dq, dk, dv)):
        assert rel(x[sl], y[0].transpose(0, 1).double()) <= 4 * u
    assert float((got[1][:, sl] - lse[0]).abs().max()) <= 1e-4


def test_scale_and_single_tokens():
    """Sequences of one token: o is v, lse the scaled score, and dS vanishes, so dq and dk are
    zero up to the float32 rounding of do.v (D products of size 1: 1e-5 after scale and k)."""
    q, k, v, do, cu = make([1] * 130, 0, 4, 2, 64, "bf16")
    o, lse, dq, dk, dv = run(q, k, v, do, cu, scale=0.3)
    assert torch.equal(o, v.repeat_interleave(2, 1))
    s = 0.3 * (q.double() * k.double().repeat_interleave(2, 1)).sum(-1).t()
    assert float((lse.double() - s).abs().max()) <= 1e-5
    assert float(dq.abs().max()) <= 1e-4 and float(dk.abs().max()) <= 1e-4
    want = do.double().unflatten(1, (2, 2)).sum(2)
    assert rel(dv, want) <= 2.0 ** -8


@pytest.mark.parametrize("hq,hkv,d,dtype", [(4, 2, 128, "bf16"), (2, 2, 64, "fp16"), (2, 1, 16, "fp32")])
def test_lone_tokens_have_no_score_gradient(hq, hkv, d, dtype):
    """One key's probability is one whatever its score: dq and dk are zero, not noise."""
    q, k, v, do, cu = make([1, 5, 1, 1], 2, hq, hkv, d, dtype)
    _, _, dq, dk, dv = run(q, k, v, do, cu)
    for row in (0, 6, 7):
        assert not bool(dq[row].any()) and not bool(dk[row].any())
        assert bool(dv[row].any())
    assert bool(dq[1:6].any()) and bool(dk[1:6].any())


@pytest.mark.parametrize("hq,hkv,d,dtype", [(4, 2, 128, "bf16"), (3, 1, 128, "bf16"), (2, 2, 64, "fp16"), (2, 1, 16, "fp32")])
def test_scores_of_minus_infinity_have_no_weight(hq, hkv, d, dtype):
    """Keys 0 .. 127 score -inf with every query: behind them, rows see only the others, also
    where a whole tile of keys comes before the first finite score."""
    from evograd_b200 import ops

    L, cut = 300, 128
    q, k, v, _, cu = make([L], 0, hq, hkv, d, dtype)
    q[:, :, 0] = q[:, :, 0].abs() + 0.5
    k[:cut, :, 0] = float("-inf")
    o, lse = ops.packed_attention_fwd(q, k, v, ops.packed_plan(cu, L))
    assert torch.isnan(o[:cut]).all()
    qd, kd, vd = q[cut:].double(), k[cut:].double(), v[cut:].double()
    kd, vd = (t.repeat_interleave(hq // hkv, 1) for t in (kd, vd))
    s = torch.einsum("ihd,jhd->hij", qd, kd) / d ** 0.5
    s = s.masked_fill(~torch.ones(L - cut, L - cut, dtype=torch.bool, device="cuda").tril(), float("-inf"))
    want = torch.einsum("hij,jhd->ihd", s.softmax(-1), vd)
    u = torch.finfo(q.dtype).eps / 2
    assert rel(o[cut:], want) <= 3 * u + 1e-5
    assert float((lse[:, cut:].double() - s.logsumexp(-1)).abs().max()) <= 1e-4


def test_many_short_sequences_among_long_ones():
    """The float32 copy of dq has no room per sequence: lengths around multiples of the tile,
    packed without gaps, must not share rows of it."""
    lens = [129, 1, 256, 257, 127, 385, 2, 128, 130, 1, 1, 640, 126, 131]
    q, k, v, do, cu = make(lens, 3, 4, 2, 64, "bf16")
    got = run(q, k, v, do, cu)
    start = 0
    for n in lens:
        one = torch.tensor([0, n], device="cuda", dtype=torch.int32)
        sl = slice(start, start + n)
        alone = run(q[sl].contiguous(), k[sl].contiguous(), v[sl].contiguous(), do[sl].contiguous(), one)
        same([t[:, sl] if i == 1 else t[sl] for i, t in enumerate(got)], alone)
        start += n


def test_invalid_offsets_make_a_plan_without_sequences():
    from evograd_b200 import ops

    q, k, v, do, _ = make([200], 0, 2, 1, 64, "bf16")
    for offsets in ([1, 200], [0, 150, 100], [0, 201], [0, -5, 200], [0, 1 << 40]):
        cu = torch.tensor(offsets, device="cuda")
        plan = ops.packed_plan(cu, 200)
        with pytest.raises(ops.EvgError, match="cu_seqlens"):
            plan.check()
        o, lse = ops.packed_attention_fwd(q, k, v, plan)
        grads = ops.packed_attention_bwd(do, q, k, v, o, lse, plan)
        assert not o.any() and bool((lse == float("-inf")).all()) and not any(g.any() for g in grads)
    ops.packed_plan(torch.tensor([0, 3, 200], device="cuda"), 200).check()
    ops.device_status()


def test_many_sequences():
    """More sequences than the plan builder has threads, most of them empty or one token."""
    g = torch.Generator().manual_seed(0)
    lens = torch.where(torch.rand(5000, generator=g) < 0.7, 0, torch.randint(1, 4, (5000,), generator=g)).tolist()
    lens[17], lens[4999] = 400, 129
    q, k, v, do, cu = make(lens, 3, 2, 1, 64, "bf16")
    o, lse, dq, dk, dv = run(q, k, v, do, cu)
    dense = [i for i, n in enumerate(lens) if n]
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    for i in dense[:3] + [17, 4999]:
        a, n = starts[i], lens[i]
        sl = slice(a, a + n)
        ro, _, grads = reference(q[sl], k[sl], v[sl], [n], do[sl])
        assert rel(o[sl], ro) <= 2 * 2.0 ** -8
        for got, (want, slack) in zip((dq, dk, dv), grads):
            assert float((got[sl].double() - want).norm()) <= 4 * 2.0 ** -8 * float(want.norm()) + slack


def test_another_stream():
    from evograd_b200 import ops

    q, k, v, do, cu = make([500, 300], 0, 4, 2, 128, "bf16")
    want = run(q, k, v, do, cu)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(a):
        one = run(q, k, v, do, cu)
    with torch.cuda.stream(b):
        two = run(q, k, v, do, cu)
    torch.cuda.synchronize()
    same(one, want)
    same(two, want)
    ops.device_status()


def test_two_streams_at_once():
    """Calls that overlap share SMs, tensor memory and nothing else."""
    sets = [make([700, 64, 300], 9, 4, 2, 128, "bf16"), make([513, 1, 90], 0, 6, 3, 64, "fp16", seed=7)]
    want = [run(*t) for t in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(run(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            same(r, want[i])


def test_tensors_of_more_than_two_to_the_31_elements():
    """135168 tokens x 128 heads x 128: offsets beyond 32 bits in q, o, do, dq and in the
    float32 copy of dq. The last sequences are compared with the same rows alone."""
    from evograd_b200 import ops

    T, hq, d = 135168, 128, 128
    assert T * hq * d > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(0)
    q, do = (torch.empty(T, hq, d, device="cuda", dtype=torch.bfloat16).normal_(generator=g) for _ in range(2))
    k, v = (torch.empty(T, 1, d, device="cuda", dtype=torch.bfloat16).normal_(generator=g) for _ in range(2))
    cu = torch.arange(0, T + 1, 128, device="cuda", dtype=torch.int32)
    cu = torch.cat([cu[:-2], cu[-1:]])  # the last sequence has 256 tokens
    got = run(q, k, v, do, cu)
    tail = slice(T - 640, T)
    small = torch.tensor([0, 128, 256, 384, 640], device="cuda", dtype=torch.int32)
    want = run(q[tail], k[tail], v[tail], do[tail], small)
    same([t[:, tail] if i == 1 else t[tail] for i, t in enumerate(got)], want)
    ops.device_status()


def test_empty_and_refusals():
    from evograd_b200 import ops

    q, k, v, do, cu = make([30], 2, 4, 2, 64, "bf16")
    plan = ops.packed_plan(cu, 32)
    o, lse = ops.packed_attention_fwd(q, k, v, plan)
    none = ops.packed_plan(torch.zeros(1, device="cuda", dtype=torch.int32), 0)
    none.check()
    eo, el = ops.packed_attention_fwd(q[:0], k[:0], v[:0], none)
    assert eo.shape == (0, 4, 64) and el.shape == (4, 0)
    grads = ops.packed_attention_bwd(do[:0], q[:0], k[:0], v[:0], eo, el, none)
    assert [tuple(t.shape) for t in grads] == [(0, 4, 64), (0, 2, 64), (0, 2, 64)]
    nobody = ops.packed_plan(torch.zeros(1, device="cuda", dtype=torch.int32), 32)
    assert not ops.packed_attention_fwd(q, k, v, nobody)[0].any()
    f, b = ops.packed_attention_fwd, ops.packed_attention_bwd
    for bad in (lambda: f(q[0], k, v, plan), lambda: f(q, k, v[:, :1], plan), lambda: f(q, k, v.half(), plan),
                lambda: f(q[:, :3], k, v, plan), lambda: f(q[:31], k[:31], v[:31], plan),
                lambda: f(q, k[..., :32], v[..., :32], plan), lambda: f(q, k, v, plan, out=o[:, :2]),
                lambda: f(q, k, v, plan, out=o[:, :1].expand(32, 4, 64)),
                lambda: b(do[:, :2], q, k, v, o, lse, plan), lambda: b(do, q, k, v, o.float(), lse, plan),
                lambda: b(do, q, k, v, o, lse.double(), plan), lambda: b(do, q, k, v, o, lse[:2], plan),
                lambda: b(do, q, k, v, o, lse, plan, outs=(q, k)),
                lambda: b(do, q, k, v, o, lse, plan, outs=(q, k, v.float())),
                lambda: ops.packed_plan(cu[None], 32), lambda: ops.packed_plan(cu[:0], 32),
                lambda: ops.packed_plan(cu, -1), lambda: ops.packed_plan(cu, (1 << 27) + 1)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: f(q, k, v, cu), lambda: ops.packed_plan(cu.float(), 32),
                lambda: f(q.double(), k.double(), v.double(), plan)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: f(q, k, v, plan, scale=0.0), lambda: f(q, k, v, plan, scale=float("nan")),
                lambda: b(do, q, k, v, o, lse, plan, scale=-1.0)):
        with pytest.raises(ops.EvgError):
            bad()
    big = torch.zeros(32, 1, 300, device="cuda")
    with pytest.raises(ops.EvgError):
        f(big, big, big, plan)
