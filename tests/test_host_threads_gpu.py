"""Calls from two host threads at once, each on its own stream, of one kernel in two sizes:
the shared memory a launch may ask for belongs to the kernel and the device, not to the
call."""

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def together(calls, rounds):
    """Every call in its own thread and stream, `rounds` times; the last results."""
    results, errors = [None] * len(calls), []
    start = threading.Barrier(len(calls))

    def work(i):
        try:
            stream = torch.cuda.Stream()
            stream.wait_stream(torch.cuda.default_stream())
            with torch.cuda.stream(stream):
                start.wait()
                for _ in range(rounds):
                    results[i] = calls[i]()
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]
    return results


@pytest.mark.parametrize("widths", [(4096, 8192), (2560, 6144)])
def test_norms_of_two_widths(widths):
    from evograd_b200 import ops

    def call(C):
        g = torch.Generator(device="cuda").manual_seed(C)
        x, h, dy, dh = (torch.randn(600, C, device="cuda", generator=g).bfloat16() for _ in range(4))
        w1, w2 = (torch.randn(C, device="cuda", generator=g).bfloat16() for _ in range(2))

        def run():
            hn, y, r1, r2 = ops.post_pre_norm_fwd(x, h, w1, w2)
            return [hn, y, *ops.post_pre_norm_bwd(dy, dh, x, hn, w1, w2, None, r1, r2)[:4]]
        return run

    calls = [call(C) for C in widths]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    for got, ref in zip(together(calls, 400), want):
        for a, b in zip(got, ref):
            assert torch.equal(a, b)


def test_packed_attention_of_two_head_sizes():
    from evograd_b200 import ops

    def call(d):
        g = torch.Generator(device="cuda").manual_seed(d)
        q, k, v, do = (torch.randn(40, 1, d, device="cuda", generator=g) for _ in range(4))
        cu = torch.tensor([0, 25, 40], device="cuda", dtype=torch.int32)

        def run():
            plan = ops.packed_plan(cu, 40)
            o, lse = ops.packed_attention_fwd(q, k, v, plan)
            return [o, lse, *ops.packed_attention_bwd(do, q, k, v, o, lse, plan)]
        return run

    calls = [call(180), call(256)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    for got, ref in zip(together(calls, 300), want):
        for a, b in zip(got, ref):
            assert torch.equal(a, b)


@pytest.mark.parametrize("op,widths", [("layernorm", (4096, 8192)), ("rmsnorm", (4096, 6144)), ("fused_add", (2048, 4096)),
                                       ("softmax", (32768, 128256))])
def test_row_operators_of_two_widths(op, widths):
    from evograd_b200 import ops

    def call(C):
        g = torch.Generator(device="cuda").manual_seed(C)
        x, r, dy = (torch.randn(300, C, device="cuda", generator=g).bfloat16() for _ in range(3))
        w, b = (torch.randn(C, device="cuda", generator=g).bfloat16() for _ in range(2))

        def run():
            if op == "layernorm":
                y, mean, rstd = ops.layernorm_fwd(x, w, b)
                return [y, *ops.layernorm_bwd(dy, x, w, mean, rstd)]
            if op == "rmsnorm":
                y, rstd = ops.rmsnorm_fwd(x, w)
                return [y, *ops.rmsnorm_bwd(dy, x, w, rstd)]
            if op == "fused_add":
                y, rstd = ops.fused_add_rmsnorm_fwd(x, r, w)
                out = ops.fused_add_rmsnorm_bwd(dy, x, r, w, rstd)
                return [y, *out]
            y = ops.softmax_fwd(x)
            return [y, ops.softmax_bwd(y, dy)]
        return run

    calls = [call(C) for C in widths]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    for got, ref in zip(together(calls, 100), want):
        for a, b in zip(got, ref):
            assert torch.equal(a, b)
