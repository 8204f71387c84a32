"""What is measured of the operators of a training step over packed sequences:
causal grouped-query attention over documents of different lengths, rotary
positions from position numbers, the norms after and before a block with its gate
and residual scale, and global gradient-norm clipping.

``own`` chooses the side: False computes the operators in elementary torch
operations (float32, float64 for rotary angles and the sum of squares, one
rounding at the end), True calls ``evograd_b200.ops``. ``exact`` states the
definitions once more in float64.
"""

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------- cases
def listed():
    return [
        # one short chat turn plus a few fragments: the call whose latency counts
        dict(name="attn_fwd_fragments", op="attn", train=False, dtype="bf16", hq=8, hkv=2, d=64,
             lens="64,1,100,0,37", pad=6),
        # a packed row of supervised fine-tuning: many answers of a few hundred tokens
        dict(name="attn_step_answers", op="attn", train=True, dtype="bf16", hq=32, hkv=8, d=128,
             lens="129,700,31,512,255,900,64,333,418,128,77,611,1,480,250,207", pad=0),
        # the same step with plain multi-head attention in fp16 at the smaller head size
        dict(name="attn_step_mha64", op="attn", train=True, dtype="fp16", hq=16, hkv=16, d=64,
             lens="1000,2048,300,748", pad=0),
        # evaluation of a long prompt packed with short ones, forward only
        dict(name="attn_fwd_long", op="attn", train=False, dtype="bf16", hq=32, hkv=8, d=128,
             lens="12001,2500,1000,883", pad=0),
        # pre-training on long documents, the decoder layer's 32/8 heads of 128
        dict(name="attn_step_documents", op="attn", train=True, dtype="bf16", hq=32, hkv=8, d=128,
             lens="8192,4100,2500,1592", pad=0),
        # the newest tokens of three running requests, a quarter of the head rotated in
        # interleaved pairs, with an attention factor: the call whose latency counts
        dict(name="rope_tokens", op="rope", train=False, dtype="fp16", tokens=3, hq=24, hkv=6, d=80, rd=20,
             interleaved=True, mscale=1.2, base=10000.0, far=131071),
        # a packed training row, whole head, half layout, context-scaled frequencies
        dict(name="rope_step_packed", op="rope", train=True, dtype="bf16", tokens=16384, hq=32, hkv=8,
             d=128, rd=128, interleaved=False, mscale=1.0, base=500000.0, far=131071),
        # one decoded token through the two norms around a block boundary
        dict(name="norms_token", op="norms", train=False, dtype="bf16", rows=1, cols=4096,
             gate="channel", alpha=0.5),
        # a training step of the decoder layer's width, gate per channel
        dict(name="norms_step", op="norms", train=True, dtype="bf16", rows=16384, cols=4096,
             gate="channel", alpha=0.5),
        # an odd number of rows, float32 stream, data-dependent gate of full width
        dict(name="norms_step_fullgate", op="norms", train=True, dtype="fp32", rows=2047, cols=1536,
             gate="full", alpha=1.0),
        # gradients of a small model's layers in three types, most of them short
        dict(name="clip_small", op="clip", dtype="mixed", hidden=257, kv=64, mlp=700, layers=5,
             max_norm=1.0),
        # every gradient of one decoder layer of width 4096 / 14336
        dict(name="clip_layer", op="clip", dtype="bf16", hidden=4096, kv=1024, mlp=14336, layers=1,
             max_norm=1.0),
    ]


def draw(rng):
    def logint(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["attn", "attn", "rope", "norms", "clip"])
    if op == "attn":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        if dtype == "fp32":  # small correctness shapes
            tokens, hkv, group, d = logint(1, 256), rng.choice([1, 2]), rng.choice([1, 2]), rng.choice([16, 64])
        else:
            tokens, hkv = logint(1, 16384), rng.choice([1, 2, 4, 8])
            group, d = rng.choice([1, 2, 3, 4]), rng.choice([64, 80, 128, 128])
        n = logint(1, min(tokens, 64))
        cuts = sorted(rng.randint(0, tokens) for _ in range(n - 1))
        lens = [b - a for a, b in zip([0] + cuts, cuts + [tokens])]
        return dict(op="attn", train=rng.random() < 0.6, dtype=dtype, hq=hkv * group, hkv=hkv, d=d,
                    lens=",".join(map(str, lens)), pad=rng.choice([0, 0, rng.randint(1, 200)]))
    if op == "rope":
        d = rng.choice([64, 80, 96, 128, 256])
        hkv = rng.choice([1, 2, 4, 8])
        rd = rng.choice([d, d, 2 * rng.randint(1, d // 2)])
        return dict(op="rope", train=rng.random() < 0.6, dtype=rng.choice(["bf16", "fp16", "fp32"]),
                    tokens=logint(1, 8192), hq=hkv * rng.choice([1, 2, 4]), hkv=hkv, d=d, rd=rd,
                    interleaved=rng.random() < 0.5, mscale=rng.choice([1.0, 1.0, 0.9, 1.3]),
                    base=rng.choice([10000.0, 500000.0, 1000000.0]), far=logint(1, 1000000))
    if op == "norms":
        cols = rng.choice([logint(16, 8192), 8 * logint(2, 1024), 1024 * rng.choice([1, 2, 4, 5, 8])])
        return dict(op="norms", train=rng.random() < 0.6, dtype=rng.choice(["bf16", "fp16", "fp32"]),
                    rows=logint(1, 8192), cols=cols, gate=rng.choice(["none", "channel", "token", "full"]),
                    alpha=rng.choice([1.0, 0.5, 0.22]))
    hidden = rng.choice([logint(16, 2048), 64 * rng.randint(1, 32)])
    return dict(op="clip", dtype=rng.choice(["bf16", "fp16", "fp32", "mixed"]), hidden=hidden,
                kv=max(1, hidden // 4), mlp=logint(16, 6000), layers=rng.randint(1, 6),
                max_norm=rng.choice([0.1, 1.0, 1.0e6]))


# ------------------------------------------------------------------------ inputs
def _lens(case):
    return [int(x) for x in case["lens"].split(",")]


def _grad_shapes(case):
    """The nine parameters of a decoder layer."""
    hid, kv, mlp = case["hidden"], case["kv"], case["mlp"]
    return [(hid,), (hid, hid), (kv, hid), (kv, hid), (hid, hid), (hid,), (mlp, hid), (mlp, hid), (hid, mlp)]


def _grad_dtype(case, k):
    return [torch.bfloat16, torch.float32, torch.float16][k % 3] if case["dtype"] == "mixed" else _DT[case["dtype"]]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def randn(*shape, dtype=None, std=1.0):
        x = torch.randn(*shape, device="cuda", generator=g, dtype=torch.float32)
        return x.mul_(std).to(dtype or _DT[case["dtype"]])

    s = dict(case=dict(case))
    if case["op"] == "attn":
        lens = _lens(case)
        T = sum(lens) + case["pad"]
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        s["cu"] = torch.tensor(cu, device="cuda", dtype=torch.int32)
        s["q"] = randn(T, case["hq"], case["d"])
        s["k"] = randn(T, case["hkv"], case["d"])
        s["v"] = randn(T, case["hkv"], case["d"])
        if case["train"]:
            s["do"] = randn(T, case["hq"], case["d"])
    elif case["op"] == "rope":
        T = case["tokens"]
        s["q"], s["k"] = randn(T, case["hq"], case["d"]), randn(T, case["hkv"], case["d"])
        if case["train"]:
            s["dq"], s["dk"] = randn(T, case["hq"], case["d"]), randn(T, case["hkv"], case["d"])
        # documents at any place of the context: positions up to `far`
        s["pos"] = torch.randint(0, case["far"] + 1, (T,), device="cuda", generator=g, dtype=torch.int32)
        i = torch.arange(0, case["rd"], 2, device="cuda", dtype=torch.float64)
        f = case["base"] ** (-i / case["rd"])
        # context scaling: slow components by 1/8, fast ones kept, a ramp between them
        wave = 8192.0 * f / (2 * math.pi)
        keep = ((wave - 1.0) / 3.0).clamp(0.0, 1.0)
        s["inv_freq"] = f * (keep + (1.0 - keep) / 8.0)
    elif case["op"] == "norms":
        R, C = case["rows"], case["cols"]
        s["x"], s["h"] = randn(R, C, std=0.7), randn(R, C, std=2.0)
        s["w_post"] = (1.0 + 0.1 * randn(C, dtype=torch.float32)).to(_DT[case["dtype"]])
        s["w_pre"] = (1.0 + 0.1 * randn(C, dtype=torch.float32)).to(_DT[case["dtype"]])
        shape = {"none": None, "channel": (C,), "token": (R, 1), "full": (R, C)}[case["gate"]]
        s["gate"] = None if shape is None else torch.sigmoid(randn(*shape, dtype=torch.float32)).to(_DT[case["dtype"]])
        if case["train"]:
            s["dy"], s["dh"] = randn(R, C), randn(R, C)
    else:
        grads = []
        for _ in range(case["layers"]):
            for k, shape in enumerate(_grad_shapes(case)):
                grads.append(randn(*shape, dtype=_grad_dtype(case, k), std=10.0 ** -(k % 3)))
        s["grads"] = grads
        s["outs"] = [torch.empty_like(x) for x in grads]
    return s


# ------------------------------------------------------------------- plain forms
def _visible(cu, T):
    """[T, T] truth: key j is in query i's sequence and not behind it; rows behind
    the last sequence see nothing."""
    t = torch.arange(T, device=cu.device)
    seq = torch.searchsorted(cu[1:].contiguous(), t.to(torch.int32), right=True)
    return (seq[:, None] == seq[None, :]) & (t[None, :] <= t[:, None]) & (t[:, None] < cu[-1])


def _plain_attention(s):
    q, k, v, cu = s["q"], s["k"], s["v"], s["cu"]
    T, hq, d = q.shape
    hkv = k.shape[1]
    group = hq // hkv
    scale = 1.0 / math.sqrt(d)
    seen = _visible(cu, T)
    train = s["case"]["train"]
    o = torch.empty_like(q)
    lse = torch.empty(hq, T, device=q.device, dtype=torch.float32)
    dq, dk, dv = (torch.empty_like(x) for x in (q, k, v))
    at_once = max(1, (1 << 30) // (group * T * T))  # k/v heads whose scores fit the memory
    for h0 in range(0, hkv, at_once):
        h1 = min(hkv, h0 + at_once)
        a, b = h0 * group, h1 * group
        qf = q[:, a:b].float().view(T, h1 - h0, group, d).permute(1, 2, 0, 3)
        kf = k[:, h0:h1].float().permute(1, 0, 2)[:, None]
        vf = v[:, h0:h1].float().permute(1, 0, 2)[:, None]
        sc = torch.matmul(qf, kf.transpose(-1, -2)).mul_(scale).masked_fill_(~seen, float("-inf"))
        m = sc.amax(-1, keepdim=True)
        m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
        p = sc.sub_(m).exp_()
        l = p.sum(-1, keepdim=True)
        lse[a:b] = (m + l.log()).reshape(b - a, T)
        p = p.div_(l.clamp_min(1e-30))
        of = torch.matmul(p, vf)
        o[:, a:b] = of.permute(2, 0, 1, 3).reshape(T, b - a, d).to(o.dtype)
        if train:
            gf = s["do"][:, a:b].float().view(T, h1 - h0, group, d).permute(1, 2, 0, 3)
            dv[:, h0:h1] = torch.matmul(p.transpose(-1, -2), gf).sum(1).permute(1, 0, 2).to(dv.dtype)
            ds = torch.matmul(gf, vf.transpose(-1, -2)).sub_((gf * of).sum(-1, keepdim=True)).mul_(p)
            dq[:, a:b] = torch.matmul(ds, kf).mul_(scale).permute(2, 0, 1, 3).reshape(T, b - a, d).to(dq.dtype)
            dk[:, h0:h1] = torch.matmul(ds.transpose(-1, -2), qf).sum(1).mul_(scale).permute(1, 0, 2).to(dk.dtype)
    return dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv) if train else dict(o=o, lse=lse)


def _plain_rotate(x, cos, sin, rd, interleaved):
    xf = x[..., :rd].float()
    if interleaved:
        x1, x2 = xf[..., 0::2], xf[..., 1::2]
    else:
        x1, x2 = xf[..., : rd // 2], xf[..., rd // 2:]
    y1, y2 = x1 * cos - x2 * sin, x2 * cos + x1 * sin
    y = torch.stack([y1, y2], -1).flatten(-2) if interleaved else torch.cat([y1, y2], -1)
    return torch.cat([y.to(x.dtype), x[..., rd:]], -1)


def _plain_rope(s):
    c = s["case"]
    angle = s["pos"].double()[:, None, None] * s["inv_freq"]
    cos, sin = (angle.cos() * c["mscale"]).float(), (angle.sin() * c["mscale"]).float()
    out = dict(q=_plain_rotate(s["q"], cos, sin, c["rd"], c["interleaved"]),
               k=_plain_rotate(s["k"], cos, sin, c["rd"], c["interleaved"]))
    if c["train"]:
        out["dq"] = _plain_rotate(s["dq"], cos, -sin, c["rd"], c["interleaved"])
        out["dk"] = _plain_rotate(s["dk"], cos, -sin, c["rd"], c["interleaved"])
    return out


_EPS = 1e-6


def _plain_norms(s):
    c, dt = s["case"], s["x"].dtype
    x, h, wp, wn = (s[n].float() for n in ("x", "h", "w_post", "w_pre"))
    gate = 1.0 if s["gate"] is None else s["gate"].float()
    r1 = torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS)
    xhat = x * r1
    n = xhat * wp
    h2 = h + c["alpha"] * gate * n
    r2 = torch.rsqrt(h2.square().mean(-1, keepdim=True) + _EPS)
    hhat = h2 * r2
    out = dict(h=h2.to(dt), y=(hhat * wn).to(dt))
    if c["train"]:
        dy, dh = s["dy"].float(), s["dh"].float()
        t = dy * wn
        G = dh + r2 * (t - hhat * (t * hhat).mean(-1, keepdim=True))
        dn = c["alpha"] * gate * G
        t = dn * wp
        out["dx"] = (r1 * (t - xhat * (t * xhat).mean(-1, keepdim=True))).to(dt)
        out["dh"] = G.to(dt)
        out["dw_post"] = (dn * xhat).sum(0).to(dt)
        out["dw_pre"] = (dy * hhat).sum(0).to(dt)
        dg = c["alpha"] * G * n
        if c["gate"] == "channel":
            out["dgate"] = dg.sum(0).to(dt)
        elif c["gate"] == "token":
            out["dgate"] = dg.sum(1, keepdim=True).to(dt)
        elif c["gate"] == "full":
            out["dgate"] = dg.to(dt)
    return out


def _plain_clip(s):
    grads = s["grads"]
    norm = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()
    coef = (s["case"]["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    return dict(norm=norm.float(), outs=[(g.float() * coef).to(g.dtype) for g in grads])


# ----------------------------------------------------------- the framework's calls
def _own(s):
    from evograd_b200 import ops

    c = s["case"]
    if c["op"] == "attn":
        plan = ops.packed_plan(s["cu"], s["q"].shape[0])
        o, lse = ops.packed_attention_fwd(s["q"], s["k"], s["v"], plan)
        if not c["train"]:
            return dict(o=o, lse=lse)
        dq, dk, dv = ops.packed_attention_bwd(s["do"], s["q"], s["k"], s["v"], o, lse, plan)
        return dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv)
    if c["op"] == "rope":
        kw = dict(interleaved=c["interleaved"], mscale=c["mscale"])
        q, k = ops.rope_positions_fwd(s["q"], s["k"], s["pos"], s["inv_freq"], **kw)
        if not c["train"]:
            return dict(q=q, k=k)
        dq, dk = ops.rope_positions_bwd(s["dq"], s["dk"], s["pos"], s["inv_freq"], **kw)
        return dict(q=q, k=k, dq=dq, dk=dk)
    if c["op"] == "norms":
        h, y, r_post, r_pre = ops.post_pre_norm_fwd(s["x"], s["h"], s["w_post"], s["w_pre"], s["gate"],
                                                    alpha=c["alpha"], eps=_EPS)
        if not c["train"]:
            return dict(h=h, y=y)
        dx, dh, dw_post, dw_pre, dgate = ops.post_pre_norm_bwd(
            s["dy"], s["dh"], s["x"], h, s["w_post"], s["w_pre"], s["gate"], r_post, r_pre,
            alpha=c["alpha"])
        out = dict(h=h, y=y, dx=dx, dh=dh, dw_post=dw_post, dw_pre=dw_pre)
        return out if dgate is None else dict(out, dgate=dgate)
    norm = ops.clip_grad_norm(s["grads"], c["max_norm"], outs=s["outs"])
    return dict(norm=norm, outs=s["outs"])


def run(state):
    if own:
        return _own(state)
    return {"attn": _plain_attention, "rope": _plain_rope, "norms": _plain_norms,
            "clip": _plain_clip}[state["case"]["op"]](state)


# -------------------------------------------------------------------------- work
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2  # clip counts its own
    if case["op"] == "attn":
        lens = _lens(case)
        T = sum(lens) + case["pad"]
        pairs = sum(n * (n + 1) // 2 for n in lens)
        q, kv = T * case["hq"] * case["d"] * e, T * case["hkv"] * case["d"] * e
        moved = 2 * q + 2 * kv + 4 * T * case["hq"]
        flops = 4 * pairs * case["d"] * case["hq"]
        if case["train"]:
            moved += 2 * q + 2 * kv
            flops += 10 * pairs * case["d"] * case["hq"]
        return dict(bytes=moved, flops=flops)
    if case["op"] == "rope":
        n = case["tokens"] * (case["hq"] + case["hkv"]) * case["d"] * (2 if case["train"] else 1)
        return dict(bytes=2 * n * e + 4 * case["tokens"] + 4 * case["rd"], flops=3 * n)
    if case["op"] == "norms":
        n = case["rows"] * case["cols"]
        full = n if case["gate"] == "full" else 0
        if not case["train"]:
            return dict(bytes=(4 * n + full) * e, flops=10 * n)
        return dict(bytes=(4 * n + full + 4 * n + full) * e, flops=40 * n)
    sizes = [math.prod(shape) for shape in _grad_shapes(case)] * case["layers"]
    widths = [_grad_dtype(case, k).itemsize for k in range(9)] * case["layers"]
    return dict(bytes=2 * sum(n * w for n, w in zip(sizes, widths)), flops=3 * sum(sizes))


# ------------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attn":
        return _exact_attention(case, s)
    if case["op"] == "rope":
        return _exact_rope(case, s)
    if case["op"] == "norms":
        leaves = {n: s[n].double().requires_grad_() for n in ("x", "h", "w_post", "w_pre")}
        gate = None if s["gate"] is None else s["gate"].double().requires_grad_()
        x, h = leaves["x"], leaves["h"]
        n = x / (x.pow(2).mean(1, keepdim=True) + _EPS).sqrt() * leaves["w_post"]
        h2 = h + case["alpha"] * (n if gate is None else n * gate)
        y = h2 / (h2.pow(2).mean(1, keepdim=True) + _EPS).sqrt() * leaves["w_pre"]
        out = dict(h=h2.detach(), y=y.detach())
        if case["train"]:
            wanted = [leaves["x"], leaves["h"], leaves["w_post"], leaves["w_pre"]] + ([] if gate is None else [gate])
            got = torch.autograd.grad([y, h2], wanted, [s["dy"].double(), s["dh"].double()])
            out.update(zip(["dx", "dh", "dw_post", "dw_pre", "dgate"], got))
        return out
    total = math.sqrt(math.fsum(float((g.double() ** 2).sum()) for g in s["grads"]))
    coef = min(1.0, case["max_norm"] / (total + 1e-6))
    return dict(norm=torch.tensor(total, dtype=torch.float64), outs=[g.double() * coef for g in s["grads"]])


def _exact_attention(case, s):
    """Sequence by sequence and k/v head by k/v head, gradients by autograd."""
    T, hq, d = s["q"].shape
    group = hq // case["hkv"]
    new = lambda t: torch.zeros(t.shape, device="cuda", dtype=torch.float64)  # noqa: E731
    out = dict(o=new(s["q"]), lse=torch.full((hq, T), float("-inf"), device="cuda", dtype=torch.float64))
    if case["train"]:
        out.update(dq=new(s["q"]), dk=new(s["k"]), dv=new(s["v"]))
    start = 0
    for n in _lens(case):
        sl = slice(start, start + n)
        start += n
        if n == 0:
            continue
        hidden = torch.ones(n, n, device="cuda", dtype=torch.bool).triu(1)
        for h in range(case["hkv"]):
            hs = slice(h * group, (h + 1) * group)
            q = s["q"][sl, hs].double().transpose(0, 1).requires_grad_()
            k = s["k"][sl, h].double().requires_grad_()
            v = s["v"][sl, h].double().requires_grad_()
            with torch.set_grad_enabled(bool(case["train"])):
                logits = (q @ k.T / math.sqrt(d)).masked_fill(hidden, float("-inf"))
                o = torch.softmax(logits, -1) @ v
            out["o"][sl, hs] = o.detach().transpose(0, 1)
            out["lse"][hs, sl] = torch.logsumexp(logits.detach(), -1)
            if case["train"]:
                dq, dk, dv = torch.autograd.grad(o, [q, k, v], s["do"][sl, hs].double().transpose(0, 1))
                out["dq"][sl, hs] = dq.transpose(0, 1)
                out["dk"][sl, h] = dk
                out["dv"][sl, h] = dv
    return out


def _exact_rope(case, s):
    """As complex numbers: y = m x exp(i pos f), the gradient with the conjugate."""
    rd = case["rd"]
    turn = torch.polar(torch.full_like(s["inv_freq"], case["mscale"]).expand(case["tokens"], 1, -1),
                       s["pos"].double()[:, None, None] * s["inv_freq"])

    def rotate(x, w):
        x = x.double()
        lo = x[..., :rd]
        z = torch.view_as_complex(lo.unflatten(-1, (rd // 2, 2)).contiguous()) if case["interleaved"] \
            else torch.complex(lo[..., : rd // 2], lo[..., rd // 2:])
        z = z * w
        lo = torch.view_as_real(z).flatten(-2) if case["interleaved"] else torch.cat([z.real, z.imag], -1)
        return torch.cat([lo, x[..., rd:]], -1)

    out = dict(q=rotate(s["q"], turn), k=rotate(s["k"], turn))
    if case["train"]:
        out.update(dq=rotate(s["dq"], turn.conj()), dk=rotate(s["dk"], turn.conj()))
    return out
