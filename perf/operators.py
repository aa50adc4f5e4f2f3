"""Workloads of the temporal operators: a selective scan with its causal convolution, a paged key-value cache of a
stream's tokens, and the attention that reads it.

A stream's frame is a set of tokens (the 17 x 30 = 510 positions of an HD frame at 1/16 scale, or one pooled token) and
every operator takes either one step of each stream or a chunk of steps.  With ``own`` false ``run`` is the operator in
elementary torch operations, with ``own`` true it is the call a user makes of ``robustvideomatting_amd.temporal``.
"""
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


# ---- cases ------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one frame of 8 streams, pooled tokens of the encoder's 960 channels: latency only
        dict(name="conv frame", op="conv", B=8, T=1, D=960, W=4, bias=True, state=True, dtype="fp16"),
        # 16 HD frames (510 tokens each) of 2 streams scanned token by token
        dict(name="conv clip", op="conv", B=2, T=8160, D=960, W=4, bias=True, state=True, dtype="bf16"),
        # one frame of 64 streams, pooled tokens
        dict(name="scan frame", op="scan", B=64, T=1, D=960, N=16, z=True, state=True, dtype="fp16"),
        # a chunk of 12 frames of 8 streams, every position of the 1/16 map a sequence of its own (where the ConvGRU stands)
        dict(name="scan positions", op="scan", B=4080, T=12, D=64, N=16, z=False, state=True, dtype="bf16"),
        # 16 HD frames of one stream scanned token by token: the parallelism has to come out of the time axis
        dict(name="scan clip", op="scan", B=1, T=8160, D=960, N=16, z=True, state=False, dtype="bf16"),
        # odd sizes in fp32
        dict(name="scan odd fp32", op="scan", B=3, T=1021, D=333, N=13, z=True, state=True, dtype="fp32"),
        # one pooled token of 64 streams after up to 300 frames
        dict(name="append frame", op="append", S=64, lo=0, hi=299, new_lo=1, new_hi=1, Hq=16, Hkv=4, Dh=128, page=16,
             interleaved=False, mix=1, dtype="fp16"),
        # chunks of very different lengths, streams that are thousands of tokens in
        dict(name="append clips", op="append", S=9, lo=0, hi=60000, new_lo=1, new_hi=8160, Hq=16, Hkv=8, Dh=128, page=64,
             interleaved=False, mix=2, dtype="bf16"),
        # one pooled token of 8 streams after up to 300 frames: latency
        dict(name="attend frame", op="attend", S=8, lo=20, hi=299, new_lo=1, new_hi=1, Hq=8, Hkv=2, Dh=64, page=16, mix=3,
             dtype="fp16"),
        # one token of 8 streams over long memories (128 HD frames of tokens)
        dict(name="attend long memory", op="attend", S=8, lo=8000, hi=65280, new_lo=1, new_hi=1, Hq=32, Hkv=8, Dh=128,
             page=64, mix=4, dtype="bf16"),
        # whole clips of different lengths, nothing in the cache before them
        dict(name="attend clips", op="attend", S=5, lo=0, hi=0, new_lo=100, new_hi=8160, Hq=16, Hkv=4, Dh=128, page=64,
             mix=6, dtype="bf16"),
        # one HD frame of tokens for each of 4 streams, on top of what they remember, in fp32
        dict(name="attend next frame fp32", op="attend", S=4, lo=500, hi=4080, new_lo=510, new_hi=510, Hq=8, Hkv=2, Dh=64,
             page=32, mix=7, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv", "scan", "append", "attend one", "attend chunk"])
    dtype = rng.choice(["fp16", "bf16", "bf16", "fp32"])
    if op == "conv":
        while True:
            c = dict(op=op, B=_log(rng, 1, 2048), T=_log(rng, 1, 8160), D=_log(rng, 16, 1500), W=rng.randint(2, 4),
                     bias=rng.random() < 0.7, state=rng.random() < 0.7, dtype=dtype)
            if c["B"] * c["T"] * c["D"] <= 15_000_000:
                return c
    if op == "scan":
        while True:
            c = dict(op=op, B=_log(rng, 1, 4080), T=_log(rng, 1, 8160), D=_log(rng, 16, 1500), N=rng.choice([4, 8, 16, 16, 24, 32, 64]),
                     z=rng.random() < 0.6, state=rng.random() < 0.7, dtype=dtype)
            if c["B"] * c["T"] * c["D"] * c["N"] <= 100_000_000 and c["B"] * c["D"] * c["N"] <= 8_000_000:
                return c
    while True:
        Hkv, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 5, 8])
        heads = dict(Hq=Hkv * group, Hkv=Hkv, Dh=rng.choice([32, 64, 64, 80, 96, 128, 128]), page=rng.choice([16, 32, 64, 128]),
                     mix=rng.randint(0, 1 << 20), dtype=dtype)
        if op == "append":
            one = rng.random() < 0.5
            new = 1 if one else _log(rng, 2, 4080)
            c = dict(op=op, S=_log(rng, 1, 256 if one else 8), lo=0, hi=_log(rng, 16, 8000), new_lo=int(one), new_hi=new,
                     interleaved=rng.random() < 0.4, **heads)
        elif op == "attend one":
            c = dict(op="attend", S=_log(rng, 1, 32), lo=0, hi=_log(rng, 16, 24000), new_lo=1, new_hi=1, **heads)
        else:
            c = dict(op="attend", S=_log(rng, 1, 6), lo=0, hi=rng.choice([0, _log(rng, 16, 3000)]), new_lo=0,
                     new_hi=_log(rng, 2, 2040), **heads)
        w = work(c)
        if w["bytes"] <= 3e8 and w["flops"] <= (2e10 if dtype == "fp32" else 2e11):
            return c


def _streams(case):
    """(tokens already remembered, new tokens) of every stream: fixed by the case, spread over its ranges, both ends hit."""
    rng = random.Random(case["mix"])
    S = case["S"]

    def spread(lo, hi):
        v = [rng.randint(lo, hi) if hi < 10 * max(lo, 1) else min(hi, max(lo, _log(rng, max(lo, 1), hi))) for _ in range(S)]
        v[rng.randrange(S)] = hi
        return v

    return spread(case["lo"], case["hi"]), spread(case["new_lo"], case["new_hi"])


# ---- inputs -----------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def rn(*shape, scale=1.0, dtype=dt):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    s = dict(case=case)
    if case["op"] == "conv":
        B, T, D, W = (case[k] for k in "BTDW")
        s["x"] = rn(B, T, 2 * D)[..., :D]               # the first half of an input projection, the second is the gate
        s["weight"] = rn(W, D, scale=W ** -0.5)
        s["bias"] = rn(D, scale=0.1) if case["bias"] else None
        s["state"] = rn(B, W - 1, D) if case["state"] else None
    elif case["op"] == "scan":
        B, T, D, N = (case[k] for k in "BTDN")
        s["x"] = rn(B, T, D)
        s["dt"] = rn(B, T, D, scale=0.5)
        # step sizes of 0.001 .. 0.1 (softplus of the bias), decay rates of 1 .. N as such models start from
        step = torch.exp(torch.rand(D, generator=g, device="cuda") * math.log(100.0) + math.log(1e-3))
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))
        s["A"] = -(torch.arange(1, N + 1, device="cuda", dtype=torch.float32)[:, None]
                   * torch.exp(0.1 * torch.randn((N, D), generator=g, device="cuda")))
        bc = rn(B, T, 2 * N)                            # both are slices of one projection
        s["B"], s["C"] = bc[..., :N], bc[..., N:]
        s["D"] = rn(D, dtype=torch.float32)
        s["z"] = rn(B, T, 2 * D)[..., D:] if case["z"] else None
        s["state"] = rn(B, N, D, scale=0.5, dtype=torch.float32) if case["state"] else None
    else:
        S, Hq, Hkv, Dh, page = (case[k] for k in ("S", "Hq", "Hkv", "Dh", "page"))
        past, new = _streams(case)
        one = case["new_hi"] == 1 and case["new_lo"] == 1
        M = sum(new)
        width = max(-(-(p + n) // page) for p, n in zip(past, new)) + 1
        used = [-(-(p + n) // page) for p, n in zip(past, new)]
        pool = sum(used) + 3
        order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
        table = torch.zeros((S, width), dtype=torch.int32, device="cuda")
        at = 0
        for i, u in enumerate(used):
            table[i, :u] = order[at:at + u]
            at += u
        s["table"] = table
        s["lengths"] = torch.tensor(past, dtype=torch.int32, device="cuda")
        off = [0]
        for n in new:
            off.append(off[-1] + n)
        s["offsets"] = None if one else torch.tensor(off, dtype=torch.int32, device="cuda")
        s["cache"] = (rn(pool, Hkv, page, Dh), rn(pool, Hkv, page, Dh))
        if case["op"] == "append":
            qkv = rn(M, Hq + 2 * Hkv, Dh)               # one projection's output
            s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
            rot = Dh // 16 * 16
            s["freqs"] = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float32) / rot)
        else:
            s["q"] = rn(M, Hq, Dh)
    return s


# ---- the operators' plain forms ----------------------------------------------------------------------------------------
def _conv_plain(s):
    x, w = s["x"].float(), s["weight"].float()
    B, T, D = x.shape
    W = w.shape[0]
    head = s["state"].float() if s["state"] is not None else torch.zeros((B, W - 1, D), device=x.device)
    xx = torch.cat([head, x], 1)
    y = (xx.unfold(1, W, 1) * w.t()).sum(-1)
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = y / (1 + torch.exp(-y))
    return y.to(s["x"].dtype), xx[:, T:].to(s["x"].dtype)


def _scan_plain(s):
    x, A = s["x"].float(), s["A"]
    B, T, D = x.shape
    pre = s["dt"].float() + s["dt_bias"]
    delta = pre.clamp(min=0) + torch.log1p(torch.exp(-pre.abs()))
    a = torch.exp(delta[:, :, None, :] * A)                                             # [B,T,N,D]
    h = (delta * x)[:, :, None, :] * s["B"].float()[..., None]
    if s["state"] is not None:
        h[:, 0] += a[:, 0] * s["state"]
    reach = 1
    while reach < T:                    # h_t = a_t h_(t-1) + u_t composed over 1, 2, 4 ... steps
        h = torch.cat([h[:, :reach], h[:, reach:] + a[:, reach:] * h[:, :-reach]], 1)
        a = torch.cat([a[:, :reach], a[:, reach:] * a[:, :-reach]], 1)
        reach *= 2
    y = (h * s["C"].float()[..., None]).sum(2) + s["D"] * x
    if s["z"] is not None:
        z = s["z"].float()
        y = y * z / (1 + torch.exp(-z))
    return y.to(s["x"].dtype), h[:, -1].contiguous()


def _owners(s):
    """Stream and position of every new token."""
    M = s["q"].shape[0]
    row = torch.arange(M, device="cuda")
    if s["offsets"] is None:
        return row, s["lengths"].long(), row * 0
    off = s["offsets"].long()
    stream = torch.searchsorted(off[1:].contiguous(), row, right=True)
    return stream, s["lengths"].long()[stream] + row - off[stream], row - off[stream]


def _rotate(x, pos, freqs, interleaved):
    angle = pos.double()[:, None] * freqs.double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    n = freqs.numel()
    x = x.float()
    if interleaved:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        r = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :n], x[..., n:2 * n]
        r = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([r, x[..., 2 * n:]], -1)


def _append_plain(s):
    stream, pos, _ = _owners(s)
    kp, vp = s["cache"]
    page = kp.shape[2]
    at, slot = s["table"][stream, pos // page].long(), pos % page
    kp[at, :, slot] = _rotate(s["k"], pos, s["freqs"], s["case"]["interleaved"]).to(kp.dtype)
    vp[at, :, slot] = s["v"]
    return _rotate(s["q"], pos, s["freqs"], s["case"]["interleaved"]).to(s["q"].dtype), kp, vp


def _attend_plain(s):
    q, (kp, vp), table = s["q"], s["cache"], s["table"]
    M, Hq, Dh = q.shape
    S, Hkv = table.shape[0], kp.shape[1]
    stream, pos, row = _owners(s)
    T = s["case"]["new_hi"]
    keys = kp[table.long()].transpose(1, 2).reshape(S, Hkv, -1, Dh).float()
    vals = vp[table.long()].transpose(1, 2).reshape(S, Hkv, -1, Dh).float()
    qq = torch.zeros((S, T, Hq, Dh), device="cuda")
    qq[stream, row] = q.float()
    pp = torch.full((S, T), -1, dtype=torch.long, device="cuda")
    pp[stream, row] = pos
    qq = qq.transpose(1, 2).reshape(S, Hkv, -1, Dh)                                     # rows (head of the group, token)
    score = qq @ keys.transpose(2, 3) / math.sqrt(Dh)
    seen = torch.arange(keys.shape[2], device="cuda") <= pp.repeat(1, Hq // Hkv)[:, None, :, None]
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(score - top)
    out = (p @ vals) / p.sum(-1, keepdim=True).clamp(min=1e-38)
    return out.reshape(S, Hq, T, Dh)[stream, :, row].to(q.dtype)


def run(s):
    op = s["case"]["op"]
    if own:
        from robustvideomatting_amd import temporal
        if op == "conv":
            return temporal.causal_conv(s["x"], s["weight"], s["bias"], state=s["state"])
        if op == "scan":
            return temporal.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
                                           state=s["state"])
        if op == "append":
            q = temporal.append_kv(s["k"], s["v"], s["cache"], s["table"], s["lengths"], s["offsets"], freqs=s["freqs"],
                                   q=s["q"], interleaved=s["case"]["interleaved"])
            return q, s["cache"][0], s["cache"][1]
        return temporal.attend(s["q"], s["cache"], s["table"], s["lengths"], s["offsets"])
    if op == "conv":
        return _conv_plain(s)
    if op == "scan":
        return _scan_plain(s)
    if op == "append":
        return _append_plain(s)
    return _attend_plain(s)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "conv":
        B, T, D, W = (case[k] for k in "BTDW")
        state = B * (W - 1) * D * e * (2 if case["state"] else 1)
        return {"bytes": 2 * B * T * D * e + W * D * e + state, "flops": B * T * D * (2 * W + 4)}
    if case["op"] == "scan":
        B, T, D, N = (case[k] for k in "BTDN")
        state = B * N * D * 4 * (2 if case["state"] else 1)
        return {"bytes": B * T * D * e * (4 if case["z"] else 3) + 2 * B * T * N * e + N * D * 4 + state,
                "flops": B * T * D * (7 * N + 8)}
    past, new = _streams(case)
    Hq, Hkv, Dh = case["Hq"], case["Hkv"], case["Dh"]
    M = sum(new)
    if case["op"] == "append":
        return {"bytes": M * (2 * Hq + 4 * Hkv) * Dh * e, "flops": M * (Hq + Hkv) * Dh * 3}
    pairs = sum(n * p + n * (n + 1) // 2 for p, n in zip(past, new))
    return {"bytes": 2 * M * Hq * Dh * e + 2 * sum(p + n for p, n in zip(past, new) if n) * Hkv * Dh * e,
            "flops": 4 * Dh * Hq * pairs}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() for k, v in s.items() if torch.is_tensor(v) and v.is_floating_point()}
    if case["op"] == "conv":
        B, T, D, W = (case[k] for k in "BTDW")
        if B * T * D > 60_000_000:
            return None
        line = torch.zeros((B, T + W - 1, D), dtype=torch.float64, device="cuda")
        line[:, W - 1:] = d["x"]
        if case["state"]:
            line[:, :W - 1] = d["state"]
        y = torch.zeros((B, T, D), dtype=torch.float64, device="cuda")
        for w in range(W):
            y += d["weight"][w] * line[:, w:w + T]
        if case["bias"]:
            y += d["bias"]
        return y * torch.sigmoid(y), line[:, T:]
    if case["op"] == "scan":
        B, T, D, N = (case[k] for k in "BTDN")
        h = d["state"] if case["state"] else torch.zeros((B, N, D), dtype=torch.float64, device="cuda")
        delta = torch.logaddexp(d["dt"] + d["dt_bias"], torch.zeros((), dtype=torch.float64, device="cuda"))
        y = torch.empty((B, T, D), dtype=torch.float64, device="cuda")
        for t in range(T):
            step = delta[:, t]
            h = (step[:, None] * d["A"]).exp() * h + (step * d["x"][:, t])[:, None] * d["B"][:, t, :, None]
            y[:, t] = torch.einsum("bnd,bn->bd", h, d["C"][:, t]) + d["D"] * d["x"][:, t]
        if case["z"]:
            y = y * d["z"] * torch.sigmoid(d["z"])
        return y, h
    past, new = _streams(case)
    page, Hq, Hkv, Dh = case["page"], case["Hq"], case["Hkv"], case["Dh"]
    keys, vals = (c.double() for c in s["cache"])
    group, row, out = Hq // Hkv, 0, []
    for i, (p, n) in enumerate(zip(past, new)):
        pages = s["table"][i].tolist()
        if case["op"] == "append":
            pos = torch.arange(p, p + n, device="cuda")
            turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), pos[:, None] * d["freqs"])[:, None]

            def turned(v):
                r = 2 * turn.shape[-1]
                w = v.clone()
                if case["interleaved"]:
                    w[..., :r] = torch.view_as_real(torch.complex(v[..., 0:r:2], v[..., 1:r:2]) * turn).flatten(-2)
                else:
                    c = torch.complex(v[..., :r // 2], v[..., r // 2:r]) * turn
                    w[..., :r // 2], w[..., r // 2:r] = c.real, c.imag
                return w

            at = torch.tensor(pages, device="cuda")[pos // page]
            keys[at, :, pos % page] = turned(d["k"][row:row + n])
            vals[at, :, pos % page] = d["v"][row:row + n]
            out.append(turned(d["q"][row:row + n]))
        elif n:
            have = pages[:-(-(p + n) // page)]
            o = torch.empty((n, Hq, Dh), dtype=torch.float64, device="cuda")
            hidden = torch.arange(p + n, device="cuda")[None] > torch.arange(p, p + n, device="cuda")[:, None]
            for kv in range(Hkv):
                K = keys[have, kv].reshape(-1, Dh)[:p + n]
                V = vals[have, kv].reshape(-1, Dh)[:p + n]
                for h in range(kv * group, (kv + 1) * group):
                    logit = (d["q"][row:row + n, h] @ K.T) * Dh ** -0.5
                    o[:, h] = logit.masked_fill_(hidden, -math.inf).softmax(-1) @ V
            out.append(o)
        row += n
    out = torch.cat(out) if out else torch.empty((0, Hq, Dh), dtype=torch.float64, device="cuda")
    return (out, keys, vals) if case["op"] == "append" else out
