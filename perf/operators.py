"""The operators of a student decoder's training step, as cases that can be timed and compared.

Three kinds of call, each through the package's public entry points:

``qk``      ``ops.attention.qk_norm_rope``: per-head RMSNorm of queries and keys and the rotation to their positions, from the packed
            projection; with ``train`` its backward pass too (the packed gradient, both weights' gradients).
``attn``    ``ops.attention.window_attention``: causal attention in which a query sees the last ``window`` keys and the first ``sinks``
            ones; ``lengths`` are the rows' lengths in a padded batch. With ``train`` the gradients of queries, keys and values.
``distill`` ``ops.train_ops.distill_loss``: cross-entropy mixed with the divergence from a teacher's top logits, loss and logit gradient.

Sizes are those of the package's model table and tests, or spread over the ranges in between by ``draw``.
"""
from __future__ import annotations

import math

import torch

own = False


def listed():
    return [
        # The tests' two-layer model on one short sequence: launches and host work. Heads of 64, windows shorter than the sequence.
        {"name": "attn_tiny_train", "kind": "attn", "batch": 1, "heads": 4, "kv": 2, "dim": 64, "seq": 128, "window": 48, "sinks": 4, "lengths": "", "train": True},
        # A layer of the 8B model on the benchmark's sequence with a window of a quarter of it, forward and backward.
        {"name": "attn_8b_train", "kind": "attn", "batch": 1, "heads": 32, "kv": 8, "dim": 128, "seq": 4096, "window": 1024, "sinks": 4, "lengths": "", "train": True},
        # The same layer evaluated on the 70B model's sequence length, forward only (held-out loss).
        {"name": "attn_8b_eval_8192", "kind": "attn", "batch": 1, "heads": 32, "kv": 8, "dim": 128, "seq": 8192, "window": 2048, "sinks": 16, "lengths": "", "train": False},
        # No window: plain causal attention with a key head for every query head (the 7B model), forward and backward.
        {"name": "attn_7b_full_train", "kind": "attn", "batch": 1, "heads": 32, "kv": 32, "dim": 128, "seq": 4096, "window": 0, "sinks": 0, "lengths": "", "train": True},
        # The 1B model (64-wide heads) on a padded batch whose rows are no multiple of anything; one row holds a single token.
        {"name": "attn_1b_ragged_train", "kind": "attn", "batch": 3, "heads": 32, "kv": 8, "dim": 64, "seq": 999, "window": 257, "sinks": 3, "lengths": "999,1,613", "train": True},
        # The tiny model's projection: one launch each way.
        {"name": "qk_tiny_train", "kind": "qk", "batch": 1, "heads": 4, "kv": 2, "dim": 64, "seq": 128, "weights": "bf16", "train": True},
        # The 8B model's projection on the benchmark's sequence, forward and backward.
        {"name": "qk_8b_train", "kind": "qk", "batch": 1, "heads": 32, "kv": 8, "dim": 128, "seq": 4096, "weights": "bf16", "train": True},
        # The 1B model's, forward only, on odd lengths with fp32 weights.
        {"name": "qk_1b_eval_ragged", "kind": "qk", "batch": 3, "heads": 32, "kv": 8, "dim": 64, "seq": 1999, "weights": "fp32", "train": False},
        # The tiny model's head: 128 tokens, a thousand logits.
        {"name": "distill_tiny", "kind": "distill", "tokens": 128, "vocab": 1024, "topk": 16, "weight": 0.5, "temperature": 2.0, "ids": "int64", "values": "fp32"},
        # The 8B model's head on the benchmark's sequence, from 64 stored teacher logits per token.
        {"name": "distill_8b", "kind": "distill", "tokens": 4096, "vocab": 128256, "topk": 64, "weight": 0.75, "temperature": 2.0, "ids": "int32", "values": "bf16"},
        # The 7B model's vocabulary, an odd number of tokens, distillation alone at temperature one.
        {"name": "distill_7b_odd", "kind": "distill", "tokens": 1997, "vocab": 32000, "topk": 7, "weight": 1.0, "temperature": 1.0, "ids": "int64", "values": "fp32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "qk", "distill"])
    if kind == "distill":
        vocab = 8 * _log(rng, 125, 16032)
        return {"kind": kind, "tokens": _log(rng, 1, 4096), "vocab": vocab, "topk": _log(rng, 1, 128), "weight": rng.choice([0.3, 0.5, 0.75, 1.0]),
                "temperature": rng.choice([1.0, 2.0, 3.5]), "ids": rng.choice(["int64", "int32"]), "values": rng.choice(["fp32", "bf16"])}
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4])
    case = {"kind": kind, "batch": rng.randint(1, 3), "heads": kv * group, "kv": kv, "dim": rng.choice([64, 128, 128, 96])}
    if kind == "qk":
        case |= {"seq": _log(rng, 1, 4096 // case["batch"]), "weights": rng.choice(["bf16", "fp32"]), "train": rng.random() < 0.6}
        return case
    seq = _log(rng, 1, 4096 // case["batch"])
    lengths = ",".join(str(rng.randint(0, seq)) for _ in range(case["batch"])) if rng.random() < 0.4 else ""
    window = 0 if rng.random() < 0.3 else _log(rng, 1, seq)
    case |= {"seq": seq, "window": window, "sinks": rng.choice([0, 1, 4, rng.randint(0, 200)]) if window else 0, "lengths": lengths, "train": rng.random() < 0.6}
    return case


def _lengths(case):
    return [int(n) for n in case["lengths"].split(",")] if case["lengths"] else [case["seq"]] * case["batch"]


def _leaf(t):
    return t.detach().requires_grad_(True)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"
    if case["kind"] == "distill":
        T, V, K = case["tokens"], case["vocab"], case["topk"]
        logits = (2.5 * torch.randn(T, V, device=dev, generator=g)).to(torch.bfloat16)
        # the teacher agrees with the student up to noise; its K largest logits are what a data set stores
        dense = logits.float().mul_(0.8).add_(torch.randn(T, V, device=dev, generator=g))
        values, ids = dense.topk(K, dim=-1)
        del dense
        targets = torch.where(torch.rand(T, device=dev, generator=g) < 0.7, ids[:, 0], torch.randint(0, V, (T,), device=dev, generator=g))
        targets[torch.rand(T, device=dev, generator=g) < 0.05] = -100  # padding
        return {"case": case, "logits": logits, "targets": targets, "ids": ids.to(torch.int32 if case["ids"] == "int32" else torch.int64).contiguous(),
                "values": values.to(torch.bfloat16 if case["values"] == "bf16" else torch.float32).contiguous(), "grad": torch.empty_like(logits), "scale": 1.0 / T}
    B, S, H, KV, D = case["batch"], case["seq"], case["heads"], case["kv"], case["dim"]
    packed = torch.randn(B, S, H + 2 * KV, D, device=dev, generator=g)
    dq, dk, dv = ((0.01 * torch.randn(B, S, n, D, device=dev, generator=g)).to(torch.bfloat16).transpose(1, 2) for n in (H, KV, KV))
    if case["kind"] == "qk":
        wt = torch.float32 if case["weights"] == "fp32" else torch.bfloat16
        wq, wk = (_leaf((1 + 0.2 * torch.randn(D, device=dev, generator=g)).to(wt)) for _ in range(2))
        # positions' (cos, sin) as the trainer keeps them: angles in 64 bits
        inv = 1.0 / (500000.0 ** (torch.arange(0, D, 2, dtype=torch.float64, device=dev) / D))
        ang = torch.outer(torch.arange(S, dtype=torch.float64, device=dev), inv)
        table = torch.stack([ang.cos(), ang.sin()], dim=-1).float().contiguous()
        return {"case": case, "qkv": _leaf((0.7 * packed).to(torch.bfloat16)), "wq": wq, "wk": wk, "table": table, "grads": (dq, dk, dv)}
    # queries and keys as the norm in front leaves them (rows of length sqrt(D) times a learned weight), values as a slice of the projection
    q, k = (1.3 * t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + 1e-5) for t in (packed[:, :, :H], packed[:, :, H:H + KV]))
    qkv = packed.to(torch.bfloat16)
    state = {"case": case, "q": _leaf(q.to(torch.bfloat16).transpose(1, 2)), "k": _leaf(k.to(torch.bfloat16).transpose(1, 2)),
             "v": _leaf(qkv[:, :, H + KV:].transpose(1, 2)), "dout": dq, "lengths": None}
    if case["lengths"]:
        state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)
    return state


def _visible(case, lengths, dev):
    """Truth values [B or 1, 1, 1, S, S]: which keys a query sees."""
    S = case["seq"]
    i = torch.arange(S, device=dev).view(S, 1)
    j = torch.arange(S, device=dev).view(1, S)
    see = j <= i
    if case["window"]:
        see = see & ((i - j < case["window"]) | (j < case["sinks"]))
    see = see.view(1, 1, 1, S, S)
    if lengths is not None:
        see = see & (i < lengths.view(-1, 1, 1, 1, 1))
    return see


def _plain_attention(st):
    case, dt = st["case"], torch.float32
    B, S, H, KV, D = case["batch"], case["seq"], case["heads"], case["kv"], case["dim"]
    G = H // KV
    scale = 1.0 / math.sqrt(D)
    q = st["q"].to(dt).reshape(B, KV, G, S, D)
    k, v = st["k"].to(dt).unsqueeze(2), st["v"].to(dt).unsqueeze(2)
    see = _visible(case, st["lengths"], q.device)
    s = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).masked_fill_(~see, float("-inf"))
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total == 0, torch.ones_like(total), total)  # a row that sees nothing answers zeros
    out = torch.matmul(p, v)
    res = {"out": out.reshape(B, H, S, D).to(torch.bfloat16)}
    if case["train"]:
        g = st["dout"].to(dt).reshape(B, KV, G, S, D)
        res["dv"] = torch.matmul(p.transpose(-1, -2), g).sum(2).to(torch.bfloat16)
        ds = torch.matmul(g, v.transpose(-1, -2)).sub_((g * out).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        res["dq"] = torch.matmul(ds, k).reshape(B, H, S, D).to(torch.bfloat16)
        res["dk"] = torch.matmul(ds.transpose(-1, -2), q).sum(2).to(torch.bfloat16)
    return res


def _plain_qk(st):
    case, dt, eps = st["case"], torch.float32, 1e-5
    H, KV, D = case["heads"], case["kv"], case["dim"]
    qkv = st["qkv"]
    x = qkv[:, :, :H + KV].to(dt)
    w = torch.cat([st["wq"].to(dt).expand(H, D), st["wk"].to(dt).expand(KV, D)])
    cos, sin = st["table"][:, None, :, 0], st["table"][:, None, :, 1]
    r = torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    a, b = (x * r * w).split(D // 2, dim=-1)
    y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(torch.bfloat16).transpose(1, 2)
    res = {"q": y[:, :H], "k": y[:, H:], "v": qkv[:, :, H + KV:].transpose(1, 2)}
    if case["train"]:
        dq, dk, dv = st["grads"]
        a, b = torch.cat([dq, dk], 1).transpose(1, 2).to(dt).split(D // 2, dim=-1)
        g = torch.cat([a * cos + b * sin, b * cos - a * sin], -1)
        dw = (g * x * r).to(torch.float64).sum((0, 1))
        g = g * w
        dx = r * (g - x * r * r * (g * x).mean(-1, keepdim=True))
        res |= {"dqkv": torch.cat([dx.to(torch.bfloat16), dv.transpose(1, 2)], 2), "dwq": dw[:H].sum(0).to(st["wq"].dtype), "dwk": dw[H:].sum(0).to(st["wk"].dtype)}
    return res


def _plain_distill(st):
    case, dt = st["case"], torch.float32
    a, tau = case["weight"], case["temperature"]
    z = st["logits"].to(dt)
    t, ids = st["targets"], st["ids"].to(torch.int64)
    live = t >= 0
    at = t.clamp(min=0).unsqueeze(1)
    m = z.amax(-1, keepdim=True)
    e = (z - m).div_(tau).exp_()
    total = e.sum(-1, keepdim=True)
    y = st["values"].to(dt) / tau
    y = y - y.amax(-1, keepdim=True)
    log_p = y - y.exp().sum(-1, keepdim=True).log()
    p = log_p.exp()
    kl = (p * (log_p - (z.gather(1, ids) - m) / tau + total.log())).sum(-1)
    loss = a * tau * tau * kl
    grad = e.mul_(a * tau / total).scatter_add_(1, ids, -a * tau * p)
    if a < 1:
        e = z.sub(m).exp_()
        total = e.sum(-1, keepdim=True)
        loss = loss + (1 - a) * (m + total.log() - z.gather(1, at)).squeeze(1)
        grad += e.mul_((1 - a) / total).scatter_add_(1, at, torch.full_like(m, -(1 - a)))
    grad *= st["scale"] * live.unsqueeze(1)
    return {"loss": torch.where(live, loss, torch.zeros_like(loss)), "grad": grad.to(torch.bfloat16)}


def _own(st):
    from rocm_systems_b200.ops import attention, train_ops

    case = st["case"]
    if case["kind"] == "distill":
        loss, grad = train_ops.distill_loss(st["logits"], st["targets"], st["ids"], st["values"], weight=case["weight"], temperature=case["temperature"],
                                            grad_scale=st["scale"], grad=st["grad"])
        return {"loss": loss, "grad": grad}
    with torch.set_grad_enabled(case["train"]):
        if case["kind"] == "qk":
            q, k, v = attention.qk_norm_rope(st["qkv"], st["wq"], st["wk"], st["table"], case["heads"], case["kv"], eps=1e-5)
            res = {"q": q, "k": k, "v": v}
            if case["train"]:
                res["dqkv"], res["dwq"], res["dwk"] = torch.autograd.grad((q, k, v), (st["qkv"], st["wq"], st["wk"]), st["grads"])
            return res
        out = attention.window_attention(st["q"], st["k"], st["v"], window=case["window"], sinks=case["sinks"], lengths=st["lengths"])
        res = {"out": out}
        if case["train"]:
            res["dv"], res["dq"], res["dk"] = torch.autograd.grad(out, (st["v"], st["q"], st["k"]), st["dout"])
        return res


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"attn": _plain_attention, "qk": _plain_qk, "distill": _plain_distill}[state["case"]["kind"]](state)


def _pairs(case):
    """Visible (query, key) pairs of one head over the whole batch."""
    n = 0
    for L in _lengths(case):
        for i in range(L):
            seen = min(i + 1, case["window"]) if case["window"] else i + 1
            n += seen + min(case["sinks"], i + 1 - seen)
    return n


def work(case):
    if case["kind"] == "distill":
        T, V, K = case["tokens"], case["vocab"], case["topk"]
        entry = (4 if case["ids"] == "int32" else 8) + (2 if case["values"] == "bf16" else 4)
        return {"bytes": 4.0 * T * V + T * K * entry + 12.0 * T, "flops": (8.0 if case["weight"] < 1 else 5.0) * T * V}
    B, S, H, KV, D = case["batch"], case["seq"], case["heads"], case["kv"], case["dim"]
    if case["kind"] == "qk":
        rows = B * S * (H + KV)
        if not case["train"]:
            return {"bytes": 4.0 * rows * D + 4.0 * S * D, "flops": 7.0 * rows * D}
        return {"bytes": 4.0 * rows * D + 4.0 * S * D + 2.0 * B * S * D * (2 * (H + KV) + 2 * KV + H), "flops": 21.0 * rows * D}
    tokens = B * S
    moved = 2.0 * tokens * D * (2 * H + 2 * KV)  # q, k, v in, the answer out
    if case["train"]:
        moved += 2.0 * tokens * D * (2 * H + 2 * KV)  # its gradient in, theirs out
    return {"bytes": moved, "flops": (14.0 if case["train"] else 4.0) * D * H * _pairs(case)}


def _exact_attention(case, st):
    dt = torch.float64
    B, S, H, KV, D = case["batch"], case["seq"], case["heads"], case["kv"], case["dim"]
    q, k, v, do = (st[n].detach().to(dt) for n in ("q", "k", "v", "dout"))
    pos = torch.arange(S, device=q.device)
    dist = pos[:, None] - pos[None, :]
    hidden = dist < 0
    if case["window"]:
        hidden |= (dist >= case["window"]) & (pos[None, :] >= case["sinks"])
    res = {"out": torch.zeros(B, H, S, D, dtype=dt, device=q.device)}
    if case["train"]:
        res |= {"dv": torch.zeros_like(v), "dq": torch.zeros_like(q), "dk": torch.zeros_like(k)}
    for b, L in enumerate(_lengths(case)):
        if L == 0:
            continue
        for h in range(H):
            kh = h // (H // KV)
            Q, K, V, dO = q[b, h, :L], k[b, kh, :L], v[b, kh, :L], do[b, h, :L]
            P = torch.softmax((Q @ K.T / math.sqrt(D)).masked_fill(hidden[:L, :L], -math.inf), dim=1)
            res["out"][b, h, :L] = P @ V
            if case["train"]:
                res["dv"][b, kh, :L] += P.T @ dO
                dP = dO @ V.T
                dS = P * (dP - (dP * P).sum(1, keepdim=True)) / math.sqrt(D)
                res["dq"][b, h, :L] = dS @ K
                res["dk"][b, kh, :L] += dS.T @ Q
    return res


def _exact_qk(case, st):
    H, KV, D = case["heads"], case["kv"], case["dim"]
    dt = torch.float64
    with torch.enable_grad():
        x, wq, wk = (st[n].detach().to(dt).requires_grad_(True) for n in ("qkv", "wq", "wk"))
        turn = torch.complex(st["table"][..., 0].to(dt), st["table"][..., 1].to(dt))[None, :, None, :]

        def place(t, w):
            n = t / (t.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w
            c = torch.complex(n[..., :D // 2], n[..., D // 2:]) * turn
            return torch.cat([c.real, c.imag], -1).transpose(1, 2)

        q, k, v = place(x[:, :, :H], wq), place(x[:, :, H:H + KV], wk), x[:, :, H + KV:].transpose(1, 2)
        res = {"q": q.detach(), "k": k.detach(), "v": v.detach()}
        if case["train"]:
            res["dqkv"], res["dwq"], res["dwk"] = torch.autograd.grad((q, k, v), (x, wq, wk), tuple(t.to(dt) for t in st["grads"]))
    return res


def _exact_distill(case, st):
    T, a, tau, dt = case["tokens"], case["weight"], case["temperature"], torch.float64
    res = {"loss": torch.zeros(T, dtype=dt, device="cuda"), "grad": torch.zeros(T, case["vocab"], dtype=dt, device="cuda")}
    for r0 in range(0, T, 512):  # some rows at a time
        rows = torch.arange(r0, min(T, r0 + 512), device="cuda")
        rows = rows[st["targets"][rows] >= 0]
        with torch.enable_grad():
            z = st["logits"][rows].to(dt).requires_grad_(True)
            log_q = torch.log_softmax(z / tau, 1).gather(1, st["ids"][rows].to(torch.int64))
            log_p = torch.log_softmax(st["values"][rows].to(dt) / tau, 1)
            loss = a * tau ** 2 * (log_p.exp() * (log_p - log_q)).sum(1)
            if a < 1:
                loss = loss - (1 - a) * torch.log_softmax(z, 1).gather(1, st["targets"][rows][:, None])[:, 0]
            (dz,) = torch.autograd.grad(loss.sum(), z)
        res["loss"][rows] = loss.detach()
        res["grad"][rows] = dz * st["scale"]
    return res


def exact(case, seed):
    st = prepare(case, seed)
    return {"attn": _exact_attention, "qk": _exact_qk, "distill": _exact_distill}[case["kind"]](case, st)
