"""The student decoder's operators in 64 bits, with how far a kernel in bf16 and fp32 may be from them.

A value rounded to bf16 is off by at most 2^-8 of itself (half a step). A sum in the tensor cores may lose one truncation (2^-23 of the
sum of magnitudes) per step of 16 products, an ordinary fp32 sum 2^-24 per addition. A power of two below fp32's smallest normal number,
2^-126, may be taken as zero: a softmax weight (at most 1 and formed against the row's maximum or its whole sum) is then off by at most TINY."""
import math

import torch

BF = 2.0 ** -8
DT = torch.float64
TINY = 2.0 ** -126


def hidden_keys(S, window, sinks, device):
    i = torch.arange(S, device=device)
    dist = i[:, None] - i[None, :]
    hid = dist < 0
    if window:
        hid = hid | ((dist >= window) & (i[None, :] >= sinks))
    return hid


def attention(q, k, v, window, sinks, lengths, scale, dout=None):
    """Windowed attention by its definition: {"out"} and with ``dout`` {"dq", "dk", "dv"}, and under "tol" how far each may be off.

    Up to 256 tokens, and where no row sees more than 64 keys, the weights and their gradients are sums of two bf16 values, off by at most 2^-16
    of themselves."""
    B, H, S, D = q.shape
    KV = k.shape[1]
    G = H // KV
    dev = q.device
    hid = hidden_keys(S, window, sinks, dev)
    few = S <= 256 or 0 < window and window + sinks <= 64
    weight = BF * BF if few else BF
    names = ("out",) if dout is None else ("out", "dq", "dk", "dv")
    like = {"out": q, "dq": q, "dk": k, "dv": k}
    res = {n: torch.zeros(like[n].shape, dtype=DT, device=dev) for n in names}
    tol = {n: torch.zeros(like[n].shape, dtype=DT, device=dev) for n in names}
    for b in range(B):
        L = S if lengths is None else min(max(int(lengths[b]), 0), S)
        if L == 0:
            continue
        sums = (L / 16 + D / 16 + 8) * 2.0 ** -22  # of a sum over the keys or queries, and of the products in front of it
        for h in range(H):
            g = h // G
            Q, K, V = (t.detach().to(DT) for t in (q[b, h, :L], k[b, g, :L], v[b, g, :L]))
            P = torch.softmax((Q @ K.T * scale).masked_fill(hid[:L, :L], -math.inf), dim=1)
            # a score is off by 2^-23 of its magnitudes per step, its power of two by 2^-20
            ds_abs = (D / 16 + 8) * 2.0 ** -22 * scale * (Q.abs() @ K.abs().T).masked_fill(hid[:L, :L], 0).amax(1, keepdim=True) + 2.0 ** -18
            O = P @ V
            A = P @ V.abs()
            res["out"][b, h, :L] = O
            # every weight rounded, the answer rounded once more; what rounding took from the answer is kept, rounded to bf16 itself, for delta
            raw = weight * A + (2 * ds_abs + sums) * A + TINY * V.abs().sum(0)
            tO = raw + BF * O.abs()
            tol["out"][b, h, :L] = tO
            if dout is None:
                continue
            dO = dout[b, h, :L].to(DT)
            dP = dO @ V.T
            delta = (dP * P).sum(1, keepdim=True)
            dS = P * (dP - delta)
            # delta is formed from the answer in two bf16 parts, dS is rounded to bf16 after fp32 arithmetic
            E = (dO.abs() * (raw + BF * BF * O.abs())).sum(1, keepdim=True) + (D / 16 + 8) * 2.0 ** -22 * (dO.abs() @ V.abs().T).amax(1, keepdim=True)
            eP = (weight + 2 * ds_abs) * P + TINY
            eS = (weight + 2 * ds_abs) * dS.abs() + P * E + TINY * (1 + dP.abs() + delta.abs() + E)
            res["dq"][b, h, :L] = dS @ K * scale
            tol["dq"][b, h, :L] = BF * res["dq"][b, h, :L].abs() + scale * ((eS + sums * dS.abs()) @ K.abs())
            res["dk"][b, g, :L] += dS.T @ Q * scale
            tol["dk"][b, g, :L] += scale * ((eS + G * sums * dS.abs()).T @ Q.abs())
            res["dv"][b, g, :L] += P.T @ dO
            tol["dv"][b, g, :L] += (eP + G * sums * P).T @ dO.abs()
    for n in ("dk", "dv"):
        if n in tol:
            tol[n] += BF * res[n].abs()
    res["tol"] = tol
    return res


def qk_norm_rope(qkv, wq, wk, table, heads, kv, eps, grads=None):
    """Per-head norms and the rotation by their definition; with ``grads`` = (dq, dk, dv) the gradients too, and under "tol" what each may be off."""
    D = qkv.shape[-1]
    half = D // 2
    S = qkv.shape[1]
    x = qkv.detach()[:, :, :heads + kv].to(DT)
    w = torch.cat([wq.detach().to(DT).expand(heads, D), wk.detach().to(DT).expand(kv, D)])
    cos, sin = table[:S, None, :, 0].to(DT), table[:S, None, :, 1].to(DT)
    r = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    n = x * r * w
    a, b = n[..., :half], n[..., half:]
    y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).transpose(1, 2)
    mag = torch.cat([a.abs() * cos.abs() + b.abs() * sin.abs(), b.abs() * cos.abs() + a.abs() * sin.abs()], -1).transpose(1, 2)
    f32 = 2.0 ** -24 * (D / 4 + 16)  # the row's sum of squares and the handful of products around it
    res = {"q": y[:, :heads], "k": y[:, heads:], "v": qkv.detach()[:, :, heads + kv:].transpose(1, 2).to(DT)}
    ty = BF * y.abs() + f32 * mag
    tol = {"q": ty[:, :heads], "k": ty[:, heads:], "v": torch.zeros_like(res["v"])}
    if grads is not None:
        dq, dk, dv = grads
        g = torch.cat([dq, dk], 1).transpose(1, 2).to(DT)
        a, b = g[..., :half], g[..., half:]
        gm = torch.cat([a.abs() * cos.abs() + b.abs() * sin.abs(), b.abs() * cos.abs() + a.abs() * sin.abs()], -1)
        g = torch.cat([a * cos + b * sin, b * cos - a * sin], -1)
        dx = r * (g * w - x * r * r * (g * w * x).mean(-1, keepdim=True))
        mx = r * (gm * w.abs() + x.abs() * r * r * (gm * w.abs() * x.abs()).mean(-1, keepdim=True))
        res["dqkv"] = torch.cat([dx, dv.transpose(1, 2).to(DT)], 2)
        tol["dqkv"] = torch.cat([BF * dx.abs() + 2 * f32 * mx, torch.zeros_like(dv.transpose(1, 2), dtype=DT)], 2)
        t, m = g * x * r, gm * x.abs() * r
        for name, cut, wt in (("dwq", slice(0, heads), wq), ("dwk", slice(heads, heads + kv), wk)):
            rows = t[:, :, cut].shape[0] * t.shape[1] * t[:, :, cut].shape[2]
            res[name] = t[:, :, cut].sum((0, 1, 2))
            tol[name] = (f32 + rows * 2.0 ** -24) * m[:, :, cut].sum((0, 1, 2)) + (BF if wt.dtype == torch.bfloat16 else 2.0 ** -24) * res[name].abs()
    res["tol"] = tol
    return res


def distill(logits, targets, ids, values, weight, tau, scale):
    """The mixed loss row by row and its gradient by their definition, in 64 bits, and under "tol" what each may be off."""
    T, V = logits.shape
    z = logits.detach().to(DT)
    loss = torch.zeros(T, dtype=DT, device=z.device)
    grad, gtol = torch.zeros_like(z), torch.zeros_like(z)
    ltol = torch.zeros_like(loss)
    for t in range(T):
        y = int(targets[t])
        if not 0 <= y < V:
            continue
        logc, logq = torch.log_softmax(z[t], 0), torch.log_softmax(z[t] / tau, 0)
        there = (ids[t] >= 0) & (ids[t] < V)
        i, u = ids[t][there].long(), values[t][there].to(DT) / tau
        a = weight if i.numel() and bool((u > -math.inf).any()) else 0.0
        loss[t] = -(1 - weight) * logc[y] if weight < 1 else 0.0
        g = (1 - weight) * logc.exp() + a * tau * logq.exp()
        # a power of two is off by 2^-22 and by its exponent's rounding, a sum over the row by one rounding per addition of a thread (256
        # threads or more side by side) and of the tree behind them
        seq = (V / 256 + 16) * 2.0 ** -24
        far = (z[t] - z[t].max()).abs().nan_to_num(posinf=0.0) * 1.45 / min(tau, 1.0) * 2.0 ** -22 + 2.0 ** -20 + seq
        # the exponents' offset, maximum / tau in powers of two, is rounded to 2^-24 of itself: once where a slice's sums are made and once for
        # the gradient
        shift = z[t].abs().nan_to_num(posinf=0.0).max() * 1.45 / min(tau, 1.0) * 2.0 ** -23
        m = g * (far + shift)
        g[y] -= 1 - weight
        ltol[t] = (1 - weight) * (2.0 ** -21 * (z[t].abs().nan_to_num(posinf=0.0).max() + 16) + seq)
        if a:
            logp = torch.log_softmax(u, 0)
            p = logp.exp()
            part = p > 0
            loss[t] += a * tau ** 2 * (p[part] * (logp[part] - logq[i[part]])).sum()
            g.index_add_(0, i, -a * tau * p)
            m.index_add_(0, i, a * tau * p * (2.0 ** -18 + (u - u.max()).abs().nan_to_num(posinf=0.0) * 2.0 ** -21))
            ltol[t] += a * tau ** 2 * (2.0 ** -18 * (p[part] * (logp[part].abs() + logq[i[part]].abs() + 16)).sum() + seq + shift)
        m[y] += 2.0 ** -22
        grad[t] = g * scale
        # the smallest results are rounded to a fixed step: half of bf16's smallest
        gtol[t] = BF * grad[t].abs() + m * abs(scale) + 2.0 ** -134 + TINY * abs(scale) * (1 + tau)
    return {"loss": loss, "grad": grad, "tol": {"loss": ltol, "grad": gtol}}


def off(name, got, ref):
    """Fails with the worst element where ``got`` is further from the definition than it may be."""
    want, tol = ref[name], ref["tol"][name]
    d = (got.detach().to(DT) - want).abs()
    assert bool(torch.isfinite(d).all()), f"{name}: not finite"
    over = d - tol
    if bool((over > 0).any()):
        at = int(over.argmax())
        idx = tuple(int(n) for n in torch.unravel_index(torch.tensor(at), d.shape))
        raise AssertionError(f"{name}{idx}: {float(got[idx])} instead of {float(want[idx])}, may be off {float(tol[idx]):.3g}; {int((over > 0).sum())} of {d.numel()} values")
