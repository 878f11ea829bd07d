"""Plain 64-bit implementations of the serving and policy-training operators, one sequence, token, row
or tensor at a time, written from the formulas; and the bounds their tests hold the kernels to."""
from __future__ import annotations

import math

import torch

# largest relative error of one rounding to nearest: 24, 11 and 8 significant bits
ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def paged_attention(q, k_pages, v_pages, table, lens, scale, eps=1e-12, window=0):
    """(S, H, D) float64: sum p v / (sum p + eps), p = relu(scale q.k)^2, over the last `window` keys."""
    S, H, D = q.shape
    P, Hkv, page, _ = k_pages.shape
    out = torch.zeros((S, H, D), dtype=torch.float64, device=q.device)
    for s in range(S):
        n = min(max(int(lens[s]), 0), table.shape[1] * page)
        keys = range(max(0, n - window) if window else 0, n)
        at = [(int(table[s, j // page]), j % page) for j in keys]
        at = [(p, r) for p, r in at if 0 <= p < P]
        if not at:
            continue
        pg = torch.tensor([p for p, _ in at], device=q.device)
        row = torch.tensor([r for _, r in at], device=q.device)
        for h in range(H):
            k = k_pages[pg, h // (H // Hkv), row].double()
            v = v_pages[pg, h // (H // Hkv), row].double()
            a = (k @ q[s, h].double()) * float(scale[h])
            p = torch.where(a <= 0, torch.zeros_like(a), a * a)
            if float(p.sum()) != 0.0:
                out[s, h] = (p[:, None] * v).sum(0) / (p.sum() + eps)
    return out


def attention_bound(ref, v_pages, dtype):
    """16-bit: each p may be rounded by r, and the normaliser sums what the product uses, so O moves by at most
    r times the weighted mean of |v - O|, itself at most max|v|; and the result is rounded once.  r is 2^-8 for
    bf16 and 2^-10 for fp16 (twice its rounding).  fp32: the framework's gate for fp32 attention."""
    if dtype == torch.float32:
        return torch.full_like(ref, 1e-4 * max(1.0, float(ref.abs().max())))
    r = {torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -8}[dtype]
    return r * float(v_pages.float().nan_to_num(0.0).abs().max()) + r * ref.abs()


def rope_l2(x, cos, sin, eps=1e-12):
    """x (..., D) float64 rotated by the angles of cos / sin (..., D / 2), then on the unit sphere."""
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    y = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return y / torch.sqrt((y * y).sum(-1, keepdim=True) + eps)


def qkv_write(qkv, cos, sin, positions, slots, k_pages, v_pages, heads, eps=1e-12):
    """float64 (q, k, v) of every token, and the pages after the write."""
    P, Hkv, page, D = k_pages.shape
    N = qkv.shape[0]
    x = qkv.double().reshape(N, heads + 2 * Hkv, D)
    q, k, v = torch.split(x, [heads, Hkv, Hkv], dim=1)
    pos = positions.long()
    known = (pos >= 0) & (pos < cos.shape[0])
    c = torch.where(known[:, None], cos.double()[pos.clamp(0, cos.shape[0] - 1)], math.nan)[:, None]
    s = torch.where(known[:, None], sin.double()[pos.clamp(0, cos.shape[0] - 1)], math.nan)[:, None]
    q, k = rope_l2(q, c, s, eps), rope_l2(k, c, s, eps)
    kp, vp = k_pages.double().clone(), v_pages.double().clone()
    for n in range(N):
        if 0 <= int(slots[n]) < P * page:
            kp[int(slots[n]) // page, :, int(slots[n]) % page] = k[n]
            vp[int(slots[n]) // page, :, int(slots[n]) % page] = v[n]
    return q, k, v, kp, vp


def logprobs(logits, targets, top_k):
    """float64 (logp, entropy, top_logp) and the int64 order: value falling, NaN first, then index."""
    x = logits.detach().double()
    N, V = x.shape
    m = x.max(dim=1, keepdim=True).values
    # (x - m) - log s, not x - (m + log s): m may be the lowest value of a type, beside which log s is lost
    lp = (x - m) - torch.log(torch.exp(x - m).sum(1, keepdim=True))
    p = torch.exp(lp)
    ent = -torch.where(x == -math.inf, p, p * lp).sum(1)  # p is 0 where x is -inf (or the row is NaN)
    ok = (targets >= 0) & (targets < V)
    logp = torch.where(ok, lp.gather(1, targets.long().clamp(0, V - 1)[:, None])[:, 0], math.nan)
    order = torch.tensor([sorted(range(V), key=lambda c: (-math.inf if r[c] != r[c] else -r[c], 0 if r[c] != r[c] else 1, c))[:top_k]
                          for r in x.tolist()], dtype=torch.int64, device=x.device).reshape(N, top_k)
    return logp, ent, lp.gather(1, order), order


def logprobs_grad(logits, targets, order, g_logp, g_entropy, g_top):
    """float64 gradient of sum(g_logp logp) + sum(g_entropy entropy) + sum(g_top top_logp)."""
    x = logits.detach().double()
    lp = torch.log_softmax(x, dim=1)
    p = lp.exp()
    ent = -torch.where(x == -math.inf, torch.zeros_like(p), p * lp).sum(1, keepdim=True)
    d = -p * (g_logp.double() + g_top.double().sum(1))[:, None]
    d -= g_entropy.double()[:, None] * torch.where(x == -math.inf, torch.zeros_like(p), p * (lp + ent))
    rows = torch.arange(x.shape[0], device=x.device)
    d[rows, targets.long()] += g_logp.double()
    for i in range(order.shape[1]):
        d[rows, order[:, i]] += g_top[:, i].double()
    return d


def clip(grads, max_norm, eps=1e-6):
    """float64 (norm, scaled gradients)."""
    norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))
    c = max_norm / (norm + eps)
    c = 1.0 if c >= 1.0 else c
    return norm, [g.double() * c for g in grads]
