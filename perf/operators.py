"""The serving and policy-training operators of the flash-Born GPT as measurable cases.

Four operators, each in a plain form (elementary torch operations in 32 bits) and through this package's
public entry points (``own = True``):

  decode   Born attention of one new token per sequence over a paged key-value cache
  write    rotary positions + L2 normalisation of new tokens' Q and K, K and V stored into the cache's pages
  score    log probabilities of given tokens with entropy and top alternatives, forward or with gradient
  clip     the global gradient norm over many tensors, and clipping

Sizes are those of this package's GPT (16 heads of 64, 1,024 tokens, a 50,257-token vocabulary padded to
50,304, 127 M parameters) and of its long-context benchmark (heads of 128, 16,384 tokens and more), with
grouped heads, odd sizes and ragged lengths between them.
"""
import math
import random

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_GOLDEN = 0.6180339887498949
EPS = 1e-12
LARGEST = 3.4e9  # bytes of the largest listed case: no drawn case moves more


# ------------------------------------------------------------------------------------------------
# Cases
# ------------------------------------------------------------------------------------------------
def listed():
    return [
        # one user, the first tokens of an answer: the call's latency is all there is
        dict(name="decode_first_tokens", op="decode", seqs=1, heads=16, kv_heads=16, head_dim=64, page=16, shortest=37,
             longest=37, window=0, dtype="bf16"),
        # a batch of conversations of every age with the GPT's own heads and context
        dict(name="decode_chat_batch", op="decode", seqs=48, heads=16, kv_heads=16, head_dim=64, page=16, shortest=1,
             longest=1024, window=0, dtype="bf16"),
        # a few documents far longer than a training row, eight query heads to a key head
        dict(name="decode_long_grouped", op="decode", seqs=6, heads=32, kv_heads=4, head_dim=128, page=64,
             shortest=16384, longest=131072, window=0, dtype="bf16"),
        # full precision, an odd head and page size, a sliding window, one sequence that has nothing yet
        dict(name="decode_window_fp32", op="decode", seqs=9, heads=6, kv_heads=3, head_dim=48, page=24, shortest=0,
             longest=5000, window=384, dtype="fp32"),
        # the same batch's new tokens on their way into the cache
        dict(name="write_step", op="write", tokens=48, heads=16, kv_heads=8, head_dim=64, page=16, padding=0,
             dtype="bf16"),
        # packed prompts of a long-context model filling the cache, some padding at the end
        dict(name="write_prompts", op="write", tokens=16389, heads=32, kv_heads=4, head_dim=128, page=64, padding=37,
             dtype="bf16"),
        # one token's alternatives shown to a user, the unpadded vocabulary in full precision
        dict(name="score_one_odd", op="score", rows=1, vocab=50257, masked=0, top_k=20, train=False, dtype="fp32"),
        # the decode batch's step: the chosen tokens' probabilities and some alternatives
        dict(name="score_step", op="score", rows=48, vocab=50304, masked=47, top_k=8, train=False, dtype="bf16"),
        # a policy-gradient batch at the GPT's training size: log probabilities and an entropy bonus, with gradient
        dict(name="score_policy_train", op="score", rows=16384, vocab=50304, masked=47, top_k=0, train=True,
             dtype="bf16"),
        # a small adapter's gradients, clipped
        dict(name="clip_adapter", op="clip", layout="ragged", tensors=12, total=98_765, clipped=True, out="fp32",
             dtype="bf16"),
        # the GPT's own gradients in place on an ordinary step: the norm is below the limit
        dict(name="clip_gpt_in_place", op="clip", layout="gpt", tensors=38, total=127_000_000, clipped=False, out="",
             dtype="fp32"),
        # 16-bit gradients of odd sizes clipped into the optimiser's 32-bit buffers
        dict(name="clip_odd_to_fp32", op="clip", layout="ragged", tensors=60, total=40_000_003, clipped=True,
             out="fp32", dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "write", "score", "score", "clip"])
    while True:
        if op == "decode":
            kv = rng.choice([1, 2, 3, 4, 8, 16])
            c = dict(op=op, seqs=_log_int(rng, 1, 200), heads=kv * rng.choice([1, 1, 2, 4, 5, 8]), kv_heads=kv,
                     head_dim=rng.choice([64, 64, 128, 128, 48, 80]), page=rng.choice([16, 16, 32, 64, 128, 24]),
                     longest=_log_int(rng, 1, 131072), window=0, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
            c["shortest"] = rng.choice([0, 1, c["longest"] // 3, c["longest"]])
            if rng.random() < 0.25:
                c["window"] = _log_int(rng, 1, max(1, c["longest"]))
            # the cache that a state holds and the padded 32-bit copy of the plain form stay within the largest case's
            if c["seqs"] * c["longest"] * kv * c["head_dim"] > 6 * 131072 * 4 * 128:
                continue
        elif op == "write":
            kv = rng.choice([1, 2, 4, 8, 16])
            c = dict(op=op, tokens=_log_int(rng, 1, 16389), heads=kv * rng.choice([1, 2, 4]), kv_heads=kv,
                     head_dim=rng.choice([64, 64, 128, 48, 80]), page=rng.choice([16, 32, 64, 24]), padding=0,
                     dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
            c["padding"] = rng.choice([0, 0, c["tokens"] // 7])
            if c["heads"] * c["head_dim"] > 4096:
                continue
        elif op == "score":
            c = dict(op=op, rows=_log_int(rng, 1, 16384), vocab=rng.choice([50304, 50257, _log_int(rng, 40, 131072)]),
                     masked=0, top_k=rng.choice([0, 1, 5, 8, 20, 32]), train=rng.random() < 0.5,
                     dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
            c["masked"] = rng.choice([0, c["vocab"] // 1000, c["vocab"] // 3])
        else:
            c = dict(op=op, layout="ragged", tensors=_log_int(rng, 1, 60), total=_log_int(rng, 1000, 127_000_000),
                     clipped=rng.random() < 0.7, out="", dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]))
            if c["clipped"]:
                c["out"] = "fp32"  # in place a second pass would find its own clipped result
        if work(c)["bytes"] <= LARGEST:
            return c


# ------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------
def _lengths(c):
    """Cache lengths spread over [shortest, longest], the longest first (they go by the case, not the seed)."""
    lo, hi = c["shortest"], c["longest"]
    return [hi] + [lo + int((hi - lo + 1) * ((i * _GOLDEN) % 1.0)) for i in range(1, c["seqs"])]


def _sizes(c):
    """Element counts of the gradient tensors of a clip case."""
    if c["layout"] == "gpt":  # d_model 1024, 6 layers, 16 heads, tied 50,304-row embedding
        d = 1024
        return [50304 * d] + [d * d * 3, d * d, 16, d, 4 * d * d, 4 * d * d] * 6 + [d]
    r = random.Random(c["tensors"] * 1_000_003 + c["total"])
    parts = [math.exp(r.uniform(0.0, 6.0)) for _ in range(c["tensors"])]
    scale = c["total"] / sum(parts)
    return [max(1, int(p * scale)) for p in parts]


def _rand(gen, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)


def _unit(x):
    return x / x.square().sum(-1, keepdim=True).sqrt()


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPE[c["dtype"]]
    if c["op"] == "decode":
        S, page, Hkv, D = c["seqs"], c["page"], c["kv_heads"], c["head_dim"]
        lens = _lengths(c)
        pages_of = [-(-n // page) for n in lens]
        width = max(1, max(pages_of))
        P = sum(pages_of) + 3
        order = torch.randperm(P, generator=gen, device="cuda", dtype=torch.int64)
        counts = torch.tensor(pages_of, device="cuda")
        used = torch.arange(width, device="cuda")[None, :] < counts[:, None]
        table = torch.full((S, width), -1, dtype=torch.int32, device="cuda")
        table[used] = order[:sum(pages_of)].to(torch.int32)
        k = torch.empty((P, Hkv, page, D), dtype=dt, device="cuda")
        v = torch.empty((P, Hkv, page, D), dtype=dt, device="cuda")
        for at in range(0, P, 4096):  # keys on the unit sphere, as the model's cache holds them
            n = min(4096, P - at)
            k[at:at + n] = _unit(torch.randn((n, Hkv, page, D), generator=gen, device="cuda")).to(dt)
            v[at:at + n] = torch.randn((n, Hkv, page, D), generator=gen, device="cuda").to(dt)
        # slots that no token has filled hold whatever was in memory: not a number, at worst
        fill = torch.zeros(P, dtype=torch.int64, device="cuda")
        n = torch.tensor(lens, device="cuda")[:, None] - torch.arange(width, device="cuda")[None, :] * page
        fill[table[used].long()] = n.clamp(0, page)[used]
        empty = torch.arange(page, device="cuda")[None, :] >= fill[:, None]
        k.masked_fill_(empty[:, None, :, None], float("nan"))
        v.masked_fill_(empty[:, None, :, None], float("nan"))
        q = _unit(torch.randn((S, c["heads"], D), generator=gen, device="cuda")).to(dt)
        scale = 4.0 + 8.0 * torch.rand(c["heads"], generator=gen, device="cuda")
        return dict(case=c, q=q, k=k, v=v, table=table, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                    scale=scale)
    if c["op"] == "write":
        N, page, H, Hkv, D = c["tokens"], c["page"], c["heads"], c["kv_heads"], c["head_dim"]
        P = -(-N // page) + 3
        qkv = _rand(gen, (N, (H + 2 * Hkv) * D), dt)
        slots = torch.randperm(P * page, generator=gen, device="cuda")[:N]
        if c["padding"]:
            slots[N - c["padding"]:] = -1
        positions = torch.randint(0, 32768, (N,), generator=gen, device="cuda")
        ang = torch.arange(32768, dtype=torch.float32, device="cuda")[:, None] * (
            10000.0 ** (-torch.arange(D // 2, dtype=torch.float32, device="cuda") / (D // 2)))[None, :]
        k, v = (torch.zeros((P, Hkv, page, D), dtype=dt, device="cuda") for _ in range(2))
        return dict(case=c, qkv=qkv, slots=slots, positions=positions, cos=ang.cos(), sin=ang.sin(), k=k, v=v)
    if c["op"] == "score":
        N, V, live = c["rows"], c["vocab"], c["vocab"] - c["masked"]
        logits = torch.empty((N, V), dtype=dt, device="cuda")
        # log-frequencies of a Zipf vocabulary in another order each seed, plus what the row adds
        base = -1.1 * torch.log(1.0 + torch.randperm(V, generator=gen, device="cuda").float())
        for at in range(0, N, 1024):
            n = min(1024, N - at)
            logits[at:at + n] = (base + 2.0 * torch.randn((n, V), generator=gen, device="cuda")).to(dt)
        logits[:, live:] = float("-inf")  # rows that only pad the output head
        targets = torch.randint(0, live, (N,), generator=gen, device="cuda")
        s = dict(case=c, logits=logits, targets=targets)
        if c["train"]:
            logits.requires_grad_(True)
            s["g_logp"] = torch.randn(N, generator=gen, device="cuda") / N
            s["g_entropy"] = torch.full((N,), -0.01 / N, device="cuda")
            s["g_top"] = torch.randn((N, c["top_k"]), generator=gen, device="cuda") / N
        return s
    grads = [_rand(gen, (n,), dt, 1e-3 * (1 + i % 5)) for i, n in enumerate(_sizes(c))]
    size = math.sqrt(sum(n * (1e-3 * (1 + i % 5)) ** 2 for i, n in enumerate(_sizes(c))))
    s = dict(case=c, grads=grads, limit=0.3 * size if c["clipped"] else 3.0 * size)
    s["out"] = [torch.empty_like(g, dtype=_DTYPE[c["out"]]) for g in grads] if c["out"] else None
    return s


# ------------------------------------------------------------------------------------------------
# One pass
# ------------------------------------------------------------------------------------------------
def run(state):
    c = state["case"]
    return (_own if own else _plain)[c["op"]](state)


def _own_decode(s):
    from quantumdlblocks_b200 import paged_born_attention

    return paged_born_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], s["scale"], eps=EPS,
                                window_size=s["case"]["window"])


def _own_write(s):
    from quantumdlblocks_b200 import paged_qkv_write

    q = paged_qkv_write(s["qkv"], s["cos"], s["sin"], s["positions"], s["slots"], s["k"], s["v"], s["case"]["heads"],
                        eps=EPS)
    return q, s["k"], s["v"]


def _own_score(s):
    from quantumdlblocks_b200 import token_logprobs

    x = s["logits"]
    r = token_logprobs(x, s["targets"], top_k=s["case"]["top_k"])
    if not s["case"]["train"]:
        return r.logp, r.entropy, r.top_logp, r.top_index
    (dx,) = torch.autograd.grad([r.logp, r.entropy, r.top_logp], [x], [s["g_logp"], s["g_entropy"], s["g_top"]])
    return r.logp.detach(), r.entropy.detach(), r.top_logp.detach(), r.top_index, dx


def _own_clip(s):
    from quantumdlblocks_b200 import clip_grad_norm_

    norm = clip_grad_norm_(s["grads"], s["limit"], out=s["out"])
    return norm, s["out"] if s["out"] is not None else s["grads"]


def _plain_decode(s):
    c, q, table, lens = s["case"], s["q"], s["table"], s["lens"]
    S, H, D = q.shape
    P, Hkv, page, _ = s["k"].shape
    G, L = H // Hkv, table.shape[1] * page
    at = torch.arange(L, device=q.device)[None, :]
    ok = at < lens[:, None]
    if c["window"]:
        ok = ok & (lens[:, None] - 1 - at < c["window"])
    rows = table.clamp(min=0).long()
    k = s["k"][rows].float().transpose(1, 2).reshape(S, Hkv, L, D)
    a = torch.matmul(q.float().view(S, Hkv, G, D) * s["scale"].view(1, Hkv, G, 1), k.transpose(2, 3))
    del k
    p = torch.where(ok[:, None, None, :] & (a > 0), a * a, torch.zeros((), device=q.device))
    v = s["v"][rows].float().transpose(1, 2).reshape(S, Hkv, L, D)
    v = torch.where(ok[:, None, :, None], v, torch.zeros((), device=q.device))
    o = torch.matmul(p, v) / (p.sum(-1, keepdim=True) + EPS)
    return o.reshape(S, H, D).to(q.dtype)


def _plain_write(s):
    c = s["case"]
    N, H, Hkv, D = c["tokens"], c["heads"], c["kv_heads"], c["head_dim"]
    x = s["qkv"].float().view(N, H + 2 * Hkv, D)
    qk, v = x[:, :H + Hkv], x[:, H + Hkv:]
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
    x1, x2 = qk[..., :D // 2], qk[..., D // 2:]
    r = torch.cat([x1 * cos - x2 * sin, x1 * sin + x2 * cos], dim=-1)
    r = r * torch.rsqrt(r.square().sum(-1, keepdim=True) + EPS)
    keep = s["slots"][:N - c["padding"]]  # the padding is at the end
    page, off = keep // c["page"], keep % c["page"]
    s["k"][page, :, off] = r[:N - c["padding"], H:].to(s["k"].dtype)
    s["v"][page, :, off] = v[:N - c["padding"]].to(s["v"].dtype)
    return r[:, :H].to(s["qkv"].dtype), s["k"], s["v"]


def _plain_score(s):
    c, t = s["case"], s["targets"][:, None]
    K = c["top_k"]
    x = s["logits"].detach().float()
    m = x.max(dim=1, keepdim=True).values
    e = torch.exp(x - m)
    z = e.sum(dim=1, keepdim=True)
    lse = m + torch.log(z)
    live = x > float("-inf")
    logp_all = torch.where(live, x - lse, torch.zeros((), device=x.device))
    p = e / z
    entropy = -(p * logp_all).sum(dim=1)
    logp = (x.gather(1, t) - lse)[:, 0]
    if K:
        values, index = torch.sort(x, dim=1, descending=True, stable=True)
        index = index[:, :K].contiguous()
        top = values[:, :K] - lse
        del values
    else:
        index = torch.empty((x.shape[0], 0), dtype=torch.int64, device=x.device)
        top = torch.empty((x.shape[0], 0), device=x.device)
    if not c["train"]:
        return logp, entropy, top, index
    g, gh, gt = s["g_logp"][:, None], s["g_entropy"][:, None], s["g_top"]
    dx = -p * (g + gt.sum(dim=1, keepdim=True) + gh * (logp_all + entropy[:, None]))
    dx.scatter_add_(1, t, g)
    if K:
        dx.scatter_add_(1, index, gt)
    return logp, entropy, top, index, dx.to(s["logits"].dtype)


def _plain_clip(s):
    norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
    c = torch.clamp(s["limit"] / (norm + 1e-6), max=1.0)
    to = s["out"] if s["out"] is not None else s["grads"]
    torch._foreach_copy_(list(to), [g.float() * c for g in s["grads"]])
    return norm, to


_own = dict(decode=_own_decode, write=_own_write, score=_own_score, clip=_own_clip)
_plain = dict(decode=_plain_decode, write=_plain_write, score=_plain_score, clip=_plain_clip)


# ------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(case):
    c, b = case, _BYTES[case["dtype"]]
    if c["op"] == "decode":
        keys = sum(min(n, c["window"]) if c["window"] else n for n in _lengths(c))
        qo = 2 * c["seqs"] * c["heads"] * c["head_dim"] * b
        pages = 4 * sum(-(-n // c["page"]) for n in _lengths(c))
        return dict(bytes=2 * keys * c["kv_heads"] * c["head_dim"] * b + qo + pages + 4 * c["seqs"],
                    flops=4 * keys * c["heads"] * c["head_dim"])
    if c["op"] == "write":
        n = c["tokens"] * (c["heads"] + 2 * c["kv_heads"]) * c["head_dim"]
        tables = c["tokens"] * c["head_dim"] * 4
        return dict(bytes=2 * n * b + tables + 16 * c["tokens"], flops=10 * n)
    if c["op"] == "score":
        n = c["rows"] * c["vocab"]
        return dict(bytes=n * b * (2 if c["train"] else 1) + c["rows"] * (16 + 12 * c["top_k"]),
                    flops=n * (10 if c["train"] else 5))
    n = sum(_sizes(c))
    return dict(bytes=n * b + (n * _BYTES[c["out"]] if c["out"] else n * b if c["clipped"] else 0), flops=3 * n)


# ------------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["op"] == "decode":
        S, H, D = s["q"].shape
        G = H // c["kv_heads"]
        out = torch.zeros((S, H, D), dtype=torch.float64, device="cuda")
        for i, n in enumerate(_lengths(c)):
            first = max(0, n - c["window"]) if c["window"] else 0
            if n == 0:
                continue
            pages = s["table"][i, :-(-n // c["page"])].long()
            for h in range(c["kv_heads"]):
                k = s["k"][pages, h].reshape(-1, D)[first:n].double()
                v = s["v"][pages, h].reshape(-1, D)[first:n].double()
                a = (s["q"][i, h * G:(h + 1) * G].double() @ k.T) * s["scale"][h * G:(h + 1) * G].double()[:, None]
                w = a.clamp(min=0) ** 2
                out[i, h * G:(h + 1) * G] = (w @ v) / (w.sum(1, keepdim=True) + EPS)
        return out
    if c["op"] == "write":
        N, H, Hkv, D = c["tokens"], c["heads"], c["kv_heads"], c["head_dim"]
        half = D // 2
        turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"]]
        rows = s["qkv"].double().reshape(N, H + 2 * Hkv, D)
        z = torch.complex(rows[:, :H + Hkv, :half], rows[:, :H + Hkv, half:]) * turn[:, None]
        z = z / torch.sqrt((z.real ** 2 + z.imag ** 2).sum(-1, keepdim=True) + EPS)
        qk = torch.cat([z.real, z.imag], dim=-1)
        k, v = s["k"].double(), s["v"].double()
        kf, vf = k.transpose(1, 2).reshape(-1, Hkv, D), v.transpose(1, 2).reshape(-1, Hkv, D)
        live = s["slots"] >= 0
        kf[s["slots"][live]] = qk[live, H:]
        vf[s["slots"][live]] = rows[live, H + Hkv:]
        shape = (-1, c["page"], Hkv, D)
        return qk[:, :H], kf.reshape(shape).transpose(1, 2), vf.reshape(shape).transpose(1, 2)
    if c["op"] == "score":
        N, K = c["rows"], c["top_k"]
        x32 = s["logits"].detach()
        logp, ent, top = [], [], []
        dx = torch.empty((N, c["vocab"]), dtype=torch.float64, device="cuda") if c["train"] else None
        for at in range(0, N, 512):
            x = x32[at:at + 512].double()
            ls = torch.log_softmax(x, dim=1)
            p = ls.exp()
            h = -torch.special.xlogy(p, p).sum(1)
            t = s["targets"][at:at + 512]
            logp.append(ls[torch.arange(len(t), device="cuda"), t])
            ent.append(h)
            best = torch.sort(ls, dim=1, descending=True, stable=True)
            top.append(best.values[:, :K].clone())
            if c["train"]:
                g, gh, gt = (s[n][at:at + 512].double() for n in ("g_logp", "g_entropy", "g_top"))
                d = torch.zeros_like(p)
                d[torch.arange(len(t), device="cuda"), t] += g
                d.scatter_add_(1, best.indices[:, :K], gt)
                d -= p * (g + gt.sum(1))[:, None]
                d -= gh[:, None] * (torch.special.xlogy(p, p) + p * h[:, None])
                dx[at:at + 512] = d
        r = (torch.cat(logp), torch.cat(ent), torch.cat(top), None)
        return r + (dx,) if c["train"] else r
    norm = torch.sqrt(sum((g.double() ** 2).sum() for g in s["grads"]))
    f = min(1.0, s["limit"] / (float(norm) + 1e-6))
    return norm, [g.double() * f for g in s["grads"]]
