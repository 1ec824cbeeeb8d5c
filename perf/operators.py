"""Rotary positions, a paged KV cache and the attention over it: what is timed, and in plain torch what it computes.

Four operators, used in this order by a decoder that reads a prompt in chunks and then writes tokens:
  rope         rotary positions of packed rows [tokens, heads, dim]
  kv_append    new keys and values into a paged cache, keys (and the queries beside them) rotated on the way
  attn_paged   attention of each sequence's new tokens over its pages (a prompt's chunk, or one token)
  attn_packed  attention inside packed documents without a cache (a prompt encoded in one go)

With ``own`` false ``run`` computes them from elementary torch operations in 32 bits (angles in 64: a far position
times a frequency loses its fraction of a turn in 32); with ``own`` true it calls the framework.
"""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
DEVICE = "cuda"


# ---------------------------------------------------------------- cases
def listed():
    """Head counts 32/8 of 128 are the text decoder's; the rest are generic."""
    return [
        # One decoded token per sequence of a small batch: launch latency.
        dict(name="rope_tokens", op="rope", dtype="fp16", tokens=4, heads=32, dim=128, rot=128, interleaved=False,
             far=4096, stretch=1.0),
        # A long prompt's queries, the interleaved layout, frequencies stretched for positions past 100000.
        dict(name="rope_prompt", op="rope", dtype="bf16", tokens=16384, heads=32, dim=128, rot=128, interleaved=True,
             far=262144, stretch=8.0),
        # Only part of the head is rotated, fp32 activations, an odd number of rows.
        dict(name="rope_partial", op="rope", dtype="fp32", tokens=3331, heads=20, dim=96, rot=32, interleaved=False,
             far=20000, stretch=1.0),
        # A decode batch's new keys and values, queries rotated in the same call.
        dict(name="append_tokens", op="kv_append", dtype="fp16", heads=32, kv_heads=8, dim=128, rot=128, page=16,
             batch=64, q_lo=1, q_hi=1, ctx_lo=100, ctx_hi=8000, spread=1, interleaved=False, stretch=1.0),
        # Chunks of several prompts on their way into the cache.
        dict(name="append_chunks", op="kv_append", dtype="bf16", heads=32, kv_heads=8, dim=128, rot=128, page=64,
             batch=6, q_lo=1000, q_hi=4096, ctx_lo=0, ctx_hi=16000, spread=2, interleaved=False, stretch=4.0),
        # One sequence writes one token over about a thousand keys (the decoder's own context).
        dict(name="paged_token", op="attn_paged", dtype="fp16", heads=32, kv_heads=8, dim=128, page=16, batch=1,
             q_lo=1, q_hi=1, ctx_lo=1023, ctx_hi=1023, spread=3, causal=True, softcap=0.0, window=0, slopes=False,
             prefix=False),
        # A serving batch, one token each, ragged contexts.
        dict(name="paged_batch", op="attn_paged", dtype="bf16", heads=32, kv_heads=8, dim=128, page=16, batch=96,
             q_lo=1, q_hi=1, ctx_lo=500, ctx_hi=16000, spread=4, causal=True, softcap=0.0, window=0, slopes=False,
             prefix=False),
        # A few tokens per sequence (drafts being checked), capped scores, a sliding window.
        dict(name="paged_drafts", op="attn_paged", dtype="fp16", heads=32, kv_heads=8, dim=128, page=32, batch=24,
             q_lo=3, q_hi=9, ctx_lo=200, ctx_hi=9000, spread=5, causal=True, softcap=30.0, window=4096, slopes=False,
             prefix=False),
        # A prompt's chunk over a long cache.
        dict(name="paged_chunk", op="attn_paged", dtype="bf16", heads=32, kv_heads=8, dim=128, page=64, batch=1,
             q_lo=2048, q_hi=2048, ctx_lo=63000, ctx_hi=63000, spread=6, causal=True, softcap=0.0, window=0,
             slopes=False, prefix=False),
        # Chunks of several prompts at once, ragged, a bias by distance, narrow heads.
        dict(name="paged_chunks", op="attn_paged", dtype="fp16", heads=16, kv_heads=4, dim=64, page=16, batch=8,
             q_lo=100, q_hi=700, ctx_lo=0, ctx_hi=6000, spread=7, causal=True, softcap=0.0, window=0, slopes=True,
             prefix=False),
        # A batch of documents packed end to end, each attending inside itself.
        dict(name="packed_documents", op="attn_packed", dtype="bf16", heads=32, kv_heads=8, dim=128, batch=12,
             q_lo=50, q_hi=4000, ctx_lo=0, ctx_hi=0, spread=8, causal=True, softcap=0.0, window=0, slopes=False,
             prefix=False),
        # Documents with a prefix every token may read, scores capped.
        dict(name="packed_prefix", op="attn_packed", dtype="fp16", heads=24, kv_heads=24, dim=128, batch=3,
             q_lo=700, q_hi=2100, ctx_lo=0, ctx_hi=0, spread=9, causal=True, softcap=50.0, window=0, slopes=False,
             prefix=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(("rope", "kv_append", "attn_paged", "attn_paged", "attn_packed"))
    case = dict(op=op, spread=rng.randrange(1 << 30))
    if op in ("rope", "kv_append"):
        dim = rng.choice((64, 96, 128, 128, 256))
        case.update(dtype=rng.choice(("fp16", "bf16", "fp32")), dim=dim, rot=rng.choice((dim, dim, dim // 2, 32)),
                    interleaved=rng.random() < 0.5, stretch=rng.choice((1.0, 2.0, 8.0)))
        if op == "rope":
            case.update(tokens=_log_int(rng, 1, 16384), heads=rng.choice((1, 5, 8, 16, 24, 32)),
                        far=_log_int(rng, 1, 500000))
            del case["spread"]
        else:
            kv_heads = rng.choice((1, 2, 4, 8))
            case.update(kv_heads=kv_heads, heads=kv_heads * rng.choice((1, 2, 3, 4, 8)))
            case.update(page=rng.choice((8, 16, 24, 32, 64, 128)), batch=_log_int(rng, 1, 64))
            hi = 1 if rng.random() < 0.4 else _log_int(rng, 2, max(2, 16384 // case["batch"]))
            case.update(q_lo=(hi + 1) // 2, q_hi=hi, ctx_lo=0, ctx_hi=_log_int(rng, 1, 8000))
        limit = max(work(c)["bytes"] for c in listed() if c["op"] == op)
        while work(case)["bytes"] > limit:
            key = "tokens" if op == "rope" else "q_hi"
            case[key] = max(1, case[key] // 2)
            if op == "kv_append":
                case["q_lo"] = min(case["q_lo"], case["q_hi"])
                case["batch"] = max(1, case["batch"] - 1)
        return case
    kv_heads = rng.choice((1, 2, 4, 8, 8))
    group = rng.choice((1, 2, 3, 4, 4, 8))
    case.update(dtype=rng.choice(("fp16", "bf16")), kv_heads=kv_heads, heads=kv_heads * group,
                dim=rng.choice((64, 128, 128)), causal=rng.random() < 0.85,
                softcap=rng.choice((0.0, 0.0, 0.0, 20.0, 50.0)), window=rng.choice((0, 0, 0, _log_int(rng, 1, 4096))),
                slopes=rng.random() < 0.25, prefix=rng.random() < 0.2)
    if op == "attn_paged":
        case.update(page=rng.choice((8, 16, 16, 24, 32, 64, 128, 256)), batch=_log_int(rng, 1, 96))
        q_hi = rng.choice((1, 1, _log_int(rng, 2, 16), _log_int(rng, 16, 2048)))
        ctx_hi = _log_int(rng, 1, 64000)
        case.update(q_lo=(q_hi + 2) // 3, q_hi=q_hi, ctx_lo=rng.randrange(ctx_hi), ctx_hi=ctx_hi)
    else:
        case.update(batch=_log_int(rng, 1, 32), q_lo=1, q_hi=_log_int(rng, 2, 6000), ctx_lo=0,
                    ctx_hi=rng.choice((0, 0, 0, _log_int(rng, 1, 1000))))
    tops = [work(c) for c in listed() if c["op"] == op]
    bytes_, flops = max(w["bytes"] for w in tops), max(w["flops"] for w in tops)
    while True:
        w = work(case)
        if w["bytes"] <= bytes_ and w["flops"] <= flops:
            return case
        for key in ("batch", "ctx_lo", "ctx_hi", "q_hi"):
            case[key] = max(0 if key.startswith("ctx") else 1, case[key] * 2 // 3)
        case["q_lo"] = min(case["q_lo"], case["q_hi"])


def _sequences(case):
    """Per sequence: (new tokens, cached keys before them). The same for every seed."""
    rng = random.Random(case["spread"])
    return [(rng.randint(case["q_lo"], case["q_hi"]), rng.randint(case["ctx_lo"], case["ctx_hi"]))
            for _ in range(case["batch"])]


def _prefixes(case, seqs):
    rng = random.Random(case["spread"] + 1)
    return [rng.randint(0, n + c) for n, c in seqs] if case["prefix"] else [0] * len(seqs)


# ---------------------------------------------------------------- work
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"]
        return {"bytes": 2 * n * case["dim"] * size + 8 * case["tokens"], "flops": 3 * n * case["rot"]}
    seqs = _sequences(case)
    tokens = sum(n for n, _ in seqs)
    if case["op"] == "kv_append":
        rows = tokens * (case["heads"] + 2 * case["kv_heads"])
        return {"bytes": 2 * rows * case["dim"] * size,
                "flops": 3 * tokens * (case["heads"] + case["kv_heads"]) * case["rot"]}
    keys = pairs = 0
    for (n, ctx), pre in zip(seqs, _prefixes(case, seqs)):
        i = torch.arange(n, dtype=torch.int64) + ctx
        hi = torch.full_like(i, n + ctx) if not case["causal"] else torch.clamp(i + 1, min=pre)
        lo = torch.clamp(i - case["window"] + 1, min=0) if case["window"] else torch.zeros_like(i)
        pairs += int((hi - lo).clamp(min=0).sum())
        keys += int(hi.max() - lo.min())
    elems = 2 * tokens * case["heads"] + 2 * keys * case["kv_heads"]
    return {"bytes": elems * case["dim"] * size, "flops": 4 * pairs * case["heads"] * case["dim"]}


# ---------------------------------------------------------------- inputs
def _randn(gen, shape, dtype, gain=1.0):
    x = torch.randn(shape, generator=gen, device=DEVICE, dtype=dtype)
    return x if gain == 1.0 else x.mul_(gain)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEVICE)


def _starts(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def _inv_freq(case):
    rot = case["rot"]
    f = 1.0 / (1000000.0 ** (torch.arange(0, rot, 2, dtype=torch.float64) / rot)) / case["stretch"]
    return f.to(device=DEVICE, dtype=torch.float32)


def _mscale(case):
    return 0.1 * math.log(case["stretch"]) + 1.0


def _pages(gen, case, seqs, dtype):
    """A pool of pages somewhat larger than the sequences need, and each sequence's pages in no order."""
    need = [-(-(n + c) // case["page"]) for n, c in seqs]
    total = sum(need) + 4
    shape = (total, case["page"], case["kv_heads"], case["dim"])
    order = torch.randperm(total, generator=gen, device=DEVICE).to(torch.int32)
    table = torch.zeros((len(seqs), max(max(need), 1)), dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return _randn(gen, shape, dtype), _randn(gen, shape, dtype), table


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    st = {"case": case}
    if own:
        from __graft_entry__ import load_package
        st["ops"] = load_package().ops
    if case["op"] == "rope":
        st["x"] = _randn(gen, (case["tokens"], case["heads"], case["dim"]), dtype)
        st["positions"] = torch.randint(0, case["far"], (case["tokens"],), generator=gen, device=DEVICE)
        st["inv_freq"], st["mscale"] = _inv_freq(case), _mscale(case)
        return st
    seqs = _sequences(case)
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    counts = [n for n, _ in seqs]
    st["seqs"] = seqs
    st["starts"] = _starts(counts)
    tokens = st["starts"][-1]
    st["cu_q"] = _ints(st["starts"])
    if case["op"] == "kv_append":
        # q, k and v as one projection writes them
        qkv = _randn(gen, (tokens, H + 2 * Hk, D), dtype)
        st["q"], st["k"], st["v"] = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
        st["k_cache"], st["v_cache"], st["table"] = _pages(gen, case, seqs, dtype)
        st["lengths"] = _ints([n + c for n, c in seqs])
        st["inv_freq"], st["mscale"] = _inv_freq(case), _mscale(case)
        return st
    st["q"] = _randn(gen, (tokens, H, D), dtype, 2.0)
    st["prefixes"] = _prefixes(case, seqs)
    st["prefix"] = _ints(st["prefixes"]) if case["prefix"] else None
    st["slopes"] = None
    if case["slopes"]:
        st["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device=DEVICE)
    st["max_q"] = max(counts)
    if case["op"] == "attn_paged":
        st["k_cache"], st["v_cache"], st["table"] = _pages(gen, case, seqs, dtype)
        st["lengths"] = _ints([n + c for n, c in seqs])
    else:
        st["k_starts"] = _starts([n + c for n, c in seqs])
        st["cu_k"] = _ints(st["k_starts"])
        st["k"] = _randn(gen, (st["k_starts"][-1], Hk, D), dtype)
        st["v"] = _randn(gen, (st["k_starts"][-1], Hk, D), dtype)
    return st


# ---------------------------------------------------------------- plain forms
def _rotate(x, positions, st):
    case = st["case"]
    rot, half = case["rot"], case["rot"] // 2
    angle = positions.to(torch.float64)[:, None] * st["inv_freq"].to(torch.float64)[None, :]
    cos = (torch.cos(angle) * st["mscale"]).to(torch.float32)[:, None, :]
    sin = (torch.sin(angle) * st["mscale"]).to(torch.float32)[:, None, :]
    f = x.to(torch.float32)
    out = f.clone()
    if case["interleaved"]:
        a, b = f[..., 0:rot:2], f[..., 1:rot:2]
        out[..., 0:rot:2] = a * cos - b * sin
        out[..., 1:rot:2] = a * sin + b * cos
    else:
        a, b = f[..., :half], f[..., half:rot]
        out[..., :half] = a * cos - b * sin
        out[..., half:rot] = a * sin + b * cos
    return out.to(x.dtype)


def _attend(q, k, v, st, first, prefix, slopes):
    """q [n, G, D] at positions first.. of one kv head, k and v [m, D]."""
    case = st["case"]
    q, k, v = q.to(torch.float32), k.to(torch.float32), v.to(torch.float32)
    n, G, D = q.shape
    m = k.shape[0]
    s = (q.reshape(n * G, D) @ k.t()).view(n, G, m) * (1.0 / math.sqrt(D))
    if case["softcap"]:
        s = case["softcap"] * torch.tanh(s / case["softcap"])
    i = torch.arange(first, first + n, device=q.device)[:, None]
    j = torch.arange(m, device=q.device)[None, :]
    if slopes is not None:
        s = s - slopes[None, :, None] * (i - j).abs().to(torch.float32)[:, None, :]
    seen = torch.ones((n, m), dtype=torch.bool, device=q.device)
    if case["causal"]:
        seen = (j <= i) | (j < prefix)
    if case["window"]:
        seen = seen & (i - j < case["window"])
    s = s.masked_fill(~seen[:, None, :], float("-inf"))
    top = s.amax(dim=-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = torch.exp(s - top)
    total = p.sum(dim=-1, keepdim=True)
    o = (p.view(n * G, m) @ v).view(n, G, D)
    return torch.where(total > 0, o / total, torch.zeros_like(o))


def _attention(st):
    case = st["case"]
    G = case["heads"] // case["kv_heads"]
    q = st["q"]
    out = torch.zeros_like(q)
    for b, (n, ctx) in enumerate(st["seqs"]):
        m = n + ctx
        q0 = st["starts"][b]
        if case["op"] == "attn_paged":
            need = -(-m // case["page"])
            rows = st["table"][b, :need].long()
            k = st["k_cache"][rows].flatten(0, 1)[:m]
            v = st["v_cache"][rows].flatten(0, 1)[:m]
        else:
            k0 = st["k_starts"][b]
            k, v = st["k"][k0:k0 + m], st["v"][k0:k0 + m]
        step = max(1, (1 << 27) // max(m * G, 1))
        for h in range(case["kv_heads"]):
            hs = slice(h * G, (h + 1) * G)
            slopes = None if st["slopes"] is None else st["slopes"][hs]
            for t in range(0, n, step):
                e = min(n, t + step)
                o = _attend(q[q0 + t:q0 + e, hs], k[:, h], v[:, h], st, ctx + t, st["prefixes"][b], slopes)
                out[q0 + t:q0 + e, hs] = o.to(q.dtype)
    return out


def _slots(st):
    """Page and row inside it of every new token, and its position."""
    case = st["case"]
    seq = torch.repeat_interleave(torch.arange(len(st["seqs"]), device=DEVICE), st["cu_q"].diff().long(),
                                  output_size=st["starts"][-1])
    at = torch.arange(st["starts"][-1], device=DEVICE)
    positions = at - st["cu_q"][seq + 1].long() + st["lengths"][seq].long()
    return st["table"][seq, positions // case["page"]].long(), positions % case["page"], positions


def run(state):
    case = state["case"]
    if own:
        return _run_own(state)
    if case["op"] == "rope":
        return _rotate(state["x"], state["positions"], state)
    if case["op"] == "kv_append":
        page, row, positions = _slots(state)
        state["k_cache"][page, row] = _rotate(state["k"], positions, state)
        state["v_cache"][page, row] = state["v"]
        return {"q": _rotate(state["q"], positions, state), "k_cache": state["k_cache"], "v_cache": state["v_cache"]}
    return _attention(state)


def _run_own(st):
    case, ops = st["case"], st["ops"]
    if case["op"] == "rope":
        return ops.rope(st["x"], st["positions"], st["inv_freq"], interleaved=case["interleaved"], mscale=st["mscale"])
    if case["op"] == "kv_append":
        q = ops.kv_append(st["k"], st["v"], st["k_cache"], st["v_cache"], st["table"], st["cu_q"], st["lengths"],
                          inv_freq=st["inv_freq"], q=st["q"], interleaved=case["interleaved"], mscale=st["mscale"])
        return {"q": q, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}
    options = dict(causal=case["causal"], softcap=case["softcap"], window=case["window"], slopes=st["slopes"],
                   prefix=st["prefix"], max_q=st["max_q"])
    if case["op"] == "attn_paged":
        return ops.attn_paged(st["q"], st["k_cache"], st["v_cache"], st["table"], st["cu_q"], st["lengths"], **options)
    return ops.attn_packed(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"], **options)


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_rotation(x, positions, case, inv_freq):
    """Each rotated pair as a complex number times mscale exp(i angle)."""
    rot = case["rot"]
    turn = torch.polar(torch.full((len(positions), rot // 2), _mscale(case), dtype=torch.float64, device=DEVICE),
                       torch.outer(positions.double(), inv_freq.double()))
    x = x.double()
    if case["interleaved"]:
        z = torch.view_as_complex(x[..., :rot].unflatten(-1, (rot // 2, 2)).contiguous()) * turn[:, None]
        head = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(x[..., :rot // 2], x[..., rot // 2:rot]) * turn[:, None]
        head = torch.cat((z.real, z.imag), dim=-1)
    return torch.cat((head, x[..., rot:]), dim=-1)


def _exact_attention(st, case):
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    out = []
    for b, (n, ctx) in enumerate(st["seqs"]):
        m = n + ctx
        key = torch.arange(m, device=DEVICE)
        if case["op"] == "attn_paged":
            slot = st["table"][b, key // case["page"]].long() * case["page"] + key % case["page"]
            K, V = st["k_cache"].view(-1, Hk, D)[slot], st["v_cache"].view(-1, Hk, D)[slot]
        else:
            K, V = st["k"][st["k_starts"][b]:][:m], st["v"][st["k_starts"][b]:][:m]
        Q = st["q"][st["starts"][b]:st["starts"][b] + n]
        heads = []
        for h in range(H):
            k, v = K[:, h * Hk // H].double(), V[:, h * Hk // H].double()
            rows = []
            for r in range(0, n, 512):
                query = torch.arange(r, min(n, r + 512), device=DEVICE)[:, None] + ctx
                score = torch.einsum("id,jd->ij", Q[r:r + 512, h].double(), k) / D ** 0.5
                if case["softcap"]:
                    score = (score / case["softcap"]).tanh() * case["softcap"]
                if case["slopes"]:
                    score = score - 2.0 ** (-8.0 * (h + 1) / H) * (query - key).abs()
                hidden = torch.zeros_like(score, dtype=torch.bool)
                if case["causal"]:
                    hidden |= (key > query) & (key >= st["prefixes"][b])
                if case["window"]:
                    hidden |= query - key >= case["window"]
                score[hidden] = -math.inf
                weight = torch.exp(score - torch.logsumexp(score, dim=1, keepdim=True))
                rows.append(torch.nan_to_num(weight, nan=0.0) @ v)
            heads.append(torch.cat(rows) if rows else torch.zeros((0, D), dtype=torch.float64, device=DEVICE))
        out.append(torch.stack(heads, dim=1))
    return torch.cat(out)


def exact(case, seed):
    if case["op"] in ("attn_paged", "attn_packed") and work(case)["flops"] > 4e12:
        return None
    global own
    kept, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = kept
    if case["op"] == "rope":
        return _exact_rotation(st["x"], st["positions"], case, st["inv_freq"])
    if case["op"] == "kv_append":
        k_cache, v_cache = st["k_cache"].double(), st["v_cache"].double()
        q = torch.empty(st["q"].shape, dtype=torch.float64, device=DEVICE)
        for b, (n, ctx) in enumerate(st["seqs"]):
            r = slice(st["starts"][b], st["starts"][b] + n)
            where = torch.arange(ctx, ctx + n, device=DEVICE)
            slot = st["table"][b, where // case["page"]].long() * case["page"] + where % case["page"]
            k_cache.flatten(0, 1)[slot] = _exact_rotation(st["k"][r], where, case, st["inv_freq"])
            v_cache.flatten(0, 1)[slot] = st["v"][r].double()
            q[r] = _exact_rotation(st["q"][r], where, case, st["inv_freq"])
        return {"q": q, "k_cache": k_cache, "v_cache": v_cache}
    return _exact_attention(st, case)
