"""Measured cases of the serving operators: the 8-bit paged KV cache (store, attention) and sampling.

Each case is one call as a serving loop makes it.  ``run`` computes it in elementary torch operations, or, where
``own`` is set, with this package's operators.  Sizes are the head layouts of the predefined geometries (9/3, 15/5
and 32/32 heads of 64 dims), their vocabulary, contexts up to the decode kernels' limit, and odd ones around them.
"""
import math

import numpy as np
import torch

own = False

D = 64                                     # head dim of every geometry of the package
LAYOUTS = ((9, 3), (15, 5), (32, 32))      # (query heads, kv heads)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one request, the usual filters as plain numbers: the last step of a single-user loop (latency)
        {"name": "sample-1", "op": "sample", "rows": 1, "vocab": 49152, "dtype": "bf16", "temperature": 0.8, "top_k": 50,
         "top_p": 0.95, "min_p": 0.0, "per_row": False, "spread": 2.5},
        # a full decode batch, every request with settings of its own
        {"name": "sample-64", "op": "sample", "rows": 64, "vocab": 49152, "dtype": "bf16", "temperature": 1.0, "top_k": 400,
         "top_p": 0.9, "min_p": 0.02, "per_row": True, "spread": 2.0},
        # nucleus sampling over flat fp32 logits of an odd, larger vocabulary
        {"name": "sample-7-fp32", "op": "sample", "rows": 7, "vocab": 100003, "dtype": "fp32", "temperature": 1.3, "top_k": 0,
         "top_p": 0.97, "min_p": 0.0, "per_row": False, "spread": 1.0},
        # many rollouts at once, temperature and min-p only
        {"name": "sample-512", "op": "sample", "rows": 512, "vocab": 49152, "dtype": "fp16", "temperature": 0.9, "top_k": 0,
         "top_p": 1.0, "min_p": 0.05, "per_row": False, "spread": 3.0},
        # one token of one request into the cache
        {"name": "append-1", "op": "append", "batch": 1, "tokens": 1, "heads": "15/5", "context": 777, "block": 16,
         "planes": False},
        # one token of each of 64 requests, pages partly filled, K and V planes apart
        {"name": "append-64", "op": "append", "batch": 64, "tokens": 1, "heads": "32/32", "context": 2000, "block": 16,
         "planes": True},
        # ragged prompts, K and V read out of the fused projection's rows
        {"name": "append-prompts", "op": "append", "batch": 8, "tokens": 3000, "heads": "32/32", "context": 3000, "block": 32,
         "planes": False},
        # decode attention of one request with a short context (latency)
        {"name": "attend-1", "op": "attend", "batch": 1, "tokens": 1, "heads": "15/5", "context": 520, "block": 16,
         "planes": False, "lse": False},
        # decode attention of a full batch at the context limit: the cache is what costs
        {"name": "attend-64-long", "op": "attend", "batch": 64, "tokens": 1, "heads": "15/5", "context": 8192, "block": 16,
         "planes": False, "lse": False},
        # a kv head for each query head, planes layout
        {"name": "attend-16-mha", "op": "attend", "batch": 16, "tokens": 1, "heads": "32/32", "context": 3001, "block": 32,
         "planes": True, "lse": True},
        # a few tokens each: drafts being verified
        {"name": "attend-8-draft", "op": "attend", "batch": 8, "tokens": 5, "heads": "9/3", "context": 2047, "block": 16,
         "planes": False, "lse": True},
        # prompt chunks behind earlier context
        {"name": "attend-prompts", "op": "attend", "batch": 4, "tokens": 2048, "heads": "15/5", "context": 6144, "block": 16,
         "planes": False, "lse": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("sample", "append", "attend", "attend"))
    if op == "sample":
        per_row = rng.random() < 0.5
        vocab = _log(rng, 1000, 130000)
        return {"op": op, "rows": _log(rng, 1, min(512, 25_000_000 // vocab)), "vocab": vocab,
                "dtype": rng.choice(tuple(DTYPES)), "temperature": round(rng.uniform(0.3, 1.6), 3),
                "top_k": rng.choice((0, _log(rng, 1, 2000))), "top_p": rng.choice((1.0, round(rng.uniform(0.3, 0.999), 3))),
                "min_p": rng.choice((0.0, round(rng.uniform(0.001, 0.3), 4))), "per_row": per_row,
                "spread": round(rng.uniform(0.5, 4.0), 2)}
    heads = rng.choice(LAYOUTS)
    case = {"op": op, "heads": "%d/%d" % heads, "block": rng.choice((16, 32, 64)), "planes": rng.random() < 0.4}
    if op == "append":
        batch = _log(rng, 1, 64)
        tokens = rng.choice((1, 1, _log(rng, 2, 3000)))
        tokens = max(1, min(tokens, 900_000 // (batch * heads[1])))
        return {**case, "batch": batch, "tokens": tokens, "context": tokens + _log(rng, 1, 5000)}
    batch = _log(rng, 1, 64)
    tokens = rng.choice((1, 1, _log(rng, 2, 16), _log(rng, 17, 2000)))
    context = tokens + _log(rng, 1, 6000)
    while batch > 1 and (batch * context * heads[1] > 2_500_000 or batch * tokens * context * heads[0] > 700_000_000):
        batch = batch // 2
    tokens = max(1, min(tokens, 700_000_000 // (batch * context * heads[0])))
    return {**case, "batch": batch, "tokens": tokens, "context": context, "lse": rng.random() < 0.5}


def _heads(case):
    a, b = case["heads"].split("/")
    return int(a), int(b)


def _lengths(case):
    """New tokens and sequence length (new ones included) of each request: plain integers that depend on the case alone."""
    b, n, ctx = case["batch"], case["tokens"], case["context"]
    new = [n if n == 1 else max(1, n - (n * 5 * i) // (8 * b)) for i in range(b)]
    seq = [max(new[i], ctx - (ctx * 3 * i) // (4 * b)) for i in range(b)]
    return new, seq


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ceil_exponent(amax):
    """Biased exponent of the smallest power of two that is at least amax / 448 (0..254)."""
    m, e = torch.frexp(amax * np.float32(1 / 448).item())
    e = torch.where(m == 0.5, e - 1, e) + 127
    return torch.where(amax > 0, e.clamp(0, 254), torch.zeros_like(e))


def _cache(case, g, pages):
    """A cache with content: values e4m3, scales e8m0, the layout that the case asks for."""
    _, kvh = _heads(case)
    bs = case["block"]
    x = torch.randn((pages, kvh, bs, 2, D), generator=g, device="cuda", dtype=torch.bfloat16)
    gain = torch.exp(0.5 * torch.randn((pages, kvh, 1, 2, 1), generator=g, device="cuda"))
    x = x * gain.to(torch.bfloat16)
    e = _ceil_exponent(x.abs().amax(dim=(2, 4)).float())                                    # [pages, kvh, 2]
    x = (x * torch.exp2(127.0 - e.float()).to(torch.bfloat16)[:, :, None, :, None]).to(torch.float8_e4m3fn)
    if case["planes"]:
        cache = x.view(torch.uint8).permute(3, 0, 2, 1, 4).contiguous().view(torch.float8_e4m3fn)
    else:
        cache = x.view(pages, kvh, bs, 2 * D)
    return cache, e.to(torch.uint8).view(torch.float8_e8m0fnu)


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "sample":
        b = case["rows"]
        logits = (torch.randn((b, case["vocab"]), generator=g, device="cuda") * case["spread"]).to(DTYPES[case["dtype"]])
        uniform = torch.rand((b,), generator=g, device="cuda")
        knobs = {k: case[k] for k in ("temperature", "top_k", "top_p", "min_p")}
        if case["per_row"]:
            i = torch.arange(b, device="cuda")
            f = 0.5 + 0.5 * (i + 1) / b                                   # settings differ from request to request
            knobs = {"temperature": torch.where(i % 8 == 7, torch.zeros_like(f), case["temperature"] * f).float(),
                     "top_k": torch.where(i % 4 == 1, torch.zeros_like(i), (case["top_k"] * f).long() + (case["top_k"] > 0)).int(),
                     "top_p": torch.where(i % 4 == 2, torch.ones_like(f), case["top_p"] * f).float(),
                     "min_p": (case["min_p"] * f).float()}
        return {"case": case, "logits": logits, "uniform": uniform, "knobs": knobs}
    qh, kvh = _heads(case)
    bs, b = case["block"], case["batch"]
    new, seq = _lengths(case)
    cols = -(-max(seq) // bs)
    need = [-(-s // bs) for s in seq]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda")
    table = torch.full((b, cols), -1, dtype=torch.int32, device="cuda")
    at = 0
    for r in range(b):
        table[r, : need[r]] = order[at: at + need[r]].int()
        at += need[r]
    cache, scales = _cache(case, g, pages)
    total = sum(new)
    qkv = torch.randn((total, (qh + 2 * kvh) * D), generator=g, device="cuda", dtype=torch.bfloat16)
    q, k, v = (qkv[:, : qh * D].view(total, qh, D), qkv[:, qh * D: (qh + kvh) * D].view(total, kvh, D),
               qkv[:, (qh + kvh) * D:].view(total, kvh, D))
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")
    return {"case": case, "q": q, "k": k, "v": v, "cache": cache, "scales": scales, "table": table,
            "seq": torch.tensor(seq, dtype=torch.int32, device="cuda"), "cu": cu if case["tokens"] > 1 else None,
            "longest": max(new)}


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if case["op"] == "sample":
        if own:
            from prime_kernels_b200 import sampling

            return sampling.sample(state["logits"], state["uniform"], return_logprobs=True, **state["knobs"])
        return _sample(state)
    if own:
        from prime_kernels_b200 import kv8

        if case["op"] == "append":
            kv8.append(state["k"], state["v"], state["cache"], state["scales"], state["table"], state["seq"], state["cu"])
            return state["cache"], state["scales"]
        return kv8.attention(state["q"], state["cache"], state["scales"], state["table"], state["seq"], state["cu"],
                             max_query_len=state["longest"], return_lse=case["lse"])
    return _append(state) if case["op"] == "append" else _attend(state)


def _sample(state):
    """Sort, cumulate, mask and draw; sums in 64 bits, since a border moves with them."""
    logits, u = state["logits"], state["uniform"]
    b, v = logits.shape
    t, k, p, mp = (x if torch.is_tensor(x) else torch.full((b,), float(x), device="cuda") for x in
                   (state["knobs"][n] for n in ("temperature", "top_k", "top_p", "min_p")))
    x, order = torch.sort(logits.float(), dim=1, descending=True, stable=True)
    greedy = t <= 0
    w = torch.exp((x.double() - x[:, :1].double()) / torch.where(greedy, torch.ones_like(t), t).double()[:, None])
    rank = torch.arange(v, device="cuda")
    w = torch.where((k[:, None] > 0) & (rank >= k[:, None]), 0.0, w)
    before = w.cumsum(1) - w
    w = torch.where((p[:, None] < 1) & (before >= p.double()[:, None] * w.sum(1, keepdim=True)), 0.0, w)
    w = torch.where(w < mp.double()[:, None], 0.0, w)
    w = torch.where(greedy[:, None] & (rank > 0), 0.0, w)
    w = torch.zeros_like(w).scatter_(1, order, w)                          # back to the order of the vocabulary
    total = w.cumsum(1)
    ids = (total > u.double()[:, None] * total[:, -1:]).int().argmax(1)
    return ids, torch.log(w.gather(1, ids[:, None])[:, 0] / total[:, -1]).float()


def _places(state):
    """Request, position, page and slot of each new token."""
    case, seq = state["case"], state["seq"].long()
    b, total = case["batch"], state["k"].shape[0]
    if state["cu"] is None:
        r, j, n = torch.arange(b, device="cuda"), torch.zeros(b, dtype=torch.long, device="cuda"), torch.ones_like(seq)
    else:
        cu = state["cu"].long()
        i = torch.arange(total, device="cuda")
        r = torch.searchsorted(cu, i, right=True) - 1
        j, n = i - cu[r], cu[1:] - cu[:-1]
    pos = seq[r] - n[r] + j
    page = state["table"][r, pos // case["block"]].long()
    return r, pos, page, pos % case["block"], n


def _append(state):
    case, scales8 = state["case"], state["scales"].view(torch.uint8)
    bs = case["block"]
    r, pos, page, slot, n = _places(state)
    flat = state["cache"].view(torch.uint8)
    # [pages, kv heads, slots, 2, 64], a view of the cache in either layout
    view = flat.permute(1, 3, 2, 0, 4) if case["planes"] else flat.view(*flat.shape[:3], 2, D)
    x = torch.stack([state["k"], state["v"]], 2).float()                                    # [T, kvh, 2, 64]
    amax = x.abs().amax(-1)
    top = torch.zeros(scales8.shape, device="cuda").index_reduce_(0, page, amax, "amax", include_self=True)
    # the page that a request had begun before
    start = state["seq"].long() - n
    first, live = state["table"].gather(1, (start // bs)[:, None])[:, 0].long(), start % bs
    e = _ceil_exponent(top)
    old = scales8[first].int()
    grown = torch.where(live[:, None, None] > 0, torch.maximum(old, e[first]), e[first])
    kept = torch.arange(bs, device="cuda") < live[:, None]                                  # [B, slots]
    had = view[first]
    moved = (had.view(torch.float8_e4m3fn).float() * torch.exp2((old - grown).float())[:, :, None, :, None]).to(torch.float8_e4m3fn)
    view[first] = torch.where(kept[:, None, :, None, None], moved.view(torch.uint8), had)
    e = e.index_copy(0, first, grown)
    scales8[page] = e[page].to(torch.uint8)
    y = (x * torch.exp2(127.0 - e[page].float())[..., None]).to(torch.float8_e4m3fn)
    view[page, :, slot] = y.view(torch.uint8)
    return state["cache"], state["scales"]


def _attend(state):
    case = state["case"]
    qh, kvh = _heads(case)
    b, longest, bs = case["batch"], state["longest"], case["block"]
    table, seq = state["table"].long().clamp(min=0), state["seq"].long()
    span = table.shape[1] * bs
    p = torch.exp2(state["scales"].view(torch.uint8)[table].float() - 127.0)                # [B, cols, kvh, 2]
    flat = state["cache"].view(torch.uint8)
    view = flat.permute(1, 3, 2, 0, 4) if case["planes"] else flat.view(*flat.shape[:3], 2, D)
    kv = view[table].view(torch.float8_e4m3fn).float()                                      # [B, cols, kvh, bs, 2, 64]
    kv = kv * p[:, :, :, None, :, None]
    k, v = (kv[..., i, :].transpose(1, 2).reshape(b, kvh, 1, span, D) for i in (0, 1))
    cu = torch.arange(b + 1, device="cuda") if state["cu"] is None else state["cu"].long()
    n = cu[1:] - cu[:-1]
    i = torch.arange(longest, device="cuda")
    at = (cu[:-1, None] + i).clamp(max=state["q"].shape[0] - 1)                             # [B, longest]
    q = state["q"][at].float().view(b, longest, kvh, qh // kvh, D).permute(0, 2, 3, 1, 4)   # [B, kvh, G, longest, 64]
    s = (q @ k.transpose(-1, -2)) * D ** -0.5
    upto = (seq - n)[:, None] + i + 1
    s = s.masked_fill(torch.arange(span, device="cuda") >= upto[:, None, None, :, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    w = torch.exp(s - top)
    total = w.sum(-1, keepdim=True)
    o = ((w @ v) / total).permute(0, 3, 1, 2, 4).reshape(b, longest, qh, D)
    lse = (top + torch.log(total))[..., 0].permute(0, 3, 1, 2).reshape(b, longest, qh)
    rows = torch.arange(state["q"].shape[0], device="cuda")
    r = torch.searchsorted(cu, rows, right=True) - 1
    out = o[r, rows - cu[r]].to(torch.bfloat16)
    return (out, lse[r, rows - cu[r]]) if case["lse"] else out


# ------------------------------------------------------------------------------------------------ cost
def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["dtype"] == "fp32" else 2) + 16 * case["rows"], "flops": 4 * n}
    qh, kvh = _heads(case)
    new, seq = _lengths(case)
    total = sum(new)
    if case["op"] == "append":
        return {"bytes": total * kvh * D * 2 * (2 + 1) + 2 * kvh * sum(-(-n // case["block"]) for n in new),
                "flops": total * kvh * D * 2 * 3}
    pairs = sum(n * (s - n) + n * (n + 1) // 2 for n, s in zip(new, seq))
    return {"bytes": sum(seq) * kvh * 2 * D + total * qh * D * 2 * 2 + (4 * total * qh if case["lse"] else 0),
            "flops": 4 * D * qh * pairs}


# ------------------------------------------------------------------------------------------------ 64-bit definition
def _e4m3(x):
    """Nearest e4m3 value of doubles with |x| <= 448, ties to even: steps of 2^(e - 3), 2^-9 below 2^-6."""
    _, e = np.frexp(np.abs(x))
    step = np.exp2(np.maximum(e - 1, -6) - 3.0)
    return np.rint(x / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    return _exact_append(s) if case["op"] == "append" else _exact_attend(s)


def _exact_sample(s):
    x, u = s["logits"].double().cpu().numpy(), s["uniform"].double().cpu().numpy()
    knob = {k: (v.double().cpu().numpy() if torch.is_tensor(v) else np.full(len(u), np.float32(v), dtype=np.float64))
            for k, v in s["knobs"].items()}
    ids, logp = np.zeros(len(u), np.int64), np.zeros(len(u))
    for r in range(len(u)):
        t, k, p, mp = (knob[n][r] for n in ("temperature", "top_k", "top_p", "min_p"))
        if t <= 0:
            ids[r] = int(np.argmax(x[r]))
            continue
        order = np.argsort(-x[r], kind="stable")
        w = np.exp((x[r][order] - x[r][order[0]]) / t)
        keep = int(min(k, len(w))) if k > 0 else len(w)
        if p < 1:
            c = np.concatenate([[0.0], np.cumsum(w[:keep])])
            keep = max(1, int(np.searchsorted(c[:-1], p * c[-1], side="left")))
        keep = max(1, min(keep, int((w >= mp).sum())))
        kept = np.sort(order[:keep])
        w = np.exp((x[r][kept] - x[r][order[0]]) / t)
        c = np.cumsum(w)
        at = min(int(np.searchsorted(c, u[r] * c[-1], side="right")), keep - 1)
        ids[r], logp[r] = kept[at], math.log(w[at] / c[-1])
    return torch.from_numpy(ids), torch.from_numpy(logp)


def _exact_append(s):
    case, bs = s["case"], s["case"]["block"]
    _, kvh = _heads(case)
    new, seq = _lengths(case)
    table = s["table"].cpu().numpy()
    raw = s["cache"].float().cpu().numpy().astype(np.float64)
    held = raw.transpose(1, 3, 2, 0, 4).copy() if case["planes"] else raw.reshape(*raw.shape[:3], 2, D).copy()
    e = s["scales"].view(torch.uint8).cpu().numpy().astype(np.int64)
    x = torch.stack([s["k"], s["v"]], 2).double().cpu().numpy()
    at = 0
    for r, (n, length) in enumerate(zip(new, seq)):
        pos, done = length - n, 0
        while done < n:
            page, slot = table[r, (pos + done) // bs], (pos + done) % bs
            m = min(bs - slot, n - done)
            part = x[at + done: at + done + m]                                             # [m, kvh, 2, 64]
            top = (np.abs(part).max(axis=(0, 3)).astype(np.float32) * np.float32(1 / 448)).astype(np.float64)
            f, ex = np.frexp(top)
            want = np.where(top > 0, np.clip(np.where(f == 0.5, ex - 1, ex) + 127, 0, 254), 0)
            now = np.maximum(e[page], want) if slot else want
            if slot:
                held[page, :, :slot] = _e4m3(held[page, :, :slot] * np.exp2(e[page] - now)[:, None, :, None])
            held[page, :, slot: slot + m] = _e4m3(part * np.exp2(127.0 - now)[None, :, :, None]).transpose(1, 0, 2, 3)
            e[page] = now
            done += m
        at += n
    cache = held.transpose(3, 0, 2, 1, 4) if case["planes"] else held.reshape(raw.shape)
    return torch.from_numpy(np.ascontiguousarray(cache)), torch.from_numpy(np.exp2(e - 127.0))


def _exact_attend(s):
    case, bs = s["case"], s["case"]["block"]
    qh, kvh = _heads(case)
    new, seq = _lengths(case)
    outs, lses, at = [], [], 0
    for r, (n, length) in enumerate(zip(new, seq)):
        pages = s["table"][r, : -(-length // bs)].long()
        e = torch.exp2(s["scales"].view(torch.uint8)[pages].double() - 127.0)              # [n pages, kvh, 2]
        if case["planes"]:
            c = s["cache"].view(torch.uint8)[:, pages].view(torch.float8_e4m3fn).double()  # [2, pages, bs, kvh, 64]
            k, v = (c[i] * e[:, None, :, i, None] for i in (0, 1))
        else:
            c = s["cache"].view(torch.uint8)[pages].view(torch.float8_e4m3fn).double()     # [pages, kvh, bs, 128]
            k, v = (c[..., i * D: (i + 1) * D].transpose(1, 2) * e[:, None, :, i, None] for i in (0, 1))
        k, v = (t.reshape(-1, kvh, D)[:length] for t in (k, v))
        out, lse = [], []
        for h in range(qh):
            kv = h // (qh // kvh)
            a = s["q"][at: at + n, h].double() @ k[:, kv].T / math.sqrt(D)
            late = torch.arange(length, device="cuda")[None] > torch.arange(length - n, length, device="cuda")[:, None]
            a[late] = -math.inf
            z = torch.logsumexp(a, 1)
            out.append(torch.exp(a - z[:, None]) @ v[:, kv])
            lse.append(z)
        outs.append(torch.stack(out, 1))
        lses.append(torch.stack(lse, 1))
        at += n
    return (torch.cat(outs), torch.cat(lses)) if case["lse"] else torch.cat(outs)
