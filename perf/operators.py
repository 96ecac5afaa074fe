"""The paged key-value cache operators as workloads: what a server calls per layer.

  append   queries, keys and values of new tokens: optional RMS norm of every query and key
           head, rotary positions, keys and values stored in the pages of their sequence
  decode   one new token per sequence attends over the sequence's pages
  prefill  several new tokens per sequence (a prompt, or a chunk of one behind a cached
           context) attend over the pages, causally or with a bidirectional prefix

Scores are scale * q.k, then optionally cap * tanh(score / cap), then optionally
- slope[head] * |position of the query - position of the key|.  Query heads share key-value
heads in groups.  Sequences of a batch never see each other.

``own`` False: plain torch operations in 32 bits (angles in 64), rounded once at the end.
``own`` True: the framework's calls.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}

# Largest plain score tensor, in elements (queries x keys x heads, padded to the longest row).
MOST_SCORES = 8192 * 8192 * 32


def _case(name, op, **over):
    c = {"name": name, "op": op, "dtype": "bf16", "heads": 16, "kv_heads": 4, "head_dim": 128,
         "page": 64, "batch": 1, "new": 1, "context": 0, "mix": 0, "softcap": 0.0, "window": 0,
         "alibi": False, "prefix": False, "norm": True, "rope_dim": 128, "interleaved": False}
    return {**c, **over}


def listed():
    return [
        # the token of one conversation: launch latency
        _case("append_one_token", "append", context=513),
        # one step of a serving batch at mixed lengths, small pages, fp16
        _case("append_batch_step", "append", dtype="fp16", heads=32, kv_heads=8, page=16, batch=64,
              context=1000, mix=5, rope_dim=64, interleaved=True),
        # a ragged batch of prompts, a key-value head for every query head
        _case("append_prompts", "append", heads=16, kv_heads=16, batch=7, new=4096, mix=3),
        # a short conversation of a small model: launch latency
        _case("decode_short", "decode", heads=8, kv_heads=8, head_dim=64, page=16, context=300),
        # one very long conversation: the cache's length is the only parallel axis
        _case("decode_long", "decode", heads=32, kv_heads=4, context=131070),
        # a serving batch at mixed lengths with idle slots, capped scores, small pages
        _case("decode_batch", "decode", heads=32, kv_heads=8, page=16, batch=64, context=8191,
              mix=11, softcap=50.0),
        # many rows, no sharing of heads, distance bias, sliding window of the long-context layers
        _case("decode_window", "decode", dtype="fp16", kv_heads=16, batch=128, context=4000,
              mix=6, window=1024, alibi=True),
        # a few short prompts at once: latency
        _case("prefill_short", "prefill", heads=8, kv_heads=8, head_dim=64, page=16, batch=3,
              new=131, mix=7),
        # a chunk of a prompt behind a long cached context: few query rows, a long key axis
        _case("prefill_chunk", "prefill", heads=32, kv_heads=4, new=200, context=32568),
        # ragged prompts, capped scores, sliding window
        _case("prefill_ragged", "prefill", page=32, batch=8, new=4096, mix=9, softcap=30.0,
              window=1024),
        # bidirectional prefixes (prompt documents) with a distance bias, fp16
        _case("prefill_prefix", "prefill", dtype="fp16", heads=12, kv_heads=12, head_dim=64,
              page=128, batch=4, new=2000, context=777, mix=4, alibi=True, prefix=True),
        # one long prompt
        _case("prefill_long", "prefill", heads=32, kv_heads=8, new=8192),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "prefill"])
    dim = rng.choice([64, 128, 128])
    kv = rng.choice([1, 2, 4, 8, 16])
    group = rng.choice([1, 2, 4, 5, 7, 8] if kv <= 4 else [1, 2, 4] if kv <= 8 else [1, 2])
    c = _case("", op, dtype=rng.choice(["bf16", "fp16"]), heads=kv * group, kv_heads=kv,
              head_dim=dim, page=rng.choice([16, 32, 64, 128]), mix=rng.randrange(1, 1 << 20),
              softcap=rng.choice([0.0, 0.0, 20.0, 50.0]), alibi=rng.random() < 0.25,
              norm=rng.random() < 0.6, rope_dim=rng.choice([0, 32, 64, dim]),
              interleaved=rng.random() < 0.4)
    del c["name"]
    if op == "append":
        c["batch"] = _log_int(rng, 1, 128)
        c["new"] = rng.choice([1, _log_int(rng, 2, max(2, 16384 // c["batch"]))])
        c["context"] = _log_int(rng, 1, 1200)
    elif op == "decode":
        c["batch"] = _log_int(rng, 1, 128)
        c["context"] = _log_int(rng, 1, min(100000, 64 * 8192 * 8 // (c["batch"] * kv)))
        c["window"] = rng.choice([0, 0, _log_int(rng, 1, 4096)])
    else:
        c["batch"] = _log_int(rng, 1, 12)
        c["new"] = _log_int(rng, 2, 6000)
        most = MOST_SCORES // (2 * c["batch"] * c["heads"])
        c["new"] = min(c["new"], int(math.sqrt(most)))
        c["context"] = rng.choice([0, _log_int(rng, 1, max(1, min(30000, most // c["new"] - c["new"])))])
        c["prefix"] = rng.random() < 0.25
        c["window"] = 0 if c["prefix"] else rng.choice([0, 0, _log_int(rng, 1, 4096)])
    return c


def _lengths(case):
    """(new tokens, length with them) of every sequence: whole numbers that follow from the case."""
    r, b = random.Random(case["mix"]), case["batch"]
    new, context = case["new"], case["context"]
    if not case["mix"]:
        return [new] * b, [new + context] * b
    n = [new] + [max(1, int(new * r.random())) for _ in range(b - 1)]
    c = [context] + [int(context * r.uniform(0.05, 1.0)) for _ in range(b - 1)]
    total = [x + y for x, y in zip(n, c)]
    if case["op"] == "decode":  # idle slots of a serving batch
        total = [0 if i and r.random() < 0.06 else t for i, t in enumerate(total)]
    return n, total


def _prefixes(case):
    r = random.Random(case["mix"] + 1)
    n, total = _lengths(case)
    return [int(t * r.random()) for t in total] if case["prefix"] else [0] * len(total)


def prepare(case, seed):
    dev, dtype = "cuda", DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(int(seed))
    new, total = _lengths(case)
    b, page, hd = case["batch"], case["page"], case["head_dim"]
    h, kv = case["heads"], case["kv_heads"]
    need = [-(-t // page) for t in total]
    pages = sum(need) + 3
    width = max(need + [1])
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    first = torch.tensor([0] + need[:-1], device=dev).cumsum(0)
    col = torch.arange(width, device=dev)
    held = col[None, :] < torch.tensor(need, device=dev)[:, None]
    table = torch.where(held, order[(first[:, None] + col[None, :]).clamp(max=pages - 1)], -1)
    shape = (pages, kv, page, hd)
    i32 = dict(dtype=torch.int32, device=dev)
    s = {"case": dict(case), "table": table.to(torch.int32).contiguous(),
         "k_pages": torch.randn(shape, generator=g, device=dev).to(dtype),
         "v_pages": torch.randn(shape, generator=g, device=dev).to(dtype),
         "lengths": torch.tensor(total, **i32),
         "cu_q": torch.tensor([0] + new, device=dev).cumsum(0).to(torch.int32),
         "slopes": None, "prefix": None, "longest": max(new)}
    n = sum(new)
    if case["op"] == "append":
        # the rows of one fused projection: queries | keys | values
        rows = torch.randn(n, (h + 2 * kv) * hd, generator=g, device=dev).to(dtype)
        s["q"] = rows[:, :h * hd].view(n, h, hd)
        s["k"] = rows[:, h * hd:(h + kv) * hd].view(n, kv, hd)
        s["v"] = rows[:, (h + kv) * hd:].view(n, kv, hd)
        half = case["rope_dim"] // 2
        s["inv_freq"] = (10000.0 ** (-torch.arange(half, device=dev, dtype=torch.float64) / max(half, 1))
                         ).float() if half else None
        s["q_norm"] = 1 + 0.1 * torch.randn(hd, generator=g, device=dev) if case["norm"] else None
        s["k_norm"] = 1 + 0.1 * torch.randn(hd, generator=g, device=dev) if case["norm"] else None
    else:
        s["q"] = torch.randn(n, h, hd, generator=g, device=dev).to(dtype)
        if case["alibi"]:
            s["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device=dev)
        if case["prefix"]:
            s["prefix"] = torch.tensor(_prefixes(case), **i32)
    return s


# ------------------------------------------------------------------ plain forms
def _where(s):
    """Row of the batch and position in its sequence of every new token."""
    cu, n = s["cu_q"].long(), s["q"].shape[0]
    token = torch.arange(n, device=cu.device)
    row = torch.searchsorted(cu, token, right=True) - 1
    return row, s["lengths"].long()[row] - cu[row + 1] + token


def _norm_rotate(x, weight, position, inv_freq, interleaved):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight
    if inv_freq is None:
        return x
    half = inv_freq.numel()
    angle = position.double()[:, None] * inv_freq.double()
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1)


def _plain_append(s):
    row, position = _where(s)
    page = s["case"]["page"]
    q = _norm_rotate(s["q"], s["q_norm"], position, s["inv_freq"], s["case"]["interleaved"])
    k = _norm_rotate(s["k"], s["k_norm"], position, s["inv_freq"], s["case"]["interleaved"])
    at, slot = s["table"][row, position // page].long(), position % page
    s["k_pages"][at, :, slot] = k.to(s["k_pages"].dtype)
    s["v_pages"][at, :, slot] = s["v"]
    return q.to(s["q"].dtype), s["k_pages"], s["v_pages"]


def _plain_attention(s):
    """Every sequence padded to the longest one."""
    c = s["case"]
    n, h, hd = s["q"].shape
    kv, b, group = c["kv_heads"], c["batch"], h // c["kv_heads"]
    row, position = _where(s)
    local = torch.arange(n, device=row.device) - s["cu_q"].long()[row]
    t = s["longest"]
    q = torch.zeros(b, t, h, hd, device=row.device)
    q[row, local] = s["q"].float()
    at = torch.full((b, t), -1, device=row.device)
    at[row, local] = position
    k, v = (p[s["table"].clamp(min=0).long()].permute(0, 2, 1, 3, 4).reshape(b, kv, -1, hd).float()
            for p in (s["k_pages"], s["v_pages"]))
    q = q.view(b, t, kv, group, hd).permute(0, 2, 3, 1, 4).reshape(b, kv, group * t, hd)
    score = (torch.matmul(q, k.transpose(-1, -2)) * hd ** -0.5).view(b, kv, group, t, -1)
    if c["softcap"]:
        score = c["softcap"] * torch.tanh(score / c["softcap"])
    key = torch.arange(k.shape[2], device=row.device)
    far = (at[:, :, None] - key)[:, None, None]          # [b, 1, 1, t, keys]
    if s["slopes"] is not None:
        score = score - s["slopes"].view(1, kv, group, 1, 1) * far.abs()
    seen = far >= 0
    if c["window"]:
        seen = seen & (far < c["window"])
    if s["prefix"] is not None:
        seen = seen | (key < s["prefix"].view(b, 1, 1, 1, 1))
    seen = seen & (key < s["lengths"].view(b, 1, 1, 1, 1)) & (at >= 0)[:, None, None, :, None]
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(score - top)
    out = torch.matmul(p.view(b, kv, group * t, -1), v).view(b, kv, group, t, hd)
    out = out / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return out.permute(0, 3, 1, 2, 4).reshape(b, t, h, hd)[row, local].to(s["q"].dtype)


# ------------------------------------------------------------------ one pass
def run(s):
    c = s["case"]
    if own:
        from hybrid_llm_b200 import kernels
        if c["op"] == "append":
            q = kernels.paged_append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"],
                                     s["lengths"], cu_q=s["cu_q"], inv_freq=s["inv_freq"],
                                     interleaved=c["interleaved"], q_norm=s["q_norm"],
                                     k_norm=s["k_norm"], eps=1e-6)
            return q, s["k_pages"], s["v_pages"]
        if c["op"] == "decode":
            return kernels.paged_decode(s["q"], s["k_pages"], s["v_pages"], s["table"],
                                        s["lengths"], softcap=c["softcap"], window=c["window"],
                                        slopes=s["slopes"])
        return kernels.paged_prefill(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"],
                                     s["cu_q"], softcap=c["softcap"], window=c["window"],
                                     slopes=s["slopes"], prefix=s["prefix"])
    return _plain_append(s) if c["op"] == "append" else _plain_attention(s)


def work(case):
    """append: every row read once and written once.  decode, prefill: the visible keys and
    values read once, queries read, outputs written; two products over the visible pairs."""
    new, total = _lengths(case)
    h, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    rows, window = sum(new), case["window"]
    if case["op"] == "append":
        values = rows * (h + 2 * kv) * hd
        return {"bytes": 4 * values, "flops": 10 * rows * (h + kv) * hd}
    pairs = keys = 0
    for n, length, prefix in zip(new, total, _prefixes(case)):
        if not length:
            continue
        first = length - n  # position of the first new token
        oldest = max(0, first - window + 1) if window else 0
        keys += length - oldest
        if window:
            rising = max(0, min(length, window) - min(first, window))  # rows that still see all before them
            lo = min(first, window)
            pairs += (lo + 1 + lo + rising) * rising // 2 + (n - rising) * window
        else:
            pairs += n * first + n * (n + 1) // 2
            ahead = max(0, min(n, prefix - first))  # rows inside the prefix see up to its end
            pairs += ahead * (prefix - first) - ahead * (ahead + 1) // 2
    return {"bytes": 2 * (2 * keys * kv * hd + 2 * rows * h * hd), "flops": 4 * hd * h * pairs}


def exact(case, seed):
    """Sequence by sequence in 64 bits, from the definition."""
    s = prepare(case, seed)
    new, total = _lengths(case)
    prefixes = _prefixes(case)
    page, hd, h, kv = case["page"], case["head_dim"], case["heads"], case["kv_heads"]
    q = s["q"].double()
    if case["op"] == "append":
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        out, begin = [], 0
        for b, (n, length) in enumerate(zip(new, total)):
            p = torch.arange(length - n, length, device=q.device)
            rows = slice(begin, begin + n)
            begin += n
            both = []
            for x, w in ((s["q"][rows].double(), s["q_norm"]), (s["k"][rows].double(), s["k_norm"])):
                if w is not None:
                    x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / hd + 1e-6) * w.double()
                if s["inv_freq"] is not None:
                    f = s["inv_freq"].double()
                    turn = torch.polar(torch.ones((), dtype=torch.float64, device=q.device),
                                       torch.outer(p.double(), f))[:, None, :]
                    m = f.numel()
                    i = torch.arange(m, device=q.device)
                    re, im = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + m)
                    z = torch.complex(x[..., re], x[..., im]) * turn
                    x = x.clone()
                    x[..., re], x[..., im] = z.real, z.imag
                both.append(x)
            out.append(both[0])
            where = s["table"][b].long()[p // page]
            k_pages[where, :, p % page] = both[1]
            v_pages[where, :, p % page] = s["v"][rows].double()
        return torch.cat(out), k_pages, v_pages
    out, begin = torch.zeros_like(q), 0
    for b, (n, length) in enumerate(zip(new, total)):
        rows = slice(begin, begin + n)
        begin += n
        if not length:
            continue
        held = s["table"][b, :-(-length // page)].long()
        i = torch.arange(length - n, length, device=q.device)[:, None]
        j = torch.arange(length, device=q.device)[None, :]
        seen = j <= i
        if case["window"]:
            seen &= j > i - case["window"]
        seen |= j < prefixes[b]
        for head in range(h):
            k = s["k_pages"][held, head // (h // kv)].reshape(-1, hd)[:length].double()
            v = s["v_pages"][held, head // (h // kv)].reshape(-1, hd)[:length].double()
            x = q[rows, head] @ k.T / math.sqrt(hd)
            if case["softcap"]:
                x = torch.tanh(x / case["softcap"]) * case["softcap"]
            if s["slopes"] is not None:
                x = x - float(s["slopes"][head]) * (i - j).abs()
            x = torch.where(seen, x, -math.inf)
            out[rows, head] = torch.softmax(x, -1) @ v
    return out
