"""The operators of the paged key-value cache, as cases that can be timed and compared: block tables and slot maps
(``paged_tables``), new keys and values written into the cache (``paged_store``) and the attention of one new token
per request over it (``attn_paged``).  Each has a plain form in elementary torch operations (``own`` false) and the
package's own call (``own`` true)."""
import math
import random

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one decoding step of a busy server: a token for each of 256 requests, pages of 16
        {"name": "tables 256 decoding", "op": "tables", "requests": 256, "held": 4000, "prompts": 0, "prompt": 0, "page": 16},
        # prompts that arrive while other requests decode, an odd page size, a padded slot map
        {"name": "tables mixed", "op": "tables", "requests": 333, "held": 9000, "prompts": 37, "prompt": 1501, "page": 48},
        # a queue of prompts taken in at once
        {"name": "tables prompts", "op": "tables", "requests": 2048, "held": 0, "prompts": 2048, "prompt": 1024, "page": 32},
        # the keys and values of a decoding step, slices of the projection's fp32 result, rounded into an fp16 cache
        {"name": "store decoding", "op": "store", "tokens": 61, "padding": 3, "kv_heads": 8, "dim": 128, "page": 16, "of": "fp32",
         "cache": "fp16", "rows": "heads"},
        # part of a prompt, a cache that keeps a token's heads together
        {"name": "store part of a prompt", "op": "store", "tokens": 1003, "padding": 21, "kv_heads": 5, "dim": 64, "page": 24,
         "of": "bf16", "cache": "bf16", "rows": "tokens"},
        # long prompts straight from the projection
        {"name": "store prompts", "op": "store", "tokens": 16384, "padding": 0, "kv_heads": 8, "dim": 128, "page": 64, "of": "fp32",
         "cache": "bf16", "rows": "heads"},
        # one short conversation: latency
        {"name": "attn one short", "op": "attn", "requests": 1, "least": 317, "most": 317, "empty": 0, "heads": 8, "kv_heads": 2,
         "dim": 64, "page": 16, "of": "fp16", "cache": "fp16", "rows": "heads"},
        # one long document: the cache's length is what there is to split
        {"name": "attn one long", "op": "attn", "requests": 1, "least": 131072, "most": 131072, "empty": 0, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "of": "bf16", "cache": "bf16", "rows": "heads"},
        # a batch of very unequal requests, padded with empty ones, q straight from the projection in fp32
        {"name": "attn unequal", "op": "attn", "requests": 23, "least": 1, "most": 6001, "empty": 2, "heads": 40, "kv_heads": 8,
         "dim": 128, "page": 32, "of": "fp32", "cache": "fp16", "rows": "tokens"},
        # one key head to each query head: the attention benchmark's heads, length and batch
        {"name": "attn every head its own", "op": "attn", "requests": 16, "least": 4096, "most": 4096, "empty": 0, "heads": 16,
         "kv_heads": 16, "dim": 128, "page": 64, "of": "fp16", "cache": "fp16", "rows": "heads"},
        # many query heads to a key head
        {"name": "attn sixteen to one", "op": "attn", "requests": 48, "least": 700, "most": 5003, "empty": 0, "heads": 32,
         "kv_heads": 2, "dim": 64, "page": 128, "of": "bf16", "cache": "bf16", "rows": "heads"},
        # a full server
        {"name": "attn full server", "op": "attn", "requests": 64, "least": 4096, "most": 8192, "empty": 0, "heads": 64,
         "kv_heads": 8, "dim": 128, "page": 32, "of": "bf16", "cache": "bf16", "rows": "heads"},
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["tables", "store", "attn", "attn"])
    page = rng.choice([8, 16, 32, 64, 128, 192, 256])
    if kind == "tables":
        requests = _spread(rng, 1, 4096)
        prompts = rng.choice([0, requests, rng.randint(0, requests)])
        return {"op": "tables", "requests": requests, "held": rng.choice([0, _spread(rng, 1, 16384)]), "prompts": prompts,
                "prompt": _spread(rng, 1, max(1, min(32768, (1 << 21) // max(1, prompts)))), "page": rng.choice([page, rng.randint(1, 100)])}
    cache = rng.choice(["fp16", "bf16"])
    of = rng.choice([cache, "fp32"])
    dim = rng.choice([64, 128])
    rows = rng.choice(["heads", "tokens"])
    if kind == "store":
        kv_heads = rng.choice([1, 2, 3, 4, 5, 8, 12, 16, 32])
        tokens = _spread(rng, 1, (1 << 24) // (kv_heads * dim))
        return {"op": "store", "tokens": tokens, "padding": rng.choice([0, rng.randint(1, 64)]), "kv_heads": kv_heads, "dim": dim,
                "page": rng.choice([page, rng.randint(1, 100)]), "of": of, "cache": cache, "rows": rows}
    kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
    group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16, 20, 32])
    while kv_heads * group > 128:
        group //= 2
    requests = _spread(rng, 1, 256)
    most = _spread(rng, 1, max(1, min(131072, (1 << 28) // (requests * kv_heads * dim))))
    return {"op": "attn", "requests": requests, "least": rng.choice([most, _spread(rng, 1, most)]), "most": most,
            "empty": rng.choice([0, rng.randint(0, requests // 4)]), "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim,
            "page": page, "of": of, "cache": cache, "rows": rows}


def _held(case):
    """What a case's requests hold in the cache before the call, and how many tokens each adds (the case's own, whatever
    the seed: ``work`` counts the same)."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    n = case["requests"]
    if case["op"] == "attn":
        lengths = [case["most"]] + [rng.randint(case["least"], case["most"]) for _ in range(n - 1)]
        for r in rng.sample(range(n), case["empty"]):
            lengths[r] = 0
        return lengths, [0] * n
    held = [rng.randint(1, case["held"]) if case["held"] else 0 for _ in range(n)]
    new = [1] * n
    for r in rng.sample(range(n), case["prompts"]):
        held[r], new[r] = 0, rng.randint(1, case["prompt"])
    return held, new


def _up(a, b):
    return -(-a // b)


# ---------------------------------------------------------------------------------------------------- inputs

def _cache(case, pages, gen):
    """A cache of (pages, kv_heads, page, dim) as the calls take it; in memory either a page's heads or its tokens come first."""
    h, p, d = case["kv_heads"], case["page"], case["dim"]
    shape = (pages, h, p, d) if case["rows"] == "heads" else (pages, p, h, d)
    c = torch.randn(shape, generator=gen, device="cuda", dtype=_TYPES[case["cache"]])
    return c if case["rows"] == "heads" else c.transpose(1, 2)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, page = case["op"], case["page"]
    state = {"op": op, "page": page}
    if op == "store":
        tokens, width = case["tokens"], case["kv_heads"] * case["dim"]
        pages = _up(tokens, page) + 3
        rows = tokens + case["padding"]
        # one row of a projection holds the queries' heads (twice as many as the keys'), then keys, then values
        qkv = torch.randn((rows, 4 * width), generator=gen, device="cuda", dtype=_TYPES[case["of"]])
        state["k"] = qkv[:, 2 * width:3 * width].unflatten(1, (case["kv_heads"], case["dim"]))
        state["v"] = qkv[:, 3 * width:].unflatten(1, (case["kv_heads"], case["dim"]))
        state["k_cache"], state["v_cache"] = _cache(case, pages, gen), _cache(case, pages, gen)
        # consecutive tokens lie in a page side by side, as a request's do; the rows of the padding have no slot
        order = torch.randperm(pages, generator=gen, device="cuda")
        at = torch.arange(tokens, device="cuda")
        state["slots"] = torch.full((rows,), -1, dtype=torch.int64, device="cuda")
        state["slots"][:tokens] = order[at // page] * page + at % page
        return state
    held, new = _held(case)
    needs = [_up(a + b, page) for a, b in zip(held, new)]
    width, pages = max(1, max(needs)), max(1, sum(needs)) + 5
    order = torch.randperm(pages, generator=gen, device="cuda", dtype=torch.int32)
    lengths = torch.tensor(held, dtype=torch.int32, device="cuda")
    has = (lengths + page - 1) // page
    first = has.cumsum(0) - has
    column = torch.arange(width, device="cuda", dtype=torch.int32)
    mine = column[None] < has[:, None]
    table = torch.where(mine, order[(first[:, None] + column[None]).clamp(max=pages - 1)], -1).to(torch.int32)
    state |= {"lengths": lengths, "table": table}
    if op == "tables":
        state["new"] = torch.tensor(new, dtype=torch.int32, device="cuda")
        used = sum(_up(a, page) for a in held)
        state["free"] = order
        state["used"] = torch.tensor([used], dtype=torch.int32, device="cuda")
        n, rows = case["requests"], sum(new) + 7  # the slot map has room for a few tokens more
        state["slots"] = torch.empty((rows,), dtype=torch.int64, device="cuda")
        state["offsets"] = torch.empty((n + 1,), dtype=torch.int32, device="cuda")
        state["after"] = torch.empty((n,), dtype=torch.int32, device="cuda")
        state["info"] = torch.empty((4,), dtype=torch.int32, device="cuda")
        return state
    n, heads, dim = case["requests"], case["heads"], case["dim"]
    # q is the first part of a projection's row
    qkv = torch.randn((n, (heads + 2 * case["kv_heads"]) * dim), generator=gen, device="cuda", dtype=_TYPES[case["of"]])
    state["q"] = qkv[:, :heads * dim].unflatten(1, (heads, dim))
    state["k_cache"], state["v_cache"] = _cache(case, pages, gen), _cache(case, pages, gen)
    state["o"] = torch.empty((n, heads, dim), dtype=_TYPES[case["cache"]], device="cuda")
    state["lse"] = torch.empty((n, heads), dtype=torch.float32, device="cuda")
    return state


# ---------------------------------------------------------------------------------------------------- plain forms

def _plain_tables(s):
    """Request r holds len[r] tokens and adds new[r]; the pages that it lacks come from the list of free pages, in the order
    of the requests.  A request whose pages or tokens do not fit is left as it was, and its tokens get no slot."""
    page, free, table = s["page"], s["free"], s["table"]
    held, new = s["lengths"].long(), s["new"].long()
    rows, width = s["slots"].numel(), table.shape[1]
    adds = new.clamp(min=0)
    ends = adds.cumsum(0)
    starts = ends - adds
    sound = (held >= 0) & (new >= 0) & ((adds == 0) | (ends <= rows)) & (held + adds <= width * page)
    old = (held.clamp(min=0) + page - 1) // page
    total = (held.clamp(min=0) + adds + page - 1) // page
    need = torch.where(sound, total - old, 0)
    until = need.cumsum(0)
    left = free.numel() - s["used"].long()
    granted = sound & ((need == 0) | (until <= left))
    base = s["used"].long() + until - need
    # the new entries of the tables
    column = torch.arange(width, device=table.device)
    fresh = granted[:, None] & (column >= old[:, None]) & (column < total[:, None])
    entry = free[(base[:, None] + column - old[:, None]).clamp(0, free.numel() - 1)]
    table.copy_(torch.where(fresh, entry, table))
    # each token's slot
    t = torch.arange(rows, device=table.device)
    r = torch.searchsorted(ends, t, right=True)
    there = r < held.numel()
    r = r.clamp(max=held.numel() - 1)
    at = (held[r] + t - starts[r]).clamp(0, width * page - 1)
    of = table[r, at // page].long()
    s["slots"].copy_(torch.where(there & granted[r] & (of >= 0), of * page + at % page, -1))
    s["offsets"][0] = 0
    s["offsets"][1:] = ends
    s["after"].copy_(torch.where(granted, held + adds, held))
    s["info"].copy_(torch.cat([s["used"].long() + torch.where(granted, need, 0).sum(), ends[-1:], (~granted).sum()[None], until[-1:]]))
    return {"slots": s["slots"], "offsets": s["offsets"], "after": s["after"], "info": s["info"], "table": table}


def _plain_store(s):
    """cache[slot // page, :, slot % page] = the token's keys (values), rounded to the cache's type; no slot, nothing written."""
    used = s["slots"] >= 0
    of, at = s["slots"][used] // s["page"], s["slots"][used] % s["page"]
    s["k_cache"][of, :, at] = s["k"][used].float().to(s["k_cache"].dtype)
    s["v_cache"][of, :, at] = s["v"][used].float().to(s["v_cache"].dtype)
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attn(s):
    """o = softmax(scale q K^T) V over the first len keys of each request; zeros (and -inf) where len is 0."""
    q, table, lengths, page = s["q"].float(), s["table"].clamp(min=0), s["lengths"], s["page"]
    n, heads, dim = q.shape
    kv_heads = s["k_cache"].shape[1]
    k = s["k_cache"][table].permute(0, 2, 1, 3, 4).reshape(n, kv_heads, -1, dim).float()
    v = s["v_cache"][table].permute(0, 2, 1, 3, 4).reshape(n, kv_heads, -1, dim).float()
    there = (torch.arange(k.shape[2], device=q.device) < lengths[:, None])[:, None, None]
    x = (q.view(n, kv_heads, -1, dim) @ k.transpose(2, 3)) * (1.0 / dim ** 0.5)
    x = torch.where(there, x, -torch.inf)
    most = x.amax(3, keepdim=True)
    p = torch.exp(x - torch.where(most == -torch.inf, 0.0, most))
    total = p.sum(3, keepdim=True)
    o = (p @ v) / torch.where(total == 0, 1.0, total)
    s["o"].copy_(o.reshape(n, heads, dim))
    s["lse"].copy_((most + torch.log(total)).reshape(n, heads))
    return {"o": s["o"], "lse": s["lse"]}


def run(state):
    if own:
        import spork_b200 as sp

        if state["op"] == "tables":
            slots, offsets, after, info = sp.paged_tables(
                state["lengths"], state["new"], state["table"], state["free"], state["used"], page_size=state["page"],
                slots=state["slots"], offsets=state["offsets"], lengths_after=state["after"], info=state["info"])
            return {"slots": slots, "offsets": offsets, "after": after, "info": info, "table": state["table"]}
        if state["op"] == "store":
            sp.paged_store(state["k"], state["v"], state["k_cache"], state["v_cache"], state["slots"])
            return {"k_cache": state["k_cache"], "v_cache": state["v_cache"]}
        o = sp.attn_paged(state["q"], state["k_cache"], state["v_cache"], state["table"], state["lengths"], state["o"],
                          lse=state["lse"])
        return {"o": o, "lse": state["lse"]}
    if state["op"] == "tables":
        return _plain_tables(state)
    if state["op"] == "store":
        return _plain_store(state)
    return _plain_attn(state)


# ---------------------------------------------------------------------------------------------------- bounds and exact values

def work(case):
    size = {"fp16": 2, "bf16": 2, "fp32": 4}
    if case["op"] == "store":
        values = 2 * case["tokens"] * case["kv_heads"] * case["dim"]
        return {"bytes": values * (size[case["of"]] + size[case["cache"]]) + 8 * (case["tokens"] + case["padding"]), "flops": 0}
    held, new = _held(case)
    page, n = case["page"], case["requests"]
    if case["op"] == "tables":
        fresh = sum(_up(a + b, page) - _up(a, page) for a, b in zip(held, new))
        last = sum(1 for a in held if a % page)  # the entry of a page that is partly full is read
        return {"bytes": 4 * (4 * n + 2 + 4 + 2 * fresh + last) + 8 * (sum(new) + 7), "flops": 0}
    keys = sum(held)
    values = keys * case["kv_heads"] * case["dim"]
    qo = n * case["heads"] * case["dim"]
    return {"bytes": 2 * values * size[case["cache"]] + qo * (size[case["of"]] + size[case["cache"]]) + 4 * n * case["heads"]
            + 4 * (n + sum(_up(a, page) for a in held)), "flops": 4 * keys * case["heads"] * case["dim"]}


def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers
    s = prepare(case, seed)
    page = case["page"]
    if case["op"] == "store":
        # token by token of the definition: slot -> (page, row), all heads; what has no slot keeps its value
        out = {}
        for name in ("k", "v"):
            c = s[name + "_cache"].double().transpose(1, 2).contiguous()  # (pages, page, kv_heads, dim)
            flat = c.view(-1, *c.shape[2:])
            flat[s["slots"][:case["tokens"]]] = s[name][:case["tokens"]].double()
            out[name + "_cache"] = c.transpose(1, 2)
        return out
    lengths, _ = _held(case)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    o = torch.zeros((len(lengths), heads, dim), dtype=torch.float64, device="cuda")
    lse = torch.full((len(lengths), heads), -math.inf, dtype=torch.float64, device="cuda")
    for r, keys in enumerate(lengths):
        if keys == 0:
            continue
        pages = s["table"][r, :_up(keys, page)].long()
        for h in range(kv_heads):
            mine = slice(h * heads // kv_heads, (h + 1) * heads // kv_heads)
            k = s["k_cache"][pages, h].reshape(-1, dim)[:keys].double()
            v = s["v_cache"][pages, h].reshape(-1, dim)[:keys].double()
            x = torch.einsum("kd,gd->gk", k, s["q"][r, mine].double()) / math.sqrt(dim)
            lse[r, mine] = torch.logsumexp(x, 1)
            o[r, mine] = torch.softmax(x, 1) @ v
    return {"o": o, "lse": lse}
