"""Plain implementations of the paged cache's operators for the tests: whole numbers in Python, attention in 64 bits."""
import math

INT_MAX = 2 ** 31 - 1


def tables(lengths, new, table, free, used, page, max_tokens):
    """The rules of spork_paged_sm100_tables, request by request, on lists (table: list of rows, changed in place)."""
    left = len(free) - used if 0 <= used <= len(free) else 0
    slots, offsets, after = [-1] * max_tokens, [], []
    tokens = pages = granted_pages = refused = 0
    for r, (held, added) in enumerate(zip(lengths, new)):
        adds = max(0, added)
        begin, tokens = tokens, tokens + adds
        offsets.append(min(begin, INT_MAX))
        width = len(table[r])
        sound = held >= 0 and added >= 0 and (adds == 0 or tokens <= max_tokens) and held + adds <= min(width * page, INT_MAX)
        if not sound:
            refused += 1
            after.append(held)
            continue
        old, total = -(-held // page), -(-(held + adds) // page)
        base, pages = pages, pages + total - old
        if total > old and pages > left:
            refused += 1
            after.append(held)
            continue
        granted_pages += total - old
        for i in range(total - old):
            table[r][old + i] = free[used + base + i]
        for i in range(adds):
            of = table[r][(held + i) // page]
            if of >= 0:
                slots[begin + i] = of * page + (held + i) % page
        after.append(held + adds)
    offsets.append(min(tokens, INT_MAX))
    return slots, offsets, after, [used + granted_pages, min(tokens, INT_MAX), refused, min(pages, INT_MAX)]


def attention(q, k, v, scale):
    """One request: q (heads, D), k and v (kv_heads, keys, D), any type; returns in 64 bits o (heads, D), lse (heads,), and
    for tolerances the weighted magnitudes sum p |v| (heads, D) and the largest sum |q k| scale of a key (heads,)."""
    import torch

    heads, dim = q.shape
    kv_heads, keys, _ = k.shape
    q, k, v = q.double(), k.double(), v.double()
    if keys == 0:
        zero = torch.zeros((heads, dim), dtype=torch.float64, device=q.device)
        return zero, torch.full((heads,), -math.inf, dtype=torch.float64, device=q.device), zero, zero[:, 0]
    group = heads // kv_heads
    kk, vv = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
    x = torch.einsum("hd,hkd->hk", q, kk) * scale
    size = torch.einsum("hd,hkd->hk", q.abs(), kk.abs()).amax(1) * scale
    lse = torch.logsumexp(x, 1)
    p = torch.softmax(x, 1)
    return (torch.einsum("hk,hkd->hd", p, vv), lse, torch.einsum("hk,hkd->hd", p, vv.abs()), size)


def tolerances(dtype, keys, dim, ref, weighted, size, fp32_q):
    """How far o and lse may be from the 64-bit values.

    Scores: dim products of 16-bit factors are exact in 32 bits, their sum is off by at most dim steps of 2^-23 (the tensor
    core may truncate) of the sum of their magnitudes; a 32-bit q is taken as two 16-bit parts, which leaves (eps / 2)^2 of
    it (for fp16 at least 2^-25 absolutely, a subnormal's half step, on q of a size around one: within the same bound
    times four); scaling, subtracting the maximum and the exponential add a few 2^-23 of the score's magnitude.  A score off by e moves a weight
    by e and, through the sum, the others by e: 2 e of the weighted magnitudes.  Weights: taken as two 16-bit parts,
    (eps / 2)^2, of numbers that are 2^6 at least for the largest weight: a key whose weight is below half the smallest step
    of fp16, 2^-25, is off by that much, 2^-31 of the largest.
    Sums over the keys: at most one step of 2^-23 for every key and joining, of the weighted magnitudes.  At the end o is
    rounded once: eps / 2 of its own value (below the normal range: half the smallest step)."""
    import torch

    half = torch.finfo(dtype).eps / 2
    e = size * ((dim + 8) * 2.0 ** -23 + (4 * half * half if fp32_q else 0.0)) + 2.0 ** -21
    inner = 2 * e + half * half + keys * 2.0 ** -31 + (keys + 64) * 2.0 ** -23
    tol_o = half * ref.abs() + (1 + half) * inner[:, None] * weighted + torch.finfo(dtype).smallest_normal * half
    tol_lse = e + (keys + 64) * 2.0 ** -23 + 2.0 ** -23 * (size + math.log(max(keys, 1)) + 1)
    return tol_o, tol_lse


def tolerances_of_fp32_queries(dtype, q, k, scale, ref, weighted, size):
    """The same for fp32 queries of any size, over the keys k (kv_heads, keys, D) of one request.

    A query's row is brought by a power of two, which is exact, to where the cache type has room below it, and taken as two
    parts of that type.  What the two leave over: the second part is off by eps / 2 of what the first one left, which is
    eps / 2 of the element, so (eps / 2)^2 of the element; and by half of the type's smallest step.  That step is fp16's
    2^-24, and the row's largest element is brought to 2^14 at least: 2^-39 of that one.  (bf16: 2^-134 beside 2^-60 at
    least, nothing; an fp32 subnormal has no more bits than the two parts.)  The rest is as above."""
    import torch

    heads, dim = q.shape
    kv_heads, keys, _ = k.shape
    half = torch.finfo(dtype).eps / 2
    sums = k.double().abs().sum(2).amax(1).repeat_interleave(heads // kv_heads)  # per head, of the key with the largest one
    least = 2.0 ** -39 if dtype == torch.float16 else 2.0 ** -74
    e = size * ((dim + 8) * 2.0 ** -23 + half * half) + least * q.double().abs().amax(1) * sums * scale + 2.0 ** -21
    inner = 2 * e + half * half + keys * 2.0 ** -31 + (keys + 64) * 2.0 ** -23
    tol_o = half * ref.abs() + (1 + half) * inner[:, None] * weighted + torch.finfo(dtype).smallest_normal * half
    tol_lse = e + (keys + 64) * 2.0 ** -23 + 2.0 ** -23 * (size + math.log(max(keys, 1)) + 1)
    return tol_o, tol_lse
