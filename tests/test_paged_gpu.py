"""The paged key-value cache on a B200: block tables and slot maps, stores, the attention of one new token per request, and
all of them together with the prompt's attention."""
import math
import random

import pytest

import paged_plain

pytestmark = pytest.mark.gpu

I32 = 2 ** 31 - 1


# ------------------------------------------------------------------------------------------------ tables

def _tables_case(rng, requests, page, held, new, spare=3, width=None):
    """A table whose rows name the pages that each request holds, in shuffled order, and the list of all pages."""
    needs = [-(-max(a, 0) // page) for a in held]
    width = width or max(1, max(-(-(max(a, 0) + max(b, 0)) // page) for a, b in zip(held, new)))
    total = sum(-(-(max(a, 0) + max(b, 0)) // page) for a, b in zip(held, new)) + spare
    order = list(range(total))
    rng.shuffle(order)
    table, used = [], 0
    for n in needs:
        n = min(n, width)
        table.append(order[used:used + n] + [-7] * (width - n))
        used += n
    return table, order, used


def _run_tables(sp, cuda, held, new, table, free, used, page, max_tokens, stride=None):
    import torch

    i32 = dict(dtype=torch.int32, device=cuda)
    rows = torch.full((len(held), stride or len(table[0])), -9, **i32)[:, :len(table[0])]
    rows.copy_(torch.tensor(table, **i32).view(rows.shape))
    got = sp.paged_tables(torch.tensor(held, **i32), torch.tensor(new, **i32), rows, torch.tensor(free, **i32),
                          torch.tensor([used], **i32), page_size=page, max_tokens=max_tokens)
    torch.cuda.synchronize()
    want_table = [list(r) for r in table]
    want = paged_plain.tables(held, new, want_table, free, used, page, max_tokens)
    for name, g, w in zip(("slots", "offsets", "lengths_after", "info"), got, want):
        assert g.tolist() == w, name
    assert rows.tolist() == want_table
    return got


@pytest.mark.parametrize("requests,page,most_held,most_new,room", [
    (1, 16, 0, 1, 0), (1, 1, 5, 9, 4), (256, 16, 4000, 1, 0), (33, 48, 500, 700, 11), (1000, 32, 300, 40, 100), (2, 7, 100, 50000, 1),
    (4097, 64, 200, 3, 0), (16384, 16, 90, 2, 5), (1025, 128, 0, 300, 1000),
    (700, 48, 500, 600, 3), (5000, 7, 30, 90, 1)])  # these two: four tokens to a thread, requests and pages that end inside
def test_tables_match_the_rules(sp, cuda, requests, page, most_held, most_new, room):
    rng = random.Random(requests * 1000 + page)
    held = [rng.randint(0, most_held) for _ in range(requests)]
    new = [rng.randint(0, most_new) for _ in range(requests)]
    table, free, used = _tables_case(rng, requests, page, held, new)
    _run_tables(sp, cuda, held, new, table, free, used, page, sum(new) + room, stride=len(table[0]) + requests % 3)


def test_tables_refuse_requests_one_by_one(sp, cuda):
    """Negative lengths, rows that are too short, a free list and a slot map that run out: those requests are left alone, and
    the rule for the ones behind them is the same at every batch size."""
    rng = random.Random(5)
    for requests in (5, 300, 5000):
        held = [rng.choice([0, 15, 16, 17, 40, -1, -I32]) if rng.random() < 0.3 else rng.randint(0, 60) for _ in range(requests)]
        new = [rng.choice([0, 1, -1, -5, 100]) if rng.random() < 0.3 else rng.randint(0, 20) for _ in range(requests)]
        table, free, used = _tables_case(rng, requests, 16, held, new, width=5)
        enough = len(free)
        tokens = sum(max(0, n) for n in new)
        for cut in (enough, used + (enough - used) // 2, used, max(0, used - 3)):
            for room in (tokens, tokens // 2, 0):
                _run_tables(sp, cuda, held, new, table, free[:cut], used, 16, room)


def test_tables_far_numbers_and_odd_lists(sp, cuda):
    # sums beyond 32 bits; a used count outside the list; free pages and entries that are negative
    _run_tables(sp, cuda, [0, I32, 3, I32], [I32, I32, 1, 0], [[-7] * 4 for _ in range(4)], [5, 6], 0, 16, 10)
    _run_tables(sp, cuda, [3, 16], [1, 1], [[1, -7], [2, -7]], [5, 6], 7, 16, 2)
    _run_tables(sp, cuda, [3, 16], [1, 1], [[1, -7], [2, -7]], [5, 6], -1, 16, 2)
    _run_tables(sp, cuda, [3, 16], [1, 4], [[-1, -7], [2, -7]], [-5, 6], 0, 16, 5)
    _run_tables(sp, cuda, [0], [3], [[-7]], [I32], 0, I32, 3)
    _run_tables(sp, cuda, [I32 - 1, I32 - 1, I32], [1, 2, 0], [[4, -7]] * 3, [I32, 8], 0, I32, 3)
    _run_tables(sp, cuda, [0, 0], [0, 0], [[], []], [], 0, 16, 2)


def test_tables_write_slots_wherever_they_begin(sp, cuda):
    # a slot map on no boundary of 16 bytes, large enough for four tokens to a thread; nothing around it is touched
    import torch

    i32 = dict(dtype=torch.int32, device=cuda)
    tokens = 160001
    around = torch.full((tokens + 2,), -9, dtype=torch.int64, device=cuda)
    slots, _, _, info = sp.paged_tables(torch.tensor([5], **i32), torch.tensor([tokens - 1], **i32),
                                        torch.zeros((1, 10001), **i32), torch.arange(1, 10001, **i32),
                                        torch.tensor([0], **i32), page_size=16, slots=around[1:-1])
    assert info.tolist() == [10000, tokens - 1, 0, 10000]
    assert torch.equal(slots[:-1], torch.arange(5, tokens + 4, device=cuda)) and slots[-1] == -1
    assert around[0] == -9 and around[-1] == -9


def test_tables_of_nearly_2_31_pages(sp, cuda):
    # pages of one token, nearly all that a step can grant: page numbers near the end of 31 bits, 34 GB of lists
    import torch

    requests, each = 16384, 131071
    pages = requests * each
    assert I32 - 148 * 1024 < pages < I32
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    lengths = torch.zeros(requests, dtype=torch.int32, device=cuda)
    new = torch.full((requests,), each, dtype=torch.int32, device=cuda)
    table = torch.full((requests, each), -7, dtype=torch.int32, device=cuda)
    free = torch.arange(pages, dtype=torch.int32, device=cuda)
    used = torch.zeros(1, dtype=torch.int32, device=cuda)
    slots, offsets, after, info = sp.paged_tables(lengths, new, table, free, used, page_size=1, max_tokens=pages)
    assert info.tolist() == [pages, pages, 0, pages]
    assert torch.equal(after, new) and offsets[-1].item() == pages
    assert torch.equal(table.view(-1), free)
    for at in range(0, pages, 1 << 28):
        assert torch.equal(slots[at:at + (1 << 28)], free[at:at + (1 << 28)].to(torch.int64)), at
    del table, free, slots
    torch.cuda.empty_cache()


def test_tables_of_no_requests(sp, cuda):
    import torch

    e = torch.empty(0, dtype=torch.int32, device=cuda)
    slots, offsets, after, info = sp.paged_tables(e, e, torch.empty((0, 4), dtype=torch.int32, device=cuda), e,
                                                  torch.tensor([0], dtype=torch.int32, device=cuda), page_size=16, max_tokens=4)
    assert slots.tolist() == [-1] * 4 and offsets.tolist() == [0] and after.tolist() == [] and info.tolist() == [0] * 4


# ------------------------------------------------------------------------------------------------ store

def _empty_cache(cuda, pages, kv_heads, page, dim, dtype, order, fill):
    """A cache (pages, kv_heads, page, dim) in memory as `order` says, inside a larger allocation for the odd strides."""
    import torch

    if order == "heads":
        return torch.full((pages, kv_heads, page, dim), fill, dtype=dtype, device=cuda)
    if order == "tokens":
        return torch.full((pages, page, kv_heads, dim), fill, dtype=dtype, device=cuda).transpose(1, 2)
    if order == "both":  # keys and values of a page side by side: this is one of the two
        return torch.full((pages, 2, kv_heads, page, dim), fill, dtype=dtype, device=cuda)[:, 1]
    assert order == "wide"  # rows with something between them
    return torch.full((kv_heads, pages, page, dim + 8), fill, dtype=dtype, device=cuda)[..., :dim].transpose(0, 1)


@pytest.mark.parametrize("src,dst", [("float32", "float16"), ("float32", "bfloat16"), ("float16", "float16"), ("bfloat16", "bfloat16")])
@pytest.mark.parametrize("tokens,kv_heads,page,dim,order,shift", [
    (1, 1, 16, 64, "heads", 0), (37, 8, 16, 128, "tokens", 0), (300, 3, 24, 64, "both", 4), (65, 5, 7, 96, "heads", 8),
    (129, 2, 32, 128, "wide", 1), (50, 4, 1, 40, "tokens", 3), (9, 1, 64, 1, "heads", 0), (2050, 2, 64, 128, "heads", 0),
    # enough blocks for four tokens to a thread: side by side in a block or not, in pieces or single elements, odd ends
    (2401, 8, 16, 128, "tokens", 0), (7203, 2, 32, 128, "both", 4), (7150, 2, 16, 128, "heads", 0), (1777, 3, 24, 64, "wide", 1)])
def test_store_puts_each_token_into_its_slot(sp, cuda, src, dst, tokens, kv_heads, page, dim, order, shift):
    import torch

    src, dst = getattr(torch, src), getattr(torch, dst)
    g = torch.Generator(device=cuda).manual_seed(tokens)
    pages = -(-tokens // page) + 2
    # tokens and heads lie apart in a projection's row, `shift` elements from an aligned place
    qkv = torch.randn((tokens, 3 * kv_heads * dim + 8), generator=g, device=cuda).mul_(100).to(src)
    k = qkv[:, shift:shift + kv_heads * dim].unflatten(1, (kv_heads, dim))
    v = qkv[:, kv_heads * dim + shift:2 * kv_heads * dim + shift].unflatten(1, (kv_heads, dim))
    qkv[0, shift], qkv[0, kv_heads * dim + shift] = math.inf, math.nan
    slots = torch.randperm(pages * page, generator=g, device=cuda)[:tokens]
    outside = torch.tensor([-1, -I32, pages * page, 2 ** 62], device=cuda)
    slots[1::5] = outside[torch.arange(slots[1::5].numel(), device=cuda) % 4]  # these tokens go nowhere
    kc, vc = (_empty_cache(cuda, pages, kv_heads, page, dim, dst, order, 7.0) for _ in range(2))
    sp.paged_store(k, v, kc, vc, slots)
    torch.cuda.synchronize()
    for x, c in ((k, kc), (v, vc)):
        want = torch.full((pages, page, kv_heads, dim), 7.0, dtype=dst, device=cuda)
        flat = want.view(pages * page, kv_heads, dim)
        inside = (slots >= 0) & (slots < pages * page)
        flat[slots[inside]] = x[inside].to(dst)
        bits = lambda t: t.contiguous().view(torch.int16)  # noqa: E731
        same = (bits(want) == bits(c.transpose(1, 2))) | (want.isnan() & c.transpose(1, 2).isnan())
        assert same.all()
    if order == "both":
        assert (kc._base[:, 0] == 7.0).all()
    if order == "wide":
        assert (kc._base[..., dim:] == 7.0).all()


def test_store_of_nothing(sp, cuda):
    import torch

    c = torch.zeros((2, 2, 16, 64), dtype=torch.float16, device=cuda)
    x = torch.ones((0, 2, 64), dtype=torch.float16, device=cuda)
    sp.paged_store(x, x, c, c.clone(), torch.empty(0, dtype=torch.int64, device=cuda))
    e = c[:0]
    y = torch.ones((1, 2, 64), dtype=torch.float16, device=cuda)
    sp.paged_store(y, y, e, e, torch.zeros(1, dtype=torch.int64, device=cuda))
    torch.cuda.synchronize()
    assert (c == 0).all()


# ------------------------------------------------------------------------------------------------ attention

class Paged:
    """Requests' keys and values laid into pages, with NaN wherever nothing may be read for a result."""

    def __init__(self, cuda, lengths, heads, kv_heads, dim, page, dtype, q_dtype=None, order="heads", seed=0, spread=1.0,
                 width=None):
        import torch

        g = torch.Generator(device=cuda).manual_seed(seed)
        self.lengths, self.page, self.dtype, self.dim = lengths, page, dtype, dim
        needs = [-(-n // page) for n in lengths]
        pages = sum(needs) + 2
        perm = torch.randperm(pages, generator=g, device=cuda).tolist()
        width = width or max(1, max(needs)) + 1
        self.kc, self.vc = (_empty_cache(cuda, pages, kv_heads, page, dim, dtype, order, math.nan) for _ in range(2))
        table, used, self.k, self.v = [], 0, [], []
        for n, need in zip(lengths, needs):
            mine = perm[used:used + need]
            used += need
            table.append(mine + [[-1, pages, I32, -I32, perm[-1]][i % 5] for i in range(width - need)])
            k, v = (torch.randn((kv_heads, n, dim), generator=g, device=cuda).mul_(spread).to(dtype) for _ in range(2))
            for i, p in enumerate(mine):
                rows = slice(i * page, min(n, (i + 1) * page))
                self.kc[p, :, :rows.stop - rows.start] = k[:, rows]
                self.vc[p, :, :rows.stop - rows.start] = v[:, rows]
            self.k.append(k)
            self.v.append(v)
        qkv = torch.randn((len(lengths), (heads + 2) * dim + 3), generator=g, device=cuda).to(q_dtype or dtype)
        self.q = qkv[:, 3:heads * dim + 3].unflatten(1, (heads, dim))  # rows of a projection, at an odd place
        wide = torch.full((len(lengths), width + 1), -3, dtype=torch.int32, device=cuda)
        self.table = wide[:, :width]
        self.table.copy_(torch.tensor(table, dtype=torch.int32))
        self.len = torch.tensor(lengths, dtype=torch.int32, device=cuda)
        self.heads = heads

    def run(self, sp, scale=None, **kw):
        import torch

        lse = torch.full((len(self.lengths), self.heads), 5.0, device=self.q.device)
        o = sp.attn_paged(self.q, self.kc, self.vc, self.table, self.len, lse=lse, scale=scale, **kw)
        torch.cuda.synchronize()
        sp.status()
        return o, lse

    def check(self, o, lse, scale=None, skip=()):
        import torch

        worst = 0.0
        for r, n in enumerate(self.lengths):
            if r in skip:
                continue
            ref, ref_lse, weighted, size = paged_plain.attention(self.q[r], self.k[r], self.v[r], scale or self.dim ** -0.5)
            if n == 0:
                assert (o[r] == 0).all() and (lse[r] == -math.inf).all(), f"request {r}"
                continue
            tol_o, tol_lse = paged_plain.tolerances(self.dtype, n, self.dim, ref, weighted, size, self.q.dtype == torch.float32)
            err = ((o[r].double() - ref).abs() / tol_o).max().item()
            err_lse = ((lse[r].double() - ref_lse).abs() / tol_lse).max().item()
            assert err <= 1 and err_lse <= 1, f"request {r} of {n} keys: o {err}, lse {err_lse} of what is allowed"
            worst = max(worst, err)
        return worst


def _types(name):
    import torch

    cache, _, q = name.partition(" of ")
    return getattr(torch, cache), getattr(torch, q) if q else None


@pytest.mark.parametrize("types", ["float16", "bfloat16", "float16 of float32", "bfloat16 of float32"])
@pytest.mark.parametrize("lengths,heads,kv_heads,dim,page,order", [
    ([1], 1, 1, 64, 16, "heads"),
    ([63, 64, 65, 0, 1, 2], 8, 2, 64, 16, "tokens"),
    ([700, 15, 16, 17, 129, 0, 0, 255], 8, 1, 128, 8, "heads"),
    ([1000, 1, 513], 12, 12, 128, 32, "both"),
    ([321, 40, 200], 15, 5, 64, 64, "wide"),
    ([2049, 100], 14, 2, 128, 128, "tokens"),
    ([500, 3], 32, 2, 64, 192, "heads"),
    ([300, 77], 40, 2, 128, 16, "heads"),
    ([200, 129, 64], 71, 1, 64, 256, "heads"),
    ([90, 1], 64, 1, 128, 64, "both"),
    ([30, 0, 128, 5000, 64], 10, 2, 128, 16, "wide")])
def test_attention_matches_the_definition(sp, cuda, types, lengths, heads, kv_heads, dim, page, order):
    dtype, q_dtype = _types(types)
    case = Paged(cuda, lengths, heads, kv_heads, dim, page, dtype, q_dtype, order, seed=len(lengths) + heads)
    case.check(*case.run(sp))
    case.check(*case.run(sp, scale=0.7), scale=0.7)


@pytest.mark.parametrize("requests,most,heads,kv_heads,dim,page", [(257, 40, 4, 4, 64, 16), (100, 900, 8, 1, 128, 32),
                                                                   (1500, 3, 6, 2, 64, 8), (40, 3000, 16, 8, 64, 64)])
def test_attention_of_many_requests(sp, cuda, requests, most, heads, kv_heads, dim, page):
    import torch

    rng = random.Random(most)
    lengths = [rng.choice([0, 1, rng.randint(0, most), rng.randint(0, most)]) for _ in range(requests)]
    case = Paged(cuda, lengths, heads, kv_heads, dim, page, torch.float16, seed=requests)
    case.check(*case.run(sp))


@pytest.mark.parametrize("keys,heads,kv_heads,dim,page", [(131072, 8, 1, 64, 16), (50001, 4, 4, 128, 64), (20000, 32, 2, 128, 32)])
def test_attention_of_one_long_request(sp, cuda, keys, heads, kv_heads, dim, page):
    import torch

    case = Paged(cuda, [keys], heads, kv_heads, dim, page, torch.bfloat16, seed=keys)
    o, lse = case.run(sp)
    case.check(o, lse)
    # the largest score last, first, and in the middle: the running maximum moves late, or never
    for at in (keys - 1, 0, keys // 2):
        k = case.k[0].clone()
        k[:, at] = case.q[0].unflatten(0, (kv_heads, -1)).sum(1)
        case.k[0], old = k, case.k[0]
        page_id = case.table[0, at // page].item()
        was = case.kc[page_id, :, at % page].clone()
        case.kc[page_id, :, at % page] = k[:, at]
        case.check(*case.run(sp))
        case.kc[page_id, :, at % page], case.k[0] = was, old


@pytest.mark.parametrize("seed", range(16))
def test_attention_of_drawn_shapes(sp, cuda, seed):
    import torch

    rng = random.Random(seed)
    dim, page = rng.choice([64, 128]), rng.choice([8, 16, 32, 64, 128, 320])
    kv_heads, group = rng.choice([(1, 3), (2, 8), (3, 9), (4, 1), (1, 17), (2, 30), (1, 40), (8, 4)])
    most = rng.choice([70, 600, 2500])
    lengths = [rng.choice([0, 1, rng.randint(0, most)]) for _ in range(rng.choice([1, 3, 17, 90]))]
    dtype = rng.choice([torch.float16, torch.bfloat16])
    case = Paged(cuda, lengths, kv_heads * group, kv_heads, dim, page, dtype, rng.choice([None, torch.float32]),
                 rng.choice(["heads", "tokens", "both", "wide"]), seed=seed, width=rng.choice([None, 1 + -(-most // page) + 40]))
    case.check(*case.run(sp))


def test_attention_of_more_requests_than_a_block_keeps_lengths_of(sp, cuda):
    import torch

    rng = random.Random(3)
    case = Paged(cuda, [rng.choice([0, 1, 130, 400]) for _ in range(1100)], 4, 1, 64, 64, torch.float16, seed=5)
    case.check(*case.run(sp))


def test_attention_large_scores_and_small_weights(sp, cuda):
    """Scores of several hundred: all but a few weights vanish, nothing overflows."""
    import torch

    for dtype in (torch.float16, torch.bfloat16):
        case = Paged(cuda, [700, 64, 3], 8, 2, 64, 16, dtype, seed=3, spread=30.0)
        case.check(*case.run(sp))


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (9, 1, 128), (40, 2, 128), (16, 16, 64)])
@pytest.mark.parametrize("dtype,size", [("float16", s) for s in (1e-3, 1e-4, 1e-5, 1e-6, 1e-9, 1e-30, 1e-38, 1e6, 1e30)]
                         + [("bfloat16", s) for s in (1e-6, 1e-30, 1e-36, 1e-38, 1e30, 3e37)])
def test_attention_of_fp32_queries_of_any_size(sp, cuda, dtype, size, heads, kv_heads, dim):
    """Queries far below or above the cache type's range, with a scale that makes scores of a size around one of them: rows
    keep their bits, each by itself (they differ by up to 2^20 here, one is zero), and so does lse."""
    import torch

    dtype = getattr(torch, dtype)
    case = Paged(cuda, [700, 1, 63, 0, 129], heads, kv_heads, dim, 16, dtype, torch.float32, seed=heads)
    row = torch.arange(len(case.lengths) * heads, device=cuda).view(-1, heads, 1) * 7 % 11
    case.q = (case.q.clamp(-4, 4).double() * 2.0 ** (-2.0 * row) * size).float()
    case.q[0, 3] = 0.0
    scale = 1.0 / dim ** 0.5 / size
    if scale > 1e38:
        scale = 1e38
    o, lse = case.run(sp, scale=scale)
    scale = torch.tensor(scale, dtype=torch.float32).item()
    for r, n in enumerate(case.lengths):
        ref, ref_lse, weighted, sizes = paged_plain.attention(case.q[r], case.k[r], case.v[r], scale)
        if n == 0:
            assert (o[r] == 0).all() and (lse[r] == -math.inf).all()
            continue
        tol_o, tol_lse = paged_plain.tolerances_of_fp32_queries(dtype, case.q[r], case.k[r], scale, ref, weighted, sizes)
        err, err_lse = (o[r].double() - ref).abs() / tol_o, (lse[r].double() - ref_lse).abs() / tol_lse
        assert err.max() <= 1 and err_lse.max() <= 1, f"request {r}: o {err.max()}, lse {err_lse.max()} of what is allowed"


def test_attention_of_fp32_queries_with_infinities(sp, cuda):
    """An element of q that is not finite says nothing about how its row is scaled: its scores are infinite or NaN as the
    definition has them, and the other rows are what they are without it."""
    import torch

    for dtype in (torch.float16, torch.bfloat16):
        case = Paged(cuda, [100, 40], 4, 2, 64, 16, dtype, torch.float32, seed=8)
        case.q = case.q * 1e-6
        case.q[0, 1, 5], case.q[0, 2, 6] = math.inf, math.nan
        case.k[0][0, :, 5] = -1.0 - case.k[0][0, :, 5].abs()  # row 1's scores: all but one are -infinity
        case.k[0][0, 33, 5] = 0.0
        for i in range(100):
            case.kc[case.table[0, i // 16].item(), 0, i % 16] = case.k[0][0, i]
        o, lse = case.run(sp, scale=1e5)
        assert o[0, 1].isnan().all() and o[0, 2].isnan().all() and lse[0, 1].isnan() and lse[0, 2].isnan()  # 0 times infinity
        case.k[0][0, 33, 5] = -2.0
        case.kc[case.table[0, 2].item(), 0, 1] = case.k[0][0, 33]
        o, lse = case.run(sp, scale=1e5)
        assert o[0, 1].isnan().all() and lse[0, 1] == -math.inf  # every key is masked: nothing to divide by
        scale = torch.tensor(1e5, dtype=torch.float32).item()
        for r, rows in ((0, [0, 3]), (1, [0, 1, 2, 3])):
            q = case.q[r].nan_to_num(0, 0, 0)
            ref, _, weighted, sizes = paged_plain.attention(q, case.k[r], case.v[r], scale)
            tol, _ = paged_plain.tolerances_of_fp32_queries(dtype, q, case.k[r], scale, ref, weighted, sizes)
            assert ((o[r].double() - ref).abs() <= tol)[rows].all()


def test_attention_infinities_and_nan_in_keys_that_count(sp, cuda):
    """An infinite score is NaN, as in the definition (infinity minus infinity); one of -infinity is a masked key; a NaN is a
    NaN; the other requests do not notice."""
    import torch

    case = Paged(cuda, [100, 100, 100, 100, 100], 4, 2, 64, 16, torch.float16, seed=9)
    case.q[:4] = case.q[:4].abs() + 0.5

    def put(r, at, value, which):
        which[case.table[r, at // 16].item(), :, at % 16] = value

    put(0, 50, math.inf, case.kc)
    put(1, 99, -math.inf, case.kc)
    put(2, 3, math.nan, case.kc)
    put(3, 7, math.inf, case.vc)
    o, lse = case.run(sp)
    assert o[0].isnan().all() and lse[0].isnan().all()
    assert o[2].isnan().all() and lse[2].isnan().all()
    assert not o[3].isfinite().any() and lse[3].isfinite().all()
    keep = [i for i in range(100) if i != 99]
    case.k[1], case.v[1] = case.k[1][:, keep], case.v[1][:, keep]
    case.lengths = [100, 99, 100, 100, 100]
    case.check(o, lse, skip=(0, 2, 3))
    # every key of a request at -infinity: nothing to divide by
    case.kc[case.table[4, :7].long()] = -math.inf
    case.q[4] = 1.0
    o, lse = case.run(sp)
    assert o[4].isnan().all()


def test_attention_bad_pages_and_lengths_are_nan_and_stay_with_their_request(sp, cuda):
    import torch

    lengths = [300, 200, 100, 64, 5, 700, 0, 90, 33]
    case = Paged(cuda, lengths, 8, 2, 128, 16, torch.bfloat16, seed=11)
    pages = case.kc.shape[0]
    for r, column, entry in ((0, 18, -1), (2, 0, pages), (4, 0, I32), (5, 20, -I32)):
        case.table[r, column] = entry
    case.len[7], case.len[8] = -5, case.table.shape[1] * 16 + 1
    o, lse = case.run(sp)
    for r in (0, 2, 4, 5, 7, 8):
        assert o[r].isnan().all() and lse[r].isnan().all(), r
    case.check(o, lse, skip=(0, 2, 4, 5, 7, 8))
    case.len[8] = I32
    case.len[7] = -I32 - 1
    o, lse = case.run(sp)
    assert o[7].isnan().all() and o[8].isnan().all()
    case.check(o, lse, skip=(0, 2, 4, 5, 7, 8))


def test_attention_without_pages_or_columns(sp, cuda):
    import torch

    q = torch.randn((3, 4, 64), device=cuda)
    c = torch.empty((0, 2, 16, 64), dtype=torch.float16, device=cuda)
    lens = torch.tensor([0, 5, 0], dtype=torch.int32, device=cuda)
    for width in (0, 3):
        table = torch.zeros((3, width), dtype=torch.int32, device=cuda)
        o = sp.attn_paged(q, c, c, table, lens)
        torch.cuda.synchronize()
        sp.status()
        assert (o[0] == 0).all() and o[1].isnan().all() and (o[2] == 0).all()
    assert sp.attn_paged(q[:0], c, c, table[:0], lens[:0]).shape == (0, 4, 64)


def test_attention_of_an_empty_request_with_2_31_words_of_output(sp, cuda):
    # (queries that are one row, and a cache without pages: only the output takes memory, 8.6 GB)
    import torch

    heads, dim = 1 << 26, 64
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GB")
    q = torch.ones((1, 1, dim), dtype=torch.float16, device=cuda).expand(1, heads, dim)
    c = torch.empty((0, heads // 32, 8, dim), dtype=torch.float16, device=cuda)
    i32 = dict(dtype=torch.int32, device=cuda)
    o = torch.full((1, heads, dim), 9.0, dtype=torch.float16, device=cuda)
    lse = torch.full((1, heads), 9.0, device=cuda)
    sp.attn_paged(q, c, c, torch.zeros((1, 0), **i32), torch.zeros(1, **i32), o, lse=lse)
    sp.status()
    assert not o.any() and (lse == -math.inf).all()
    del o, lse
    torch.cuda.empty_cache()


def test_attention_writes_its_outputs_and_nothing_else(sp, cuda):
    import torch

    case = Paged(cuda, [100, 0, 3000, 7], 8, 4, 64, 32, torch.float16, seed=2)
    room = torch.full((4 * 8 * 64 + 128,), 9.0, dtype=torch.float16, device=cuda)
    before = [t.clone() for t in (case.q, case.kc, case.vc, case.table, case.len)]
    need = sp.attn_paged_workspace(8, 4, 64)
    work = torch.full((need + 64,), 123, dtype=torch.uint8, device=cuda)
    work[:65536] = 0
    for _ in range(3):
        o, lse = case.run(sp, o=room[64:-64].view(4, 8, 64), workspace=work[:need])
        case.check(o, lse)
        assert (work[:65536] == 0).all()
    assert (room[:64] == 9).all() and (room[-64:] == 9).all() and (work[need:] == 123).all()
    for t, b in zip((case.q, case.kc, case.vc, case.table, case.len), before):
        assert torch.equal(t.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
    with pytest.raises(sp.SporkError):
        case.run(sp, workspace=work[:need - 16])


def test_attention_is_the_same_in_every_run(sp, cuda):
    import torch

    case = Paged(cuda, [5000, 3, 0, 777, 2048], 16, 2, 128, 16, torch.bfloat16, seed=4)
    first = case.run(sp)
    for _ in range(20):
        again = case.run(sp)
        assert torch.equal(first[0].view(torch.int16), again[0].view(torch.int16)) and torch.equal(first[1], again[1])


def test_attention_far_into_a_cache(sp, cuda):
    """Pages whose elements lie beyond 2^32 bytes and beyond 2^31 elements."""
    import torch

    page, kv_heads, dim = 64, 4, 128
    pages = (2 ** 31) // (page * kv_heads * dim) + 40
    kc, vc = (torch.empty((pages, kv_heads, page, dim), dtype=torch.float16, device=cuda) for _ in range(2))
    n = 300
    mine = [pages - 1, pages - 37, 5, pages - 2, pages - 20]
    k, v = (torch.randn((n, kv_heads, dim), device=cuda) for _ in range(2))
    at = torch.arange(n, device=cuda)
    slots = torch.tensor(mine, device=cuda)[at // page] * page + at % page
    sp.paged_store(k, v, kc, vc, slots)
    q = torch.randn((1, 8, dim), device=cuda)
    table = torch.tensor([mine], dtype=torch.int32, device=cuda)
    o = sp.attn_paged(q, kc, vc, table, torch.tensor([n], dtype=torch.int32, device=cuda))
    torch.cuda.synchronize()
    ref, _, weighted, size = paged_plain.attention(q[0], k.half().transpose(0, 1), v.half().transpose(0, 1), dim ** -0.5)
    tol, _ = paged_plain.tolerances(torch.float16, n, dim, ref, weighted, size, True)
    assert ((o[0].double() - ref).abs() <= tol).all()


# ------------------------------------------------------------------------------------------------ streams and graphs

def test_another_stream_and_the_wrong_device(sp, cuda):
    import torch

    case = Paged(cuda, [900, 40], 8, 2, 64, 16, torch.float16, seed=6)
    want, _ = case.run(sp)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = [sp.attn_paged(case.q, case.kc, case.vc, case.table, case.len, stream=side) for _ in range(5)]
    torch.cuda.current_stream().wait_stream(side)
    for g in got:
        assert torch.equal(g, want)
    with pytest.raises(TypeError):
        sp.attn_paged(case.q, case.kc, case.vc, case.table.cpu(), case.len)
    with pytest.raises(TypeError):
        sp.paged_store(case.k[0].transpose(0, 1), case.v[0].transpose(0, 1), case.kc, case.vc,
                       torch.zeros(900, dtype=torch.int64))


def test_launches_of_other_shapes_share_a_streams_workspace(sp, cuda):
    """The kept workspace grows with what a launch needs, and every launch leaves its counters at zero for the next one."""
    import torch

    cases = [Paged(cuda, [2000, 5, 700], h, kv, d, 16, torch.float16, seed=h) for h, kv, d in
             ((4, 4, 64), (32, 1, 128), (16, 2, 64), (8, 8, 128), (71, 1, 128))]
    for _ in range(3):
        for c in cases:
            c.check(*c.run(sp))


def test_two_streams_at_once(sp, cuda):
    """Calls that overlap have workspaces of their own."""
    import torch

    cases = [Paged(cuda, [4000, 17, 800], 8, 2, 128, 16, torch.bfloat16, seed=s) for s in (1, 2)]
    want = [c.run(sp)[0] for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(30):
        for i, (c, s) in enumerate(zip(cases, streams)):
            got[i].append(sp.attn_paged(c.q, c.kc, c.vc, c.table, c.len, stream=s))
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        assert all(torch.equal(g, w) for g in gs)


def test_captured_graphs_follow_the_lengths(sp, cuda):
    """Two graphs, replayed in turn, with other lengths, tables and slots in the same buffers than at capture."""
    import torch

    cases = [Paged(cuda, [700, 64, 33], 8, 2, 64, 16, torch.float16, seed=s, width=60) for s in (1, 2)]
    graphs, outs = [], []
    for c in cases:
        sp.attn_paged(c.q, c.kc, c.vc, c.table, c.len)
    torch.cuda.synchronize()
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(sp.attn_paged(c.q, c.kc, c.vc, c.table, c.len))
        graphs.append(g)
    for lengths in ([700, 64, 33], [1, 0, 33], [699, 63, 0], [0, 0, 0]):
        want = []
        for c in cases:
            c.len.copy_(torch.tensor(lengths, dtype=torch.int32))
            want.append(c.run(sp)[0])
        for g in graphs + graphs:
            g.replay()
        torch.cuda.synchronize()
        for w, o in zip(want, outs):
            assert torch.equal(w, o)


def test_streams_that_torch_did_not_make(sp, cuda):
    """The per-thread default stream, one handle for a stream of each thread, and streams that come and go under one handle:
    no workspace is kept by such a handle, and launches that have one in common follow one another."""
    import ctypes
    import threading

    import torch

    from spork_b200 import api

    cases = [Paged(cuda, [4000, 17, 800], 8, 2, 128, 16, torch.bfloat16, seed=s) for s in (1, 2, 3)]
    want = [c.run(sp)[0] for c in cases]
    kept = dict(api._workspaces)
    outs = [[torch.empty_like(w) for _ in range(40)] for w in want]
    torch.cuda.synchronize()
    failed = []

    def decode(i):
        try:
            c, s = cases[i], torch.cuda.ExternalStream(2, device=cuda)  # cudaStreamPerThread
            for o in outs[i]:
                sp.attn_paged(c.q, c.kc, c.vc, c.table, c.len, o, stream=s)
            s.synchronize()
        except Exception as e:
            failed.append(e)

    threads = [threading.Thread(target=decode, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    sp.status()
    for w, os in zip(want, outs):
        assert all(torch.equal(o, w) for o in os)

    cudart = torch.cuda.cudart()
    again = []
    for i in range(12):  # more than there are workspaces; each is destroyed while its launch may still be under way
        c, handle = cases[i % 3], ctypes.c_uint64()
        assert int(cudart.cudaStreamCreate(ctypes.addressof(handle))) == 0
        s = torch.cuda.ExternalStream(handle.value, device=cuda)
        o = torch.empty_like(want[0])
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            sp.attn_paged(c.q, c.kc, c.vc, c.table, c.len, o)
        assert int(cudart.cudaStreamDestroy(handle.value)) == 0
        again.append(o)
    torch.cuda.synchronize()
    sp.status()
    assert all(torch.equal(o, want[i % 3]) for i, o in enumerate(again))
    assert api._workspaces == kept and 1 <= len(api._lent[0]) <= 4

    # after a launch that was given up the counters are cleared before the next use
    for entry in api._lent[0]:
        entry.workspace[:65536] = 1
    assert sp.lib().spork_selftest_bounded_wait(1000, torch.cuda.current_stream().cuda_stream) == 0
    with pytest.raises(sp.SporkError):
        sp.status()
    for o in outs[0]:
        o.fill_(9.0)
    torch.cuda.synchronize()
    decode(0)
    assert not failed and all(torch.equal(o, want[0]) for o in outs[0])


def test_after_a_wait_that_ran_out(sp, cuda):
    """A launch that was given up may leave its workspace's counters as they were: once status() has said so, no kept
    workspace is used again, and the next calls of every stream are right."""
    import torch

    from spork_b200 import api

    case = Paged(cuda, [3000, 17, 800], 8, 2, 128, 16, torch.bfloat16, seed=12)
    side = torch.cuda.Stream()
    want = case.run(sp)[0]
    side.wait_stream(torch.cuda.current_stream())
    sp.attn_paged(case.q, case.kc, case.vc, case.table, case.len, stream=side)
    torch.cuda.synchronize()
    kept = list(api._workspaces.values())
    assert len(kept) >= 2
    for workspace in kept:
        workspace[:65536] = 1  # as a launch would that stopped half way
    assert sp.lib().spork_selftest_bounded_wait(1000, torch.cuda.current_stream().cuda_stream) == 0
    with pytest.raises(sp.SporkError):
        sp.status()
    assert not api._workspaces
    case.check(*case.run(sp))
    with torch.cuda.stream(side):
        assert torch.equal(sp.attn_paged(case.q, case.kc, case.vc, case.table, case.len), want)
    torch.cuda.synchronize()


def test_the_range_checked_build_agrees(sp, cuda):
    """Every kernel through libspork_b200_checked.so, in a process of its own: no range check fires, results are right."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    checked = os.path.join(root, "spork_b200", "libspork_b200_checked.so")
    if not os.path.exists(checked):
        pytest.skip("libspork_b200_checked.so was not built (python -m spork_b200.build --checked)")
    if os.environ.get("SPORK_B200_LIBRARY") == checked:
        pytest.skip("this is that process")
    names = "attention_matches or many_requests or one_long or bad_pages or captured or test_store or tables_match"
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "-m", "gpu", "-k", names, os.path.abspath(__file__)],
                       capture_output=True, text=True, env=dict(os.environ, SPORK_B200_LIBRARY=checked), timeout=600, cwd=root)
    assert r.returncode == 0 and "passed" in r.stdout, r.stdout[-3000:] + r.stderr[-2000:]


# ------------------------------------------------------------------------------------------------ all together

@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("graph", [False, True])
def test_prompts_and_decoding_together(sp, cuda, dtype, graph):
    """Prompts through attn_fwd and into the cache, then steps of one token each (the whole step captured in a graph, where
    asked): every step's output is the last row of a causal attn_fwd over all tokens so far, within both sides' rounding."""
    import torch

    dtype = getattr(torch, dtype)
    heads = kv_heads = 4
    dim, page, steps = 128, 16, 20
    prompts = [37, 1, 130, 64]
    n, most = len(prompts), max(prompts) + steps
    g = torch.Generator(device=cuda).manual_seed(1)
    tokens = [torch.randn((p + steps, 3, heads, dim), generator=g, device=cuda).to(dtype) for p in prompts]
    i32 = dict(dtype=torch.int32, device=cuda)
    pages = sum(-(-(p + steps) // page) for p in prompts) + 1
    free = torch.randperm(pages, generator=g, device=cuda).to(torch.int32)
    kc, vc = (torch.full((pages, kv_heads, page, dim), math.nan, dtype=dtype, device=cuda) for _ in range(2))
    table = torch.full((n, -(-most // page)), -1, **i32)
    # the prompts: the slot map serves q, k and v of all of them, packed one behind the other
    slots, offsets, lengths, info = sp.paged_tables(torch.zeros(n, **i32), torch.tensor(prompts, **i32), table, free,
                                                    torch.zeros(1, **i32), page_size=page, max_tokens=sum(prompts) + 9)
    packed = torch.cat([t[:p] for t, p in zip(tokens, prompts)] + [torch.full((9, 3, heads, dim), math.nan, device=cuda).to(dtype)])
    sp.paged_store(packed[:, 1], packed[:, 2], kc, vc, slots)
    assert info.tolist()[1:3] == [sum(prompts), 0]
    # one decoding step on fixed buffers; lengths and the free list's counter move to the next step at its end
    x = torch.empty((n, 3, heads, dim), dtype=dtype, device=cuda)
    used, ones = info[:1].clone(), torch.ones(n, **i32)

    def step():
        s, _, after, now = sp.paged_tables(lengths, ones, table, free, used, page_size=page, max_tokens=n)
        sp.paged_store(x[:, 1], x[:, 2], kc, vc, s)
        o = sp.attn_paged(x[:, 0], kc, vc, table, after)
        lengths.copy_(after)
        used.copy_(now[:1])
        return o, now

    run = step
    if graph:
        keep = [t.clone() for t in (table, lengths, used, kc, vc)]
        x.zero_()
        step()
        torch.cuda.synchronize()
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            out = step()
        for t, b in zip((table, lengths, used, kc, vc), keep):
            t.copy_(b)

        def run():
            captured.replay()
            return out

    half = torch.finfo(dtype).eps / 2
    for i in range(steps):
        for r, p in enumerate(prompts):
            x[r].copy_(tokens[r][p + i])
        o, now = run()
        torch.cuda.synchronize()
        assert now.tolist()[2] == 0
        for r, p in enumerate(prompts):
            q, k, v = (tokens[r][:p + i + 1, j].transpose(0, 1).contiguous() for j in range(3))
            ref, _, weighted, size = paged_plain.attention(q[:, -1], k, v, dim ** -0.5)
            tol, _ = paged_plain.tolerances(dtype, p + i + 1, dim, ref, weighted, size, False)
            assert ((o[r].double() - ref).abs() <= tol).all()
            whole = sp.attn_fwd(q, k, v, causal=True)[:, -1]
            # the prompt's kernel rounds its weights to 16 bits (half a step of each) and uses a cubic of relative error
            # 7e-5 for some exponentials: both move the weights, and through their sum the others
            assert ((o[r].double() - whole.double()).abs() <= 2 * tol + weighted * 2 * (half + 1e-4)).all()
    sp.status()
    assert lengths.tolist() == [p + steps for p in prompts]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("graph", [False, True])
def test_projection_store_and_attention_behind_one_another(sp, cuda, dtype, graph):
    """The fp32 result of matmul_sm100 straight into the cache and the attention, step after step with nothing in between and
    one buffer for the projection of all steps: each launch may begin before the one in front of it has ended, and waits
    for it before it touches memory.  The outputs are those of steps that are waited for, bit for bit, and these are the
    definition's."""
    import torch

    dtype = getattr(torch, dtype)
    n, heads, kv_heads, dim, page, steps, width = 6, 8, 2, 64, 16, 40, 512
    g = torch.Generator(device=cuda).manual_seed(3)
    i32 = dict(dtype=torch.int32, device=cuda)
    x = torch.randn((steps, n, width), generator=g, device=cuda).half()
    w = torch.randn(((heads + 2 * kv_heads) * dim, width), generator=g, device=cuda).mul_(width ** -0.5).half()
    blocks = -(-steps // page)
    free = torch.randperm(n * blocks, generator=g, device=cuda).to(torch.int32)
    qkv = torch.empty((n, w.shape[0]), dtype=torch.float32, device=cuda)
    q, k, v = (t.unflatten(1, (-1, dim)) for t in qkv.split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
    kc, vc = (torch.empty((n * blocks, kv_heads, page, dim), dtype=dtype, device=cuda) for _ in range(2))
    table = torch.empty((n, blocks), **i32)
    zeros, ones, none = torch.zeros(n, **i32), torch.ones(n, **i32), torch.zeros(1, **i32)

    def decode(between):
        lengths, used, outs = zeros, none, []
        for i in range(steps):
            sp.matmul_sm100(x[i], w, qkv, split_k=1)
            slots, _, lengths, info = sp.paged_tables(lengths, ones, table, free, used, page_size=page, max_tokens=n)
            sp.paged_store(k, v, kc, vc, slots)
            outs.append(sp.attn_paged(q, kc, vc, table, lengths))
            used = info[:1]
            between()
        return outs

    def clear():
        qkv.fill_(math.nan)
        kc.fill_(math.nan)
        vc.fill_(math.nan)
        table.fill_(-1)
        torch.cuda.synchronize()

    projections = []

    def keep():
        torch.cuda.synchronize()
        projections.append(qkv.clone())

    clear()
    want = decode(keep)
    torch.cuda.synchronize()
    sp.status()
    for r in (0, n - 1):
        for i in (0, 15, 16, steps - 1):
            qs, ks, vs = torch.stack(projections[:i + 1])[:, r].split([heads * dim, kv_heads * dim, kv_heads * dim], 1)
            keys, values = (t.unflatten(1, (kv_heads, dim)).transpose(0, 1).to(dtype) for t in (ks, vs))
            query = qs[i].unflatten(0, (heads, dim))
            ref, _, weighted, size = paged_plain.attention(query, keys, values, dim ** -0.5)
            tol, _ = paged_plain.tolerances_of_fp32_queries(dtype, query, keys, dim ** -0.5, ref, weighted, size)
            assert ((want[i][r].double() - ref).abs() <= tol).all(), (r, i)
    # and the projection itself: 16-bit factors, exact products, sums of `width` of them in 32 bits
    exact = x[steps - 1].double() @ w.double().t()
    assert ((projections[-1].double() - exact).abs() <= width * 2.0 ** -23 * (x[steps - 1].double().abs() @ w.double().abs().t())).all()
    if graph:
        clear()
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            outs = decode(lambda: None)
    for _ in range(3):
        clear()
        if graph:
            for o in outs:
                o.fill_(9.0)
            captured.replay()
            got = outs
        else:
            got = decode(lambda: None)
        torch.cuda.synchronize()
        sp.status()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
