"""CPU tests of the paged cache's entry points: refusals, before anything is launched."""
import struct

import pytest

FAKE = 0x7F0000000000  # an aligned address that no check follows


def tables_args(**kw):
    a = dict(lengths=FAKE, new_tokens=FAKE + 4096, block_table=FAKE + 2 * 4096, free_pages=FAKE + 3 * 4096,
             free_used=FAKE + 4 * 4096, slots=FAKE + 5 * 4096, offsets=FAKE + 6 * 4096, lengths_after=FAKE + 7 * 4096,
             info=FAKE + 8 * 4096, table_stride=8, max_tokens=16, requests=4, max_blocks=8, page_size=16, free_count=32)
    a.update(kw)
    return struct.pack("=9Q2q4i", *a.values())


def cache(**kw):
    a = dict(k=FAKE, v=FAKE + (1 << 30), kp=2 * 16 * 64, kh=16 * 64, kr=64, vp=2 * 16 * 64, vh=16 * 64, vr=64, type=0,
             num_pages=8, kv_heads=2, page_size=16, head_dim=64, reserved=0)
    a.update(kw)
    return struct.pack("=QQ6q6i", *a.values())


def store_args(c=None, **kw):
    a = dict(k=FAKE, v=FAKE, slots=FAKE, kt=128, kh=64, vt=128, vh=64, tokens=4, src_type=0, reserved=0)
    a.update(kw)
    return (c or cache()) + struct.pack("=3Q5q2i", *a.values())


def attn_args(c=None, **kw):
    a = dict(q=FAKE, block_table=FAKE, lengths=FAKE, o=FAKE, lse=0, workspace=FAKE, workspace_bytes=1 << 40, qr=4 * 64, qh=64,
             table_stride=8, requests=4, heads=4, max_blocks=8, q_type=0, scale=0.125, reserved=0)
    a.update(kw)
    return (c or cache()) + struct.pack("=6Q4q4ifi", *a.values())


@pytest.mark.parametrize("change,code", [
    (dict(requests=-1), 10002), (dict(page_size=0), 10002), (dict(max_tokens=-1), 10002), (dict(table_stride=7), 10002),
    (dict(free_count=-1), 10002), (dict(max_blocks=-1), 10002), (dict(requests=16385, table_stride=8), 10006),
    (dict(max_tokens=(1 << 31) - 1), 10006), (dict(free_count=(1 << 31) - 1), 10006), (dict(lengths=0), 10001), (dict(slots=FAKE + 5 * 4096 + 4), 10001),
    (dict(lengths_after=FAKE), 10001), (dict(lengths_after=FAKE + 12), 10001), (dict(info=FAKE + 4 * 4096), 10001),
    (dict(offsets=FAKE + 5 * 4096 + 64), 10001), (dict(free_pages=FAKE + 2 * 4096 + 64), 10001), (dict(info=FAKE + 2), 10001)])
def test_tables_refuses(sp, change, code):
    assert sp.lib().spork_paged_sm100_tables(tables_args(**change), None) == code


@pytest.mark.parametrize("change,code", [
    (dict(num_pages=-1), 10002), (dict(page_size=0), 10002), (dict(head_dim=0), 10002), (dict(type=2), 10001),
    (dict(k=0), 10001), (dict(v=FAKE + 1), 10001), (dict(kp=0), 10001), (dict(kh=63), 10001), (dict(vr=63), 10001),
    (dict(kp=2 * 16 * 64 - 8), 10001), (dict(vp=-2048), 10001), (dict(kh=64, kr=64), 10001)])
def test_store_and_attention_refuse_a_cache(sp, change, code):
    assert sp.lib().spork_paged_sm100_store(store_args(cache(**change)), None) == code
    assert sp.lib().spork_attn_sm100_paged(attn_args(cache(**change)), None) == code


@pytest.mark.parametrize("change,code", [
    (dict(tokens=-1), 10002), (dict(tokens=1 << 31), 10006), (dict(src_type=1), 10001), (dict(k=0), 10001),
    (dict(v=FAKE + 1), 10001), (dict(slots=0), 10001), (dict(slots=FAKE + 4), 10001), (dict(src_type=2, k=FAKE + 2), 10001),
    (dict(tokens=0), 0)])
def test_store_refuses(sp, change, code):
    assert sp.lib().spork_paged_sm100_store(store_args(**change), None) == code


INT_MAX = 2 ** 31 - 1


@pytest.mark.parametrize("kv_heads,head_dim,shift", [
    (1, INT_MAX, 0), (1 << 30, 1, 0), (1 << 15, 1 << 15, 1), (INT_MAX, INT_MAX, 0), (3, 715827883, 0), ((1 << 30) - 100, 1, 0),
    (1 << 16, 1 << 17, 0)])  # the last one in pieces of 8 elements
def test_store_refuses_rows_of_more_pieces_than_32_bits_count(sp, kv_heads, head_dim, shift):
    # (one row to a page, so that no stride comes into it but that of the heads)
    c = cache(kv_heads=kv_heads, head_dim=head_dim, page_size=1, num_pages=1, kh=head_dim, vh=head_dim, k=FAKE + 2 * shift)
    assert sp.lib().spork_paged_sm100_store(store_args(c, kh=head_dim, vh=head_dim, tokens=1), None) == 10006


@pytest.mark.parametrize("halves", ["k", "v", "kv"])
@pytest.mark.parametrize("change", [
    # rows that cover 2^71 elements, which 64 bits would wrap to less than nothing, and pages that lie inside them
    dict(page_size=INT_MAX - 63, r=1 << 40, p=1 << 40, num_pages=INT_MAX), dict(page_size=1 << 30, r=1 << 40, p=1 << 40),
    dict(page_size=1 << 20, r=1 << 40), dict(num_pages=INT_MAX, p=1 << 40), dict(num_pages=1 << 24, p=1 << 40, h=1 << 40)])
def test_a_cache_that_covers_more_than_an_address_space_is_refused(sp, change, halves):
    sizes = {k: v for k, v in change.items() if len(k) > 1}
    c = cache(**sizes, **{half + k: v for half in halves for k, v in change.items() if len(k) == 1})
    assert sp.lib().spork_paged_sm100_store(store_args(c), None) in (10001, 10006)
    assert sp.lib().spork_attn_sm100_paged(attn_args(c), None) in (10001, 10006)


@pytest.mark.parametrize("change,code", [
    (dict(requests=-1), 10002), (dict(heads=3), 10002), (dict(heads=-2), 10002), (dict(max_blocks=-1), 10002),
    (dict(table_stride=7), 10002), (dict(q=0), 10001), (dict(q=FAKE + 1), 10001), (dict(q_type=1), 10001),
    (dict(q_type=2, q=FAKE + 2), 10001), (dict(lengths=0), 10001), (dict(lengths=FAKE + 2), 10001), (dict(o=0), 10001),
    (dict(o=FAKE + 8), 10001), (dict(lse=FAKE + 2), 10001), (dict(block_table=0), 10001), (dict(scale=0.0), 10001),
    (dict(scale=-1.0), 10001), (dict(scale=float("nan")), 10001), (dict(scale=float("inf")), 10001),
    (dict(workspace=FAKE + 8), 10001), (dict(requests=0), 0), (dict(heads=0), 0)])
def test_attention_refuses(sp, change, code):
    assert sp.lib().spork_attn_sm100_paged(attn_args(**change), None) == code


@pytest.mark.parametrize("change,code", [
    (dict(k=FAKE + 8), 10001), (dict(kr=68, kh=16 * 68, kp=2 * 16 * 68), 10001), (dict(head_dim=96, kr=96, kh=16 * 96, kp=2 * 16 * 96,
     vr=96, vh=16 * 96, vp=2 * 16 * 96), 10002), (dict(page_size=24, kh=24 * 64, kp=48 * 64, vh=24 * 64, vp=48 * 64), 10002),
    (dict(kv_heads=0), 10002)])
def test_attention_refuses_what_the_store_takes(sp, change, code):
    assert sp.lib().spork_attn_sm100_paged(attn_args(cache(**change)), None) == code


def test_null_structures_are_refused(sp):
    L = sp.lib()
    for fn in (L.spork_paged_sm100_tables, L.spork_paged_sm100_store, L.spork_attn_sm100_paged):
        assert fn(None, None) == 10001


def test_supports(sp):
    assert sp.attn_paged_supports(32, 8, 128, 16) and sp.attn_paged_supports(7, 1, 64, 192) and sp.attn_paged_supports(8, 8, 64, 8)
    assert not sp.attn_paged_supports(32, 5, 128, 16)
    assert not sp.attn_paged_supports(32, 0, 128, 16)
    assert not sp.attn_paged_supports(32, 8, 96, 16)
    for page in (0, 1, 4, 24, 48, 96, -64):
        assert not sp.attn_paged_supports(32, 8, 128, page)


def test_streams_that_torch_did_not_make_take_turns():
    """Which workspace a launch gets: its stream's last one, else one that has no memory yet, else the one that was not used for
    the longest time.  (Every launch waits for the event of the one before it with the same workspace.)"""
    from spork_b200 import api

    pool = []
    first = [api._whose_turn(pool, h) for h in (2, 64, 128, 192)]
    assert len({id(e) for e in first}) == 4 and not any(e.clean or e.workspace for e in first)
    for e in first:
        e.workspace, e.clean = object(), True
    assert api._whose_turn(pool, 2) is first[0] and api._whose_turn(pool, 64) is first[1]
    assert api._whose_turn(pool, 256) is first[2] and first[2].handle == 256  # 128's was used longest ago
    assert api._whose_turn(pool, 128) is first[3] and api._whose_turn(pool, 2) is first[0]
    assert len(pool) == 4 and all(e.clean for e in pool)


def test_wrappers_refuse_shapes_types_and_host_tensors(sp):
    import torch

    i32 = dict(dtype=torch.int32)
    lens, table, free, used = torch.zeros(3, **i32), torch.zeros((3, 4), **i32), torch.zeros(9, **i32), torch.zeros(1, **i32)

    def tables(lengths=lens, new=lens, table=table, free=free, used=used, **kw):
        return sp.paged_tables(lengths, new, table, free, used, **{**dict(page_size=16, max_tokens=5), **kw})

    for kw in (dict(new=lens[:2]), dict(table=table[:2]), dict(table=table[0]), dict(used=free), dict(page_size=0),
               dict(max_tokens=None), dict(max_tokens=-1), dict(slots=torch.zeros(4, dtype=torch.int64)), dict(free=free[::2]),
               dict(table=table.t().contiguous().t()), dict(offsets=lens), dict(info=lens), dict(lengths_after=free),
               dict(lengths=lens[None]), dict(page_size=1 << 31)):
        with pytest.raises(ValueError):
            tables(**kw)
    for kw in (dict(lengths=lens.long()), dict(free=free.long()), dict(table=table.long()),
               dict(slots=torch.zeros(5, **i32)), dict()):  # the last: all as it should be, but not on a GPU
        with pytest.raises(TypeError):
            tables(**kw)

    c = torch.zeros((6, 2, 16, 64), dtype=torch.float16)
    x, slots = torch.zeros((3, 2, 64), dtype=torch.float16), torch.zeros(3, dtype=torch.int64)

    def store(k=x, v=x, kc=c, vc=c, slots=slots):
        return sp.paged_store(k, v, kc, vc, slots)

    for kw in (dict(v=x[:2]), dict(k=x[:, :1], v=x[:, :1]), dict(vc=c[:3]), dict(kc=c[0], vc=c[0]), dict(slots=slots[:2]),
               dict(k=x.transpose(1, 2).contiguous().transpose(1, 2)), dict(kc=c.transpose(2, 3).contiguous().transpose(2, 3)),
               dict(slots=torch.zeros(6, dtype=torch.int64)[::2])):
        with pytest.raises(ValueError):
            store(**kw)
    for kw in (dict(k=x.bfloat16()), dict(k=x.bfloat16(), v=x.bfloat16()), dict(vc=c.bfloat16()), dict(kc=c.float(), vc=c.float()),
               dict(slots=slots.int()), dict(k=x.double(), v=x.double()), dict()):
        with pytest.raises(TypeError):
            store(**kw)

    q = torch.zeros((3, 4, 64), dtype=torch.float16)

    def attn(q=q, kc=c, vc=c, table=table, lengths=lens, **kw):
        return sp.attn_paged(q, kc, vc, table, lengths, **kw)

    for kw in (dict(q=q[0]), dict(q=q[:, :, :32]), dict(lengths=lens[:2]), dict(table=table[:1]), dict(o=q[:2]),
               dict(lse=torch.zeros((3, 3))), dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)),
               dict(o=torch.zeros((3, 4, 128), dtype=torch.float16)[:, :, ::2])):
        with pytest.raises(ValueError):
            attn(**kw)
    for kw in (dict(q=q.bfloat16()), dict(q=q.double()), dict(o=q.bfloat16()), dict(lengths=lens.long()), dict(table=table.long()),
               dict(o=q)):
        with pytest.raises(TypeError):
            attn(**kw)


# ------------------------------------------------------------------------------------------------ how a launch is cut

def _plan(sp, lengths, **kw):
    args = dict(heads=8, kv_heads=2, head_dim=128, page_size=16, max_blocks=1 << 14, sm_count=148) | kw
    return [sp.attn_paged_plan(lengths, b, **args) for b in range(2 * args["sm_count"])], args


@pytest.mark.parametrize("seed", range(12))
def test_every_unit_is_in_one_run_and_every_part_has_a_place(sp, seed):
    """The kernel's own cutting, on the host: all units of each (request, key head, unit of query heads) once, in the order
    of the blocks; the parts of one that is cut are those of neighbouring blocks, each in a slot of its own, the first one
    in the slot that the others' joining computes for it and all others in slot 0; short ones are not cut; runs are of one
    size."""
    import random

    rng = random.Random(seed)
    dim = rng.choice([64, 128])
    tile = 8192 // dim
    kv_heads, group = rng.choice([(1, 1), (2, 5), (8, 8), (4, 16), (1, 71), (3, 33)])
    most = rng.choice([1, 3, 40, 700, 5000, 100000])
    lengths = [rng.choice([0, 1, tile, tile + 1, rng.randint(0, most), -3, 1 << 30]) for _ in range(rng.choice([1, 2, 23, 300, 1000]))]
    blocks, args = _plan(sp, lengths, heads=kv_heads * group, kv_heads=kv_heads, head_dim=dim, sm_count=rng.choice([148, 3, 64]))
    capacity = args["max_blocks"] * args["page_size"]
    head_units = -(-group // (8 if group <= 8 else 16 if group <= 16 else 32))
    found, slots = {}, set()
    for b, runs in enumerate(blocks):
        for run in runs:
            found.setdefault((run["request"], run["kv_head"], run["head_unit"]), []).append((b, run))
    want = {(r, kv, hu): -(-n // tile) for r, n in enumerate(lengths) if 0 < n <= capacity
            for kv in range(kv_heads) for hu in range(head_units)}
    assert set(found) == set(want)
    for key, parts in found.items():
        at = 0
        for i, (b, run) in enumerate(parts):
            assert run["first"] == at and run["units"] == want[key] and run["count"] > 0
            at += run["count"]
            if len(parts) > 1:
                assert run["blocks"] == len(parts) and run["first_block"] + i == b
                assert i == 0 or run["slot"] == 0
                assert (b, run["slot"]) not in slots
                slots.add((b, run["slot"]))
        assert at == want[key]
        assert len(parts) == 1 or want[key] > 4
    # a run: its units and what a (request, head unit) costs besides, one unit; those that are not cut lie to either side
    sizes = [sum(run["count"] + 1 for run in runs) for runs in blocks]
    total = sum(n + 1 for n in want.values())
    assert max(sizes, default=0) <= -(-total // len(blocks)) + 2 + 2 * 5


def test_small_launches_are_not_cut_into_crumbs(sp):
    blocks, _ = _plan(sp, [64 * 6])
    busy = [runs for runs in blocks if runs]
    assert len(busy) <= 8 and all(sum(r["count"] for r in runs) >= 1 for runs in busy)
    blocks, _ = _plan(sp, [64 * 4, 1, 100], heads=2)
    assert all(run["count"] == run["units"] for runs in blocks for run in runs)


def test_plan_refuses(sp):
    for kw in (dict(heads=7), dict(head_dim=96), dict(page_size=24), dict(sm_count=0), dict(max_blocks=-1)):
        with pytest.raises(ValueError):
            sp.attn_paged_plan([100], 0, **(dict(heads=8, kv_heads=2, head_dim=128, page_size=16, max_blocks=64) | kw))
    with pytest.raises(ValueError):
        sp.attn_paged_plan([100], 296, heads=8, kv_heads=2, head_dim=128, page_size=16, max_blocks=64)
    # more places in the list than 32 bits number: 2^25 units a request
    with pytest.raises(ValueError):
        sp.attn_paged_plan([100] * 100, 0, heads=8, kv_heads=2, head_dim=128, page_size=64, max_blocks=1 << 25)


@pytest.mark.parametrize("requests,kv_heads,dim,blocks", [(4096, 1 << 30, 128, (1 << 25) - 2), (4096, INT_MAX, 128, 1 << 20),
                                                          (32768, 1 << 24, 128, (1 << 25) - 2), (8192, INT_MAX, 64, 1 << 20)])
def test_plan_refuses_more_places_than_64_bits_number(sp, requests, kv_heads, dim, blocks):
    # the product wraps 64 bits, to zero or less (lengths of zero, so that nothing is walked through where it is not refused)
    with pytest.raises(ValueError):
        sp.attn_paged_plan([0] * requests, 0, heads=kv_heads, kv_heads=kv_heads, head_dim=dim, page_size=64, max_blocks=blocks)
