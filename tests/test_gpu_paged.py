"""Paged cache and windowed attention on the GPU against the 64-bit statements of tests/paged_reference.py."""
import os
import random
import subprocess
import sys

import pytest
import torch

import paged_reference as R
from shareprefill_b200 import native

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------------ plan
def _random_plan(seed, requests, page, spare, ctx, new, pad, width_cut=0, short_rows=0):
    rng = random.Random(seed)
    cached = [rng.choice([0, 1, page - 1, page, page + 1, rng.randint(0, ctx)]) for _ in range(requests)]
    fresh = [rng.choice([0, 1, 1, page, rng.randint(0, new)]) for _ in range(requests)]
    held = [-(-c // page) for c in cached]
    width = max(-(-(c + n) // page) for c, n in zip(cached, fresh)) + 1 - width_cut
    width = max(width, max(held), 1)
    ids = list(range(sum(held) + spare))
    rng.shuffle(ids)
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-7] * (width - h))
        at += h
    head = rng.randrange(len(ids) or 1)
    ring = [-9] * max(len(ids), 1)
    for i, x in enumerate(ids[at:]):
        ring[(head + i) % len(ring)] = x
    return cached, fresh, table, width, ring, head, spare, max(0, sum(fresh) + pad - short_rows)


@pytest.mark.parametrize("seed,requests,page,spare,ctx,new,pad,width_cut,short_rows", [
    (1, 1, 16, 4, 40, 3, 0, 0, 0), (2, 7, 16, 200, 300, 70, 5, 0, 0), (3, 33, 32, 9, 500, 200, 0, 0, 0),
    (4, 64, 64, 0, 900, 100, 3, 0, 0), (5, 513, 16, 700, 700, 60, 11, 2, 0), (6, 1500, 256, 500, 5000, 20, 0, 0, 300),
    (7, 4096, 16, 9000, 100, 40, 1, 1, 17), (8, 3, 128, 50, 40, 9000, 0, 0, 0),
])
def test_plan_equals_the_statement(seed, requests, page, spare, ctx, new, pad, width_cut, short_rows):
    cached, fresh, table, width, ring, head, count, n_rows = _random_plan(seed, requests, page, spare, ctx, new, pad,
                                                                          width_cut, short_rows)
    want = R.plan(cached, fresh, table, width, ring, head, count, n_rows, page)
    t = _ints(table)
    got = native.paged_plan(_ints(cached), _ints(fresh), t, _ints(ring), _ints([head, count]), n_rows, page)
    assert t.tolist() == want["table"]
    for name in ("cu_new", "seq_len", "refused", "slot_map", "positions", "ring_state"):
        assert getattr(got, name).tolist() == want[name], name
    # once more over its own result: the entries are found again, not taken anew
    again = native.paged_plan(_ints(cached), _ints(fresh), t, _ints(ring), _ints([head, count]), n_rows, page)
    assert t.tolist() == want["table"] and again.slot_map.tolist() == want["slot_map"]


def test_plan_in_place_state_odd_lengths_and_padded_table_rows():
    page, cap = 16, 10
    ring, state = _ints(list(range(100, 100 + cap))), _ints([8, 5])
    table = torch.full((3, 9), -1, dtype=torch.int32, device="cuda")[:, :6]      # rows further apart than wide
    cached, fresh = _ints([-4, 0, 16]), _ints([17, -3, 1])
    table[2, 0] = 55
    p = native.paged_plan(cached, fresh, table, ring, state, 20, page, ring_state_out=state)
    want = R.plan([-4, 0, 16], [17, -3, 1], [[-1] * 6, [-1] * 6, [55] + [-1] * 5], 6, list(range(100, 110)), 8, 5, 20, page)
    assert p.ring_state.data_ptr() == state.data_ptr() and state.tolist() == want["ring_state"] == [1, 2]
    assert table.tolist() == want["table"] and p.slot_map.tolist() == want["slot_map"]
    assert p.seq_len.tolist() == [17, 0, 17] and p.refused.tolist() == [0, 0, 0]


@pytest.mark.parametrize("requests", [4073, 4074, 4075, 4095])
def test_plan_of_nearly_the_most_requests_in_a_fresh_process(requests):
    # (a call with more requests before it in the process would raise the kernel's limit of shared memory for this one)
    program = f"""
import torch
from shareprefill_b200 import native
i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
r = {requests}
table = torch.full((r, 1), -1, dtype=torch.int32, device="cuda")
p = native.paged_plan(i([0] * r), i([1] * r), table, torch.arange(r, dtype=torch.int32, device="cuda"), i([0, r]), r, 16)
assert p.slot_map.tolist() == [16 * x for x in range(r)] and p.ring_state.tolist() == [0, 0] and not p.refused.any()
"""
    done = subprocess.run([sys.executable, "-c", program], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_plan_from_the_end_of_a_ring_of_more_than_2_to_the_30_ids():
    # head + capacity is more than an int holds
    cap = (1 << 30) + 16
    ring = torch.empty(cap, dtype=torch.int32, device="cuda")
    ring[-2:], ring[:3] = _ints([7, 5]), _ints([9, 4, 6])
    for head in (cap - 2, -2):
        table = torch.full((2, 3), -1, dtype=torch.int32, device="cuda")
        p = native.paged_plan(_ints([0, 0]), _ints([33, 17]), table, ring, _ints([head, 5]), 50, 16)
        assert table.tolist() == [[7, 5, 9], [4, 6, -1]] and p.ring_state.tolist() == [3, 0] and p.refused.tolist() == [0, 0]
        assert p.slot_map.tolist() == [16 * page + i for page, n in ((7, 16), (5, 16), (9, 1), (4, 16), (6, 1)) for i in range(n)]


def test_plan_may_put_its_outputs_where_its_inputs_were():
    lib, page, rows = native.load(), 16, 40
    cached, new = [15, 0, 16, 100], [2, 17, 0, 9]
    table = [[4, -1, -1], [-1] * 3, [6, -1, -1], [-1] * 3]
    want = R.plan(cached, new, table, 3, [9, 8, 7, 5], 2, 4, rows, page)
    seq, fresh, t, ring, state = _ints(cached), _ints(new), _ints(table), _ints([9, 8, 7, 5]), _ints([2, 4])
    cu, slots, positions = _ints([0] * 5), torch.empty(rows, dtype=torch.int64, device="cuda"), _ints([0] * rows)
    assert lib.spf_paged_plan(seq.data_ptr(), fresh.data_ptr(), 4, page, t.data_ptr(), 3, 3, ring.data_ptr(), 4, state.data_ptr(), state.data_ptr(),
                              cu.data_ptr(), seq.data_ptr(), slots.data_ptr(), positions.data_ptr(), fresh.data_ptr(), rows,
                              torch.cuda.current_stream().cuda_stream) == 0
    got = dict(table=t, cu_new=cu, seq_len=seq, refused=fresh, slot_map=slots, positions=positions, ring_state=state)
    assert {name: x.tolist() for name, x in got.items()} == want


def test_plan_with_extreme_lengths_refuses_and_stays_inside():
    page, top = 16, 2 ** 31 - 1
    table = torch.full((4, 3), -1, dtype=torch.int32, device="cuda")
    ring, state = _ints(list(range(8))), _ints([2 ** 31 - 1, 2 ** 31 - 1])       # head and count past the ring
    p = native.paged_plan(_ints([top, 0, top, 3]), _ints([1, top, top, 2]), table, ring, state, 5, page)
    assert p.refused.tolist() == [1, 1, 1, 1]      # the rows of the last lie behind the batch
    assert p.cu_new.tolist() == [0, 1, 5, 5, 5] and p.slot_map.tolist() == [-1] * 5
    assert bool((table == -1).all())


# ----------------------------------------------------------------------------------------- write
@pytest.mark.parametrize("rows,kv_heads,dim,page,dtype,layout", [
    (1, 1, 64, 16, BF16, "token"), (37, 8, 128, 16, FP16, "head"), (1000, 4, 128, 64, BF16, "joined"),
    (257, 3, 64, 256, FP16, "token"), (5000, 8, 128, 32, BF16, "token"),
])
def test_write_puts_rows_in_their_slots_and_nothing_else(rows, kv_heads, dim, page, dtype, layout):
    g = torch.Generator().manual_seed(rows)
    lengths = [rows]
    pool = R.Pool(lengths, page, kv_heads, dim, dtype, g, layout)
    k_cache, v_cache = pool.cuda()
    k_cache.fill_(3.0), v_cache.fill_(4.0)
    k = torch.randn(rows, kv_heads + 2, dim, generator=g).to(dtype).cuda()[:, 1:-1]     # strided rows
    v = torch.randn(kv_heads, rows, dim, generator=g).to(dtype).cuda().transpose(0, 1)
    n_slots = k_cache.shape[0] * page
    slots = torch.randperm(n_slots, generator=g)[:rows]
    bad = torch.rand(rows, generator=g) < 0.1
    slots[bad] = torch.tensor([-1, n_slots, n_slots + 5, -2 ** 40, 2 ** 62])[torch.randint(0, 5, (int(bad.sum()),), generator=g)]
    want_k, want_v = k_cache.clone(), v_cache.clone()
    keep = slots[~bad].cuda()
    want_k[keep // page, keep % page] = k[~bad.cuda()]
    want_v[keep // page, keep % page] = v[~bad.cuda()]
    native.paged_write(k, v, slots.cuda(), k_cache, v_cache)
    assert torch.equal(k_cache, want_k) and torch.equal(v_cache, want_v)


def test_write_refuses_expanded_caches_and_takes_one_page_or_head_of_any_stride():
    rows = torch.randn(16, 2, 64, device="cuda").to(BF16)
    slots = torch.arange(16, device="cuda")
    cache = torch.zeros(2, 16, 2, 64, dtype=BF16, device="cuda")
    for view in (cache[:1].expand(2, -1, -1, -1), cache[:, :1].expand(-1, 16, -1, -1), cache[:, :, :1].expand(-1, -1, 2, -1)):
        for pair in ((view, cache), (cache, view)):
            with pytest.raises(native.SpfError):
                native.paged_write(rows, rows, slots, *pair)
    assert not cache.any()
    one = cache.as_strided((1, 16, 1, 64), (0, 128, 0, 1))
    native.paged_write(rows[:, :1], rows[:, :1], slots, one, one)
    assert torch.equal(cache[0, :, :1], rows[:, :1]) and not cache[1].any() and not cache[:, :, 1].any()


# ------------------------------------------------------------------------------------- attention
CASES = [
    # (cached, new) per request, page, heads, kv heads, head size, type, window, sinks, cache layout
    ([(0, 1)], 16, 32, 8, 128, BF16, 0, 0, "token"),
    ([(15, 1), (16, 1), (0, 1), (700, 1), (63, 1)], 16, 32, 8, 128, BF16, 0, 0, "head"),
    ([(2000, 1), (31, 1)], 32, 28, 4, 128, FP16, 0, 0, "token"),
    ([(900, 1), (5, 1), (130, 1)], 64, 64, 8, 64, BF16, 100, 4, "joined"),
    ([(900, 1), (5, 1)], 256, 8, 2, 128, BF16, 1, 0, "token"),
    ([(777, 1), (300, 1)], 16, 16, 1, 128, FP16, 33, 200, "token"),
    ([(100, 4), (0, 3), (47, 1), (200, 2)], 16, 8, 2, 128, BF16, 0, 0, "token"),
    ([(0, 130)], 16, 8, 2, 64, BF16, 0, 0, "token"),
    ([(0, 1), (0, 0), (500, 77), (3, 0), (64, 64)], 64, 8, 2, 128, BF16, 0, 0, "head"),
    ([(1000, 300), (0, 257), (33, 1)], 128, 14, 2, 128, FP16, 0, 0, "joined"),
    ([(1000, 300), (0, 257), (33, 1), (5, 40)], 32, 8, 2, 64, FP16, 70, 5, "token"),
    ([(600, 500)], 16, 4, 4, 128, BF16, 128, 130, "head"),
    ([(130, 260), (7, 9)], 16, 40, 1, 128, BF16, 0, 0, "token"),        # 40 heads on one KV head
    ([(50, 3), (0, 20)], 16, 200, 1, 64, BF16, 0, 0, "token"),
    ([(0, 1000)], 256, 6, 2, 128, BF16, 8, 1, "token"),
    ([(3000, 64)] + [(i * 37, 1) for i in range(40)], 16, 8, 2, 128, BF16, 0, 0, "token"),
    ([(i * 29, 1 + 41 * (i % 3)) for i in range(45)], 32, 8, 2, 64, BF16, 90, 2, "head"),
    ([(700, 5), (0, 5), (33, 5)], 64, 16, 2, 128, FP16, 0, 0, "token"),                # all bring as many
    ([(i * i % 700, i % 7 > 0) for i in range(70)], 16, 16, 8, 128, BF16, 0, 0, "token"),      # a worker per warp
    ([(i * 13 % 900, 1 + i % 2) for i in range(260)], 16, 16, 2, 128, FP16, 120, 20, "head"),
    ([(3000 + i, 1) for i in range(300)], 64, 2, 2, 128, BF16, 0, 0, "token"),
    ([(5, 2), (900, 1)], 16, 12, 1, 128, BF16, 0, 0, "token"),                         # 12 rows and 24
]


def _batch(spec, page, heads, kv_heads, dim, dtype, layout, seed):
    g = torch.Generator().manual_seed(seed)
    pool = R.Pool([c + n for c, n in spec], page, kv_heads, dim, dtype, g, layout)
    cu = [0]
    for _, n in spec:
        cu.append(cu[-1] + n)
    q = (1.5 * torch.randn(cu[-1], heads, dim, generator=g)).to(dtype)
    return pool, cu, q


def _check_batch(got, spec, pool, cu, q, scale, window, sinks, dtype, present=None):
    for r, (c, n) in enumerate(spec):
        k, v = pool.rows[r]
        out, mass = R.attention(q[cu[r]:cu[r + 1]], k, v, c, scale, window, sinks, None if present is None else present[r])
        if n:
            R.check(got[cu[r]:cu[r + 1]], out, mass, dtype, c + n, float(v.abs().max()), f"request {r}")


@pytest.mark.parametrize("case", range(len(CASES)))
def test_paged_attention_matches_the_statement(case):
    spec, page, heads, kv_heads, dim, dtype, window, sinks, layout = CASES[case]
    pool, cu, q = _batch(spec, page, heads, kv_heads, dim, dtype, layout, 100 + case)
    k, v = pool.cuda()
    scale = dim ** -0.5
    got = native.paged_attention(q.cuda(), k, v, pool.table.cuda(), _ints(cu), _ints([c + n for c, n in spec]),
                                 max(n for _, n in spec), scale, window, sinks)
    _check_batch(got, spec, pool, cu, q, scale, window, sinks, dtype)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("spec,heads,kv_heads,dim,dtype,window,sinks", [
    ([(700, 90), (40, 200), (0, 3), (5, 0)] + [(i * 29 % 600, 1) for i in range(20)], 8, 2, 128, BF16, 0, 0),
    ([(300, 7), (900, 6), (0, 1), (33, 5)] + [(i * 17, 1) for i in range(20)], 28, 4, 64, FP16, 0, 0),
    ([(2300, 40), (2500, 1)] + [(i * 7, 1) for i in range(60)], 16, 8, 64, BF16, 2100, 4),
])
def test_chunks_and_single_tokens_in_one_pass_or_two(spec, heads, kv_heads, dim, dtype, window, sinks, wide):
    # a table that could hold long sequences makes a batch of tokens and chunks run through both kernels
    pool, cu, q = _batch(spec, 16, heads, kv_heads, dim, dtype, "token", 31)
    k, v = pool.cuda()
    table = torch.nn.functional.pad(pool.table, (0, 6000 if wide else 0), value=-1).cuda()
    out = torch.full((cu[-1] + 3, heads, dim), 7.0, dtype=dtype, device="cuda")
    padded = torch.cat([q, q[:3]]).cuda()
    lengths = _ints([c + n for c, n in spec])
    native.paged_attention(padded, k, v, table, _ints(cu), lengths, max(n for _, n in spec), dim ** -0.5, window, sinks, out)
    _check_batch(out, spec, pool, cu, q, dim ** -0.5, window, sinks, dtype)
    assert (out[cu[-1]:] == 7.0).all()


@pytest.mark.parametrize("new", [1, 3, 90])
def test_rows_without_keys_absent_pages_and_rows_behind_the_batch(new):
    page, heads, kv_heads, dim, dtype = 16, 8, 2, 128, BF16
    spec = [(100, new), (200, new), (40, new)]
    pool, cu, q = _batch(spec, page, heads, kv_heads, dim, dtype, "token", new)
    k, v = pool.cuda()
    # request 0 loses pages 1 and 4 (ids outside the pool), request 1 is refused, request 2 keeps only absent pages
    table = pool.table.clone()
    table[0, 1], table[0, 4] = -3, k.shape[0]
    table[2] = 2 ** 31 - 1
    present = torch.ones(100 + new, dtype=torch.bool)
    present[16:32] = False
    present[64:80] = False
    rows = torch.cat([q, q[:5]]).cuda()
    out = torch.full_like(rows, 7.0)
    got = native.paged_attention(rows, k, v, table.cuda(), _ints(cu), _ints([100 + new, 0, 40 + new]), new, dim ** -0.5,
                                 out=out)
    assert got.data_ptr() == out.data_ptr()
    _check_batch(got, spec[:1], pool, cu, q, dim ** -0.5, 0, 0, dtype, [present])
    assert bool((got[cu[1]:cu[3]] == 0).all()), "refused and absent: zeros"
    assert bool((got[cu[3]:] == 7).all()), "rows behind the batch were touched"


@pytest.mark.parametrize("new,page,window,sinks", [(1, 16, 90, 20), (50, 16, 90, 20), (50, 64, 90, 70), (200, 32, 120, 5), (60, 128, 100, 150)])
def test_absent_pages_among_sinks_and_window(new, page, window, sinks):
    heads, kv_heads, dim, dtype = 8, 2, 64, FP16
    spec = [(400, new), (700, new)]
    pool, cu, q = _batch(spec, page, heads, kv_heads, dim, dtype, "token", new)
    k, v = pool.cuda()
    table, present = pool.table.clone(), []
    for r, gone in enumerate(([0, 2], [0, (700 - 60) // page, (700 - 20) // page])):
        present.append(torch.ones(spec[r][0] + new, dtype=torch.bool))
        for i in gone:
            table[r, i] = -1
            present[r][i * page:(i + 1) * page] = False
    got = native.paged_attention(q.cuda(), k, v, table.cuda(), _ints(cu), _ints([c + n for c, n in spec]), new, 0.125, window, sinks)
    _check_batch(got, spec, pool, cu, q, 0.125, window, sinks, dtype, present)


def test_sinks_and_windows_of_every_relation():
    # window edges and sinks on, before and behind the places where units, pages and copies begin
    dim, g = 64, torch.Generator().manual_seed(71)
    for new, keys in ((1, 400), (30, 400), (400, 400)):
        q = torch.randn(new, 4, dim, generator=g).to(BF16)
        k, v = (torch.randn(keys, 2, dim, generator=g).to(BF16) for _ in range(2))
        for window in (1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200, 399, 400, 401):
            for sinks in (0, 1, 16, 31, 32, 33, 64, 127, 129, 390):
                out, mass = R.attention(q, k, v, keys - new, 0.125, window, sinks)
                got = native.window_attention(q.cuda(), k.cuda(), v.cuda(), 0.125, window, sinks)
                R.check(got, out, mass, BF16, keys, 5.0, f"{new} new, window {window}, sinks {sinks}")


def test_offsets_and_lengths_that_lie_are_clipped():
    page, heads, kv_heads, dim = 16, 8, 2, 64
    spec = [(30, 2)]
    pool, cu, q = _batch(spec, page, heads, kv_heads, dim, BF16, "token", 5)
    k, v = pool.cuda()
    table = pool.table.cuda().expand(3, -1).contiguous()
    for cu_bad in ([0, 2, 2, 400], [-9, 2, 2, 2], [0, 2, 2, 1]):
        got = native.paged_attention(q.cuda(), k, v, table, _ints(cu_bad), _ints([32, 2 ** 31 - 1, -1]), 2, dim ** -0.5)
        _check_batch(got, spec, pool, cu, q, dim ** -0.5, 0, 0, BF16)


@pytest.mark.parametrize("requests", [5, 40, 300])
def test_a_request_longer_than_max_new_says_leaves_the_others_right(requests):
    # 16 rows a tile are two tokens of eight heads: three tokens are more than one tile where one token was promised
    spec = [(10 + 7 * i, 3 if i == 3 else 1) for i in range(requests)]
    pool, cu, q = _batch(spec, 16, 8, 1, 64, BF16, "token", requests)
    k, v = pool.cuda()
    got = native.paged_attention(q.cuda(), k, v, pool.table.cuda(), _ints(cu), _ints([c + n for c, n in spec]), 1, 0.125)
    for r, (c, n) in enumerate(spec):
        if r != 3:
            out, mass = R.attention(q[cu[r]:cu[r + 1]], *pool.rows[r], c, 0.125)
            R.check(got[cu[r]:cu[r + 1]], out, mass, BF16, c + n, 5.0, f"request {r}")


@pytest.mark.parametrize("new", [1, 200])
def test_cache_of_more_than_32_bits_of_elements(new):
    page, heads, kv_heads, dim = 64, 8, 8, 128
    n_pages = (2 ** 32 // (page * kv_heads * dim)) + 40
    if torch.cuda.mem_get_info()[0] < 3 * n_pages * page * kv_heads * dim * 2:
        pytest.skip("not enough free memory")
    spec = [(500, new)]
    pool, cu, q = _batch(spec, page, heads, kv_heads, dim, BF16, "token", 11)
    k, v = (torch.empty(n_pages, page, kv_heads, dim, dtype=BF16, device="cuda") for _ in range(2))
    table = torch.full_like(pool.table, -1)
    for i in range(-(-(500 + new) // page)):
        table[0, i] = n_pages - 1 - 2 * i
        k[table[0, i]] = pool.k[pool.table[0, i]].cuda()
        v[table[0, i]] = pool.v[pool.table[0, i]].cuda()
    got = native.paged_attention(q.cuda(), k, v, table.cuda(), _ints(cu), _ints([500 + new]), new, dim ** -0.5)
    _check_batch(got, spec, pool, cu, q, dim ** -0.5, 0, 0, BF16)


# ---------------------------------------------------------------------------------------- window
@pytest.mark.parametrize("new,keys,heads,kv_heads,dim,dtype,window,sinks,layout", [
    (1, 1, 32, 8, 128, BF16, 4, 0, "token"), (1, 5000, 32, 8, 128, BF16, 1000, 4, "token"),
    (1, 3001, 28, 4, 64, FP16, 37, 300, "head"), (5, 5, 8, 2, 128, BF16, 2, 1, "token"),
    (129, 129, 8, 2, 128, FP16, 64, 0, "head"), (1000, 1000, 8, 2, 64, BF16, 256, 4, "token"),
    (700, 1500, 14, 2, 128, BF16, 300, 140, "token"), (257, 900, 4, 4, 128, BF16, 5000, 3, "head"),
    (640, 640, 8, 1, 128, BF16, 1, 0, "token"), (300, 1000, 40, 1, 64, FP16, 129, 1, "token"),
    (513, 513, 8, 2, 128, BF16, 0, 9, "token"), (1500, 1500, 32, 8, 64, BF16, 128, 128, "token"),
    (2100, 2100, 64, 1, 64, BF16, 100, 3, "token"), (1200, 2000, 64, 1, 64, BF16, 0, 0, "token"),    # more than 512 tiles, and less
])
def test_window_attention_matches_the_statement(new, keys, heads, kv_heads, dim, dtype, window, sinks, layout):
    g = torch.Generator().manual_seed(new + keys)
    q = (1.5 * torch.randn(new, heads, dim, generator=g)).to(dtype)
    k, v = (torch.randn(keys, kv_heads, dim, generator=g).to(dtype) for _ in range(2))
    dq, dk, dv = q.cuda(), k.cuda(), v.cuda()
    if layout == "head":        # [heads, tokens, D] storage seen token-major
        dq, dk, dv = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (dq, dk, dv))
    got = native.window_attention(dq, dk, dv, dim ** -0.5, window, sinks)
    out, mass = R.attention(q, k, v, keys - new, dim ** -0.5, window, sinks)
    R.check(got, out, mass, dtype, keys, float(v.abs().max()))


@pytest.mark.parametrize("new", [1, 40])
def test_values_that_no_query_sees_may_be_anything(new):
    dim, keys, window, sinks = 128, 900, 100, 4
    g = torch.Generator().manual_seed(3)
    q = torch.randn(new, 8, dim, generator=g).to(BF16)
    k, v = (torch.randn(keys, 2, dim, generator=g).to(BF16) for _ in range(2))
    out, mass = R.attention(q, k, v, keys - new, dim ** -0.5, window, sinks)
    hidden = slice(sinks, keys - new - window + 1)
    for bad in (float("nan"), float("inf"), torch.finfo(BF16).min):
        k[hidden], v[hidden] = bad, bad
        got = native.window_attention(q.cuda(), k.cuda(), v.cuda(), dim ** -0.5, window, sinks)
        R.check(got, out, mass, BF16, keys, 5.0)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,keys,window,sinks", [(64, 64, 0, 0), (300, 300, 0, 0), (40, 700, 0, 0), (300, 700, 90, 0), (300, 700, 70, 20),
                                                   (3, 600, 50, 4), (200, 200, 1, 0)])
def test_large_values_of_keys_that_a_token_does_not_see_have_no_weight(new, keys, window, sinks, dim):
    # every key is hidden from some tokens of a tile and seen by others, and every third has a value 10^30 times
    # as large: a weight of 2^-57 where there should be none would show
    g = torch.Generator().manual_seed(new + keys + dim)
    q = torch.randn(new, 8, dim, generator=g).to(BF16)
    k, v = (torch.randn(keys, 2, dim, generator=g).to(BF16) for _ in range(2))
    hidden_first = torch.arange(keys) % 3 == 1
    hidden_first &= torch.arange(keys) > keys - new          # the first token sees none of them in its future
    v[hidden_first] *= 1e30
    out, mass = R.attention(q, k, v, keys - new, dim ** -0.5, window, sinks)
    assert float(mass[0].max()) < 10 and (window == 1 or float(mass.max()) > 1e20)
    got = native.window_attention(q.cuda(), k.cuda(), v.cuda(), dim ** -0.5, window, sinks)
    R.check(got, out, mass, BF16, keys, 1e31)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("new,keys,heads,dim", [(1, 300, 4, 128), (1, 9000, 4, 64), (64, 200, 4, 128), (64, 200, 4, 64), (200, 9000, 2, 128), (200, 9000, 2, 64)])
def test_scores_that_are_not_finite_are_seen_wherever_their_key_stands(new, keys, heads, dim, dtype):
    # a key of NaN makes every row NaN that sees it, an infinite score too; a score of -infinity is a weight of 0
    g = torch.Generator().manual_seed(new + keys + dim)
    q = torch.randn(new, heads, dim, generator=g).to(dtype)
    k, v = (torch.randn(keys, 1, dim, generator=g).to(dtype) for _ in range(2))
    q[:, 0::2, 0], q[:, 1::2, 0] = 1.0, -1.0                # heads to which a key's infinity is +infinity and -infinity
    before, scale = keys - new, dim ** -0.5
    out, mass = R.attention(q, k, v, before, scale)
    dq, dk, dv = q.cuda(), k.cuda(), v.cuda()
    for at in [*range(before - 20, before + new, 3), *range(68), keys - 1]:
        sees = before + torch.arange(new) >= at
        for bad in (float("nan"), float("inf")):
            dk.copy_(k)
            dk[at, 0, 0] = bad
            got = native.window_attention(dq, dk, dv, scale, 0).cpu()
            spoiled = sees[:, None] & (torch.tensor([True, False] * (heads // 2)) | (bad != bad))
            assert bool((got.isnan().all(-1) == spoiled).all()), f"{bad} at {at}"
            fine = got.double().nan_to_num(0.0)
            fine[spoiled] = out[spoiled]
            if bad == bad and keys < 1000:
                present = torch.ones(keys, dtype=torch.bool)
                present[at] = False
                want, weight = R.attention(q[:, 1::2], k, v, before, scale, present=present)
                R.check(fine[:, 1::2], want, weight, dtype, keys, 5.0, f"-inf at {at}")
            R.check(fine[~sees], out[~sees], mass[~sees], dtype, keys, 5.0, f"rows before {at}") if not bool(sees.all()) else None


@pytest.mark.parametrize("new,dim", [(1, 64), (1, 128), (5, 64), (5, 128)])
def test_fp16_weights_far_below_the_largest_still_add_up(new, dim):
    # one key 17 nats (2^24.5) above 30000 others that hold a thousandth of the mass together, and only they have values.
    # 64 requests over the same pages, so that a request's keys stay with one CTA.
    page, heads, kv_heads, keys, requests, scale = 16, 32, 8, 30000, 64, 0.125
    g = torch.Generator().manual_seed(new + dim)
    q = (0.3 * torch.randn(new, heads, dim, generator=g)).to(FP16)
    k = torch.randn(keys, kv_heads, dim, generator=g).to(FP16)
    v = (1 + 0.1 * torch.randn(keys, kv_heads, dim, generator=g)).to(FP16)
    q[:, :, 0], k[:, :, 0] = 8.0, 0.0
    k[0], v[0] = 0.0, 0.0
    k[0, :, 0] = 17.0
    out, mass = R.attention(q, k, v, keys - new, scale)
    assert 5e-4 < float(out.min()) and float(out.max()) < 5e-3
    table = torch.arange(keys // page).to(torch.int32).expand(requests, -1).contiguous()
    got = native.paged_attention(q.repeat(requests, 1, 1).cuda(), k.view(-1, page, kv_heads, dim).cuda(), v.view(-1, page, kv_heads, dim).cuda(),
                                 table.cuda(), _ints([i * new for i in range(requests + 1)]), _ints([keys] * requests), new, scale)
    # as R.tolerance, but the largest weight of a unit is 2^8 or more, so that multiples of 2^-24 are 2^-33 of it per key
    u = 2 ** -11
    tol = u * (mass + out.abs()) * (1 + 2 ** -6) + 2 ** -11 * mass + keys * 2 ** -33 * float(v.abs().max())
    off = (got.view(requests, new, heads, dim).double().cpu() - out).abs() / tol
    assert float(off.max()) <= 1.0, f"{float(off.max()):.3g} times the tolerance"


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,keys,heads", [(1, 300, 4), (1, 5000, 4), (40, 300, 4), (200, 5000, 2)])
def test_values_up_to_the_largest_of_the_type_do_not_overflow(new, keys, heads, dim):
    # scores that rise along the sequence by 2^60 in all (the tcgen05 kernel keeps a row's reference point while it can), and
    # values of 3e38, of which two do not add up in fp32
    g = torch.Generator().manual_seed(keys + dim)
    before, scale = keys - new, 0.125
    q = torch.randn(new, heads, dim, generator=g).to(BF16)
    k, v = (torch.randn(keys, 1, dim, generator=g).to(BF16) for _ in range(2))
    q[:, :, 0], k[:, :, 0] = 8.0, torch.linspace(0, 41, keys).to(BF16)[:, None]
    for size in (1e-20, 1e25, 3e38):
        big = (v.sign() * size).to(BF16) if size > 1e30 else (v.double() * size).to(BF16)
        big[:, :, 1] = torch.tensor(size, dtype=BF16)                 # the same value everywhere: their mean is it
        for rising in (True, False):
            if not rising:
                k[:, :, 0] = 0.0
            out, mass = R.attention(q, k, big, before, scale)
            got = native.window_attention(q.cuda(), k.cuda(), big.cuda(), scale, 0)
            R.check(got, out, mass, BF16, keys, 5.0, f"{size} {rising}")
        k[:, :, 0] = torch.linspace(0, 41, keys).to(BF16)[:, None]


@pytest.mark.parametrize("new", [1, 200])
@pytest.mark.parametrize("gain", [30.0, 1e4])
def test_peaked_scores_and_expanded_caches(new, gain):
    # scores far apart (the reference point of the exponentials moves often) and one KV row shared by views
    dim = 128
    g = torch.Generator().manual_seed(17)
    q = (gain * torch.randn(new, 4, dim, generator=g)).to(BF16)
    k, v = (torch.randn(1000, 1, dim, generator=g).to(BF16) for _ in range(2))
    out, _ = R.attention(q, k, v, 1000 - new, dim ** -0.5, 0, 0)
    got = native.window_attention(q.cuda(), k.cuda().expand(-1, 2, -1), v.cuda().expand(-1, 2, -1), dim ** -0.5, 0)
    # weights differ by e^(score error): 128 products of size gain * 4 sum up with errors of 128 * 2^-24 * their size
    s_err = 128 * 2.0 ** -24 * gain * 4 * 4 * dim ** 0.5
    mass = R.attention(q, k, v, 1000 - new, dim ** -0.5, 0, 0)[1]
    tol = R.tolerance(out, mass, BF16, 1000, 5.0) + 2 * min(s_err, 1.0) * (mass + out.abs())
    assert bool(((got.double().cpu() - out).abs() <= tol).all())


@pytest.mark.parametrize("new,heads", [(1, 2), (90, 2), (33, 80)])
def test_caches_that_no_tensor_map_describes(new, heads):
    # keys expanded over heads and tokens (strides of 0) take the other kernel, at any number of rows
    dim = 64
    g = torch.Generator().manual_seed(19)
    q = torch.randn(new, heads, dim, generator=g).to(FP16)
    k, v = (torch.randn(300, 1, dim, generator=g).to(FP16) for _ in range(2))
    out, mass = R.attention(q, k.expand(-1, 2, -1), v.expand(-1, 2, -1), 300 - new, 0.2, 50, 3)
    got = native.window_attention(q.cuda(), k.cuda().expand(-1, 2, -1), v.cuda().expand(-1, 2, -1), 0.2, 50, 3)
    R.check(got, out, mass, FP16, 300, 5.0)
    one = k[:1].cuda().expand(300, 2, -1)                 # every token the same key and value
    got = native.window_attention(q.cuda(), one, one, 0.2, 50, 3)
    assert float((got.cpu().double() - k[0].double()).abs().max()) <= 2 ** -10 * float(k[0].abs().max())


@pytest.mark.parametrize("new", [1, 100])
def test_numbers_of_other_types_and_beyond_an_int(new):
    import numpy as np
    g = torch.Generator().manual_seed(29)
    q = torch.randn(new, 4, 64, generator=g).to(BF16)
    k, v = (torch.randn(200, 2, 64, generator=g).to(BF16) for _ in range(2))
    out, mass = R.attention(q, k, v, 200 - new, 0.125, 0, 0)
    for window, sinks in ((2 ** 31, 0), (2 ** 32 + 1, 2 ** 40), (np.int64(2 ** 30), np.int32(3)), (np.int64(0), 5), (1, 2 ** 33)):
        got = native.window_attention(q.cuda(), k.cuda(), v.cuda(), np.float64(0.125), window, sinks)
        R.check(got, out, mass, BF16, 200, 5.0, f"{window} {sinks}")


# ---------------------------------------------------------------------------------- run together
def test_a_serving_loop_plan_write_attend_over_pages():
    page, heads, kv_heads, dim, dtype, window, sinks = 16, 8, 2, 128, BF16, 60, 3
    g = torch.Generator().manual_seed(23)
    steps = [[40, 0, 7], [33, 100, 1], [1, 1, 1], [1, 17, 0], [1, 1, 1], [0, 300, 2]]
    n_pages = 64
    shape = (n_pages, page, kv_heads, dim)
    k_cache, v_cache = (torch.full(shape, float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    table = torch.full((3, 40), -1, dtype=torch.int32, device="cuda")
    ring, state = torch.randperm(n_pages, generator=g).to(torch.int32).cuda(), _ints([5, n_pages])
    seq = _ints([0, 0, 0])
    history = [(torch.empty(0, kv_heads, dim, dtype=dtype),) * 2 for _ in range(3)]
    for new in steps:
        rows = sum(new) + 3                                   # a padded batch
        q = torch.randn(rows, heads, dim, generator=g).to(dtype)
        k, v = (torch.randn(rows, kv_heads, dim, generator=g).to(dtype) for _ in range(2))
        plan = native.paged_plan(seq, _ints(new), table, ring, state, rows, page, ring_state_out=state)
        native.paged_write(k.cuda(), v.cuda(), plan.slot_map, k_cache, v_cache)
        out = native.paged_attention(q.cuda(), k_cache, v_cache, table, plan.cu_new, plan.seq_len, max(new), dim ** -0.5,
                                     window, sinks)
        seq = plan.seq_len
        at = 0
        for r, n in enumerate(new):
            hk, hv = history[r]
            history[r] = (torch.cat([hk, k[at:at + n]]), torch.cat([hv, v[at:at + n]]))
            if n:
                want, mass = R.attention(q[at:at + n], *history[r], len(hk), dim ** -0.5, window, sinks)
                R.check(out[at:at + n], want, mass, dtype, len(hk) + n, 5.0, f"step {new} request {r}")
            at += n
        assert seq.tolist() == [len(h[0]) for h in history] and plan.refused.tolist() == [0, 0, 0]
    assert state[1].item() == n_pages - sum(-(-len(h[0]) // page) for h in history)


@pytest.mark.parametrize("new", [1, 70])
def test_captured_graphs_replay_with_new_lengths_side_by_side(new):
    page, heads, kv_heads, dim = 16, 8, 2, 128
    spec = [(300, new), (77, new)]
    pool, cu, q = _batch(spec, page, heads, kv_heads, dim, BF16, "token", 31)
    k, v = pool.cuda()
    table = pool.table.cuda()
    graphs = []
    for _ in range(2):
        s = dict(q=torch.zeros_like(q).cuda(), cu=_ints([0, 0, 0]), seq=_ints([0, 0]), stream=torch.cuda.Stream())
        with torch.cuda.stream(s["stream"]):
            native.paged_attention(s["q"], k, v, table, s["cu"], s["seq"], new, dim ** -0.5)
        torch.cuda.synchronize()
        s["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(s["graph"]):
            s["out"] = native.paged_attention(s["q"], k, v, table, s["cu"], s["seq"], new, dim ** -0.5)
        graphs.append(s)
    for cut in (0, 33):
        want = []
        for i, s in enumerate(graphs):
            lens = [c + n - cut * (i + 1) for c, n in spec]
            s["q"].copy_(q * (1 + i)), s["cu"].copy_(_ints(cu)), s["seq"].copy_(_ints(lens))
            want.append([R.attention(q[cu[r]:cu[r + 1]] * (1 + i), *(x[:lens[r]] for x in pool.rows[r]),
                                     lens[r] - spec[r][1], dim ** -0.5) for r in range(2)])
        torch.cuda.synchronize()
        for _ in range(5):
            for s in graphs:
                with torch.cuda.stream(s["stream"]):
                    s["graph"].replay()
        torch.cuda.synchronize()
        for i, s in enumerate(graphs):
            for r in range(2):
                R.check(s["out"][cu[r]:cu[r + 1]], *want[i][r], BF16, 400, 5.0, f"graph {i} request {r} cut {cut}")


def test_a_whole_step_captured_and_replayed():
    # plan, write and attention in one graph: lengths, rows and the ring's state live in its buffers
    page, heads, kv_heads, dim, dtype, rows = 16, 8, 2, 64, BF16, 24
    g = torch.Generator().manual_seed(37)
    k_cache, v_cache = (torch.full((40, page, kv_heads, dim), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    table = torch.full((3, 12), -1, dtype=torch.int32, device="cuda")
    ring, state, seq, fresh = torch.randperm(40, generator=g).to(torch.int32).cuda(), _ints([38, 40]), _ints([0, 0, 0]), _ints([0, 0, 0])
    q = torch.zeros(rows, heads, dim, dtype=dtype, device="cuda")
    k, v = (torch.zeros(rows, kv_heads, dim, dtype=dtype, device="cuda") for _ in range(2))

    def step():
        plan = native.paged_plan(seq, fresh, table, ring, state, rows, page, ring_state_out=state)
        native.paged_write(k, v, plan.slot_map, k_cache, v_cache)
        out = native.paged_attention(q, k_cache, v_cache, table, plan.cu_new, plan.seq_len, 10, 0.125, 40, 2)
        seq.copy_(plan.seq_len)
        return out

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()                                            # no tokens: warms up, changes nothing
    torch.cuda.synchronize()
    assert state.tolist() == [38, 40]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    history = [(torch.empty(0, kv_heads, dim, dtype=dtype),) * 2 for _ in range(3)]
    for new in ([10, 3, 0], [1, 1, 9], [10, 1, 10], [1, 0, 1], [7, 10, 1]):
        rows_q = torch.randn(rows, heads, dim, generator=g).to(dtype)
        rows_k, rows_v = (torch.randn(rows, kv_heads, dim, generator=g).to(dtype) for _ in range(2))
        q.copy_(rows_q), k.copy_(rows_k), v.copy_(rows_v), fresh.copy_(_ints(new))
        graph.replay()
        at = 0
        for r, n in enumerate(new):
            hk, hv = history[r]
            history[r] = (torch.cat([hk, rows_k[at:at + n]]), torch.cat([hv, rows_v[at:at + n]]))
            if n:
                want, mass = R.attention(rows_q[at:at + n], *history[r], len(hk), 0.125, 40, 2)
                R.check(out[at:at + n], want, mass, dtype, 100, 5.0, f"{new} request {r}")
            at += n
    assert seq.tolist() == [len(h[0]) for h in history]


@pytest.mark.parametrize("requests", [20, 60])
def test_captured_batches_of_tokens_and_chunks_in_two_passes(requests):
    # a wide table sends tokens and chunks through both kernels; 60 requests are scheduled by a kernel of their own
    page, heads, kv_heads, dim = 16, 8, 2, 64
    spec = [(i * 23 % 500, 1 if i % 9 else 30 + i) for i in range(requests)]
    pool, cu, q = _batch(spec, page, heads, kv_heads, dim, BF16, "token", requests)
    k, v = pool.cuda()
    table = torch.nn.functional.pad(pool.table, (0, 12000), value=-1).cuda()
    live = dict(q=torch.zeros_like(q).cuda(), cu=_ints([0] * (requests + 1)), seq=_ints([0] * requests))
    most = max(n for _, n in spec)
    for window in (0, 90):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            native.paged_attention(live["q"], k, v, table, live["cu"], live["seq"], most, 0.125, window, 2)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = native.paged_attention(live["q"], k, v, table, live["cu"], live["seq"], most, 0.125, window, 2)
        for cut in (0, 1):
            lens = [max(c + n - cut * 7, n) for c, n in spec]
            live["q"].copy_(q), live["cu"].copy_(_ints(cu)), live["seq"].copy_(_ints(lens))
            graph.replay()
            for r, (_, n) in enumerate(spec):
                want, mass = R.attention(q[cu[r]:cu[r + 1]], *(x[:lens[r]] for x in pool.rows[r]), lens[r] - n, 0.125, window, 2)
                R.check(out[cu[r]:cu[r + 1]], want, mass, BF16, lens[r], 5.0, f"request {r} window {window} cut {cut}")


@pytest.mark.parametrize("new", [1, 60])
def test_calls_on_two_streams_at_once(new):
    batches = []
    for i in range(2):
        pool, cu, q = _batch([(900 + 300 * i, new), (50, new)], 16, 8, 2, 128, BF16, "token", 50 + i)
        k, v = pool.cuda()
        args = (q.cuda(), k, v, pool.table.cuda(), _ints(cu), _ints([900 + 300 * i + new, 50 + new]), new, 128 ** -0.5)
        batches.append((args, native.paged_attention(*args), torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, (args, _, stream) in enumerate(batches):
            with torch.cuda.stream(stream):
                outs[i].append(native.paged_attention(*args))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, batches[i][1]) for x in outs[i])


def test_results_do_not_depend_on_the_run_or_the_stream():
    pool, cu, q = _batch([(3000, 1), (777, 1), (20, 1)], 16, 32, 8, 128, BF16, "token", 41)
    k, v = pool.cuda()
    args = (q.cuda(), k, v, pool.table.cuda(), _ints(cu), _ints([3001, 778, 21]), 1, 128 ** -0.5)
    first = native.paged_attention(*args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(side):
            again = native.paged_attention(*args)
        side.synchronize()
        assert torch.equal(first, again)


@pytest.mark.parametrize("requests,new", [(2, 1), (40, 1), (300, 1), (3, 90), (45, 30)])
def test_lengths_and_queries_written_by_the_kernel_just_before(requests, new):
    # the attention kernels are launched under the end of the kernel before: what that one writes must be seen
    steps = []
    pool = _batch([(400, new)] * requests, 16, 8, 2, 128, BF16, "token", 77)[0]
    k, v = pool.cuda()
    table = pool.table.cuda()
    for i in range(3):
        spec = [((37 * r + 131 * i) % 400, 1 + (r + i) % new) for r in range(requests)]
        cu = [0]
        for _, n in spec:
            cu.append(cu[-1] + n)
        q = torch.randn(requests * new, 8, 128, device="cuda").to(BF16)
        data = (q, _ints(cu), _ints([c + n for c, n in spec]))
        torch.cuda.synchronize()
        want = [native.paged_attention(data[0], k, v, table, data[1], data[2], new, 0.1, window)[:cu[-1]] for window in (0, 50)]
        torch.cuda.synchronize()
        steps.append((data, want))
    live = [x.clone() for x in steps[0][0]]
    got = []
    for i in range(30):
        for which in ((0, 1, 2), (2, 0, 1), (1, 2, 0))[i // 3 % 3]:      # each of them once the last to be written
            live[which].copy_(steps[i % 3][0][which])
        got.append(native.paged_attention(live[0], k, v, table, live[1], live[2], new, 0.1, 50 * (i % 2)))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        want = steps[i % 3][1][i % 2]
        assert torch.equal(x[:len(want)], want), i


@pytest.mark.parametrize("requests,new,dim", [(1, 1, 128), (40, 1, 64), (300, 1, 128), (3, 90, 128), (45, 30, 64)])
def test_tables_and_queries_written_by_the_kernel_just_before(requests, new, dim):
    g = torch.Generator().manual_seed(requests)
    k, v = (torch.randn(64, 16, 2, dim, generator=g).to(BF16).cuda() for _ in range(2))
    cu, seq = _ints([i * new for i in range(requests + 1)]), _ints([new + (37 * r) % 300 for r in range(requests)])
    steps = []
    for i in range(3):
        table = torch.randint(0, 64, (requests, 25), generator=g).to(torch.int32).cuda()
        q = torch.randn(requests * new, 8, dim, generator=g).to(BF16).cuda()
        torch.cuda.synchronize()
        steps.append((table, q, native.paged_attention(q, k, v, table, cu, seq, new, 0.1)))
        torch.cuda.synchronize()
    table, q = steps[0][0].clone(), steps[0][1].clone()
    got = []
    for i in range(30):
        for which in ((0, 1), (1, 0))[i // 3 % 2]:
            (table, q)[which].copy_(steps[i % 3][which])
        got.append(native.paged_attention(q, k, v, table, cu, seq, new, 0.1))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert torch.equal(x, steps[i % 3][2]), i


@pytest.mark.parametrize("new,dim", [(1, 128), (3, 64), (90, 128), (700, 64)])
def test_windowed_inputs_written_by_the_kernel_just_before(new, dim):
    g = torch.Generator().manual_seed(new)
    steps = []
    for i in range(3):
        data = [torch.randn(n, heads, dim, generator=g).to(BF16).cuda() for n, heads in ((new, 8), (900, 2), (900, 2))]
        torch.cuda.synchronize()
        steps.append((data, native.window_attention(*data, 0.1, 200, 3)))
        torch.cuda.synchronize()
    live = [x.clone() for x in steps[0][0]]
    got = []
    for i in range(30):
        for which in ((0, 1, 2), (2, 0, 1), (1, 2, 0))[i // 3 % 3]:      # each of them once the last to be written
            live[which].copy_(steps[i % 3][0][which])
        got.append(native.window_attention(*live, 0.1, 200, 3))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert torch.equal(x, steps[i % 3][1]), i


def test_a_device_that_is_not_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    q = torch.randn(3, 4, 64, device="cuda:1").to(BF16)
    k = torch.randn(30, 2, 64, device="cuda:1").to(BF16)
    got = native.window_attention(q, k, k, 0.125, 10)
    assert got.device == q.device and torch.cuda.current_device() == 0


def test_wrong_arguments_are_refused():
    q = torch.zeros(4, 8, 128, dtype=BF16, device="cuda")
    c = torch.zeros(6, 16, 2, 128, dtype=BF16, device="cuda")
    t, cu, seq = _ints([[0, 1], [2, 3]]), _ints([0, 2, 4]), _ints([20, 20])
    ok = dict(q=q, k_cache=c, v_cache=c, block_table=t, cu_new=cu, seq_len=seq, max_new=2, softmax_scale=0.1)
    native.paged_attention(ok.pop("q"), **ok)
    for change in (dict(q=q.half()), dict(k_cache=c.half()), dict(q=q[:, :7]), dict(q=q.float()), dict(cu_new=_ints([0, 4])),
                   dict(cu_new=cu.long()), dict(seq_len=seq.cpu()), dict(block_table=t[:1]), dict(block_table=t.t()),
                   dict(max_new=0), dict(softmax_scale=float("nan")), dict(softmax_scale=-1.0), dict(window=-1), dict(sinks=-1),
                   dict(k_cache=c[:, :10], v_cache=c[:, :10]), dict(k_cache=c[..., :96], v_cache=c[..., :96]),
                   dict(out=torch.zeros(4, 8, 64, dtype=BF16, device="cuda")), dict(out=q), dict(q=q[..., ::2]),
                   dict(k_cache=c[..., 4:68], v_cache=c[..., 4:68], q=q[..., :64])):
        with pytest.raises(native.SpfError):
            native.paged_attention(change.pop("q", q), **{**ok, **change})
    with pytest.raises(native.SpfError):
        native.window_attention(q, c[0], c[0][:8], 0.1, 4)
    with pytest.raises(native.SpfError):
        native.window_attention(q, c[0, :3], c[0, :3], 0.1, 4)         # more queries than keys
    with pytest.raises(native.SpfError):
        native.paged_write(c[0], c[0], torch.zeros(15, dtype=torch.int64, device="cuda"), c, c)
    with pytest.raises(native.SpfError):
        native.paged_plan(seq, seq, t, seq, seq, -1, 16)
    with pytest.raises(native.SpfError):
        native.paged_plan(seq, seq, t, seq, seq, 40, 24)
    empty = native.paged_attention(q[:0], c, c, t, _ints([0, 0, 0]), seq, 1, 0.1)
    assert empty.shape == (0, 8, 128)
