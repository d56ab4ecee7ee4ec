"""Cases for the serving operators: the step plan of a paged cache, the write into it, attention of a
chunk of new tokens (or of single tokens) over it, and attention with a sliding window and visible
first tokens over a contiguous cache.

``run`` computes each operator in elementary torch operations, or - where ``own`` is set - through
``shareprefill_b200.native``.  ``exact`` states the same results in 64 bits, request by request.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decoding step of a small batch: eight requests, a token each
        dict(name="plan_step", op="plan", requests=8, chunks=0, new=1, ctx=4096, page=16, pad=0, spare=64, mix=1),
        # a full server: 512 requests, most decode, eight bring 4K-token chunks, the batch is padded and the
        # pool runs out of pages before the last requests
        dict(name="plan_mixed", op="plan", requests=512, chunks=8, new=4096, ctx=32768, page=16, pad=257, spare=1900, mix=2),
        # a decoding step's rows: 64 tokens
        dict(name="write_step", op="write", rows=64, kv_heads=8, dim=128, page=16, dtype="bf16", mix=3),
        # a 32K prompt
        dict(name="write_prompt", op="write", rows=32768, kv_heads=8, dim=128, page=64, dtype="bf16", mix=4),
        # one user, one token: latency
        dict(name="token_one", op="paged", requests=1, chunks=0, new=1, ctx=4096, page=16, heads=32, kv_heads=8, dim=128,
             dtype="bf16", window=0, sinks=0, mix=5),
        # a decoding batch of ragged lengths up to 8K
        dict(name="token_batch", op="paged", requests=64, chunks=0, new=1, ctx=8192, page=16, heads=32, kv_heads=8, dim=128,
             dtype="bf16", window=0, sinks=0, mix=6),
        # one token at 128K, groups of seven, fp16, the last page holds one token less than it could
        dict(name="token_long", op="paged", requests=1, chunks=0, new=1, ctx=131070, page=64, heads=28, kv_heads=4, dim=128,
             dtype="fp16", window=0, sinks=0, mix=7),
        # the last 2K-token chunk of a 34K prompt
        dict(name="chunk_prompt", op="paged", requests=1, chunks=1, new=2048, ctx=32768, page=64, heads=32, kv_heads=8, dim=128,
             dtype="bf16", window=0, sinks=0, mix=8),
        # decoding requests and two chunks in one batch, with a window and sinks, head size 64
        dict(name="chunk_mixed", op="paged", requests=16, chunks=2, new=509, ctx=16000, page=32, heads=32, kv_heads=8, dim=64,
             dtype="bf16", window=4096, sinks=4, mix=9),
        # a 32K prompt through a layer with a 2K window and four visible first tokens
        dict(name="window_prompt", op="window", new=32768, keys=32768, heads=32, kv_heads=8, dim=128, dtype="bf16",
             window=2048, sinks=4),
        # a short odd prompt behind a cached prefix, fp16, head size 64
        dict(name="window_short", op="window", new=777, keys=1301, heads=8, kv_heads=2, dim=64, dtype="fp16", window=250,
             sinks=3),
        # one token of such a layer over a 128K cache
        dict(name="window_token", op="window", new=1, keys=131072, heads=32, kv_heads=8, dim=128, dtype="bf16", window=4096,
             sinks=4),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "write", "paged", "paged", "paged", "window", "window"])
    page = rng.choice([16, 32, 64, 128])
    mix = rng.randrange(1, 1 << 20)
    if op == "plan":
        requests = _log_uniform(rng, 1, 512)
        return dict(op=op, requests=requests, chunks=rng.randint(0, min(requests, 8)), new=_log_uniform(rng, 2, 4096),
                    ctx=_log_uniform(rng, 16, 32768), page=page, pad=rng.choice([0, rng.randint(1, 300)]),
                    spare=_log_uniform(rng, 1, 3000), mix=mix)
    heads, kv_heads = rng.choice([(32, 8), (28, 4), (64, 8), (8, 2)])
    dim = rng.choice([128, 128, 64])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "write":
        return dict(op=op, rows=_log_uniform(rng, 1, 32768), kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, mix=mix)
    windowed = rng.random() < 0.5
    if op == "paged":
        if rng.random() < 0.5:      # single tokens
            requests, chunks, new = _log_uniform(rng, 1, 96), 0, 1
            ctx = _log_uniform(rng, 16, min(131072, (1 << 19) // requests))
        else:
            requests, new = _log_uniform(rng, 1, 12), _log_uniform(rng, 2, 2048)
            chunks = rng.randint(1, requests)
            # the plain form pads every request to the longest: requests * new * ctx bounds what it holds
            ctx = _log_uniform(rng, 16, max(17, min(32768, (1 << 25) // (requests * new))))
        return dict(op=op, requests=requests, chunks=chunks, new=new, ctx=ctx, page=page, heads=heads, kv_heads=kv_heads,
                    dim=dim, dtype=dtype, window=_log_uniform(rng, 8, 8192) if windowed else 0,
                    sinks=rng.choice([0, 4, rng.randint(1, 150)]) if windowed else 0, mix=mix)
    keys = _log_uniform(rng, 16, 32768)
    return dict(op=op, new=rng.choice([keys, keys, 1, rng.randint(1, keys)]), keys=keys, heads=min(heads, 32),
                kv_heads=kv_heads if heads <= 32 else 4, dim=dim, dtype=dtype, window=_log_uniform(rng, 8, 2048),
                sinks=rng.choice([0, 4, rng.randint(1, 150)]))


# ---------------------------------------------------------------------------------------- lengths
def _lengths(case):
    """Cached and new tokens of every request: the first `chunks` requests bring chunks of up to `new`
    tokens (the first one exactly that), the others one token; the first context is the longest."""
    rng = random.Random(case["mix"])
    cached, new = [], []
    for r in range(case["requests"]):
        cached.append(case["ctx"] if r == 0 else rng.randint(case["ctx"] // 8, case["ctx"]))
        new.append(case["new"] if r == 0 and case["chunks"] else
                   rng.randint(max(1, case["new"] // 2), case["new"]) if r < case["chunks"] else 1)
    return cached, new


def _pages(tokens, page):
    return -(-tokens // page)


def work(case):
    if case["op"] == "plan":
        cached, new = _lengths(case)
        rows = sum(new) + case["pad"]
        taken = sum(_pages(c + n, case["page"]) - _pages(c, case["page"]) for c, n in zip(cached, new))
        # lengths in; offsets, lengths and flags out; per row a slot and a position; ids read and put in the table
        return {"bytes": case["requests"] * (8 + 4 + 4 + 4) + rows * 12 + 8 * min(taken, case["spare"]), "flops": 0}
    if case["op"] == "write":
        return {"bytes": case["rows"] * (case["kv_heads"] * case["dim"] * 2 * 4 + 8), "flops": 0}
    h, hkv, d, w, s = case["heads"], case["kv_heads"], case["dim"], case["window"], case["sinks"]
    cached, new = _lengths(case) if case["op"] == "paged" else ([case["keys"] - case["new"]], [case["new"]])
    pairs = keys = 0
    for c, n in zip(cached, new):
        # query i sees min(c + i + 1, window) keys, and the first tokens that lie before its window
        if w:
            pairs += sum(min(c + i + 1, w) + min(s, max(0, c + i + 1 - w)) for i in range(n))
            keys += min(c + n, n + w - 1 + min(s, max(0, c + 1 - w)))
        else:
            pairs += n * c + n * (n + 1) // 2
            keys += c + n
    return {"bytes": sum(new) * h * d * 4 + keys * hkv * d * 4, "flops": 4 * pairs * h * d}


# ---------------------------------------------------------------------------------------- prepare
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "window":
        dt = DTYPES[case["dtype"]]
        q = _randn(gen, case["new"], case["heads"], case["dim"]).mul_(1.5).to(dt)
        k = _randn(gen, case["keys"], case["kv_heads"], case["dim"])
        k[:4] += 0.2                                   # first tokens that many queries look at
        v = _randn(gen, case["keys"], case["kv_heads"], case["dim"]).to(dt)
        return dict(case=case, q=q, k=k.to(dt), v=v, scale=case["dim"] ** -0.5)
    if case["op"] == "write":
        dt, page, rows = DTYPES[case["dtype"]], case["page"], case["rows"]
        n_pages = _pages(rows, page) * 5 // 4 + 2
        slots = torch.randperm(n_pages, generator=gen, device="cuda")[:, None] * page + torch.arange(page, device="cuda")
        slots = slots.reshape(-1)[:rows].clone()
        slots[torch.rand(rows, generator=gen, device="cuda") < 0.05] = -1       # rows of a padded batch
        shape = (n_pages, page, case["kv_heads"], case["dim"])
        k, v = (_randn(gen, rows, case["kv_heads"], case["dim"]).to(dt) for _ in range(2))
        return dict(case=case, k=k, v=v, slots=slots, k_cache=torch.zeros(shape, dtype=dt, device="cuda"),
                    v_cache=torch.zeros(shape, dtype=dt, device="cuda"))
    page = case["page"]
    cached, new = _lengths(case)
    held = [_pages(c, page) for c in cached]
    most = max(_pages(c + n, page) for c, n in zip(cached, new))
    if case["op"] == "plan":
        n_pages = sum(held) + case["spare"]
        ids = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
        table = torch.full((case["requests"], most), -1, dtype=torch.int32, device="cuda")
        owns = torch.arange(most, device="cuda") < torch.tensor(held, device="cuda")[:, None]
        table[owns] = ids[:sum(held)]
        # the free list is a ring over the whole pool: it starts somewhere and may wrap
        head = int(torch.randint(0, n_pages, (1,), generator=gen, device="cuda"))
        ring = torch.full((n_pages,), -1, dtype=torch.int32, device="cuda")
        ring[(head + torch.arange(case["spare"], device="cuda")) % n_pages] = ids[sum(held):]
        return dict(case=case, cached=_ints(cached), new=_ints(new), table=table, ring=ring,
                    ring_state=_ints([head, case["spare"]]), n_rows=sum(new) + case["pad"])
    # a pool in which only what the requests hold was ever written: the rest is NaN
    dt = DTYPES[case["dtype"]]
    owned = [_pages(c + n, page) for c, n in zip(cached, new)]
    n_pages = sum(owned) + 3
    ids = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((case["requests"], most), -1, dtype=torch.int32, device="cuda")
    col = torch.arange(most, device="cuda")
    table[col < torch.tensor(owned, device="cuda")[:, None]] = ids[:sum(owned)]
    seq = torch.tensor([c + n for c, n in zip(cached, new)], device="cuda")
    live = torch.zeros(n_pages, page, dtype=torch.bool, device="cuda")
    inside = (col[None, :, None] * page + torch.arange(page, device="cuda")) < seq[:, None, None]
    held = col < torch.tensor(owned, device="cuda")[:, None]
    live[table[held].long()] = inside[held]
    k = _randn(gen, n_pages, page, case["kv_heads"], case["dim"])
    k[table[:, 0].long(), :4] += 0.2
    k = k.masked_fill_(~live[:, :, None, None], math.nan).to(dt)
    v = _randn(gen, n_pages, page, case["kv_heads"], case["dim"]).masked_fill_(~live[:, :, None, None], math.nan).to(dt)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = _randn(gen, sum(new), case["heads"], case["dim"]).mul_(1.5).to(dt)
    return dict(case=case, q=q, k=k, v=v, table=table, starts=_ints(starts), seq=seq.to(torch.int32), max_new=max(new),
                scale=case["dim"] ** -0.5)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# -------------------------------------------------------------------------------------------- run
def run(s):
    op = s["case"]["op"]
    if own:
        from shareprefill_b200 import native
        if op == "plan":
            p = native.paged_plan(s["cached"], s["new"], s["table"], s["ring"], s["ring_state"], s["n_rows"],
                                  s["case"]["page"])
            return dict(table=s["table"], cu_new=p.cu_new, seq_len=p.seq_len, slot_map=p.slot_map, positions=p.positions,
                        refused=p.refused, ring_state=p.ring_state)
        if op == "write":
            native.paged_write(s["k"], s["v"], s["slots"], s["k_cache"], s["v_cache"])
            return s["k_cache"], s["v_cache"]
        if op == "paged":
            return native.paged_attention(s["q"], s["k"], s["v"], s["table"], s["starts"], s["seq"], s["max_new"],
                                          s["scale"], window=s["case"]["window"], sinks=s["case"]["sinks"])
        return native.window_attention(s["q"], s["k"], s["v"], s["scale"], s["case"]["window"], s["case"]["sinks"])
    return {"plan": _plan, "write": _write, "paged": _paged, "window": _window}[op](s)


def _plan(s):
    page, n_rows = s["case"]["page"], s["n_rows"]
    table, ring = s["table"], s["ring"]
    cached, new = s["cached"].long().clamp(min=0), s["new"].long().clamp(min=0)
    ends = torch.cumsum(new, 0)
    held, total = (cached + page - 1) // page, (cached + new + page - 1) // page
    fits = (total <= table.shape[1]) & (ends <= n_rows)
    need = torch.where(fits, total - held, 0)
    upto = torch.cumsum(need, 0)
    head, count = s["ring_state"][0].long(), s["ring_state"][1].long()
    ok = fits & ((need == 0) | (upto <= count))
    taken = torch.where(ok & (need > 0), upto, 0).max()
    # the ids of the new pages, column by column of the table
    col = torch.arange(table.shape[1], device=table.device)
    fresh = ok[:, None] & (col >= held[:, None]) & (col < total[:, None])
    ids = ring[(head + (upto - need)[:, None] + col - held[:, None]) % ring.shape[0]]
    table.copy_(torch.where(fresh, ids, table))
    cu_new = torch.cat([ends.new_zeros(1), ends.clamp(max=n_rows)])
    row = torch.arange(n_rows, device=table.device)
    r = torch.searchsorted(ends, row, right=True)
    inside, r = r < ends.shape[0], r.clamp(max=ends.shape[0] - 1)
    pos = cached[r] + row - cu_new[r]
    where = table[r, (pos // page).clamp(max=table.shape[1] - 1)].long()
    slot = torch.where(inside & ok[r] & (where >= 0), where * page + pos % page, -1)
    return dict(table=table, cu_new=cu_new.to(torch.int32), seq_len=torch.where(ok, cached + new, 0).to(torch.int32),
                slot_map=slot, positions=torch.where(inside, pos, 0).to(torch.int32), refused=(~ok).to(torch.int32),
                ring_state=torch.stack([(head + taken) % ring.shape[0], count - taken]).to(torch.int32))


def _write(s):
    rows = s["slots"] >= 0
    at = s["slots"][rows]
    s["k_cache"].view(-1, *s["k"].shape[1:])[at] = s["k"][rows]
    s["v_cache"].view(-1, *s["v"].shape[1:])[at] = s["v"][rows]
    return s["k_cache"], s["v_cache"]


def _softmax_product(scores, seen, v, product):
    """softmax over the last axis of `scores` where `seen`, times v; a row that sees nothing gives zeros."""
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    return torch.einsum(product, p.div_(torch.where(total > 0, total, 1.0)), v)


def _paged(s):
    """Every request padded to the most new tokens and the most keys of the batch."""
    case, (rows, heads, dim) = s["case"], s["q"].shape
    page, kv_heads = s["k"].shape[1], s["k"].shape[2]
    seq, starts = s["seq"].long(), s["starts"].long()
    new = starts[1:] - starts[:-1]
    width = s["table"].shape[1] * page
    t = torch.arange(s["max_new"], device="cuda")
    j = torch.arange(width, device="cuda")
    there = (j < seq[:, None]) & (s["table"] >= 0).repeat_interleave(page, 1)
    at = (s["table"].clamp(min=0).long()[:, :, None] * page + torch.arange(page, device="cuda")).flatten(1)
    k, v = (torch.where(there[:, :, None, None], x.view(-1, kv_heads, dim)[at].float(), 0.0) for x in (s["k"], s["v"]))
    q = s["q"][(starts[:-1, None] + t).clamp(max=rows - 1)].float().unflatten(2, (kv_heads, heads // kv_heads))
    pos = (seq - new)[:, None] + t
    seen = there[:, None, :] & (j <= pos[:, :, None])
    if case["window"]:
        seen &= (j > pos[:, :, None] - case["window"]) | (j < case["sinks"])
    scores = torch.einsum("rthgd,rjhd->rhgtj", q, k).mul_(s["scale"])
    o = _softmax_product(scores, seen[:, None, None], v, "rhgtj,rjhd->rthgd").flatten(2, 3)
    return o[t < new[:, None]].to(s["q"].dtype)


def _window(s):
    """Blocks of as many queries as the window is long: a block sees its own keys, the window before it
    and the first tokens."""
    (new, heads, dim), (keys, kv_heads, _) = s["q"].shape, s["k"].shape
    w, sinks = min(s["case"]["window"], keys), min(s["case"]["sinks"], keys)
    b = min(w, new)
    n = -(-new // b)
    row = torch.arange(n * b, device="cuda").view(n, b)
    pos = row + keys - new
    near = pos[:, :1] - w + 1 + torch.arange(b + w - 1, device="cuda")
    first = torch.arange(sinks, device="cuda").expand(n, sinks)
    j = torch.cat([near, first], 1)[:, None, :]
    is_near = (torch.arange(j.shape[-1], device="cuda") < b + w - 1)
    old = j <= pos[:, :, None] - w
    seen = torch.where(is_near, (j >= 0) & (j < keys) & (j <= pos[:, :, None]) & ~old, old)
    at = j[:, 0].clamp(0, keys - 1)
    q = s["q"][row.clamp(max=new - 1)].float().unflatten(2, (kv_heads, heads // kv_heads))
    scores = torch.einsum("nthgd,njhd->nhgtj", q, s["k"][at].float()).mul_(s["scale"])
    o = _softmax_product(scores, seen[:, None, None], s["v"][at].float(), "nhgtj,njhd->nthgd")
    return o.reshape(n * b, heads, dim)[:new].to(s["q"].dtype)


# ------------------------------------------------------------------------------------------ exact
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return _exact_plan(s)
    if case["op"] == "write":
        slots = s["slots"].tolist()
        out = []
        for x, cache in ((s["k"], s["k_cache"]), (s["v"], s["v_cache"])):
            flat = cache.double().flatten(0, 1)
            source = [i for i, at in enumerate(slots) if at >= 0]
            flat.index_copy_(0, torch.tensor([slots[i] for i in source], device="cuda", dtype=torch.long),
                             x.double()[torch.tensor(source, device="cuda", dtype=torch.long)])
            out.append(flat.view(cache.shape))
        return tuple(out)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    if case["op"] == "window":
        _exact_rows(s["q"], s["k"], s["v"], case["keys"] - case["new"], s["scale"], case["window"], case["sinks"], out)
        return out
    starts, seq = s["starts"].tolist(), s["seq"].tolist()
    for r in range(case["requests"]):
        a, b = starts[r], starts[r + 1]
        pages = s["table"][r, :_pages(seq[r], case["page"])].long()
        k, v = (x[pages].flatten(0, 1)[:seq[r]] for x in (s["k"], s["v"]))
        _exact_rows(s["q"][a:b], k, v, seq[r] - (b - a), s["scale"], case["window"], case["sinks"], out[a:b])
    return out


def _exact_rows(q, k, v, before, scale, window, sinks, out):
    """One request: query i stands at position before + i."""
    group = q.shape[1] // k.shape[1]
    for i0 in range(0, q.shape[0], 2048):
        i1 = min(i0 + 2048, q.shape[0])
        pos = torch.arange(before + i0, before + i1, device="cuda")[:, None]
        lo, hi = max(0, before + i0 + 1 - window) if window else 0, before + i1
        j = torch.arange(lo, hi, device="cuda")
        if lo > 0 and sinks > 0:
            j = torch.cat([torch.arange(min(sinks, lo), device="cuda"), j])
        hidden = j > pos
        if window:
            hidden |= (j <= pos - window) & (j >= sinks)
        for h in range(k.shape[1]):
            kh, vh = k[j, h].double(), v[j, h].double()
            for g in range(h * group, (h + 1) * group):
                x = (q[i0:i1, g].double() @ kh.T) * scale
                x[hidden] = -math.inf
                out[i0:i1, g] = torch.softmax(x, -1) @ vh


def _exact_plan(s):
    page, n_rows = s["case"]["page"], s["n_rows"]
    table, ring = s["table"].tolist(), s["ring"].tolist()
    head, count = s["ring_state"].tolist()
    cu, seq, refused, slots, positions, used = [0], [], [], [], [], 0
    blocked = False                    # pages are given in the order of the requests: nobody overtakes
    wanted = end = 0
    for r, (c, n) in enumerate(zip(s["cached"].tolist(), s["new"].tolist())):
        held, total = _pages(c, page), _pages(c + n, page)
        end += n
        fits = total <= len(table[r]) and end <= n_rows
        if fits:
            wanted += total - held
            blocked = wanted > count
        ok = fits and (total == held or not blocked)
        if ok:
            for col in range(held, total):
                table[r][col] = ring[(head + used) % len(ring)]
                used += 1
        first = cu[-1]
        cu.append(min(end, n_rows))
        seq.append(c + n if ok else 0)
        refused.append(0 if ok else 1)
        for i in range(cu[-1] - first):
            at = table[r][(c + i) // page] if ok else -1
            slots.append(at * page + (c + i) % page if at >= 0 else -1)
            positions.append(c + i)
    slots += [-1] * (n_rows - len(slots))
    positions += [0] * (n_rows - len(positions))
    return dict(table=_ints(table), cu_new=_ints(cu), seq_len=_ints(seq), refused=_ints(refused), positions=_ints(positions),
                slot_map=torch.tensor(slots, device="cuda"), ring_state=_ints([(head + used) % len(ring), count - used]))
