"""Plain 64-bit statements of the paged and windowed operators, for the tests."""
import math

import torch


def attention(q, k, v, before, scale, window=0, sinks=0, present=None):
    """One request: q [n,H,D] at positions before..., k/v [N,Hkv,D] -> (out, mass) in fp64, mass = sum of weight * |v|:
    what the roundings of the weights are relative to.  `present` [N]: keys that are there."""
    n, heads, d = q.shape
    group = heads // k.shape[1]
    pos = before + torch.arange(n)[:, None]
    j = torch.arange(k.shape[0])
    seen = j <= pos
    if window:
        seen &= (j > pos - window) | (j < sinks)
    if present is not None:
        seen &= present
    any_seen = seen.any(0)
    out = torch.zeros(n, heads, d, dtype=torch.float64)
    mass = torch.zeros_like(out)
    for h in range(heads):
        kh = torch.where(any_seen[:, None], k[:, h // group].double(), 0.0)
        vh = torch.where(any_seen[:, None], v[:, h // group].double(), 0.0)
        s = (q[:, h].double() @ kh.T) * scale
        s = s.masked_fill(~seen, -math.inf)
        top = s.amax(1, keepdim=True) if s.shape[1] else torch.zeros(n, 1, dtype=torch.float64)
        p = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
        total = p.sum(1, keepdim=True)
        p = p / torch.where(total > 0, total, 1.0)
        out[:, h], mass[:, h] = p @ vh, p @ vh.abs()
    return out, mass


def tolerance(out, mass, dtype, n_keys, v_max):
    """The kernels round each weight to `dtype` (half a step u of it: u * mass), the result once (u * |out|) and compute
    scores, exponentials and sums in fp32: 128 products of a few units off by 2^-24 each and exponentials by at most
    2^-13 relative move a weight by less than 2^-12, numerator and sum together by 2^-11 * mass.  fp16 weights below
    2^-14 of the largest are rounded to multiples of 2^-24 of it: 2^-25 per key."""
    u = torch.finfo(dtype).eps / 2
    t = u * (mass + out.abs()) * (1 + 2 ** -6) + 2 ** -11 * mass + 1e-30
    return t + n_keys * 2 ** -25 * v_max if dtype == torch.float16 else t


def check(got, out, mass, dtype, n_keys, v_max, what=""):
    got = got.double().cpu()
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    over = (got - out).abs() / tolerance(out, mass, dtype, n_keys, v_max)
    assert float(over.max()) <= 1.0, f"{what}: {float(over.max()):.3g} times the tolerance at {over.argmax().item()}"


def plan(cached, new, table, width, ring, head, count, n_rows, page):
    """The step plan on Python lists; returns what spf_paged_plan leaves."""
    table = [list(row) for row in table]
    cu, seq, refused, slots, positions = [0], [], [], [], []
    used = wanted = end = 0
    for r, (c, n) in enumerate(zip(cached, new)):
        c, n = max(c, 0), max(n, 0)
        held, total = -(-c // page), -(-(c + n) // page)
        end += n
        fits = total <= width and end <= n_rows and c + n <= 1 << 28
        wanted += total - held if fits else 0
        ok = fits and (total == held or wanted <= count)
        if ok:
            for i in range(held, total):
                table[r][i] = ring[(head + used) % len(ring)]
                used += 1
        cu.append(min(end, n_rows))
        seq.append(c + n if ok else 0)
        refused.append(0 if ok else 1)
        for i in range(cu[-1] - cu[-2]):
            at = table[r][(c + i) // page] if ok else -1
            slots.append(at * page + (c + i) % page if at >= 0 else -1)
            positions.append(c + i)
    slots += [-1] * (n_rows - len(slots))
    positions += [0] * (n_rows - len(positions))
    return dict(table=table, cu_new=cu, seq_len=seq, refused=refused, slot_map=slots, positions=positions,
                ring_state=[(head + used) % len(ring), count - used])


class Pool:
    """A paged cache in which only live keys were ever written: everything else is NaN."""

    def __init__(self, lengths, page, kv_heads, dim, dtype, gen, layout="token"):
        self.page, self.lengths = page, lengths
        owned = [-(-n // page) for n in lengths]
        n_pages = sum(owned) + 2
        shape = (n_pages, kv_heads, page, dim) if layout == "head" else (n_pages, page, kv_heads, dim)
        both = torch.full((n_pages, 2) + shape[1:], math.nan, dtype=dtype)
        self.k, self.v = (both[:, 0], both[:, 1]) if layout == "joined" else (both[:, 0].clone(), both[:, 1].clone())
        if layout == "head":
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        ids = torch.randperm(n_pages, generator=gen)
        width = max(max(owned), 1) + 1
        self.table = torch.full((len(lengths), width), -1, dtype=torch.int32)
        self.rows = []
        at = 0
        for r, n in enumerate(lengths):
            self.table[r, :owned[r]] = ids[at:at + owned[r]].to(torch.int32)
            at += owned[r]
            k = torch.randn(n, kv_heads, dim, generator=gen).to(dtype)
            v = torch.randn(n, kv_heads, dim, generator=gen).to(dtype)
            for i in range(owned[r]):
                a, b = i * page, min(n, (i + 1) * page)
                self.k[self.table[r, i], :b - a] = k[a:b]
                self.v[self.table[r, i], :b - a] = v[a:b]
            self.rows.append((k, v))

    def cuda(self):
        """The caches on the GPU with the strides they have here."""
        def move(x):
            full = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda")
            return full.copy_(x)
        if self.k.stride() == self.v.stride() and self.k.stride(0) == 2 * self.k.shape[1:].numel():
            both = torch.stack([self.k, self.v], 1).cuda()
            return both[:, 0], both[:, 1]
        return move(self.k), move(self.v)
