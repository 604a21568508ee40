"""Plain float64 forms of the key/value cache operators, and batches with
everything poisoned that an operator must not read."""

from __future__ import annotations

import torch

GROUP = 64
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}  # half a step, relative


class Batch:
    """Sequences of rows[b] new rows after past[b] cached ones. Pages are dealt
    in random order; slots and pages that no position uses hold `poison`, page
    numbers past a sequence's end are garbage."""

    def __init__(self, rows, past, page_tokens, kv_heads, head_dim, storage, seed=0, poison=float("nan"), device="cuda",
                 extra_rows=0, strided=False):
        g = torch.Generator().manual_seed(seed)
        self.rows, self.past, self.page = list(rows), list(past), page_tokens
        self.kv_heads, self.d, self.storage, self.device = kv_heads, head_dim, storage, device
        used = [-(-(n + p) // page_tokens) for n, p in zip(rows, past)]
        pages = sum(used) + 2
        order = torch.randperm(pages, generator=g)
        width = max(used + [1]) + 1
        table = torch.full((len(rows), width), 2 ** 30, dtype=torch.int32)
        at = 0
        for b, n in enumerate(used):
            table[b, :n] = order[at:at + n].int()
            at += n
        starts = [0]
        for n in rows:
            starts.append(starts[-1] + n)
        self.total, self.first = starts[-1], starts
        self.table = table.to(device)
        self.starts = torch.tensor(starts, dtype=torch.int32, device=device)
        self.past_t = torch.tensor(past, dtype=torch.int32, device=device)
        shape = (pages, kv_heads, page_tokens)
        # every slot poisoned, then the positions that exist
        live = torch.zeros(shape[0], page_tokens, dtype=torch.bool)
        for b, (n, p) in enumerate(zip(rows, past)):
            j = torch.arange(n + p)
            live[table[b].long()[j // page_tokens], j % page_tokens] = True
        live = live[:, None, :, None]
        self.params = (None, None)
        if storage == "int4":
            self.k, self.v = (torch.randint(0, 256, shape + (head_dim // 2,), generator=g, dtype=torch.uint8).to(device)
                              for _ in range(2))
            par = []
            for _ in range(2):
                scale = 0.2 + 0.1 * torch.rand(shape + (head_dim // GROUP,), generator=g)
                both = torch.stack([scale, -7.5 * scale], -1)
                par.append(torch.where(live[..., None], both, torch.full_like(both, poison)).bfloat16().to(device))
            self.params = tuple(par)
        else:
            dtype = torch.bfloat16 if storage == "bf16" else torch.float32
            k, v = (torch.randn(shape + (head_dim,), generator=g) for _ in range(2))
            k, v = (torch.where(live, x, torch.full_like(x, poison)).to(dtype).to(device) for x in (k, v))
            if strided:  # keys and values of a page side by side
                both = torch.stack([k, v], 1)
                k, v = both[:, 0], both[:, 1]
            self.k, self.v = k, v
        self.extra = extra_rows
        self.generator = g

    def new_rows(self, heads, dtype, poison=float("nan")):
        """[total + extra, heads, d], the extra rows (of no sequence) poisoned."""
        x = torch.randn(self.total + self.extra, heads, self.d, generator=self.generator)
        x[self.total:] = poison
        return x.to(dtype).to(self.device)

    def handles(self, awa, max_rows=None):
        cache = awa.KvCache(self.k, self.v, *self.params)
        batch = awa.CacheBatch(self.starts, self.past_t, self.table, self.total + self.extra,
                               max(self.rows + [0]) if max_rows is None else max_rows)
        return cache, batch

    def slots(self, b, positions):
        j = torch.as_tensor(positions, device=self.device)
        return self.table[b].long()[j // self.page], j % self.page

    def cached(self, b, name):
        """Positions 0 .. past + rows - 1 of sequence b, float64 [n, kv_heads, d]."""
        page, slot = self.slots(b, torch.arange(self.rows[b] + self.past[b]))
        x = getattr(self, name)[page, :, slot]
        if self.storage == "int4":
            x = unpack(x, self.params[0 if name == "k" else 1][page, :, slot])
        return x.double()


def unpack(packed, params):
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).float()
    par = params.float().repeat_interleave(GROUP, -2)
    return codes * par[..., 0] + par[..., 1]


def seen_keys(p, length, sinks, window, frame):
    """The definition, position by position: a bool per key."""
    j = torch.arange(length)
    if p < sinks:
        return j < min(sinks, (p // frame + 1) * frame)
    f, fj = (p - sinks) // frame, torch.div(j - sinks, frame, rounding_mode="floor")
    ok = (j < sinks) | ((fj <= f) & (j >= sinks))
    if window:
        ok &= (j < sinks) | (fj > f - window)
    return ok


def attention(case: Batch, q, sinks, window, frame, scale):
    """(out, tolerance) in float64 for the rows that belong to a sequence.

    Tolerance, element by element: with A = sum p |v| / l and B the largest
    scale sum |q k| of the row,
      scores: fp32 sums of d products (exact in fp32 for bf16): (d + 4) 2^-24 B,
              which moves p, and with it out, by twice that times A;
      p: 2^-22 for exp2, one rounding to bf16 (2^-8) where the products run on
         bf16 operands; sums over n keys in fp32: n 2^-24 A, the division 2^-23;
      out: half a step of its type.
    A 4-bit cache's rows may be rounded to bf16 once (2^-8 of every k and v)
    ahead of the products."""
    half = HALF[q.dtype]
    f32 = q.dtype == torch.float32
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    group = q.shape[1] // case.kv_heads
    for b, (n, p) in enumerate(zip(case.rows, case.past)):
        if not n:
            continue
        k = case.cached(b, "k").repeat_interleave(group, 1)
        v = case.cached(b, "v").repeat_interleave(group, 1)
        x = q[case.first[b]:case.first[b] + n].double()
        seen = torch.stack([seen_keys(p + i, n + p, sinks, window, frame) for i in range(n)]).to(q.device)
        s = torch.einsum("ihd,jhd->hij", x, k) * scale
        s.masked_fill_(~seen, float("-inf"))
        big = torch.einsum("ihd,jhd->hij", x.abs(), k.abs()) * scale
        big = big.masked_fill(~seen, 0).amax(-1)  # [heads, rows]
        prob = torch.softmax(s, -1).nan_to_num(0.0)
        r = slice(case.first[b], case.first[b] + n)
        out[r] = torch.einsum("hij,jhd->ihd", prob, v)
        a = torch.einsum("hij,jhd->ihd", prob, v.abs())
        score = (case.d + 4) * 2.0 ** -24 * big
        per = 2.0 ** -22 + (n + p + 8) * 2.0 ** -24
        if not f32:
            per += 2.0 ** -8
        if case.storage == "int4":
            score = score + 2.0 ** -8 * big
            per += 2.0 ** -8
        tol[r] = a * (per + 2 * torch.expm1(score).T[..., None]) + half * out[r].abs() + 1e-30
    return out, tol


def rotate(x, table, coords):
    """fp32 rotation, every product and sum rounded on its own."""
    x = x.float().clone()
    axes, pairs = coords.shape[1], table.shape[1]
    for a in range(axes):
        cs = table[coords[:, a].long()][:, None]
        lo = 2 * a * pairs
        x0, x1 = x[..., lo:lo + 2 * pairs:2].clone(), x[..., lo + 1:lo + 2 * pairs:2].clone()
        x[..., lo:lo + 2 * pairs:2] = x0 * cs[..., 0] - x1 * cs[..., 1]
        x[..., lo + 1:lo + 2 * pairs:2] = x1 * cs[..., 0] + x0 * cs[..., 1]
    return x


def bf16_next(x, up):
    """The bf16 value at or beyond x (fp32), bit by bit."""
    bits = x.contiguous().view(torch.int32)
    cut = bits & -65536
    away = (bits != cut) & ((bits >= 0) if up else (bits < 0))
    return (cut + away.to(torch.int32) * 65536).view(torch.float32)


def quantize(x):
    """(packed, params) of fp32 rows [..., d], as the header defines them."""
    x = x.unflatten(-1, (-1, GROUP))
    low = bf16_next(x.amin(-1), False)
    scale = bf16_next((x.amax(-1) - low) / torch.full_like(low, 15.0), True)
    inverse = torch.where(scale > 0, torch.ones_like(scale) / scale, torch.zeros_like(scale))
    codes = torch.round((x - low[..., None]) * inverse[..., None]).clamp(0, 15).flatten(-2).to(torch.uint8)
    return codes[..., 0::2] | (codes[..., 1::2] << 4), torch.stack([scale, low], -1).bfloat16()
