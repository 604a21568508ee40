"""The paged key/value cache on a B200 against plain float64 forms."""

from __future__ import annotations

import pytest
import torch

import awa_b200
from cache_testlib import Batch, attention, quantize, rotate, unpack

pytestmark = pytest.mark.gpu


def same(a, b):
    """Bit for bit, NaN where NaN."""
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


# ---------------------------------------------------------------- append and read
# (rows, past, page, kv heads, q heads, head_dim, axes, pairs)
APPEND = [
    ([1], [0], 16, 1, 1, 64, 1, 32),
    ([1, 1, 1], [5, 16, 100], 16, 20, 20, 128, 3, 21),
    ([0, 37, 0, 5, 0], [3, 31, 0, 64, 9], 32, 4, 12, 128, 1, 64),
    ([1300], [58], 64, 2, 2, 128, 3, 21),       # the tile of several rows
    ([3, 1181], [0, 7], 256, 1, 7, 64, 2, 9),   # rotated part ends inside a 16-byte piece
]


@pytest.mark.parametrize("storage", ["bf16", "f32", "int4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16rows", "f32rows"])
@pytest.mark.parametrize("case", APPEND, ids=lambda c: f"{len(c[0])}x{max(c[0])}d{c[5]}p{c[2]}")
def test_append_bit_exact(case, dtype, storage):
    rows, past, page, kv, heads, d, axes, pairs = case
    c = Batch(rows, past, page, kv, d, storage, seed=1, extra_rows=3)
    cache, batch = c.handles(awa_b200)
    q, k, v = (c.new_rows(h, dtype) for h in (heads, kv, kv))
    table = awa_b200.rope_table(2000, pairs)
    pos = torch.cat([p + torch.arange(n) for n, p in zip(rows, past)] + [torch.full((3,), -5)]).cuda()
    coords = None
    if axes > 1:
        coords = torch.stack([(pos * (a + 2)) % 2000 for a in range(axes)], 1).int().contiguous()
        coords[c.total:] = 1 << 30  # of rows that belong to nobody: not read
    q_out = torch.full_like(q, 3.0)
    before = [t.clone() for t in (c.k, c.v)]
    got = cache.append(batch, k, v, q=q, rope=awa_b200.CacheRope(table, coords), q_out=q_out)
    torch.cuda.synchronize()
    awa_b200.device_status()
    at = (pos[:, None] if coords is None else coords)[:c.total]
    n = c.total
    assert got is q_out and torch.equal(q_out[:n], rotate(q[:n], table, at).to(dtype))
    assert (q_out[n:] == 3.0).all()
    want = {"k": rotate(k[:n], table, at), "v": v[:n].float()}
    untouched = torch.ones(c.k.shape[0], page, dtype=torch.bool, device="cuda")
    back = cache.read(batch, torch.float32)
    for i, name in enumerate(("k", "v")):
        for b in range(len(rows)):
            slots = c.slots(b, past[b] + torch.arange(rows[b]))
            untouched[slots] = False
            r = slice(c.first[b], c.first[b] + rows[b])
            stored = getattr(c, name)[slots[0], :, slots[1]]
            if storage == "int4":
                packed, params = quantize(want[name][r])
                assert torch.equal(stored, packed)
                assert torch.equal(c.params[i][slots[0], :, slots[1]], params)
                assert torch.equal(back[i][r], unpack(packed, params))
                # within half a step of the row itself (and the roundings of the fp32 arithmetic on it)
                step = params[..., :1].float()
                off = (back[i][r] - want[name][r]).abs().unflatten(-1, (-1, 64))
                assert (off <= step * (0.5 + 2.0 ** -16) + 2.0 ** -22 * want[name][r].abs().unflatten(-1, (-1, 64))).all()
            else:
                assert torch.equal(stored, want[name][r].to(stored.dtype))
                assert torch.equal(back[i][r], stored.float())
    for t, was in zip((c.k, c.v), before):
        keep = untouched[:, None, :, None].expand_as(t)
        assert same(t[keep].float(), was[keep].float())


def test_append_unaligned_strided_in_place_and_without_q():
    c = Batch([5, 9], [2, 30], 16, 3, 24, "bf16", seed=2, strided=True)
    cache, batch = c.handles(awa_b200)
    wide = torch.randn(14, 200, device="cuda").bfloat16()
    k, v = wide[:, 1:73].unflatten(1, (3, 24)), wide[:, 77:149].unflatten(1, (3, 24))  # rows at odd elements
    cache.append(batch, k, v)
    got = cache.read(batch)
    assert torch.equal(got[0], k) and torch.equal(got[1], v)
    q = torch.randn(14, 6, 24, device="cuda").bfloat16()
    table = awa_b200.rope_table(40, 12)
    pos = torch.cat([2 + torch.arange(5), 30 + torch.arange(9)]).cuda()[:, None]
    want = rotate(q, table, pos).bfloat16()
    assert cache.append(batch, k, v, q=q, rope=awa_b200.CacheRope(table), q_out=q) is q
    assert torch.equal(q, want)


def test_constant_and_extreme_groups_of_a_4bit_cache():
    c = Batch([6], [0], 16, 1, 64, "int4", seed=3)
    cache, batch = c.handles(awa_b200)
    x = torch.zeros(6, 1, 64, device="cuda")
    x[1] = 1.0          # constant, a bf16 value: scale 0
    x[2] = 1.001        # constant, no bf16 value
    x[3, 0, 7] = 3e38   # one huge feature
    x[4] = torch.linspace(-1e-30, 1e-30, 64, device="cuda")
    x[5] = 1000 + torch.linspace(0, 1e-3, 64, device="cuda")  # range below a step of the minimum's type
    cache.append(batch, x, x)
    k, v = cache.read(batch, torch.float32)
    packed, params = quantize(x)
    assert torch.equal(k, unpack(packed, params)) and torch.equal(v, k)
    assert torch.equal(k[0], x[0]) and torch.equal(k[1], x[1])
    step = params[..., 0].float()
    assert ((k - x).abs() <= step * (0.5 + 2.0 ** -16) + 2.0 ** -22 * x.abs()).all()


def test_bad_pages_and_coordinates_are_reported_and_skipped():
    c = Batch([3, 2], [0, 14], 16, 2, 64, "bf16", seed=4)
    cache, batch = c.handles(awa_b200)
    q, k, v = (c.new_rows(2, torch.bfloat16) for _ in range(3))
    c.table[0, 0] = c.k.shape[0]  # one past the last page
    before = c.k.clone()
    cache.append(batch, k, v)
    with pytest.raises(awa_b200.AwaError, match="71"):
        awa_b200.device_status()
    page, slot = c.slots(1, [14, 15])
    assert torch.equal(c.k[page, :, slot], k[3:])
    before[page, :, slot] = k[3:]
    assert same(c.k, before)
    cache.attention(batch, q)
    with pytest.raises(awa_b200.AwaError, match="71"):
        awa_b200.device_status()
    coords = torch.tensor([[0], [4], [-1], [1], [3]], dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 9.0)
    c.table[0, 0] = 0 if c.table[1, 0] != 0 else 1
    cache.append(batch, k, v, q=q, rope=awa_b200.CacheRope(awa_b200.rope_table(4, 8), coords), q_out=out)
    with pytest.raises(awa_b200.AwaError, match="72"):
        awa_b200.device_status()
    assert (out[1:3] == 9.0).all() and not (out[[0, 3, 4]] == 9.0).all()
    # a sequence longer than its page table
    c.past_t[0] = 10 ** 6
    cache.attention(batch, q)
    with pytest.raises(awa_b200.AwaError, match="71"):
        awa_b200.device_status()
    c.past_t[0] = 2 ** 31 - 2
    cache.append(batch, k, v)
    cache.attention(batch, q)
    with pytest.raises(awa_b200.AwaError, match="71"):
        awa_b200.device_status()


# ---------------------------------------------------------------- attention
# (rows, past, page, kv heads, q heads, sinks, window, frame)
ATTEND = [
    ([1], [0], 16, 1, 1, 0, 0, 1),                          # one row that sees itself
    ([1], [700], 64, 20, 20, 58, 0, 1),
    ([1, 1, 1, 1], [0, 15, 16, 777], 16, 2, 8, 4, 100, 1),
    ([0, 1, 0, 3], [9, 40, 0, 130], 32, 1, 16, 0, 1, 1),    # window of one: each row itself
    ([1, 2], [5000, 3333], 128, 4, 4, 5, 1500, 1),
    ([1, 1, 0, 2], [5000, 131, 40, 9000], 64, 2, 6, 4, 0, 1),  # long: the work dealt out over the blocks
    ([4, 3, 1, 4], [6001, 17, 4500, 0], 32, 1, 8, 70, 6000, 1),  # two tiles a sequence
    ([2], [12345], 256, 1, 1, 0, 0, 1),
    ([4, 2, 1], [60, 300, 0], 16, 2, 14, 17, 33, 1),        # prefix ends inside a page and a block
    ([17], [0], 16, 1, 1, 0, 0, 1),
    ([200], [0], 64, 2, 6, 0, 0, 1),
    ([129, 0, 300, 64], [0, 5, 77, 640], 16, 2, 8, 4, 100, 1),
    ([333, 1], [1000, 4000], 64, 3, 3, 70, 257, 1),
    ([128], [190], 64, 2, 2, 62, 2, 64),                    # frames; the batch ends with a frame
    ([300, 90], [58, 0], 32, 4, 4, 58, 3, 100),             # frames that end inside a page, a short last one
    ([150], [0], 16, 2, 2, 40, 1, 16),                      # rows of the prefix itself, in frames
    ([257], [2], 256, 1, 5, 300, 7, 1),                     # everything is prefix
    ([70], [1500], 16, 1, 3, 0, 4, 300),
]


def attend(c, heads, sinks, window, frame, dtype, scale=None, q_scale=1.5, **kw):
    q = q_scale * c.new_rows(heads, dtype)
    cache, batch = c.handles(awa_b200, kw.pop("max_rows", None))
    out = torch.full_like(q, 5.0)
    cache.attention(batch, q, sinks=sinks, window=window, frame_tokens=frame, scale=scale, out=out, **kw)
    torch.cuda.synchronize()
    awa_b200.device_status()
    assert (out[c.total:] == 5.0).all()  # rows behind the last sequence
    want, tol = attention(c, q[:c.total], sinks, window, frame, c.d ** -0.5 if scale is None else scale)
    off = (out[:c.total].double() - want).abs()
    assert not off.isnan().any()
    assert (off <= tol).all(), f"{(off / tol).max().item():.3g} of the tolerance"
    return q, out


@pytest.mark.parametrize("storage", ["bf16", "f32", "int4"])
@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("case", ATTEND, ids=lambda c: f"{len(c[0])}x{max(c[0])}+{max(c[1])}p{c[2]}h{c[4]}-{c[3]}s{c[5]}w{c[6]}f{c[7]}")
def test_attention(case, d, storage):
    rows, past, page, kv, heads, sinks, window, frame = case
    c = Batch(rows, past, page, kv, d, storage, seed=5, extra_rows=2, strided=storage != "int4")
    attend(c, heads, sinks, window, frame, torch.float32 if storage == "f32" else torch.bfloat16)


@pytest.mark.parametrize("d", [8, 24, 96, 120])
@pytest.mark.parametrize("storage", ["bf16", "f32"])
def test_other_head_sizes(d, storage):
    dtype = torch.float32 if storage == "f32" else torch.bfloat16
    for rows, past in (([1, 2], [40, 300]), ([90], [33])):
        attend(Batch(rows, past, 16, 2, d, storage, seed=6), 6, 3, 50, 1, dtype)


@pytest.mark.parametrize("storage", ["bf16", "f32", "int4"])
def test_many_sequences(storage):
    g = torch.Generator().manual_seed(1)
    rows = torch.randint(0, 4, (150,), generator=g).tolist()
    past = torch.randint(0, 200, (150,), generator=g).tolist()
    c = Batch(rows, past, 16, 2, 64, storage, seed=7, extra_rows=5)
    attend(c, 8, 4, 64, 1, torch.float32 if storage == "f32" else torch.bfloat16)


@pytest.mark.parametrize("storage", ["bf16", "f32", "int4"])
@pytest.mark.parametrize("rows,told", [([200, 3], 1), ([1, 2], 500), ([2], 0)])
def test_max_rows_chooses_only_the_kernel(rows, told, storage):
    c = Batch(rows, [70] * len(rows), 16, 2, 128, storage, seed=8)
    attend(c, 4, 4, 90, 1, torch.float32 if storage == "f32" else torch.bfloat16, max_rows=told)


@pytest.mark.parametrize("storage", ["bf16", "f32", "int4"])
@pytest.mark.parametrize("rows", [1, 150])
@pytest.mark.parametrize("scale", [3.0, 1e-4, 1e-38])
def test_peaked_and_flat_softmax(rows, scale, storage):
    # scores up to a few hundred, and all but equal
    c = Batch([rows], [900], 32, 2, 128, storage, seed=9)
    attend(c, 2, 0, 0, 1, torch.float32 if storage == "f32" else torch.bfloat16, scale=scale)


@pytest.mark.parametrize("storage", ["bf16", "f32", "int4"])
@pytest.mark.parametrize("rows", [2, 140])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -3.0e38])
def test_pages_behind_the_window_may_be_gone(rows, poison, storage):
    past, page, sinks, window = 1000, 16, 20, 100
    c = Batch([rows], [past], page, 2, 128, storage, seed=10, poison=poison)
    full = c.table.clone()
    # positions sinks .. past - window are seen by no row; pages wholly among them are given away
    for e in range(-(-sinks // page), (past - window + 1) // page):
        gone = full[0, e].item()
        for t in ((c.k, c.v) if storage != "int4" else c.params):
            t[gone] = poison
        c.table[0, e] = -1 if e % 2 else 2 ** 31 - 1
    dtype = torch.float32 if storage == "f32" else torch.bfloat16
    q = c.new_rows(4, dtype)
    cache, batch = c.handles(awa_b200)
    out = cache.attention(batch, q, sinks=sinks, window=window)
    awa_b200.device_status()
    c.table = full
    for t in ((c.k, c.v) if storage != "int4" else c.params):
        t.nan_to_num_(0.0, 0.0, 0.0)
        t.clamp_(-100, 100)
    want, tol = attention(c, q, sinks, window, 1, 128 ** -0.5)
    assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("storage", ["bf16", "int4"])
def test_a_page_shared_by_sequences_and_a_past_of_garbage(storage):
    c = Batch([3, 3], [32, 32], 16, 2, 128, storage, seed=11)
    c.table[1, :2] = c.table[0, :2]  # a common prefix
    attend(c, 2, 0, 0, 1, torch.bfloat16)
    # a negative past is no past: the rows stand at 0, 1, 2
    cache, batch = c.handles(awa_b200)
    q = c.new_rows(2, torch.bfloat16)
    c.past_t[0] = -7
    got = cache.attention(batch, q)
    torch.cuda.synchronize()
    c.past[0] = 0
    want, tol = attention(c, q, 0, 0, 1, 128 ** -0.5)
    assert ((got.double() - want).abs() <= tol).all()


def test_4bit_groups_of_one_value_and_far_from_zero():
    """Scale 0, a minimum many steps from 0, huge and tiny groups."""
    c = Batch([2], [94], 16, 1, 128, "int4", seed=17)
    x = torch.randn(96, 1, 128, device="cuda")
    x[:20] = 3.0
    x[20:30, :, :64] = 100 + 0.01 * x[20:30, :, :64]
    x[30:40] *= 1e-30
    x[40:50] = 0.0
    x[50:60] = -1.001
    packed, params = quantize(x)
    page, slot = c.slots(0, torch.arange(96))
    for t, p in ((c.k, c.params[0]), (c.v, c.params[1])):
        t[page, :, slot], p[page, :, slot] = packed, params
    for window in (0, 45, 60, 80):
        attend(c, 4, 0, window, 1, torch.bfloat16, q_scale=0.3)


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("storage", ["bf16", "f32", "int4"])
def test_frames_through_append_and_attention(storage):
    """Text, then frame after frame, as a stream of latents comes: each step's
    rows are rotated into the cache and attend to the last frames."""
    text, frame, window, heads, d, page = 10, 48, 2, 4, 128, 16
    dtype = torch.float32 if storage == "f32" else torch.bfloat16
    pages = 40
    cache = awa_b200.KvCache.empty(pages, page, heads, d, storage)
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).int().cuda()[None]
    angles = awa_b200.rope_table(64, 21)
    c = Batch([0], [0], page, heads, d, storage, seed=12)
    c.k, c.v, c.params, c.table = cache.k, cache.v, (cache.k_params, cache.v_params), table
    past = 0
    for step in range(6):
        n = text if step == 0 else frame
        q, k, v = (torch.randn(n, heads, d, device="cuda").to(dtype) for _ in range(3))
        i = torch.arange(n, device="cuda", dtype=torch.int32)
        coords = torch.stack([i, i, i] if step == 0 else [0 * i + text + step, i // 8, i % 8], 1).contiguous()
        starts = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        batch = awa_b200.CacheBatch(starts, torch.tensor([past], dtype=torch.int32, device="cuda"), table, n, n)
        turned = cache.append(batch, k, v, q=q, rope=awa_b200.CacheRope(angles, coords))
        assert torch.equal(turned, rotate(q, angles, coords).to(dtype))
        out = cache.attention(batch, turned, sinks=text, window=window, frame_tokens=frame)
        awa_b200.device_status()
        c.rows, c.past, c.first, c.total = [n], [past], [0, n], n
        want, tol = attention(c, turned, text, window, frame, d ** -0.5)
        assert ((out.double() - want).abs() <= tol).all(), step
        past += n


@pytest.mark.parametrize("storage", ["bf16", "f32", "int4"])
@pytest.mark.parametrize("width", [14, 1000])  # a table with room for long sequences takes other kernels
def test_captured_step_serves_later_steps(width, storage):
    """One captured step of append and attention, replayed with other lengths,
    pages and rows, gives what eager calls give; two graphs may run at once."""
    dtype = torch.float32 if storage == "f32" else torch.bfloat16
    c = Batch([1, 1, 1], [207, 207, 207], 16, 2, 128, storage, seed=13)  # 13 pages each, of 41
    c.table = torch.nn.functional.pad(c.table, (0, width - c.table.shape[1]), value=-1)
    cache, batch = c.handles(awa_b200)
    q, k, v = (c.new_rows(h, dtype) for h in (8, 2, 2))
    rope = awa_b200.CacheRope(awa_b200.rope_table(400, 64))

    def step():
        return cache.attention(batch, cache.append(batch, k, v, q=q, rope=rope), sinks=4, window=50 if width < 99 else 0)

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    side = torch.cuda.Stream()
    for past in ([71, 6, 201], [10, 0, 63], [207, 15, 90]):
        c.past_t.copy_(torch.tensor(past, dtype=torch.int32))
        c.table[:, :13] = torch.randperm(41, generator=c.generator)[:39].reshape(3, 13).int().cuda()
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=c.generator).to(dtype))
        for t in ((c.k, c.v) if storage != "int4" else c.params):
            t.nan_to_num_(0.25)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0][0].replay()
        graphs[1][0].replay()
        torch.cuda.synchronize()
        want = step()
        assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want)
        assert not want.isnan().any()
    awa_b200.device_status()


@pytest.mark.parametrize("storage", ["bf16", "f32", "int4"])
def test_captured_prompt(storage):
    """Many rows in a graph, replayed with other lengths and page numbers."""
    dtype = torch.float32 if storage == "f32" else torch.bfloat16
    c = Batch([150, 90], [200, 300], 16, 2, 128, storage, seed=18)
    cache, batch = c.handles(awa_b200)
    q = c.new_rows(4, dtype)

    def step():
        return cache.attention(batch, q, sinks=4, window=60)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for starts, past in (([0, 150, 240], [200, 300]), ([0, 3, 240], [340, 100]), ([0, 240, 240], [90, 0])):
        c.starts.copy_(torch.tensor(starts, dtype=torch.int32))
        c.past_t.copy_(torch.tensor(past, dtype=torch.int32))
        q.copy_(torch.randn(q.shape, generator=c.generator).to(dtype))
        for t in ((c.k, c.v) if storage != "int4" else c.params):
            t.nan_to_num_(0.25)
        graph.replay()
        got = out.clone()
        assert torch.equal(got, step()) and not got.isnan().any()
    awa_b200.device_status()


@pytest.mark.parametrize("storage", ["bf16", "f32", "int4"])
@pytest.mark.parametrize("rows,past", [([1, 1], [300, 40]), ([1, 2], [7000, 5500]), ([70, 130], [300, 40])])
def test_another_stream_and_repeatable(rows, past, storage):
    dtype = torch.float32 if storage == "f32" else torch.bfloat16
    c = Batch(rows, past, 16, 2, 128, storage, seed=14)
    cache, batch = c.handles(awa_b200)
    q = c.new_rows(8, dtype)
    want = cache.attention(batch, q, sinks=4)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    many = [cache.attention(batch, q, sinks=4, stream=stream) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in many)


@pytest.mark.parametrize("storage", ["bf16", "int4"])
def test_positions_past_four_gigabytes(storage):
    """Pages whose byte offsets pass 32 bits."""
    d, page, heads = 128, 256, 8
    pages = 9000 if storage == "bf16" else 34000
    cache = awa_b200.KvCache.empty(pages, page, heads, d, storage)
    assert cache.k.numel() * cache.k.element_size() > 2 ** 32
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
    n = 600
    q, k, v = (torch.randn(n, heads, d, device="cuda").bfloat16() for _ in range(3))
    zero, starts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0], [0, n]))
    batch = awa_b200.CacheBatch(starts, zero, table, n, n)
    cache.append(batch, k, v)
    c = Batch([0], [0], page, heads, d, storage)
    c.k, c.v, c.params, c.table = cache.k, cache.v, (cache.k_params, cache.v_params), table
    c.rows, c.past, c.first, c.total = [n], [0], [0, n], n
    back = cache.read(batch, torch.float32)
    assert torch.equal(back[0].double(), c.cached(0, "k")) and torch.equal(back[1].double(), c.cached(0, "v"))
    out = cache.attention(batch, q)
    one = awa_b200.CacheBatch(torch.tensor([0, 1], dtype=torch.int32, device="cuda"),
                              torch.tensor([n - 1], dtype=torch.int32, device="cuda"), table, 1, 1)
    last = cache.attention(one, q[-1:])
    awa_b200.device_status()
    want, tol = attention(c, q, 0, 0, 1, d ** -0.5)
    assert ((out.double() - want).abs() <= tol).all()
    assert ((last.double() - want[-1:]).abs() <= tol[-1:]).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [1, 20, 150])
def test_f32_values_of_a_single_key_come_back_exactly(rows, d):
    """A row that sees one key gets p = 1: its value, bit for bit, up to the largest floats and over 160 binades."""
    c = Batch([rows], [40], 16, 2, d, "f32", seed=5)
    cache, batch = c.handles(awa_b200)
    q = c.new_rows(2, torch.float32)
    page, slot = c.slots(0, torch.arange(40, 40 + rows))
    v = c.cached(0, "v")[40:].float()
    v *= torch.exp2(torch.arange(rows * d * 2, device=v.device).reshape(rows, 2, d) % 161 - 80.0)
    v[0, 0, 0], v[-1, 1, 1] = torch.finfo(torch.float32).max, torch.finfo(torch.float32).min
    c.v[page, :, slot] = v
    out = cache.attention(batch, q, window=1)
    awa_b200.device_status()
    assert torch.equal(out, v)
