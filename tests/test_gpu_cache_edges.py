"""The paged key/value cache on a B200: calls that its documentation allows and
that come near an edge (memory, magnitudes, sizes, masks)."""

from __future__ import annotations

import ctypes

import pytest
import torch

import awa_b200
from awa_b200 import cache as binding
import test_gpu_cache as others
from cache_testlib import Batch, attention, quantize, rotate, seen_keys, unpack

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- the memory
def create(k, v, pages=4):
    handle = ctypes.c_void_p()
    params = binding._CacheParams(awa_b200.AWA_BF16, 2, 64, 16, pages, k, v, 2 * 16 * 64, 16 * 64, None, None, 0, 0)
    lib = binding._cache_library()
    rc = lib.awa_cache_create(ctypes.byref(params), ctypes.byref(handle))
    if handle.value:
        lib.awa_cache_destroy(handle)
    return rc, lib.awa_last_error().decode()


def test_memory_that_the_gpu_cannot_reach_is_refused():
    """Refused when the handle is made: no kernel runs."""
    on_gpu = torch.empty(4, 2, 16, 64, dtype=torch.bfloat16, device="cuda")
    on_host = torch.empty(4, 2, 16, 64, dtype=torch.bfloat16)
    pointer = (on_host.data_ptr() + 15) // 16 * 16
    assert create(on_gpu.data_ptr(), on_gpu.data_ptr())[0] == awa_b200.AWA_OK
    for k, v in ((pointer, on_gpu.data_ptr()), (on_gpu.data_ptr(), pointer)):
        rc, error = create(k, v)
        assert rc == awa_b200.AWA_ERR_INVALID and "GPU" in error


# ---------------------------------------------------------------- 4 bits, as close as the kernels are
def four_bit_attention(c, q, sinks, window, frame, scale, many):
    """(out, tolerance) of a 4-bit cache in float64, row by row.

    A row of values is minimum + scale * code; with K^ = |minimum| + scale * code
    for keys, V^ for values, p the probabilities, d features, n keys:
      few rows: codes are exact operands, so scores carry fp32 sums of d products
        of both parts: (d + 4) 2^-24 sum |q| K^. p times the scale is rounded to
        bf16 once: 2^-8 p |v|. The sums over n keys: n 2^-24 p V^. A scale
        below 2^-80 max(1, |minimum|) is raised to that, which moves a value by up
        to 15 2^-80 max(1, |minimum|), and products whose share of the result is
        below 2^-126 / (2^-133 2^90) = 2^-83 may be cut: together 2^-75
        max(1, |minimum|) a key, weighed by p (at most 1) and by 1 for n < 2^8 keys.
      many rows: keys, values and p in fp16: 2^-11 sum |q k| on the scores, 2^-11
        twice on p |v| (q, 8 bits, is exact); p below 2^-32 of the row's largest
        is dropped: 2^-31 V^ a key. The sums as above.
    exp2: 2^-22, the division 2^-23; out: half a step of bf16."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    group = q.shape[1] // c.kv_heads
    for b, (n, p) in enumerate(zip(c.rows, c.past)):
        if not n:
            continue
        k, v, k_up, v_up = (x.repeat_interleave(group, 1) for x in
                            (c.cached(b, "k"), c.cached(b, "v"), magnitude(c, b, "k"), magnitude(c, b, "v")))
        r = slice(c.first[b], c.first[b] + n)
        x = q[r].double()
        seen = torch.stack([seen_keys(p + i, n + p, sinks, window, frame) for i in range(n)]).to(q.device)
        s = torch.einsum("ihd,jhd->hij", x, k) * scale
        prob = torch.softmax(s.masked_fill(~seen, float("-inf")), -1).nan_to_num(0.0)
        top = lambda y: (torch.einsum("ihd,jhd->hij", x.abs(), y) * scale).masked_fill(~seen, 0).amax(-1)
        out[r] = torch.einsum("hij,jhd->ihd", prob, v)
        a, a_up = (torch.einsum("hij,jhd->ihd", prob, y) for y in (v.abs(), v_up))
        score = (c.d + 4) * 2.0 ** -24 * top(k_up) + (2.0 ** -11 * top(k.abs()) if many else 0)
        tol[r] = a * (2 * 2.0 ** -11 if many else 2.0 ** -8) + a_up * (2.0 ** -22 + (n + p + 8) * 2.0 ** -24)
        tol[r] += a_up * 2 * torch.expm1(score).T[..., None] + 2.0 ** -8 * out[r].abs() + 1e-37
        if not many:
            tol[r] += 2.0 ** -75 * max(1.0, v_up.max().item()) * (1 + (n + p) / 256)
        if many:
            most = prob.amax(-1).T[..., None]
            tol[r] += 2.0 ** -31 * most * torch.einsum("hij,jhd->ihd", seen[None].expand_as(prob).double(), v_up)
    return out, tol


def magnitude(c, b, name):
    page, slot = c.slots(b, torch.arange(c.rows[b] + c.past[b]))
    params = c.params[0 if name == "k" else 1][page, :, slot].abs()
    return unpack(getattr(c, name)[page, :, slot], params).double()


def fill_four_bit(c, k, v):
    """The rows [past + rows, heads, d] of c's only sequence, packed."""
    page, slot = c.slots(0, torch.arange(k.shape[0]))
    for t, p, x in ((c.k, c.params[0], k), (c.v, c.params[1], v)):
        t[page, :, slot], p[page, :, slot] = quantize(x)


def check_four_bit(c, q, sinks=0, window=0, frame=1, scale=None, most=0.003):
    """most: of the error's norm, relative to the result's. bf16's rounding of
    the output is up to 2^-8 / sqrt(3) = 0.0023 of it; keys and values rounded to
    bf16 would come to 0.0048."""
    cache, batch = c.handles(awa_b200)
    scale = c.d ** -0.5 if scale is None else scale
    out = cache.attention(batch, q, sinks=sinks, window=window, frame_tokens=frame, scale=scale)
    torch.cuda.synchronize()
    awa_b200.device_status()
    many = max(c.rows) * (q.shape[1] // c.kv_heads) > 32
    want, tol = four_bit_attention(c, q[:c.total], sinks, window, frame, scale, many)
    out = out[:c.total].double()
    assert not out.isnan().any()
    off = (out - want).abs()
    assert (off <= tol).all(), f"{(off / tol).max().item():.3g} of the tolerance"
    if most and (many or want.abs().max() > 2.0 ** -60):
        assert (off.norm() <= most * want.norm()), f"{(off.norm() / want.norm()).item():.3g} of the norm"
        # the bound tells these from the result
        assert (want.abs() > tol).any() and (2 * want.abs() > tol).float().mean() > 0.5


ROWS = [1, 8, 9, 150]  # 8 rows of a group of 4: the last that the kernel for few rows takes


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("size_k,size_v,size_q", [
    (1, 1, 1), (1e-4, 1, 1e4), (1, 1e-4, 1), (1e-6, 1e-6, 1e6), (1e-8, 1e-8, 1e6), (1, 1e-12, 1), (1, 1e-30, 1),
    (3e4, 3e4, 1e-4), (1e4, 1, 1e-4), (1, 1, 1e-3)])
def test_four_bit_values_of_any_size(size_k, size_v, size_q, rows, d):
    """What a row gets does not depend on how many rows come with it, for tiny values as well."""
    c = Batch([rows], [200], 16, 2, d, "int4", seed=21)
    x = torch.randn(2, 200 + rows, 2, d, generator=c.generator).cuda()
    fill_four_bit(c, size_k * x[0], size_v * x[1])
    q = (size_q * c.new_rows(8, torch.float32)).bfloat16()
    check_four_bit(c, q, window=150, sinks=3, scale=min(1.0, 1 / (size_k * size_q)) * d ** -0.5)


@pytest.mark.parametrize("rows", ROWS)
def test_four_bit_groups_of_different_sizes(rows):
    """Heads, groups of 64 features and rows of q far apart in size."""
    c = Batch([rows], [120], 32, 2, 128, "int4", seed=22)
    x = torch.randn(2, 120 + rows, 2, 128, generator=c.generator).cuda()
    x[0, :, 0, :64] *= 1e-7
    x[0, :, 1, 64:] *= 1e3
    x[1, :, 0, 64:] *= 1e-9
    x[1, :, 1, :64] *= 1e4
    fill_four_bit(c, x[0], x[1])
    q = c.new_rows(8, torch.float32)
    q[..., :64] *= torch.tensor([1e7, 1.0]).repeat_interleave(4)[:, None].cuda()
    q[..., 64:] *= torch.tensor([1.0, 1e-3]).repeat_interleave(4)[:, None].cuda()
    q[::3] *= 1e-5
    check_four_bit(c, q.bfloat16())


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("below", [20, 24, 27, 30])
def test_four_bit_keys_far_below_the_largest(below, rows):
    """One key holds all but 2^-below of a row, and 0 as its value: the others make the result."""
    c = Batch([rows], [300], 16, 1, 64, "int4", seed=23)
    k = torch.zeros(300 + rows, 1, 64, device="cuda")
    v = 1 + torch.rand(300 + rows, 1, 64, generator=c.generator).cuda()
    k[5], v[5] = 1.0, 0.0
    fill_four_bit(c, k, v)
    q = torch.full((rows, 4, 64), below / 64, device="cuda").bfloat16()  # exact: a multiple of 2^-6 below 2^8
    check_four_bit(c, q, scale=0.6931471805599453, most=0.005)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("sinks,window,frame", [(0, 0, 1), (20, 90, 1), (20, 2, 33)])
@pytest.mark.parametrize("d", [64, 128])
def test_four_bit_attention_as_close_as_it_is(d, sinks, window, frame, rows):
    c = Batch([rows, 0, max(1, rows // 2)], [400, 7, 33], 16, 2, d, "int4", seed=24, extra_rows=2)
    check_four_bit(c, 1.5 * c.new_rows(8, torch.bfloat16), sinks, window, frame)


@pytest.mark.parametrize("rows", ROWS)
def test_four_bit_peaked_softmax(rows):
    c = Batch([rows], [500], 32, 2, 128, "int4", seed=25)
    check_four_bit(c, 1.5 * c.new_rows(2 if rows == 1 else 8, torch.bfloat16), scale=0.5, most=0)


def test_four_bit_sequences_of_different_sizes():
    """The largest values of one sequence take nothing from another's."""
    c = Batch([60, 50, 40], [100, 30, 77], 16, 2, 128, "int4", seed=26)
    for b, (k_size, v_size) in enumerate(((1.0, 1.0), (1e-3, 1e-6), (30.0, 1e4))):
        page, slot = c.slots(b, torch.arange(c.rows[b] + c.past[b]))
        for t, p, size in ((c.k, c.params[0], k_size), (c.v, c.params[1], v_size)):
            x = size * torch.randn(page.shape[0], 2, 128, generator=c.generator).cuda()
            t[page, :, slot], p[page, :, slot] = quantize(x)
    q = c.new_rows(8, torch.float32)
    q[60:110] *= 1e3
    q[110:] *= 0.03
    check_four_bit(c, q.bfloat16(), most=0)


@pytest.mark.parametrize("width", [700, 840])  # x 3 sequences: fewer pages than the cache has, and more
def test_four_bit_heads_in_several_passes(width):
    """Unpacked pages of more than 2 GiB: some heads at a time. The table has room
    for far more rows than there are."""
    pages, heads = 2500, 10
    c = Batch([40, 3, 30], [600, 300, 0], 256, heads, 128, "int4", seed=27, extra_rows=1)
    for name in ("k", "v"):
        x = torch.zeros((pages,) + getattr(c, name).shape[1:], dtype=torch.uint8, device="cuda")
        x[:getattr(c, name).shape[0]] = getattr(c, name)
        setattr(c, name, x)
    params = []
    for p in c.params:
        x = torch.full((pages,) + p.shape[1:], float("nan"), dtype=p.dtype, device="cuda")
        x[:p.shape[0]] = p
        params.append(x)
    c.params = tuple(params)
    c.table = torch.nn.functional.pad(c.table, (0, width - c.table.shape[1]), value=2 ** 31 - 1)
    cache, batch = c.handles(awa_b200)
    need = cache.attention_workspace_bytes(batch, 4 * heads)
    assert need < 2 ** 31 < heads * min(pages, 3 * width) * 256 * 128 * 4
    check_four_bit(c, 1.5 * c.new_rows(4 * heads, torch.bfloat16), sinks=5, most=0.003)


def test_four_bit_pages_shared_by_sequences():
    """More table entries than pages: the unpacked ones are the cache's, whoever sees them."""
    c = Batch([40, 40, 40], [96, 96, 96], 16, 2, 64, "int4", seed=28)
    c.table[1:, :6] = c.table[0, :6]  # a common prefix
    c.table = torch.nn.functional.pad(c.table, (0, 100), value=-1)
    check_four_bit(c, 1.5 * c.new_rows(8, torch.bfloat16))
    # a page that the cache does not have counts as zero keys and values, and is reported
    page = c.table[2, 7].item()
    c.table[2, 7] = c.k.shape[0]
    cache, batch = c.handles(awa_b200)
    q = c.new_rows(8, torch.bfloat16)
    got = cache.attention(batch, q)
    with pytest.raises(awa_b200.AwaError, match="71"):
        awa_b200.device_status()
    c.table[2, 7] = page
    for p in c.params:
        p[page] = 0
    want, tol = four_bit_attention(c, q, 0, 0, 1, 64 ** -0.5, True)
    assert ((got.double() - want).abs() <= tol).all()


# ---------------------------------------------------------------- sizes
@pytest.mark.parametrize("storage", ["bf16", "f32", "int4"])
def test_append_of_many_rows(storage):
    """9472 rows and more go 16 to a block; the last tile is short."""
    others.test_append_bit_exact(([9500, 3], [37, 0], 64, 2, 3, 128, 3, 21), torch.bfloat16, storage)


@pytest.mark.parametrize("storage", ["bf16", "f32", "int4"])
@pytest.mark.parametrize("rows", [1, 2, 40])
def test_groups_of_more_than_128_heads(rows, storage):
    c = Batch([rows, 1], [70, 200], 16, 1, 64, storage, seed=31, extra_rows=1)
    others.attend(c, 130, 4, 100, 1, torch.float32 if storage == "f32" else torch.bfloat16)


@pytest.mark.parametrize("storage", ["bf16", "f32", "int4"])
@pytest.mark.parametrize("rows", [1, 40])
def test_more_than_16384_sequences(rows, storage):
    """Most of them without rows; those that have some are spread."""
    sequences = 16500
    has = [rows if b % 700 == 5 else 0 for b in range(sequences)]
    past = [37 * (b % 5) if n else 0 for b, n in enumerate(has)]
    c = Batch(has, past, 16, 1, 64, storage, seed=32)
    others.attend(c, 2, 0, 60, 1, torch.float32 if storage == "f32" else torch.bfloat16)


def side_by_side(c):
    """Keys and values, and their params, of a page next to one another."""
    both, params = torch.stack([c.k, c.v], 1), torch.stack(c.params, 1)
    c.k, c.v, c.params = both[:, 0], both[:, 1], (params[:, 0], params[:, 1])


def heads_outside(c):
    """The pages of a head next to one another."""
    turn = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
    c.k, c.v, c.params = turn(c.k), turn(c.v), tuple(turn(p) for p in c.params)


@pytest.mark.parametrize("layout", [side_by_side, heads_outside])
@pytest.mark.parametrize("rows", [[1, 2], [60, 3]])
@pytest.mark.parametrize("d", [64, 128])
def test_four_bit_layouts(d, rows, layout):
    c = Batch(rows, [130, 77], 16, 3, d, "int4", seed=33)
    layout(c)
    check_four_bit(c, 1.5 * c.new_rows(6, torch.bfloat16), sinks=3, window=90)
    cache, batch = c.handles(awa_b200)
    k, v = (c.new_rows(3, torch.bfloat16) for _ in range(2))
    cache.append(batch, k, v)
    back = cache.read(batch, torch.float32)
    for x, got in ((k, back[0]), (v, back[1])):
        assert torch.equal(got, unpack(*quantize(x.float())))


# ---------------------------------------------------------------- beside the framework's other operators
def test_append_turns_rows_as_mmrope_does():
    """With the layer's own angles, row by row the same bits."""
    plan = awa_b200.AwaPlan(2, 4, 6, 1, 1, 1)
    info = plan.info
    text, n, heads = info.text_tokens, info.source_tokens, 2
    x = torch.randn(n, 3, heads, 128, device="cuda")
    t = torch.randn(text, 3, heads, 128, device="cuda")
    packed, starts = plan.pack(x, t)
    starts = starts.int().tolist()
    turned = plan.mmrope(packed)
    unit = torch.zeros_like(packed)
    unit[..., 0::2] = 1.0  # comes back as (cos, sin)
    angles = plan.mmrope(unit)[:, 0, 0, :126].view(-1, 3, 21, 2)
    for window in range(info.window_count):
        rows = slice(starts[window], starts[window + 1])
        count = rows.stop - rows.start
        # a table with one entry for each row and axis
        table = angles[rows].reshape(count * 3, 21, 2).contiguous()
        coords = torch.arange(3 * count, dtype=torch.int32, device="cuda").view(count, 3).contiguous()
        c = Batch([count], [0], 64, heads, 128, "f32", seed=34)
        cache, batch = c.handles(awa_b200)
        q, k, v = packed[rows].unbind(1)
        got = cache.append(batch, k, v, q=q, rope=awa_b200.CacheRope(table, coords))
        back = cache.read(batch)
        want = turned[rows]
        assert torch.equal(got, want[:, 0]) and torch.equal(back[0], want[:, 1]) and torch.equal(back[1], want[:, 2])
    awa_b200.device_status()


@pytest.mark.parametrize("storage", ["bf16", "int4"])
def test_frames_from_projection_to_projection(storage):
    """A block's step over a stream: QKV projection, append, attention, output projection; text, then frames."""
    heads, d, model, text, frame, page = 3, 128, 192, 10, 40, 16
    g = torch.Generator().manual_seed(35)
    normal = lambda *shape: torch.randn(*shape, generator=g).cuda()
    w_in, w_out = (normal(3 * heads * d, model) / model ** 0.5).bfloat16(), (normal(256, heads * d) / 20).bfloat16()
    gamma_q, gamma_k, bias, gate = 1 + 0.2 * normal(d), 1 + 0.2 * normal(d), 0.1 * normal(256), 0.2 * normal(256)
    cache = awa_b200.KvCache.empty(30, page, heads, d, storage)
    table = torch.randperm(30, generator=g).int().cuda()[None]
    angles = awa_b200.rope_table(64, 21)
    c = Batch([0], [0], page, heads, d, storage)
    c.k, c.v, c.params, c.table = cache.k, cache.v, (cache.k_params, cache.v_params), table
    past = 0
    for step in range(4):
        n = text if step == 0 else frame
        x, residual = normal(n, model).bfloat16(), normal(n, 256).bfloat16()
        qkv = awa_b200.qkv_project(x, w_in, gamma_q, gamma_k, 1e-5, heads)
        q, k, v = qkv.unbind(1)  # views: rows 3 * heads * d apart
        i = torch.arange(n, device="cuda", dtype=torch.int32)
        coords = torch.stack([i, i, i] if step == 0 else [0 * i + text + step, i // 8, i % 8], 1).contiguous()
        batch = awa_b200.CacheBatch(torch.tensor([0, n], dtype=torch.int32, device="cuda"),
                                    torch.tensor([past], dtype=torch.int32, device="cuda"), table, n, n)
        turned = cache.append(batch, k, v, q=q, rope=awa_b200.CacheRope(angles, coords))
        assert torch.equal(turned, rotate(q, angles, coords).bfloat16())
        out = cache.attention(batch, turned, sinks=text, window=2, frame_tokens=frame)
        got = awa_b200.out_project(out.flatten(1), w_out, bias, gate, residual)
        awa_b200.device_status()
        c.rows, c.past, c.first, c.total = [n], [past], [0, n], n
        if storage == "int4":
            want, tol = four_bit_attention(c, turned, text, 2, frame, d ** -0.5, n * 1 > 32)
        else:
            want, tol = attention(c, turned, text, 2, frame, d ** -0.5)
        assert ((out.double() - want).abs() <= tol).all(), step
        # the projection of these rows: products exact in fp32, sums of heads * d of them, two
        # roundings to bf16 (product, output) of up to 2^-8 each
        y = out.flatten(1).double() @ w_out.double().T + bias
        size = out.flatten(1).double().abs() @ w_out.double().abs().T + bias.abs()
        final = residual.double() + y * gate
        bound = gate.abs() * (2.0 ** -8 * y.abs() + heads * d * 2.0 ** -23 * size) + 2.0 ** -8 * final.abs()
        bound += 2.0 ** -22 * (residual.double().abs() + (y * gate).abs()) + 2.0 ** -8 * bound
        assert ((got.double() - final).abs() <= bound).all(), step
        past += n


@pytest.mark.parametrize("storage", ["bf16", "f32", "int4"])
@pytest.mark.parametrize("rows", [[1, 2], [70, 0, 45]])
def test_rows_ahead_of_the_first_sequence(rows, storage):
    """row_starts that begin behind 0: the rows before belong to nobody, as those behind the last."""
    dtype = torch.float32 if storage == "f32" else torch.bfloat16
    c = Batch(rows, [60] * len(rows), 16, 2, 128, storage, seed=36)
    ahead, behind, n = 5, 4, sum(rows)
    c.starts += ahead
    q, k, v = (torch.full((ahead + n + behind, h, 128), float("nan"), device="cuda").to(dtype) for h in (4, 2, 2))
    for t in (q, k, v):
        t[ahead:ahead + n] = torch.randn(n, t.shape[1], 128, generator=c.generator).to(dtype)
    cache = awa_b200.KvCache(c.k, c.v, *c.params)
    batch = awa_b200.CacheBatch(c.starts, c.past_t, c.table, ahead + n + behind, max(rows))
    table = awa_b200.rope_table(200, 64)
    turned = torch.full_like(q, 7.0)
    cache.append(batch, k, v, q=q, rope=awa_b200.CacheRope(table), q_out=turned)
    out = torch.full_like(q, 5.0)
    cache.attention(batch, turned, sinks=3, window=50, out=out)
    awa_b200.device_status()
    pos = torch.cat([60 + torch.arange(m) for m in rows]).cuda()[:, None]
    mine = slice(ahead, ahead + n)
    assert torch.equal(turned[mine], rotate(q[mine], table, pos).to(dtype))
    for t, kept in ((turned, 7.0), (out, 5.0)):
        assert (t[:ahead] == kept).all() and (t[ahead + n:] == kept).all()
    if storage == "int4":
        want, tol = four_bit_attention(c, turned[mine], 3, 50, 1, 128 ** -0.5, max(rows) * 2 > 32)
    else:
        want, tol = attention(c, turned[mine], 3, 50, 1, 128 ** -0.5)
    assert ((out[mine].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("storage", ["bf16", "f32", "int4"])
@pytest.mark.parametrize("most", [1, 100])
@pytest.mark.parametrize("rows,sequences", [(0, 0), (0, 2), (4, 0), (4, 2)])
def test_batches_without_work(rows, sequences, most, storage):
    dtype = torch.float32 if storage == "f32" else torch.bfloat16
    cache = awa_b200.KvCache.empty(4, 16, 2, 64, storage)
    for t in (cache.k, cache.v):
        t.zero_()
    ints = dict(dtype=torch.int32, device="cuda")
    batch = awa_b200.CacheBatch(torch.zeros(sequences + 1, **ints), torch.zeros(sequences, **ints),
                                torch.full((sequences, 3), -1, **ints), rows, most)
    q, k, v = (torch.ones(rows, h, 64, device="cuda").to(dtype) for h in (4, 2, 2))
    out = torch.full_like(q, 3.0)
    turned = cache.append(batch, k, v, q=q, q_out=out.clone())
    assert cache.attention(batch, q, out=out) is out
    cache.read(batch)
    awa_b200.device_status()
    assert (out == 3.0).all() and (turned == 3.0).all() and not cache.k.any() and not cache.v.any()


@pytest.mark.parametrize("storage", ["bf16", "f32", "int4"])
@pytest.mark.parametrize("rows", [1, 9, 150])
def test_lengths_that_change_behind_a_call(rows, storage):
    """The next step's lengths and rows are written right behind the call, on its stream:
    kernels that start early must not take them, nor later ones miss them."""
    dtype = torch.float32 if storage == "f32" else torch.bfloat16
    c = Batch([rows] * 3, [9000, 4000, 6000], 64, 2, 128, storage, seed=37)
    for t in ((c.k, c.v) if storage != "int4" else c.params):
        t.nan_to_num_(0.25)
    cache, batch = c.handles(awa_b200)
    q = c.new_rows(8, dtype)
    pasts = [torch.tensor(p, dtype=torch.int32, device="cuda") for p in
             ([9000, 4000, 6000], [10, 500, 5900], [8000, 0, 77])]  # within the pages that each has
    rowss = [q.clone(), q.flip(0).contiguous(), (0.5 * q)]
    want = []
    for p, x in zip(pasts, rowss):
        c.past_t.copy_(p)
        q.copy_(x)
        want.append(cache.attention(batch, q, sinks=4))
        torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for p, x in zip(pasts, rowss):
            c.past_t.copy_(p)
            q.copy_(x)
            got.append(cache.attention(batch, q, sinks=4))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    awa_b200.device_status()


@pytest.mark.parametrize("window", [0, 60])
@pytest.mark.parametrize("storage", ["bf16", "f32", "int4"])
def test_many_rows_with_a_page_that_is_not_there(storage, window):
    """Its rows are zeros to the attention, keys and values, and are reported."""
    dtype = torch.float32 if storage == "f32" else torch.bfloat16
    c = Batch([90], [200], 16, 2, 64, storage, seed=38)
    real = c.table[0, 14].item()
    c.table[0, 14] = -5
    cache, batch = c.handles(awa_b200)
    q = c.new_rows(8, dtype)
    got = cache.attention(batch, q, sinks=4, window=window)
    with pytest.raises(awa_b200.AwaError, match="71"):
        awa_b200.device_status()
    c.table[0, 14] = real
    for t in ((c.k, c.v) if storage != "int4" else c.params):
        t[real] = 0
    if storage == "int4":
        want, tol = four_bit_attention(c, q, 4, window, 1, 64 ** -0.5, True)
    else:
        want, tol = attention(c, q, 4, window, 1, 64 ** -0.5)
    assert ((got.double() - want).abs() <= tol).all()
