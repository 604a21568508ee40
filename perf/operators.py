"""Workloads of the key/value cache operators: appending rotated rows to a paged
cache (f32, bf16 or 4 bits) and attention over it with a sliding window and a
prefix that stays visible.

``run`` computes one pass either in elementary torch operations or, with
``own``, through the library. Lengths of a case come from the case alone,
values and the order of the pages from the seed.
"""

import math
import os
import random
import sys

import torch

own = False

GROUP = 64  # features that share a scale and a minimum in a 4-bit cache


def listed():
    video = dict(q_heads=20, kv_heads=20, dim=128)  # the 3B model's heads
    return [
        # a frame-by-frame step of eight streams: one row each, launch latency
        dict(name="append_step_bf16", kind="append", storage="bf16", input="bf16", **video, sequences=8, rows_min=1,
             rows_max=1, past_min=100, past_max=5000, shape=1, page=64, axes=3, pairs=21),
        # the whole 21 x 64 x 64 latent clip with its 58 text rows into an empty cache
        dict(name="append_clip_bf16", kind="append", storage="bf16", input="bf16", **video, sequences=1,
             rows_min=86074, rows_max=86074, past_min=0, past_max=0, shape=2, page=64, axes=3, pairs=21),
        # an fp32 block's rows, ragged, grouped heads of 64 features, positions as coordinates
        dict(name="append_ragged_f32", kind="append", storage="f32", input="f32", q_heads=32, kv_heads=8, dim=64,
             sequences=7, rows_min=1, rows_max=1531, past_min=0, past_max=900, shape=3, page=16, axes=1, pairs=32),
        # prompts of several streams into a 4-bit cache, and the stored rows read back
        dict(name="append_ragged_int4", kind="append", storage="int4", input="bf16", q_heads=32, kv_heads=8, dim=128,
             sequences=16, rows_min=40, rows_max=2100, past_min=0, past_max=3000, shape=4, page=32, axes=1, pairs=64),
        # one new token of one short stream: latency alone
        dict(name="step_one_bf16", kind="attend", storage="bf16", **video, sequences=1, rows_min=1, rows_max=1,
             past_min=700, past_max=700, shape=5, page=64, sinks=58, window=0, frame=1),
        # a serving step: 64 streams of uneven length, grouped heads, window of 8192 tokens
        dict(name="step_batch_bf16", kind="attend", storage="bf16", q_heads=32, kv_heads=8, dim=128, sequences=64,
             rows_min=1, rows_max=1, past_min=500, past_max=32000, shape=6, page=64, sinks=4, window=8192, frame=1),
        # two 64 x 64 latent frames attend to five frames each and the text prefix
        dict(name="frames_bf16", kind="attend", storage="bf16", **video, sequences=1, rows_min=8192, rows_max=8192,
             past_min=20538, past_max=20538, shape=7, page=64, sinks=58, window=5, frame=4096),
        # prompts of uneven length (some of no rows), causal window of 1024 tokens, small pages
        dict(name="ragged_bf16", kind="attend", storage="bf16", q_heads=32, kv_heads=8, dim=128, sequences=12,
             rows_min=0, rows_max=1999, past_min=0, past_max=1500, shape=8, page=16, sinks=5, window=1024, frame=1),
        # heads of 64 features in groups of seven, plain causal attention
        dict(name="causal_d64_bf16", kind="attend", storage="bf16", q_heads=14, kv_heads=2, dim=64, sequences=3,
             rows_min=900, rows_max=4001, past_min=0, past_max=2000, shape=9, page=128, sinks=0, window=0, frame=1),
        # an fp32 block: two of the 16 x 16 latent frames over three frames and the text
        dict(name="frames_f32", kind="attend", storage="f32", **video, sequences=1, rows_min=512, rows_max=512,
             past_min=1082, past_max=1082, shape=10, page=64, sinks=58, window=3, frame=256),
        # a serving step over long 4-bit caches
        dict(name="step_batch_int4", kind="attend", storage="int4", q_heads=32, kv_heads=8, dim=128, sequences=32,
             rows_min=1, rows_max=1, past_min=4000, past_max=32700, shape=11, page=64, sinks=0, window=0, frame=1),
        # one 32 x 32 latent frame over a 4-bit cache of nine
        dict(name="frame_int4", kind="attend", storage="int4", **video, sequences=1, rows_min=1024, rows_max=1024,
             past_min=9274, past_max=9274, shape=12, page=64, sinks=58, window=9, frame=1024),
    ]


def spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["append", "step", "step", "rows", "rows", "rows"])
    kv_heads, group = rng.choice([(20, 1), (8, 4), (4, 8), (2, 7), (1, 16), (5, 3), (10, 2)])
    case = dict(kind="append" if kind == "append" else "attend", storage=rng.choice(["bf16", "bf16", "int4", "f32"]),
                q_heads=kv_heads * group, kv_heads=kv_heads, dim=rng.choice([128, 128, 64]),
                shape=rng.randrange(1 << 30), page=rng.choice([16, 32, 64, 128]))
    if kind == "append":
        rows = spread(rng, 1, 20000)
        case.update(input="f32" if case["storage"] == "f32" else rng.choice(["bf16", "f32"]),
                    sequences=rng.randint(1, max(1, min(32, 30000 // rows))), rows_min=rng.choice([0, 1, rows]),
                    rows_max=rows, past_min=0, past_max=spread(rng, 1, 3000))
        axes = rng.choice([1, 3])
        case.update(axes=axes, pairs=case["dim"] // 2 // axes)
    elif kind == "step":
        past = spread(rng, 1, 32000)
        rows = rng.choice([1, 1, 1, 2, 4])
        case.update(sequences=spread(rng, 1, max(2, min(64, 120000 // past))), rows_min=rng.choice([0, rows]),
                    rows_max=rows, past_min=max(1, past // 8), past_max=past)
    else:
        rows, past = spread(rng, 5, 3000), spread(rng, 1, 12000)
        most = 1 if case["storage"] == "f32" else 6
        rows = min(rows, 700) if case["storage"] == "f32" else rows
        past = min(past, 2500) if case["storage"] == "f32" else past
        scores = case["q_heads"] * rows * (rows + past)
        case.update(sequences=rng.randint(1, max(1, min(most, int(1.5e9 // scores)))), rows_min=rng.choice([0, 1, rows]),
                    rows_max=rows, past_min=rng.choice([0, past]), past_max=past)
    if case["kind"] == "attend":
        frame = rng.choice([1, 1, 1, spread(rng, 2, 1100)])
        case.update(sinks=rng.choice([0, 4, rng.randint(1, 130)]), frame=frame,
                    window=rng.choice([0, spread(rng, 1, 9000) if frame == 1 else rng.randint(1, 9)]))
    return case


def lengths(case):
    """(rows, past) of each sequence; the first is the longest."""
    r = random.Random(case["shape"])

    def lens(low, high):
        got = [high] + [spread(r, max(low, 1), max(high, 1)) for _ in range(case["sequences"] - 1)]
        if low == 0 and case["sequences"] > 2:
            got[-1] = 0
        return [min(n, high) for n in got]

    return lens(case["rows_min"], case["rows_max"]), lens(case["past_min"], case["past_max"])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, past = lengths(case)
    d, page, kv, heads = case["dim"], case["page"], case["kv_heads"], case["q_heads"]
    bf16 = torch.bfloat16
    used = [-(-(n + p) // page) for n, p in zip(rows, past)]
    pages, width, total = sum(used) + 3, max(used), sum(rows)
    order = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
    table = torch.full((len(rows), width), -1, dtype=torch.int32, device="cuda")
    begin = 0
    for b, n in enumerate(used):
        table[b, :n] = order[begin:begin + n]
        begin += n
    starts = [0]
    for n in rows:
        starts.append(starts[-1] + n)
    ints = dict(dtype=torch.int32, device="cuda")
    state = dict(case=case, table=table, starts=torch.tensor(starts, **ints), past=torch.tensor(past, **ints),
                 sequence=torch.repeat_interleave(torch.arange(len(rows), device="cuda"),
                                                  torch.tensor(rows, device="cuda")))
    state["index"] = torch.arange(total, device="cuda") - state["starts"][state["sequence"]]

    def normal(*shape, dtype):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    shape = (pages, kv, page)
    if case["storage"] == "int4":
        for name in ("k", "v"):
            state[name] = torch.randint(0, 256, shape + (d // 2,), generator=g, device="cuda", dtype=torch.uint8)
            scale = 0.2 + 0.1 * torch.rand(shape + (d // GROUP,), generator=g, device="cuda")
            state[name + "_params"] = torch.stack([scale, -7.5 * scale], -1).to(bf16)
    else:
        dtype = bf16 if case["storage"] == "bf16" else torch.float32
        state.update(k=normal(*shape, d, dtype=dtype), v=normal(*shape, d, dtype=dtype))
    if case["kind"] == "append":
        dtype = bf16 if case["input"] == "bf16" else torch.float32
        qkv = normal(total, heads + 2 * kv, d, dtype=dtype)  # one row per token, as a projection writes it
        state.update(new_q=qkv[:, :heads], new_k=qkv[:, heads:heads + kv], new_v=qkv[:, heads + kv:])
        if case["axes"] == 1:
            most, coords = max(n + p for n, p in zip(rows, past)), None
        else:  # (t, h, w) of a clip behind 58 text rows
            most, at = 160, state["past"].long()[state["sequence"]] + state["index"] - 58
            t = 58 + torch.clamp(at, min=0) // 4096 % 100
            coords = torch.stack([t, at % 4096 // 64, at % 64], 1)
            coords = torch.where(at[:, None] < 0, (at + 58)[:, None], coords).to(torch.int32).contiguous()
        angle = torch.arange(most, dtype=torch.float64, device="cuda")[:, None] * torch.pow(
            10000.0, -torch.arange(case["pairs"], dtype=torch.float64, device="cuda") / case["pairs"])
        state.update(rope=torch.stack([angle.cos(), angle.sin()], -1).float().contiguous(), coords=coords)
    else:
        state["q"] = 2 * normal(total, heads, d, dtype=torch.float32 if case["storage"] == "f32" else bf16)
    if own:
        keep_handles(state, total, max(rows))
    return state


def keep_handles(state, rows, max_rows):
    package = os.path.join(os.getcwd(), "seedvr2-ncnn_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import awa_b200

    state["cache"] = awa_b200.KvCache(state["k"], state["v"], state.get("k_params"), state.get("v_params"))
    state["batch"] = awa_b200.CacheBatch(state["starts"], state["past"], state["table"], rows, max_rows)
    if state["case"]["kind"] == "append":
        state["rotation"] = awa_b200.CacheRope(state["rope"], state["coords"])


def run(state):
    case = state["case"]
    if not own:
        return plain_append(state) if case["kind"] == "append" else plain_attention(state)
    cache, batch = state["cache"], state["batch"]
    if case["kind"] == "attend":
        return cache.attention(batch, state["q"], sinks=case["sinks"], window=case["window"],
                               frame_tokens=case["frame"])
    q = cache.append(batch, state["new_k"], state["new_v"], q=state["new_q"], rope=state["rotation"])
    if case["storage"] != "int4":
        return {"q": q, "k": state["k"], "v": state["v"]}
    k, v = cache.read(batch, torch.float32)
    return {"q": q, "k": k, "v": v}


def slots(state):
    """(page, slot) of each new row."""
    at = state["past"].long()[state["sequence"]] + state["index"]
    page = state["case"]["page"]
    return state["table"].long()[state["sequence"], at // page], at % page


def rotate(state, x):
    case = state["case"]
    if state["coords"] is None:
        coords = (state["past"].long()[state["sequence"]] + state["index"])[:, None]
    else:
        coords = state["coords"].long()
    cos, sin = state["rope"][coords].flatten(1, 2)[:, None].unbind(-1)  # [rows, 1, axes * pairs]
    x = x.float()
    n = 2 * cos.shape[-1]
    x0, x1 = x[..., 0:n:2], x[..., 1:n:2]
    turned = torch.stack([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1).flatten(-2)
    return torch.cat([turned, x[..., n:]], -1)


def to_bf16(x, up):
    """x rounded to bf16 towards +inf or -inf."""
    bits = x.view(torch.int32)
    cut = bits & -65536
    away = (bits != cut) & ((bits >= 0) if up else (bits < 0))
    return (cut + away.to(torch.int32) * 65536).view(torch.float32)


def quantize(x):
    """(codes, scale, minimum) of the groups of 64 features."""
    x = x.unflatten(-1, (-1, GROUP))
    low = to_bf16(x.amin(-1), up=False)
    fifteen = torch.full_like(low, 15)  # by a tensor: division by a number may multiply by its reciprocal
    scale = to_bf16((x.amax(-1) - low) / fifteen, up=True)
    inverse = torch.where(scale > 0, 1 / scale, torch.zeros_like(scale))
    codes = torch.round((x - low[..., None]) * inverse[..., None]).clamp(0, 15)
    return codes.flatten(-2).to(torch.uint8), scale, low


def plain_append(state):
    page, slot = slots(state)
    q, k, v = rotate(state, state["new_q"]), rotate(state, state["new_k"]), state["new_v"].float()
    q = q.to(state["new_q"].dtype)
    if state["case"]["storage"] != "int4":
        state["k"][page, :, slot] = k.to(state["k"].dtype)
        state["v"][page, :, slot] = v.to(state["v"].dtype)
        return {"q": q, "k": state["k"], "v": state["v"]}
    back = {"q": q}
    for name, x in (("k", k), ("v", v)):
        codes, scale, low = quantize(x)
        state[name][page, :, slot] = codes[..., 0::2] | codes[..., 1::2] << 4
        state[name + "_params"][page, :, slot] = torch.stack([scale, low], -1).to(torch.bfloat16)
        back[name] = values(state[name][page, :, slot], state[name + "_params"][page, :, slot])
    return back


def values(packed, params):
    """What 4-bit rows stand for."""
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).float().unflatten(-1, (-1, GROUP))
    scale, low = params.float()[..., None].unbind(-2)
    return (scale * codes + low).flatten(-2)


def gather(state, name):
    """The cached rows of every sequence in order, [sequences, heads, longest, dim] in f32."""
    page, table = state["case"]["page"], state["table"].long().clamp(min=0)
    rows = state[name][table]
    rows = values(rows, state[name + "_params"][table]) if state["case"]["storage"] == "int4" else rows.float()
    return rows.transpose(1, 2).flatten(2, 3)


def plain_attention(state):
    case = state["case"]
    kv, group, d = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["dim"]
    sinks, window, frame = case["sinks"], case["window"], case["frame"]
    starts, past = state["starts"].long(), state["past"].long()
    rows = starts[1:] - starts[:-1]
    i = torch.arange(case["rows_max"], device="cuda")
    at = (starts[:-1, None] + i).clamp(max=max(0, state["q"].shape[0] - 1))
    q = state["q"][at].float().unflatten(2, (kv, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    k, v = gather(state, "k"), gather(state, "v")
    scores = (q * (1 / math.sqrt(d))) @ k.transpose(2, 3)
    scores = scores.unflatten(2, (group, -1))
    p = past[:, None, None] + i[:, None]
    length = (past + rows)[:, None, None]
    j = torch.arange(k.shape[2], device="cuda")
    f = (p - sinks).clamp(min=0) // frame
    high = torch.where(p < sinks, ((p // frame + 1) * frame).clamp(max=sinks), sinks + (f + 1) * frame)
    low = sinks + (f - window + 1).clamp(min=0) * frame if window > 0 else torch.zeros_like(f)
    seen = (j < torch.minimum(high, length)) & ((j >= low) | (j < sinks))
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True).clamp(min=-1e30)
    scores.exp_()
    total = scores.sum(-1)
    out = (scores.flatten(2, 3) @ v).unflatten(2, (group, -1)) / total[..., None]
    out = out.permute(0, 3, 1, 2, 4).flatten(2, 3)
    return out[state["sequence"], state["index"]].to(state["q"].dtype)


def work(case):
    rows, past = lengths(case)
    d, kv, heads = case["dim"], case["kv_heads"], case["q_heads"]
    size = {"bf16": 2.0, "f32": 4.0, "int4": 0.5 + 4.0 / GROUP}[case["storage"]]
    if case["kind"] == "append":
        n, e = sum(rows), 2 if case["input"] == "bf16" else 4
        moved = n * d * (2 * heads * e + 2 * kv * (e + size))
        if case["storage"] == "int4":
            moved += n * d * 2 * kv * (size + 4)
        return {"bytes": moved, "flops": 3 * n * (heads + kv) * case["axes"] * case["pairs"] * 2}
    pairs, read = 0, 0
    for n, p in zip(rows, past):
        spans = [span(case, p + i, p + n) for i in range(n)]
        pairs += sum(high - low + min(case["sinks"], low) for low, high in spans)
        if n:  # every token that some row sees
            low, high = min(s[0] for s in spans), max(s[1] for s in spans)
            read += high - low + min(case["sinks"], low)
    e = 4 if case["storage"] == "f32" else 2
    return {"bytes": 2 * sum(rows) * heads * d * e + 2 * read * kv * d * size, "flops": 4.0 * pairs * heads * d}


def span(case, p, length):
    """[low, high) of the window that the row at position p sees (the prefix apart)."""
    sinks, frame = case["sinks"], case["frame"]
    if p < sinks:
        return 0, min(sinks, (p // frame + 1) * frame, length)
    f = (p - sinks) // frame
    low = sinks + max(0, f - case["window"] + 1) * frame if case["window"] else 0
    return low, min(length, sinks + (f + 1) * frame)


def exact(case, seed):
    """The operators' definition row by row in float64: sequence after sequence and head after head."""
    s = prepare(case, seed)
    return exact_append(s) if case["kind"] == "append" else exact_attention(s)


def exact_values(s, name, page, slot):
    """Stored rows [n, heads, dim] in float64."""
    x = s[name][page, :, slot]
    if s["case"]["storage"] != "int4":
        return x.double()
    out = torch.empty(x.shape[:-1] + (s["case"]["dim"],), dtype=torch.float64, device="cuda")
    out[..., 0::2], out[..., 1::2] = (x % 16).double(), (x // 16).double()
    par = s[name + "_params"][page, :, slot].double()
    return par[..., 1].repeat_interleave(GROUP, -1) + out * par[..., 0].repeat_interleave(GROUP, -1)


def exact_append(s):
    case = s["case"]
    rows, past = lengths(case)
    out = {"q": torch.empty(s["new_q"].shape, dtype=torch.float64, device="cuda")}
    pages = {n: s[n].double() for n in ("k", "v")} if case["storage"] != "int4" else None
    if pages is None:
        out.update({n: torch.empty(s["new_" + n].shape, dtype=torch.float64, device="cuda") for n in ("k", "v")})
    first = 0
    for b, (n, p) in enumerate(zip(rows, past)):
        at = p + torch.arange(n, device="cuda")
        r = slice(first, first + n)
        first += n
        where = at[:, None] if s["coords"] is None else s["coords"][r].long()
        new = {}
        for name in ("q", "k", "v"):
            # products and sums round to f32 by definition: both are exact in f64 before that rounding
            x = s["new_" + name][r].double().clone()
            for a in range(case["axes"] if name != "v" else 0):
                cs = s["rope"][where[:, a]].double()[:, None]
                f = 2 * (a * case["pairs"] + torch.arange(case["pairs"], device="cuda"))
                x0, x1 = x[..., f].clone(), x[..., f + 1].clone()
                c, t = cs[..., 0], cs[..., 1]
                x[..., f] = ((x0 * c).float().double() - (x1 * t).float().double()).float().double()
                x[..., f + 1] = ((x1 * c).float().double() + (x0 * t).float().double()).float().double()
            new[name] = x
        out["q"][r] = new["q"]
        page, slot = s["table"][b].long()[at // case["page"]], at % case["page"]
        for name in ("k", "v"):
            if pages is not None:
                pages[name][page, :, slot] = new[name]
            else:
                out[name][r] = exact_codes(new[name])
    return out if pages is None else {**out, **pages}


def exact_codes(x):
    """The nearest of the 16 values that a group's minimum and scale allow, roundings as defined."""
    x = x.unflatten(-1, (-1, GROUP))

    def bf16(y, up):  # the next bf16 value at or beyond y
        near = y.bfloat16().double()
        wrong = near < y if up else near > y
        step = torch.exp2(torch.floor(torch.log2(near.abs().clamp(min=1e-38))) - 7)
        # one step of the binade below where the magnitude falls to a power of two
        step = torch.where((near.abs() == torch.exp2(torch.round(torch.log2(near.abs().clamp(min=1e-38))))) &
                           ((near > 0) != up), step / 2, step)
        return torch.where(wrong, near + (step if up else -step), near)

    low = bf16(x.amin(-1), False)[..., None]
    scale = bf16(((x.amax(-1)[..., None] - low).float().double() / 15).float().double(), True)
    inverse = (1 / scale).float().double()
    code = ((x - low).float().double() * inverse).float().double().round().clamp(0, 15)
    return torch.where(scale > 0, low + scale * code, low.expand_as(code)).flatten(-2)


def exact_attention(s):
    case = s["case"]
    rows, past = lengths(case)
    group = case["q_heads"] // case["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for b, (n, p) in enumerate(zip(rows, past)):
        j = torch.arange(n + p, device="cuda")
        page, slot = s["table"][b].long()[j // case["page"]], j % case["page"]
        k, v = (exact_values(s, name, page, slot) for name in ("k", "v"))
        for r in range(0, n, 2048):
            m = min(2048, n - r)
            spans = torch.tensor([span(case, p + r + i, p + n) for i in range(m)], device="cuda")
            hidden = (j >= spans[:, 1:]) | ((j < spans[:, :1]) & (j >= case["sinks"]))
            for h in range(case["q_heads"]):
                z = s["q"][first + r:first + r + m, h].double() @ k[:, h // group].T / case["dim"] ** 0.5
                z.masked_fill_(hidden, -math.inf)
                out[first + r:first + r + m, h] = torch.softmax(z, -1) @ v[:, h // group]
        first += n
    return out
