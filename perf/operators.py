"""The operators of the 8-bit paged K/V cache, as cases that can be timed.

- "append": new tokens' keys (rotated to their positions) and values into the
  pages, the queries rotated on the way; then the tokens of the touched pages
  read back as floats, which is what the pages hold;
- "decode": attention of one query row per sequence over its pages;
- "prefill": causal attention of packed rows, `count` new ones per sequence
  behind `used` tokens that were there before.

A page is `bt` tokens of one layer. Per KV head it holds a byte per element
and a power of two, its scale, for keys and one for values. Bytes stand for
byte - 128 ("int8") or for an E4M3 number ("e4m3"). Order of a head's bytes:
tiles of 16 tokens; in a tile keys are [dim/16][slot][16 dims] and values
[dim/64][slot/4][dim%16][dim%64/16][slot%4].
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _case(name, kind, dtype, fmt, shape, bt, sequences, used, count, rot=0, interleaved=False):
    """shape: (heads, kv_heads, dim); used and count: (smallest, largest) tokens of a sequence before the call and
    in it."""
    return dict(name=name, kind=kind, dtype=dtype, fmt=fmt, heads=shape[0], kv_heads=shape[1], dim=shape[2], bt=bt,
                sequences=sequences, used_low=used[0], used_high=used[1], count_low=count[0], count_high=count[1],
                rot=rot, interleaved=interleaved)


SMALL = (9, 3, 64)    # the SmolLM2-135M layer
WIDE = (32, 8, 128)   # a layer of a model of several billion parameters


def listed():
    return [
        # One user chatting: the next token's K/V. A call's latency.
        _case("append_1", "append", "f32", "int8", SMALL, 16, 1, (190, 190), (1, 1), 64),
        # A server's decode step: 64 ragged sequences, most in the middle of a page.
        _case("append_64", "append", "f32", "int8", SMALL, 16, 64, (255, 2174), (1, 1), 64),
        # Eight chunks of long documents that prefill together.
        _case("append_8x512", "append", "f32", "int8", SMALL, 16, 8, (8192, 8192), (512, 512), 64),
        # Whole prompts of different lengths in one batch of a wider model, half of the head rotated.
        _case("append_prompts", "append", "bf16", "e4m3", WIDE, 64, 16, (0, 0), (100, 2000), 64, True),
        # The single attention operation at its usual size, one row of 503 tokens: a call's latency.
        _case("decode_1x503", "decode", "f32", "int8", SMALL, 16, 1, (502, 502), (1, 1)),
        # A server's decode step: 64 ragged sequences.
        _case("decode_64", "decode", "f32", "int8", SMALL, 16, 64, (255, 2174), (1, 1)),
        # Eight long documents decoding together.
        _case("decode_8_long", "decode", "f32", "int8", SMALL, 16, 8, (14336, 16638), (1, 1)),
        # The widest batch, 256 sequences of about a thousand tokens, in a wider model.
        _case("decode_256_wide", "decode", "bf16", "e4m3", WIDE, 64, 256, (1023, 1086), (1, 1)),
        # One request's prompt chunk while nothing else runs: time to the first token.
        _case("prefill_1x256", "prefill", "f32", "int8", SMALL, 16, 1, (768, 768), (256, 256)),
        # The ragged last chunks of three prompts.
        _case("prefill_3x61", "prefill", "f32", "e4m3", SMALL, 16, 3, (1003, 1013), (37, 61)),
        # Long prompts prefilling together, in the middle of 16k tokens.
        _case("prefill_8x512", "prefill", "f32", "int8", SMALL, 16, 8, (8192, 8192), (512, 512)),
        # Whole prompts of different lengths, packed, in a wider model.
        _case("prefill_prompts", "prefill", "bf16", "e4m3", WIDE, 64, 16, (0, 0), (100, 2000)),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _drawn(rng):
    heads = rng.choice([(1, 1), (3, 3), (4, 1), (6, 2), (8, 1), (9, 3), (12, 4), (16, 1), (16, 4), (24, 8), (32, 8)])
    shape = (*heads, rng.choice([64, 64, 128]))
    dtype, fmt, bt = rng.choice(["f32", "f32", "bf16", "f16"]), rng.choice(["int8", "e4m3"]), rng.choice([16, 32, 64])
    pick = rng.random()
    if pick < 0.3:
        rot = rng.choice([0, 16, 32, 64, shape[2]])
        if rng.random() < 0.4:  # decoding sequences
            low, high = sorted((rng.randint(0, 4000), rng.randint(0, 16000)))
            return _case("", "append", dtype, fmt, shape, bt, _log(rng, 1, 256), (low, high), (1, 1), rot,
                         rng.random() < 0.5)
        longest = _log(rng, 2, 2000)
        low, high = (0, 0) if rng.random() < 0.5 else sorted((rng.randint(0, 4000), rng.randint(0, 16000)))
        return _case("", "append", dtype, fmt, shape, bt, _log(rng, 1, 16), (low, high),
                     (max(1, int(longest * rng.uniform(0.1, 1))), longest), rot, rng.random() < 0.5)
    if pick < 0.65:
        longest = _log(rng, 1, 16640)
        sequences = _log(rng, 1, 256)
        return _case("", "decode", dtype, fmt, shape, bt, sequences,
                     (int((longest - 1) * rng.uniform(0.1, 1)), longest - 1), (1, 1))
    longest = _log(rng, 2, 2000)
    low, high = (0, 0) if rng.random() < 0.5 else sorted((rng.randint(0, 4000), rng.randint(0, 8192)))
    return _case("", "prefill", dtype, fmt, shape, bt, _log(rng, 1, 16), (low, high),
                 (max(1, int(longest * rng.uniform(0.1, 1))), longest))


def draw(rng):
    largest = {}
    for case in listed():
        w = work(case)
        for key in w:
            kind = (case["kind"], key)
            largest[kind] = max(largest.get(kind, 0), w[key])
    while True:
        case = _drawn(rng)
        w = work(case)
        sequences, _, _ = _ranges(case)
        most = max(u + c for u, c in sequences)
        # The plain form's padded scores stay below those of the largest listed case.
        padded = len(sequences) * case["heads"] * case["count_high"] * most
        if all(w[key] <= largest[case["kind"], key] for key in w) and \
                (case["kind"] == "append" or padded <= 16 * 32 * 2000 * 2000):
            del case["name"]
            return case


def _spread(low, high, n):
    """n whole numbers over [low, high], in an order that is not sorted; the first n has both ends among them."""
    if n == 1:
        return [high]
    order = sorted(range(n), key=lambda i: (0.5 + 0.6180339887 * i) % 1.0)
    return [low + (high - low) * order[i] // (n - 1) for i in range(n)]


def _ranges(case):
    """[(used, count)] of the sequences, all rows, all tokens attended or held."""
    n = case["sequences"]
    used = _spread(case["used_low"], case["used_high"], n)
    count = _spread(case["count_low"], case["count_high"], n)[::-1]
    return list(zip(used, count)), sum(count), sum(u + c for u, c in zip(used, count))


def work(case):
    sequences, rows, held = _ranges(case)
    size = 4 if case["dtype"] == "f32" else 2
    heads, kv_heads, dim, bt = case["heads"], case["kv_heads"], case["dim"], case["bt"]
    if case["kind"] == "append":
        # Reads q, k, v and the rotations, writes q, the new tokens' bytes and the floats that are read back.
        back = sum(u % bt + c for u, c in sequences)
        elements = rows * (2 * heads + 2 * kv_heads) * dim + back * 2 * kv_heads * dim
        return {"bytes": size * elements + rows * (2 * kv_heads * dim + 4 * case["rot"]),
                "flops": 3 * rows * (heads + kv_heads) * case["rot"] + 2 * rows * kv_heads * dim * 2}
    pages = sum(-(-(u + c) // bt) for u, c in sequences)
    attended = sum(c * u + c * (c + 1) // 2 for u, c in sequences)
    return {"bytes": held * 2 * kv_heads * dim + pages * (8 * kv_heads + 4) + 2 * size * rows * heads * dim,
            "flops": 4 * attended * heads * dim}


# ---- the cache in plain torch -------------------------------------------------


def _to_bytes(codes, fmt):
    """Whole codes or E4M3 values, as floats, to the bytes that hold them."""
    if fmt == "int8":
        return (codes + 128).to(torch.uint8)
    return codes.to(torch.float8_e4m3fn).view(torch.uint8)


def _to_codes(data, fmt):
    return data.float() - 128 if fmt == "int8" else data.view(torch.float8_e4m3fn).float()


def _key_order(x):
    """[..., bt, dim] to the page's key order [..., bt * dim]."""
    *lead, bt, dim = x.shape
    return x.reshape(*lead, bt // 16, 16, dim // 16, 16).transpose(-3, -2).reshape(*lead, bt * dim)


def _value_order(x):
    *lead, bt, dim = x.shape
    x = x.reshape(*lead, bt // 16, 4, 4, dim // 64, 4, 16)  # tile, slot/4, slot%4, dim/64, dim%64/16, dim%16
    n = len(lead)
    return x.permute(*range(n), n, n + 3, n + 1, n + 5, n + 4, n + 2).reshape(*lead, bt * dim)


def _natural_keys(x, bt, dim):
    """The page's key order [..., bt * dim] to [..., bt, dim]."""
    lead = x.shape[:-1]
    return x.reshape(*lead, bt // 16, dim // 16, 16, 16).transpose(-3, -2).reshape(*lead, bt, dim)


def _natural_values(x, bt, dim):
    lead = x.shape[:-1]
    n = len(lead)
    x = x.reshape(*lead, bt // 16, dim // 64, 4, 16, 4, 4)  # tile, dim/64, slot/4, dim%16, dim%64/16, slot%4
    return x.permute(*range(n), n, n + 2, n + 5, n + 1, n + 4, n + 3).reshape(*lead, bt, dim)


def _scale_of(amax, fmt):
    """The smallest power of two s, from 2^-126 on, with amax <= M s (M: 127 or 448)."""
    mantissa, exponent = torch.frexp(amax)
    top, bits = (0.9921875, 7) if fmt == "int8" else (0.875, 9)
    e = (exponent - bits + (mantissa > top).int()).clamp(min=-126)
    e = torch.where(amax > 0, e, torch.full_like(e, -126))
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _round(x, fmt):
    return x.round() if fmt == "int8" else x.to(torch.float8_e4m3fn).float()


# ---- the state before the call --------------------------------------------


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _pages(case, gen, blocks):
    """Filled pages [blocks, 1 layer, kv_heads, bytes] of keys and values, and their scales."""
    kv_heads, dim, bt, fmt = case["kv_heads"], case["dim"], case["bt"], case["fmt"]
    channel = torch.exp(0.5 * _normal(gen, kv_heads, 1, dim))
    keys = torch.empty((blocks, 1, kv_heads, bt * dim), dtype=torch.uint8, device="cuda")
    values = torch.empty_like(keys)
    scales = torch.empty((blocks, 1, kv_heads, 2), device="cuda")
    for first in range(0, blocks, 4096):  # in parts, so that the floats stay small
        n = min(4096, blocks - first)
        for i, (to, order, by) in enumerate(((keys, _key_order, channel), (values, _value_order, 0.5))):
            x = _normal(gen, n, kv_heads, bt, dim) * by
            s = _scale_of(x.abs().amax((-1, -2)), fmt)
            scales[first:first + n, 0, :, i] = s
            to[first:first + n, 0] = order(_to_bytes(_round(x / s[..., None, None], fmt), fmt))
    return keys, values, scales, channel


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * seed + 29)
    sequences, rows, _ = _ranges(case)
    n, bt, dtype = len(sequences), case["bt"], TYPES[case["dtype"]]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    used = torch.tensor([u for u, _ in sequences], dtype=torch.int32)
    count = torch.tensor([c for _, c in sequences], dtype=torch.int32)
    pages = [-(-(u + c) // bt) for u, c in sequences]
    # An append touches the last pages only: the others are left out of the pool, their entries name page 0.
    skip = [u // bt if case["kind"] == "append" else 0 for u, _ in sequences]
    stride = max(pages)
    need = sum(p - s for p, s in zip(pages, skip))
    blocks = 1 + need + need // 8
    order = torch.randperm(blocks - 1, generator=gen, device="cuda").to(torch.int32) + 1
    tables = torch.zeros((n, stride), dtype=torch.int32, device="cuda")
    at = 0
    for row, p, s in zip(tables, pages, skip):
        row[s:p] = order[at:at + p - s]
        at += p - s
    keys, values, scales, channel = _pages(case, gen, blocks)
    starts = torch.zeros(n + 1, dtype=torch.int32)
    starts[1:] = count.cumsum(0)
    qkv = _normal(gen, rows, heads + 2 * kv_heads, dim)
    qkv[:, heads:heads + kv_heads] *= channel[:, 0]
    qkv[:, heads + kv_heads:] *= 0.5
    qkv = qkv.to(dtype).view(rows, -1)
    state = dict(case=case, rows=rows, sequences=n, longest=max(u + c for u, c in sequences),
                 most=max(c for _, c in sequences), tables=tables, stride=stride, keys=keys, values=values,
                 scales=scales, starts=starts.cuda(), used=used.cuda(), lengths=(used + count).cuda(), qkv=qkv,
                 out=torch.empty((rows, heads * dim), dtype=dtype, device="cuda"))
    if case["kind"] == "append":
        half = max(1, case["rot"] // 2)
        angles = torch.arange(state["longest"], dtype=torch.float64, device="cuda")[:, None] * \
            100000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
        state |= {"cos": angles.cos().float(), "sin": angles.sin().float()}
        # Every token of the touched pages, for the reading back.
        from_page = used // bt * bt
        back = torch.zeros(n + 1, dtype=torch.int32)
        back[1:] = (used + count - from_page).cumsum(0)
        state |= {"back_starts": back.cuda(), "back_used": from_page.cuda(), "back_rows": int(back[-1])}
        for name in ("back_keys", "back_values"):
            state[name] = torch.empty((state["back_rows"], kv_heads * dim), dtype=dtype, device="cuda")
    if own:
        from tinyinfer_amd import backend as mp
        cache = mp.Kv8Cache(keys.data_ptr(), values.data_ptr(), scales.data_ptr(), blocks, 1, bt, kv_heads, dim,
                            mp.KV8_INT8 if case["fmt"] == "int8" else mp.KV8_E4M3)
        state["cache"] = cache
        state["type"] = {"f32": mp.TYPE_F32, "bf16": mp.TYPE_BF16, "f16": mp.TYPE_F16}[case["dtype"]]
        if case["kind"] == "append":
            state["rope"] = mp.Rope(state["cos"].data_ptr(), state["sin"].data_ptr(), state["longest"], case["rot"],
                                    int(case["interleaved"]))
        else:
            size = mp.kv8_attention_workspace(cache, rows, n, heads, state["longest"])
            state["workspace"] = torch.empty(max(1, size), dtype=torch.uint8, device="cuda")
            state["workspace_bytes"] = size
    return state


# ---- the calls --------------------------------------------------------------


def _run_own(state):
    from tinyinfer_amd import backend as mp
    case = state["case"]
    stream = torch.cuda.current_stream().cuda_stream
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    q, width = state["qkv"].data_ptr(), state["qkv"].shape[1]
    cache, kind, out = state["cache"], state["type"], state["out"].data_ptr()
    tables, stride = state["tables"].data_ptr(), state["stride"]
    if case["kind"] == "append":
        element = state["qkv"].element_size()
        k = q + heads * dim * element
        mp.kv8_append(cache, 0, k, width, k + kv_heads * dim * element, width, kind, tables, stride,
                      state["starts"].data_ptr(), state["used"].data_ptr(), state["sequences"], state["rows"],
                      rope=state["rope"], q=q, q_stride=width, q_out=out, q_out_stride=heads * dim, heads=heads,
                      stream=stream)
        mp.kv8_read(cache, 0, tables, stride, state["back_starts"].data_ptr(), state["back_used"].data_ptr(),
                    state["sequences"], state["back_rows"], kind, state["back_keys"].data_ptr(), kv_heads * dim,
                    state["back_values"].data_ptr(), kv_heads * dim, stream=stream)
        return {"q": state["out"], "keys": state["back_keys"], "values": state["back_values"]}
    scale = 1 / math.sqrt(dim)
    if case["kind"] == "decode":
        mp.kv8_attention_decode(cache, 0, q, width, kind, tables, stride, state["lengths"].data_ptr(), state["rows"],
                                heads, state["longest"], scale, out, heads * dim, state["workspace"].data_ptr(),
                                state["workspace_bytes"], stream=stream)
    else:
        mp.kv8_attention_prefill(cache, 0, q, width, kind, tables, stride, state["starts"].data_ptr(),
                                 state["used"].data_ptr(), state["sequences"], state["rows"], heads,
                                 state["longest"], scale, out, heads * dim, state["workspace"].data_ptr(),
                                 state["workspace_bytes"], stream=stream)
    return {"out": state["out"]}


def _places(starts, used, rows):
    """Sequence and position of every packed row."""
    row = torch.arange(rows, device="cuda")
    sequence = torch.searchsorted(starts[1:].long(), row, right=True)
    return sequence, used.long()[sequence] + row - starts.long()[sequence]


def _rotated(x, cos, sin, rot, interleaved):
    """x [rows, heads, dim] with its first `rot` dims rotated by cos and sin [rows, 1, rot/2]."""
    if not rot:
        return x
    turned, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned[..., :rot // 2], turned[..., rot // 2:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1)


def _append_plain(state):
    case = state["case"]
    heads, kv_heads, dim, bt, fmt = case["heads"], case["kv_heads"], case["dim"], case["bt"], case["fmt"]
    rows, dtype = state["rows"], state["qkv"].dtype
    sequence, position = _places(state["starts"], state["used"], rows)
    x = state["qkv"].view(rows, heads + 2 * kv_heads, dim).float()
    cos, sin = state["cos"][position][:, None], state["sin"][position][:, None]
    q = _rotated(x[:, :heads], cos, sin, case["rot"], case["interleaved"])
    k = _rotated(x[:, heads:heads + kv_heads], cos, sin, case["rot"], case["interleaved"])
    v = x[:, heads + kv_heads:]
    page, slot = state["tables"][sequence, position // bt].long(), position % bt
    blocks = state["keys"].shape[0]
    first = torch.full((blocks,), bt, device="cuda").scatter_reduce(0, page, slot, "amin")
    touched, old = (first < bt)[:, None], torch.arange(bt, device="cuda") < first[:, None]
    state["keys"][:, 0], state["scales"][:, 0, :, 0] = _page_plain(
        state["keys"][:, 0], state["scales"][:, 0, :, 0], k, page, slot, first, touched, old, fmt, _natural_keys,
        _key_order, bt, dim)
    state["values"][:, 0], state["scales"][:, 0, :, 1] = _page_plain(
        state["values"][:, 0], state["scales"][:, 0, :, 1], v, page, slot, first, touched, old, fmt, _natural_values,
        _value_order, bt, dim)
    sequence, position = _places(state["back_starts"], state["back_used"], state["back_rows"])
    page, slot = state["tables"][sequence, position // bt].long(), position % bt
    natural = (_natural_keys(state["keys"][:, 0], bt, dim), _natural_values(state["values"][:, 0], bt, dim))
    back = [(_to_codes(data.transpose(1, 2)[page, slot].contiguous(), fmt) * state["scales"][page, 0, :, i, None])
            for i, data in enumerate(natural)]
    return {"q": q.reshape(rows, -1).to(dtype), "keys": back[0].reshape(state["back_rows"], -1).to(dtype),
            "values": back[1].reshape(state["back_rows"], -1).to(dtype)}


def _page_plain(data, scales, x, page, slot, first, touched, old, fmt, natural, order, bt, dim):
    """Bytes and scales of the pages with the new rows x in them."""
    kv_heads = x.shape[1]
    amax = torch.zeros((data.shape[0], kv_heads), device="cuda").scatter_reduce(
        0, page[:, None].expand(-1, kv_heads), x.abs().amax(-1), "amax")
    held = torch.where((first > 0)[:, None], scales, torch.zeros_like(scales))
    scale = torch.where(touched, torch.maximum(held, _scale_of(amax, fmt)), scales)
    codes = _to_codes(natural(data, bt, dim).contiguous(), fmt)
    moved = _round(codes * (scales / scale)[..., None, None], fmt)
    codes = torch.where((old & touched)[:, None, :, None], moved, codes)
    codes.transpose(1, 2)[page, slot] = _round(x / scale[page][..., None], fmt)
    return order(_to_bytes(codes, fmt)), scale


def _attention_plain(state):
    case = state["case"]
    heads, kv_heads, dim, bt, fmt = case["heads"], case["kv_heads"], case["dim"], case["bt"], case["fmt"]
    rows, n, most, dtype = state["rows"], state["sequences"], state["most"], state["qkv"].dtype
    pages = state["tables"].long()
    scales = state["scales"][pages, 0]  # [sequence, page, head, 2]
    keys = _to_codes(_natural_keys(state["keys"][pages, 0], bt, dim).contiguous(), fmt) * scales[..., 0, None, None]
    values = _to_codes(_natural_values(state["values"][pages, 0], bt, dim).contiguous(), fmt) * \
        scales[..., 1, None, None]
    tokens = pages.shape[1] * bt
    keys = keys.permute(0, 2, 4, 1, 3).reshape(n, kv_heads, dim, tokens)
    values = values.permute(0, 2, 1, 3, 4).reshape(n, kv_heads, tokens, dim)
    # Rows padded to the longest sequence's count.
    starts, used = state["starts"].long(), state["used"].long()
    sequence, position = _places(starts, used, rows)
    inside = position - used[sequence]
    q = torch.zeros((n, most, heads * dim), device="cuda")
    q[sequence, inside] = state["qkv"][:, :heads * dim].float()
    group = heads // kv_heads
    q = q.view(n, most, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(n, kv_heads, group * most, dim)
    scores = torch.matmul(q * (1 / math.sqrt(dim)), keys).view(n, kv_heads, group, most, tokens)
    last = used[:, None] + torch.arange(most, device="cuda")
    hidden = torch.arange(tokens, device="cuda") > last[..., None]
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    scores.exp_()
    total = scores.sum(-1, keepdim=True)
    # Slots behind a row's length weigh nothing, and what they hold is finite.
    out = torch.matmul(scores.view(n, kv_heads, group * most, tokens), values).view(n, kv_heads, group, most, dim)
    out = (out / total).permute(0, 3, 1, 2, 4).reshape(n, most, heads * dim)
    return {"out": out[sequence, inside].to(dtype)}


def run(state):
    if own:
        return _run_own(state)
    return _append_plain(state) if state["case"]["kind"] == "append" else _attention_plain(state)


# ---- in 64 bits -----------------------------------------------------------


def _byte_values(fmt):
    if fmt == "int8":
        return torch.arange(256, dtype=torch.float64) - 128
    def e4m3(b):
        e, m = b >> 3 & 15, b & 7
        x = math.nan if e == 15 and m == 7 else m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        return -x if b & 128 else x
    return torch.tensor([e4m3(b) for b in range(256)], dtype=torch.float64)


def _byte_places(bt, dim):
    """Where in a head's bytes of a page the element (slot, dim) is, for keys and for values."""
    slot, d = torch.arange(bt)[:, None], torch.arange(dim)[None]
    tile, s = slot // 16 * 16 * dim, slot % 16
    return (tile + d // 16 * 256 + s * 16 + d % 16).cuda(), \
        (tile + d // 64 * 1024 + s // 4 * 256 + d % 16 * 16 + d % 64 // 16 * 4 + s % 4).cuda()


def _rotated64(x, position, rot, interleaved, cos, sin):
    out = x.clone()
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        c, s = cos[position, i][:, None], sin[position, i][:, None]
        out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return out


def _nearest64(x, fmt):
    """x rounded to the numbers a byte can hold, ties to even."""
    if fmt == "int8":
        return torch.round(x)
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -20))).clamp(min=-6)
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _power64(amax, fmt):
    top = 127.0 if fmt == "int8" else 448.0
    if amax == 0:
        return 2.0 ** -126
    e = math.floor(math.log2(amax / top)) - 1
    while amax > top * 2.0 ** e:
        e += 1
    return 2.0 ** max(e, -126)


def _append_exact(case, state):
    heads, kv_heads, dim, bt, fmt = case["heads"], case["kv_heads"], case["dim"], case["bt"], case["fmt"]
    sequences, rows, _ = _ranges(case)
    cos, sin = state["cos"].double(), state["sin"].double()
    x = state["qkv"].double().view(rows, -1, dim)
    position = torch.cat([torch.arange(u, u + c) for u, c in sequences]).cuda()
    turned = _rotated64(x[:, :heads + kv_heads], position, case["rot"], case["interleaved"], cos, sin)
    new = (turned[:, heads:], x[:, heads + kv_heads:])
    table, values = state["tables"].tolist(), _byte_values(fmt).cuda()
    scales = state["scales"].double()
    top = [[], []]
    spans = []
    row = 0
    for s, (u, c) in enumerate(sequences):
        p = u
        while p < u + c:
            n = min(u + c, p // bt * bt + bt) - p
            spans.append((table[s][p // bt], p % bt, n, row))
            row, p = row + n, p + n
    for i in range(2):
        top[i] = torch.stack([new[i][r:r + n].abs().amax((0, 2)) for _, _, n, r in spans]).tolist()
    back = ([], [])
    old_scales = scales[[b for b, _, _, _ in spans], 0].tolist()
    for i, (data, where) in enumerate(zip((state["keys"], state["values"]), _byte_places(bt, dim))):
        held = values[data[[b for b, _, _, _ in spans], 0].long()][:, :, where]  # [span, head, bt, dim]
        for j, (_, slot, n, r) in enumerate(spans):
            was = [old_scales[j][h][i] for h in range(kv_heads)]
            now = [max(was[h] if slot else 0.0, _power64(top[i][j][h], fmt)) for h in range(kv_heads)]
            was, now = (torch.tensor(t, dtype=torch.float64, device="cuda")[:, None, None] for t in (was, now))
            old = _nearest64(held[j, :, :slot] * (was / now), fmt) * now
            fresh = _nearest64(new[i][r:r + n].transpose(0, 1) / now, fmt) * now
            back[i].append(torch.cat((old, fresh), 1).transpose(0, 1).reshape(slot + n, -1))
    return {"q": turned[:, :heads].reshape(rows, -1), "keys": torch.cat(back[0]), "values": torch.cat(back[1])}


def _attention_exact(case, state):
    heads, kv_heads, dim, bt = case["heads"], case["kv_heads"], case["dim"], case["bt"]
    sequences, rows, _ = _ranges(case)
    table_of, (key_at, value_at) = _byte_values(case["fmt"]).cuda(), _byte_places(bt, dim)
    out = torch.empty((rows, kv_heads, heads // kv_heads, dim), dtype=torch.float64, device="cuda")
    q = state["qkv"][:, :heads * dim].double().view(rows, kv_heads, heads // kv_heads, dim)
    row = 0
    for s, (u, c) in enumerate(sequences):
        pages = state["tables"][s, :-(-(u + c) // bt)].long()
        scale = state["scales"][pages, 0].double()
        k = table_of[state["keys"][pages, 0].long()[:, :, key_at]] * scale[:, :, None, None, 0]
        v = table_of[state["values"][pages, 0].long()[:, :, value_at]] * scale[:, :, None, None, 1]
        k, v = (t.transpose(0, 1).reshape(kv_heads, -1, dim)[:, :u + c] for t in (k, v))
        later = torch.arange(u + c, device="cuda") > torch.arange(u, u + c, device="cuda")[:, None]
        for h in range(kv_heads):
            z = torch.matmul(q[row:row + c, h], k[h].T.contiguous()) / math.sqrt(dim)  # [row, group, token]
            z = torch.softmax(z.masked_fill(later[:, None], -math.inf), -1)
            out[row:row + c, h] = torch.matmul(z, v[h])
        row += c
    return {"out": out.view(rows, -1)}


def exact(case, seed):
    state = prepare(case, seed)
    return _append_exact(case, state) if case["kind"] == "append" else _attention_exact(case, state)
