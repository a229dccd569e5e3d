"""The operators of a model with 4-bit weights, as cases that can be timed.

- "pack": a weight matrix to 4 bits, and its rows read back as floats, which is what the codes stand for;
- "norm": root-mean-square norm of rows with the residual's addition, to floats or to rows of 8 bits;
- "convert": rows of floats to rows of 8 bits and back;
- "product": rows of floats or of 8 bits times a 4-bit matrix, alone or as the gated pair silu(x G^T) * (x W^T).

A 4-bit weight is an E2M1 number times the power of two of its group, 32 weights along a row. An element of an 8-bit
row is a whole number, -127 to 127, times the power of two of its group of 32. A scale byte b stands for 2^(b - 127):
the smallest power, from 2^-100 on, with which the group's largest magnitude is in range (6 and 127).

Order of a matrix's bytes: codes by tiles of 16 rows and 128 columns, [rows/16][columns/128][columns%128/32][rows%16]
[16 bytes], a byte holding an even column in its low half and the next in its high half; scales [rows/16][columns/512]
[columns%128/32][rows%16][columns%512/128]. Rows and columns are filled up with zeros. Rows of 8 bits lie row by row,
their scales in rows of whole words of four.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _norm(name, rows, width, dtype, out, residual=True):
    return dict(name=name, kind="norm", rows=rows, width=width, dtype=dtype, out=out, residual=residual)


def _convert(name, rows, width, dtype):
    return dict(name=name, kind="convert", rows=rows, width=width, dtype=dtype)


def _pack(name, n, k, dtype):
    return dict(name=name, kind="pack", n=n, k=k, dtype=dtype)


def _product(name, rows, k, n, x, out, gated=False):
    """x: the rows' type, "i8" for 8 bits; out: the results'."""
    return dict(name=name, kind="product", rows=rows, n=n, k=k, x=x, out=out, gated=gated)


def listed():
    return [
        # The norm between two layers of the SmolLM2-135M shape while one user chats: a call's latency.
        _norm("norm_1", 1, 576, "f32", "f32"),
        # The final norm of a batch whose rows are not a multiple of anything, without a residual.
        _norm("norm_odd", 777, 2047, "f16", "f16", False),
        # Prompts of a wider model packed in one batch, to rows of 8 bits for the products behind it.
        _norm("norm_prompts", 4096, 4096, "bf16", "i8"),
        # The attention's output of a decode step of 64 sequences, to 8 bits for the projection.
        _convert("convert_64", 64, 576, "f32"),
        # The same of packed prompts in a wider model.
        _convert("convert_prompts", 4096, 4096, "bf16"),
        # The embedding table of the SmolLM2-135M shape, as a model is loaded.
        _pack("pack_table", 49152, 576, "f32"),
        # A projection of a wider model.
        _pack("pack_wide", 12288, 4096, "bf16"),
        # One user chatting: the down projection of the SmolLM2-135M shape. A call's latency.
        _product("down_1", 1, 1536, 576, "f32", "f32"),
        # The gated pair of a wider model for a single token: the weights' bytes are what counts.
        _product("gated_1_wide", 1, 4096, 12288, "bf16", "bf16", True),
        # The language-model head of a server's decode step: 64 rows.
        _product("head_64", 64, 576, 49152, "f32", "f32"),
        # The last, ragged chunk of a prompt, query, key and value projections in one.
        _product("qkv_203", 203, 576, 960, "f32", "f32"),
        # Packed prompts through a wider model's gated pair, 8 bits in and out: the matrix cores are what counts.
        _product("gated_prompts", 4096, 4096, 12288, "i8", "i8", True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _drawn(rng):
    dtype = rng.choice(["f32", "bf16", "f16"])
    pick = rng.random()
    if pick < 0.25:
        out = rng.choice([dtype, dtype, "i8", rng.choice(["f32", "bf16", "f16"])])
        width = 32 * _log(rng, 1, 512) if out == "i8" else _log(rng, 1, 16384)
        return _norm("", _log(rng, 1, 16384), width, dtype, out, rng.random() < 0.6)
    if pick < 0.35:
        return _convert("", _log(rng, 1, 16384), 32 * _log(rng, 1, 512), dtype)
    if pick < 0.45:
        return _pack("", _log(rng, 1, 50000), 32 * _log(rng, 1, 512), dtype)
    x = rng.choice([dtype, "i8"])
    gated = rng.random() < 0.4
    # A row of 8 bits out of a product is what the gated pair gives the next one.
    out = "i8" if gated and rng.random() < 0.4 else dtype
    n = 32 * _log(rng, 1, 512) if out == "i8" else _log(rng, 1, 50000)
    rows = _log(rng, 1, 300) if rng.random() < 0.6 else _log(rng, 1, 5000)
    return _product("", rows, 32 * _log(rng, 1, 512), n, x, out, gated)


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
        # The plain form of a product holds the weights and the results in 32 bits.
        whole = case["n"] * max(case["k"], case["rows"]) if case["kind"] == "product" else 0
        if all(w[key] <= largest[case["kind"], key] for key in w) and whole <= 12288 * 8192:
            del case["name"]
            return case


def _size(dtype):
    return {"f32": 4, "bf16": 2, "f16": 2, "i8": 1 + 1 / 32}[dtype]


def work(case):
    kind = case["kind"]
    if kind == "norm":
        n = case["rows"] * case["width"]
        each = _size(case["dtype"]) * (3 if case["residual"] else 1) + _size(case["out"])
        back = _size("i8") + 4 if case["out"] == "i8" else 0  # read back as floats
        return {"bytes": n * (each + back) + 4 * case["width"], "flops": 5 * n}
    if kind == "convert":
        n = case["rows"] * case["width"]
        return {"bytes": n * 2 * (_size(case["dtype"]) + _size("i8")), "flops": 3 * n}
    if kind == "pack":
        n = case["n"] * case["k"]
        return {"bytes": n * 2 * (_size(case["dtype"]) + 17 / 32), "flops": 3 * n}
    matrices = 2 if case["gated"] else 1
    rows, n, k = case["rows"], case["n"], case["k"]
    back = rows * n * (_size("i8") + 2) if case["out"] == "i8" else 0
    return {"bytes": matrices * n * k * 17 / 32 + rows * k * _size(case["x"]) + rows * n * _size(case["out"]) + back,
            "flops": 2 * matrices * rows * n * k}


# ---- the formats in plain torch ----------------------------------------------


def _scale_bytes(amax, top, bits):
    """Bytes of the smallest powers of two s, from 2^-100 on, with amax <= top * 2^bits * s."""
    mantissa, exponent = torch.frexp(amax)
    e = (exponent - bits + (mantissa > top).int()).clamp(min=-100)
    e = torch.where(amax > 0, e, torch.full_like(e, -100))
    return (e + 127).to(torch.uint8)


def _power(scales, dtype):
    return torch.ldexp(torch.ones((), dtype=dtype, device=scales.device), scales.int() - 127)


def _to_rows8(x):
    """Rows of 8 bits of x [rows, width]: codes, scale bytes in rows of whole words."""
    rows, width = x.shape
    groups = x.reshape(rows, width // 32, 32)
    scales = _scale_bytes(groups.abs().amax(-1), 0.9921875, 7)
    codes = torch.round(groups / _power(scales, x.dtype)[..., None])
    padded = torch.zeros((rows, -(-width // 128) * 4), dtype=torch.uint8, device=x.device)
    padded[:, :width // 32] = scales
    return codes.to(torch.int8).reshape(rows, width), padded


def _from_rows8(codes, scales):
    rows, width = codes.shape
    x = codes.float().view(rows, width // 32, 32)
    return (x * _power(scales[:, :width // 32], torch.float32)[..., None]).reshape(rows, width)


def _to_codes4(x):
    """Codes 0 .. 15 of the E2M1 numbers nearest to x, ties to the even code."""
    a = x.abs()
    _, exponent = torch.frexp(a)
    step = torch.ldexp(torch.ones((), dtype=x.dtype, device=x.device), (exponent - 2).clamp(min=-1))
    v = torch.round(a / step) * step  # 0, 0.5, 1, 1.5, 2, 3, 4 or 6
    code = torch.where(v <= 2, 2 * v, torch.where(v < 4, v + 2, v / 2 + 4))
    return code.to(torch.uint8) + 8 * (x < 0)


def _to_matrix(x):
    """The bytes of a 4-bit matrix of x [n, k]: codes and scales in their order."""
    n, k = x.shape
    tiles, steps, words = -(-n // 16), -(-k // 128), -(-k // 512)
    groups = x.reshape(n, k // 32, 32)
    scale = _scale_bytes(groups.abs().amax(-1), 0.75, 3)
    codes = torch.zeros((tiles * 16, steps * 4, 32), dtype=torch.uint8, device=x.device)
    codes[:n, :k // 32] = _to_codes4(groups / _power(scale, x.dtype)[..., None])
    scales = torch.zeros((tiles * 16, words * 16), dtype=torch.uint8, device=x.device)
    scales[:n, :k // 32] = scale
    codes = codes.view(tiles, 16, steps, 4, 16, 2).permute(0, 2, 3, 1, 4, 5)
    scales = scales.view(tiles, 16, words, 4, 4).permute(0, 2, 4, 1, 3)
    return (codes[..., 0] + 16 * codes[..., 1]).reshape(-1), scales.reshape(-1)


def _from_matrix(codes, scales, n, k):
    """The weights [n, k] that a 4-bit matrix stands for."""
    tiles, steps, words = -(-n // 16), -(-k // 128), -(-k // 512)
    numbers = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    numbers = torch.cat((numbers, -numbers))
    both = torch.stack((numbers[(codes & 15).int()], numbers[(codes >> 4).int()]), -1)
    x = both.view(tiles, steps, 4, 16, 32).permute(0, 3, 1, 2, 4).reshape(tiles * 16, steps * 4, 32)
    power = _power(scales, torch.float32).view(tiles, words, 4, 16, 4).permute(0, 3, 1, 4, 2)
    power = power.reshape(tiles * 16, words * 16)[:, :steps * 4]
    return (x * power[..., None]).reshape(tiles * 16, steps * 128)[:n, :k]


# ---- the state before the call ------------------------------------------------


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _activations(gen, rows, width, dtype):
    """Rows of hidden states: a few channels are much larger than the others."""
    channel = torch.exp(0.7 * _normal(gen, width))
    return (_normal(gen, rows, width) * channel).to(TYPES[dtype])


def _weights(gen, n, k):
    """A projection's weights: their size varies from row to row."""
    return _normal(gen, n, k) * (0.02 * torch.exp(0.3 * _normal(gen, n, 1)))


def _rows8_buffers(rows, width):
    return torch.empty((rows, width), dtype=torch.int8, device="cuda"), \
        torch.empty((rows, -(-width // 128) * 4), dtype=torch.uint8, device="cuda")


def _matrix_buffers(n, k):
    tiles = -(-n // 16)
    return torch.empty(tiles * -(-k // 128) * 1024, dtype=torch.uint8, device="cuda"), \
        torch.empty(tiles * -(-k // 512) * 256, dtype=torch.uint8, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * seed + 41)
    state = dict(case=case)
    if case["kind"] in ("norm", "convert"):
        rows, width = case["rows"], case["width"]
        state["x"] = _activations(gen, rows, width, case["dtype"])
        out = case.get("out", "i8")
        if case["kind"] == "norm":
            state["weight"] = 1 + 0.1 * _normal(gen, width)
            if case["residual"]:
                state["residual"] = (4 * _normal(gen, rows, width)).to(TYPES[case["dtype"]])
                state["sum"] = torch.empty_like(state["residual"])
        if out == "i8":
            state["codes"], state["scales"] = _rows8_buffers(rows, width)
            back = torch.float32 if case["kind"] == "norm" else TYPES[case["dtype"]]
            state["out"] = torch.empty((rows, width), dtype=back, device="cuda")
        else:
            state["out"] = torch.empty((rows, width), dtype=TYPES[out], device="cuda")
    elif case["kind"] == "pack":
        n, k = case["n"], case["k"]
        state["x"] = _weights(gen, n, k).to(TYPES[case["dtype"]])
        state["matrix"] = _matrix_buffers(n, k)
        state["ids"] = torch.arange(n, dtype=torch.int32, device="cuda")
        state["out"] = torch.empty_like(state["x"])
    else:
        rows, n, k = case["rows"], case["n"], case["k"]
        if case["x"] == "i8":
            state["x"] = _to_rows8(_activations(gen, rows, k, "f32"))
        else:
            state["x"] = _activations(gen, rows, k, case["x"])
        state["matrix"] = _to_matrix(_weights(gen, n, k))
        if case["gated"]:
            state["gate"] = _to_matrix(_weights(gen, n, k))
        if case["out"] == "i8":
            state["codes"], state["scales"] = _rows8_buffers(rows, n)
            state["out"] = torch.empty((rows, n), dtype=torch.bfloat16, device="cuda")
        else:
            state["out"] = torch.empty((rows, n), dtype=TYPES[case["out"]], device="cuda")
    if own:
        _handles(state)
    return state


def _handles(state):
    """The descriptors and the workspace that a program keeps."""
    from tinyinfer_amd import backend as mp
    case = state["case"]
    types = {torch.float32: mp.TYPE_F32, torch.bfloat16: mp.TYPE_BF16, torch.float16: mp.TYPE_F16}

    def floats(t):
        return mp.Rows(t.data_ptr(), t.shape[1], None, 0, types[t.dtype])

    def rows8(codes, scales):
        return mp.Rows(codes.data_ptr(), codes.shape[1], scales.data_ptr(), scales.shape[1], mp.TYPE_I8)

    def matrix(m):
        return mp.W4Matrix(m[0].data_ptr(), m[1].data_ptr(), case["n"], case["k"])

    own_rows = {"out": floats(state["out"])}
    own_rows["x"] = rows8(*state["x"]) if isinstance(state["x"], tuple) else floats(state["x"])
    if "codes" in state:
        own_rows["i8"] = rows8(state["codes"], state["scales"])
    for name in ("residual", "sum"):
        own_rows[name] = floats(state[name]) if name in state else None
    for name in ("matrix", "gate"):
        own_rows[name] = matrix(state[name]) if name in state else None
    if case["kind"] == "product":
        size = mp.w4_product_workspace(own_rows["matrix"], own_rows["x"].type, case["rows"], case["gated"])
        state["workspace"] = torch.empty(max(1, size), dtype=torch.uint8, device="cuda")
        state["workspace_bytes"] = size
    state["own"] = own_rows


# ---- the calls -----------------------------------------------------------------


def _run_own(state):
    from tinyinfer_amd import backend as mp
    case, at = state["case"], state["own"]
    stream = torch.cuda.current_stream().cuda_stream
    to = at.get("i8", at["out"])
    if case["kind"] == "pack":
        mp.w4_pack(at["matrix"], 0, at["x"], case["n"], stream=stream)
        mp.w4_read(at["matrix"], state["ids"].data_ptr(), case["n"], at["out"], stream=stream)
        return {"out": state["out"]}
    rows = case["rows"]
    if case["kind"] == "norm":
        mp.rms_norm(at["x"], state["weight"].data_ptr(), 1e-5, rows, case["width"], to, residual=at["residual"],
                    sum=at["sum"], stream=stream)
    elif case["kind"] == "convert":
        mp.convert_rows(at["x"], rows, case["width"], to, stream=stream)
    else:
        mp.w4_product(at["matrix"], at["x"], rows, to, gate=at["gate"], workspace=state["workspace"].data_ptr(),
                      workspace_bytes=state["workspace_bytes"], stream=stream)
    if "i8" in at:
        mp.convert_rows(to, rows, state["out"].shape[1], at["out"], stream=stream)
    return {"out": state["out"], "sum": state["sum"]} if "sum" in state else {"out": state["out"]}


def _run_plain(state):
    case = state["case"]
    out = state["out"].dtype
    if case["kind"] == "pack":
        codes, scales = _to_matrix(state["x"].float())
        return {"out": _from_matrix(codes, scales, case["n"], case["k"]).to(out)}
    if case["kind"] == "convert":
        return {"out": _from_rows8(*_to_rows8(state["x"].float())).to(out)}
    if case["kind"] == "norm":
        # Values next to the border of two codes need more than 32 bits.
        wide = torch.float64 if case["out"] == "i8" else torch.float32
        x = state["x"].to(wide)
        if case["residual"]:
            x = x + state["residual"].to(wide)
        y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) * state["weight"].to(wide)
        found = {"out": _from_rows8(*_to_rows8(y)) if case["out"] == "i8" else y.to(out)}
        return found | {"sum": x.to(state["sum"].dtype)} if case["residual"] else found
    x = _from_rows8(*state["x"]) if case["x"] == "i8" else state["x"].float()
    y = torch.matmul(x, _from_matrix(*state["matrix"], case["n"], case["k"]).T)
    if case["gated"]:
        g = torch.matmul(x, _from_matrix(*state["gate"], case["n"], case["k"]).T)
        y = g / (1 + torch.exp(-g)) * y
    return {"out": _from_rows8(*_to_rows8(y)).to(out) if case["out"] == "i8" else y.to(out)}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- in 64 bits ------------------------------------------------------------------


def _numbers4(device):
    """The E2M1 numbers by code: sign, two bits of exponent, one of mantissa."""
    found = []
    for code in range(16):
        e, m = code >> 1 & 3, code & 1
        x = m / 2 if e == 0 else math.ldexp(2 + m, e - 2)
        found.append(-x if code & 8 else x)
    return torch.tensor(found, dtype=torch.float64, device=device)


def _held(x, numbers, most):
    """x [..., groups of 32] as a format holds it whose numbers from 0 up are `numbers`."""
    rows, width = x.shape
    x = x.reshape(rows, -1, 32)
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -110) / most)) - 1
    for _ in range(2):  # the logarithm may be off by a rounding
        e = torch.where(top > most * torch.exp2(e), e + 1, e)
    e = e.clamp(min=-100)
    y = x / torch.exp2(e)
    above = torch.searchsorted(numbers, y.abs().contiguous()).clamp(max=len(numbers) - 1)
    below = (above - 1).clamp(min=0)
    up, down = numbers[above] - y.abs(), y.abs() - numbers[below]
    code = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
    return (numbers[code] * torch.sign(y) * torch.exp2(e)).reshape(rows, width)


def _rows64(x):
    """The values of rows: floats, or codes and scales."""
    if not isinstance(x, tuple):
        return x.double()
    codes, scales = x
    width = codes.shape[1]
    column = torch.arange(width, device="cuda")
    return codes.double() * torch.exp2(scales[:, column // 32].double() - 127)


def _matrix64(matrix, n, k):
    codes, scales = matrix
    column = torch.arange(k, device="cuda")
    steps, words = -(-k // 128), -(-k // 512)
    table = _numbers4("cuda")
    parts = []
    for first in range(0, n, 4096):  # in parts, so that the places stay small
        row = torch.arange(first, min(n, first + 4096), device="cuda")[:, None]
        lane = column % 128 // 32 * 16 + row % 16
        byte = codes[(row // 16 * steps + column // 128) * 1024 + lane * 16 + column % 32 // 2].int()
        code = torch.where(column % 2 == 1, byte >> 4, byte & 15)
        scale = scales[(row // 16 * words + column // 512) * 256 + lane * 4 + column % 512 // 128]
        parts.append(table[code.long()] * torch.exp2(scale.double() - 127))
    return torch.cat(parts)


def exact(case, seed):
    state = prepare(case, seed)
    eight = torch.arange(128, dtype=torch.float64, device="cuda")
    if case["kind"] == "pack":
        four = _numbers4("cuda")[:8]
        x = state["x"]
        return {"out": torch.cat([_held(x[i:i + 4096].double(), four, 6.0) for i in range(0, case["n"], 4096)])}
    x = _rows64(state["x"])
    if case["kind"] == "convert":
        return {"out": _held(x, eight, 127.0)}
    if case["kind"] == "norm":
        if case["residual"]:
            x = x + state["residual"].double()
        y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["width"] + 1e-5) * state["weight"].double()
        found = {"out": _held(y, eight, 127.0) if case["out"] == "i8" else y}
        return found | {"sum": x} if case["residual"] else found
    # Made contiguous first, as elsewhere: the product's right operand is no transposed view.
    y = torch.mm(x, _matrix64(state["matrix"], case["n"], case["k"]).T.contiguous())
    if case["gated"]:
        g = torch.mm(x, _matrix64(state["gate"], case["n"], case["k"]).T.contiguous())
        y = y * g * torch.sigmoid(g)
    return {"out": _held(y, eight, 127.0) if case["out"] == "i8" else y}
