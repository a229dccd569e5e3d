"""The 8-bit paged K/V cache on the GPU, through its C entries, against the
definition in numpy (kv8_reference.py): bytes and scales bit for bit, attention
within the bound that its arithmetic gives (kv8_reference.bound, plus the
rounding of the row type: half a step of the result, and for FP16 and BF16
prefill rows half an FP16 step of every probability)."""
import numpy as np
import pytest

from tinyinfer_amd import backend as mp

from .kv8_reference import BF16, E4M3, F16, F32, INT8, VALUES, Cache, attention_close, rounded
from .kv8_sizes import WALKS

pytestmark = pytest.mark.gpu

FORMATS = pytest.mark.parametrize("fmt", [INT8, E4M3], ids=["int8", "e4m3"])
TYPES = {F32: "float32", BF16: "bfloat16", F16: "float16"}
HALF_STEP = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}


class Device:
    """A numpy Cache's pools on the GPU, and calls on them."""

    def __init__(self, torch, cache: Cache):
        self.torch, self.cache = torch, cache
        self.bytes = [torch.from_numpy(b.copy()).cuda() for b in cache.bytes]
        self.scales = torch.from_numpy(cache.scales.copy()).cuda()
        self.view = mp.Kv8Cache(self.bytes[0].data_ptr(), self.bytes[1].data_ptr(), self.scales.data_ptr(),
                                cache.blocks, cache.layers, cache.bt, cache.kv_heads, cache.dim, cache.fmt)

    def ints(self, a):
        return self.torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()

    def rows(self, x, kind, pad=0, shift=0):
        """x [rows, width] float32 as a row matrix of a type: (tensor kept alive, address, stride); `pad` elements
        behind every row, the first `shift` elements from the buffer's start. Padding is NaN."""
        t = self.torch
        n, width = x.shape
        buffer = t.full((n * (width + pad) + shift,), float("nan"), dtype=getattr(t, TYPES[kind]), device="cuda")
        matrix = buffer[shift:].view(n, width + pad)
        matrix[:, :width] = t.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).cuda()
        return matrix, matrix.data_ptr(), width + pad

    def back(self, matrix, width):
        self.torch.cuda.synchronize()
        return matrix[:, :width].float().cpu().numpy()

    def check_bytes(self, want: Cache):
        """Scales and bytes equal, but for the bytes of what reads as NaN."""
        self.torch.cuda.synchronize()
        scales = self.scales.cpu().numpy()
        assert np.array_equal(scales, want.scales, equal_nan=True)
        for kind in range(2):
            got, readable = self.bytes[kind].cpu().numpy(), ~np.isnan(want.scales[..., kind])
            assert np.array_equal(got[readable], want.bytes[kind][readable]), f"kind {kind}"


def tables_for(rng, blocks, lengths, bt, spare=1):
    pages = [-(-max(n, 1) // bt) for n in lengths]
    order = rng.permutation(blocks)
    assert sum(pages) <= blocks
    tables = np.full((len(lengths), max(pages) + spare), -1, dtype=np.int32)
    at = 0
    for s, p in enumerate(pages):
        tables[s, :p] = order[at:at + p]
        at += p
    return tables


def blocks_for(lengths, bt):
    return sum(-(-max(n, 1) // bt) for n in lengths) + 2


def angles(positions, dims):
    a = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(max(dims // 2, 1)) / max(dims // 2, 1))
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def starts_of(counts, first=0):
    return np.concatenate(([first], first + np.cumsum(counts))).astype(np.int32)


# ---- appending and reading ----------------------------------------------------

APPENDS = [
    # kv_heads, heads, dim, bt, rotated, interleaved, type, pad, shift
    (3, 9, 64, 16, 64, False, F32, 0, 0),
    (3, 9, 64, 16, 64, True, BF16, 4, 0),
    (1, 2, 64, 32, 20, False, F32, 1, 1),   # rows and pairs that are not aligned
    (2, 2, 64, 64, 6, True, F16, 0, 1),
    (2, 6, 128, 64, 64, False, BF16, 8, 0),
    (1, 4, 128, 128, 128, False, F32, 0, 0),
    (1, 3, 256, 32, 32, True, F16, 12, 0),
    (2, 4, 256, 16, 0, False, F32, 0, 0),
    # queries by 16 bytes: every arrangement of turning and passing dims
    (2, 32, 128, 64, 64, True, BF16, 0, 0),
    (1, 7, 128, 16, 128, False, F16, 8, 0),
    (3, 9, 64, 32, 16, False, BF16, 0, 0),
    (1, 3, 64, 16, 24, True, F32, 0, 0),
    (1, 5, 256, 16, 256, False, F32, 4, 0),
    (1, 1, 64, 16, 0, False, F16, 0, 0),
]


@FORMATS
@pytest.mark.parametrize("kv_heads, heads, dim, bt, dims, interleaved, kind, pad, shift", APPENDS)
def test_append_and_read(torch_cuda, fmt, kv_heads, heads, dim, bt, dims, interleaved, kind, pad, shift):
    """Three calls in a row, each going on where the one before ended (in the middle of pages, with larger tokens, so
    that scales grow): counts of 0, 1 and more than two pages, rows before the first and behind the last sequence,
    layer 1 of 2. Then everything read back."""
    rng = np.random.default_rng(dim + bt + fmt)
    total = [0, 2 * bt + 5, 3, bt, 1, 3 * bt - 1]
    steps = [[0, bt + 3, 1, bt - 1, 0, bt], [0, 1, 1, 1, 1, bt + 2], [0, bt + 1, 1, 0, 0, bt - 3]]
    assert [sum(s) for s in zip(*steps)] == total
    cache = Cache(blocks_for(total, bt), 2, kv_heads, bt, dim, fmt, rng)
    device = Device(torch_cuda, cache)
    tables = tables_for(rng, cache.blocks, total, bt)
    cos, sin = angles(max(total), dims)
    d_tables, d_cos, d_sin = device.ints(tables), torch_cuda.from_numpy(cos).cuda(), torch_cuda.from_numpy(sin).cuda()
    rope = mp.Rope(d_cos.data_ptr(), d_sin.data_ptr(), len(cos), dims, int(interleaved))
    used = np.zeros(len(total), dtype=np.int32)
    for step, counts in enumerate(steps):
        starts = starts_of(counts, first=2)
        rows = int(starts[-1]) + 3
        q, k, v = (rounded(rng.standard_normal((rows, h, dim)) * 3.0 ** step, kind)
                   for h in (heads, kv_heads, kv_heads))
        mq, q_at, q_stride = device.rows(q.reshape(rows, -1), kind, pad, shift)
        mk, k_at, k_stride = device.rows(k.reshape(rows, -1), kind, pad, shift)
        mv, v_at, v_stride = device.rows(v.reshape(rows, -1), kind, pad, shift)
        mo, o_at, o_stride = device.rows(np.full((rows, heads * dim), 7.0), kind, pad, shift)
        d_starts, d_used = device.ints(starts), device.ints(used)
        mp.kv8_append(device.view, 1, k_at, k_stride, v_at, v_stride, kind, d_tables.data_ptr(), tables.shape[1],
                      d_starts.data_ptr(), d_used.data_ptr(), len(total), rows, rope=rope, q=q_at, q_stride=q_stride,
                      q_out=o_at, q_out_stride=o_stride, heads=heads)
        cache.append(1, k, v, tables, starts, used, (cos, sin, dims, interleaved))
        device.check_bytes(cache)
        # Queries: rotated in float32, rounded once; other rows as they were.
        from .kv8_reference import rotate
        want = np.full((rows, heads, dim), 7.0, dtype=np.float32)
        for s in range(len(total)):
            for i in range(counts[s]):
                r, position = starts[s] + i, used[s] + i
                want[r] = rounded(rotate(q[r], cos[position], sin[position], dims, interleaved), kind) if dims else q[r]
        assert np.array_equal(device.back(mo, heads * dim), want.reshape(rows, -1))
        assert bool(mo[:, heads * dim:].isnan().all())
        used = used + np.array(counts, dtype=np.int32)
    # Reading: every token, and the ends alone.
    for first in (np.zeros(len(total), dtype=np.int32), np.array([max(n - 2, 0) for n in total], dtype=np.int32)):
        counts = np.array(total) - first
        starts = starts_of(counts, first=1)
        rows = int(starts[-1]) + 2
        out = [device.rows(np.full((rows, kv_heads * dim), 5.0), kind, pad, shift) for _ in range(2)]
        d_starts, d_used = device.ints(starts), device.ints(first)
        mp.kv8_read(device.view, 1, d_tables.data_ptr(), tables.shape[1], d_starts.data_ptr(), d_used.data_ptr(),
                    len(total), rows, kind, out[0][1], out[0][2], out[1][1], out[1][2])
        for which in range(2):
            want = np.full((rows, kv_heads, dim), 5.0)
            for s in range(len(total)):
                values = cache.tokens(1, which, tables[s], total[s])[:, first[s]:]
                want[starts[s]:starts[s + 1]] = values.transpose(1, 0, 2)
            assert np.array_equal(device.back(out[which][0], kv_heads * dim), rounded(want.reshape(rows, -1), kind))


def append_plain(device, layer, k, v, tables, starts, used, rope=None, keep=None):
    """FP32 rows without padding or queries."""
    rows = k.shape[0]
    mk, k_at, k_stride = device.rows(k.reshape(rows, -1), F32)
    mv, v_at, v_stride = device.rows(v.reshape(rows, -1), F32)
    ints = [device.ints(a) for a in (tables, starts, used)]
    mp.kv8_append(device.view, layer, k_at, k_stride, v_at, v_stride, F32, ints[0].data_ptr(), tables.shape[1],
                  ints[1].data_ptr(), ints[2].data_ptr(), len(used), rows, rope=rope)
    device.torch.cuda.synchronize()


@FORMATS
def test_append_extremes(torch_cuda, fmt):
    """Zeros, denormals, the largest numbers, and magnitudes on both sides of where the scale steps."""
    rng = np.random.default_rng(3)
    top = 127.0 if fmt == INT8 else 448.0
    peaks = [0.0, 2.0 ** -149, 2.0 ** -130, 2.0 ** -126, top * 2.0 ** -126, np.nextafter(np.float32(top / 8), np.float32(1e9)),
             top / 8, np.nextafter(np.float32(top / 8), np.float32(0)), 1.0, 3e38, float(np.finfo(np.float32).max)]
    cache = Cache(len(peaks) + 1, 1, 1, 16, 64, fmt, rng)
    device = Device(torch_cuda, cache)
    tables = np.arange(len(peaks), dtype=np.int32)[:, None]
    x = rng.uniform(-1, 1, (len(peaks), 1, 64))
    x[:, 0, 17] = -1
    x = (x * np.array(peaks, dtype=np.float64)[:, None, None]).astype(np.float32)
    starts, used = starts_of([1] * len(peaks)), np.zeros(len(peaks), dtype=np.int32)
    append_plain(device, 0, x, -x, tables, starts, used)
    cache.append(0, x, -x, tables, starts, used)
    device.check_bytes(cache)
    for at, s in enumerate(cache.scales[:len(peaks), 0, 0, 0]):
        assert s >= 2.0 ** -126 and np.frexp(s)[0] == 0.5 and peaks[at] <= top * float(s)


@FORMATS
def test_token_by_token_is_within_a_step_of_a_chunk(torch_cuda, fmt):
    """Rounded again at each growth, a token's INT8 code is off its own rounding by less than one step of the final
    scale (1/2 + 1/4 + ...); an E4M3 value by half a step of 2^-3 twice at most where it falls below the normal range."""
    rng = np.random.default_rng(4)
    x = (rng.standard_normal((32, 2, 64)) * 2.0 ** (np.arange(32) % 16 / 3)[:, None, None]).astype(np.float32)
    tables = np.array([[1, 2]], dtype=np.int32)
    whole, single = (Cache(3, 1, 2, 16, 64, fmt, rng) for _ in range(2))
    a, b = Device(torch_cuda, whole), Device(torch_cuda, single)
    append_plain(a, 0, x, x, tables, np.array([0, 32]), np.array([0]))
    whole.append(0, x, x, tables, [0, 32], [0])
    a.check_bytes(whole)
    for i in range(32):
        append_plain(b, 0, x[i:i + 1], x[i:i + 1], tables, np.array([0, 1]), np.array([i]))
        single.append(0, x[i:i + 1], x[i:i + 1], tables, [0, 1], [i])
    b.check_bytes(single)
    assert np.array_equal(whole.scales[1:], single.scales[1:])
    scale = np.repeat(whole.scales[1:, 0, :, 0], 16, axis=0)[..., None].astype(np.float64)
    for cache in (whole, single):
        got = cache.tokens(0, 0, tables[0], 32).transpose(1, 0, 2)
        off = np.abs(got - x)
        if fmt == INT8:
            assert np.all(off < (0.5 if cache is whole else 1.0) * scale)
        else:
            assert np.all(off <= np.maximum(np.abs(x) * 2.0 ** -4, scale * 2.0 ** -9))


@FORMATS
def test_a_step_taken_back_and_a_poisoned_page(torch_cuda, fmt):
    """NaN and infinity make a head's keys of the page NaN and nothing else; writing the page from slot 0 heals it;
    a token written again gives its codes again."""
    rng = np.random.default_rng(5)
    cache = Cache(4, 2, 2, 16, 64, fmt, rng)
    device = Device(torch_cuda, cache)
    tables = np.array([[2, 0]], dtype=np.int32)
    x = rng.standard_normal((20, 2, 64)).astype(np.float32)

    def step(rows, at, k, v):
        append_plain(device, 1, k, v, tables, np.array([0, rows]), np.array([at]))
        cache.append(1, k, v, tables, [0, rows], [at])
        device.check_bytes(cache)

    step(20, 0, x, x)
    step(1, 5, x[5:6], x[5:6])
    bad = x[6:7].copy()
    bad[0, 1, 3] = np.nan
    step(1, 6, bad, x[6:7])
    assert np.isnan(cache.scales[2, 1, 1, 0]) and np.isnan(cache.scales).sum() == 1
    step(1, 6, x[6:7], x[6:7])
    assert np.isnan(cache.scales[2, 1, 1, 0]) and np.isnan(cache.scales).sum() == 1
    step(20, 0, x, x)
    assert not np.isnan(cache.scales).any()
    bad = x[:1].copy()
    bad[0, 0, 0] = -np.inf
    step(1, 19, x[19:20], bad)
    assert np.isnan(cache.scales[0, 1, 0, 1]) and np.isnan(cache.scales).sum() == 1


def test_append_beyond_pages_and_angles(torch_cuda):
    """Page ids outside the pool, pages past the table and positions past the rotation tables: those tokens are not
    written, all others are; a query past the tables is NaN. Sequences that start below 0 are left out."""
    rng = np.random.default_rng(6)
    cache = Cache(6, 1, 1, 16, 64, INT8, rng)
    device = Device(torch_cuda, cache)
    tables = np.array([[0, -1, 1], [2, 6, 3], [4, 2147483647, 5], [1, 1, 1]], dtype=np.int32)
    counts, used = [40, 60, 20, 3], np.array([0, 0, 25, -7], dtype=np.int32)
    starts = starts_of(counts)
    rows = int(starts[-1])
    k, v, q = (rng.standard_normal((rows, 1, 64)).astype(np.float32) for _ in range(3))
    cos, sin = angles(38, 64)
    d_cos, d_sin = torch_cuda.from_numpy(cos).cuda(), torch_cuda.from_numpy(sin).cuda()
    rope = mp.Rope(d_cos.data_ptr(), d_sin.data_ptr(), 38, 64, 0)
    mk, k_at, _ = device.rows(k.reshape(rows, -1), F32)
    mv, v_at, _ = device.rows(v.reshape(rows, -1), F32)
    mq, q_at, _ = device.rows(q.reshape(rows, -1), F32)
    ints = [device.ints(a) for a in (tables, starts, used)]
    mp.kv8_append(device.view, 0, k_at, 64, v_at, 64, F32, ints[0].data_ptr(), 3, ints[1].data_ptr(),
                  ints[2].data_ptr(), 4, rows, rope=rope, q=q_at, q_stride=64, q_out=q_at, q_out_stride=64, heads=1)
    cache.append(0, k, v, tables[:3], starts[:4], used[:3], (cos, sin, 64, False))
    device.check_bytes(cache)
    got = device.back(mq, 64)
    position = np.concatenate([u + np.arange(c) for u, c in zip(used, counts)])
    lost = (position >= 38) | (np.arange(rows) >= starts[3])
    assert np.array_equal(np.isnan(got).all(1), lost) and np.array_equal(np.isnan(got).any(1), lost)
    # Reading gives NaN for the same pages.
    out = [device.rows(np.zeros((rows, 64)), F32) for _ in range(2)]
    mp.kv8_read(device.view, 0, ints[0].data_ptr(), 3, ints[1].data_ptr(), ints[2].data_ptr(), 3, rows, F32,
                out[0][1], 64, out[1][1], 64)
    got = device.back(out[0][0], 64)
    page = position // 16
    sequence = np.repeat(np.arange(4), counts)
    missing = np.array([p >= 3 or not 0 <= tables[s, min(p, 2)] < 6 for s, p in zip(sequence, page)])
    inside = np.arange(rows) < starts[3]
    assert np.array_equal(np.isnan(got).all(1)[inside], missing[inside])
    assert np.all(got[~inside] == 0)


# ---- attention ------------------------------------------------------------------


def fill(cache, rng, tables, lengths, spread=1.0):
    """Tokens of all layers appended by the reference; in the slots behind them stays whatever there was."""
    for layer in range(cache.layers):
        for s, n in enumerate(lengths):
            if n > 0:
                k, v = (rng.standard_normal((n, cache.kv_heads, cache.dim)).astype(np.float32) for _ in range(2))
                k *= spread * np.exp(0.5 * rng.standard_normal(cache.dim)).astype(np.float32)
                cache.append(layer, k, v, tables[s:s + 1], [0, n], [0])


def workspace_for(device, rows, sequences, heads, max_length):
    size = mp.kv8_attention_workspace(device.view, rows, sequences, heads, max_length)
    return device.torch.full((max(size, 1),), 255, dtype=device.torch.uint8, device="cuda"), size


def run_decode(device, layer, q, kind, tables, lengths, max_length, scale, pad=0, shift=0):
    rows, width = q.shape[0], q.shape[1] * q.shape[2]
    mq, q_at, q_stride = device.rows(q.reshape(rows, -1), kind, pad, shift)
    mo, o_at, o_stride = device.rows(np.full((rows, width), 7.0), kind, pad, shift)
    d_tables, d_lengths = device.ints(tables), device.ints(lengths)
    space, size = workspace_for(device, rows, rows, q.shape[1], max_length)
    mp.kv8_attention_decode(device.view, layer, q_at, q_stride, kind, d_tables.data_ptr(), tables.shape[1],
                            d_lengths.data_ptr(), rows, q.shape[1], max_length, scale, o_at, o_stride,
                            space.data_ptr(), size)
    got = device.back(mo, width)
    assert bool(mo[:, width:].isnan().all())
    return got.reshape(q.shape)


def run_prefill(device, layer, q, kind, tables, starts, used, max_length, scale, pad=0, shift=0):
    rows, width = q.shape[0], q.shape[1] * q.shape[2]
    mq, q_at, q_stride = device.rows(q.reshape(rows, -1), kind, pad, shift)
    mo, o_at, o_stride = device.rows(np.full((rows, width), 7.0), kind, pad, shift)
    ints = [device.ints(a) for a in (tables, starts, used)]
    space, size = workspace_for(device, rows, len(used), q.shape[1], max_length)
    mp.kv8_attention_prefill(device.view, layer, q_at, q_stride, kind, ints[0].data_ptr(), tables.shape[1],
                             ints[1].data_ptr(), ints[2].data_ptr(), len(used), rows, q.shape[1], max_length, scale,
                             o_at, o_stride, space.data_ptr(), size)
    got = device.back(mo, width)
    assert bool(mo[:, width:].isnan().all())
    return got.reshape(q.shape)


def check_row(got, want, err, kind, v_max, prefill, what):
    limit = err + HALF_STEP[kind] * np.abs(want) + (HALF_STEP[F16] * v_max if prefill and kind != F32 else 0)
    off = np.abs(got - want)
    assert np.all(off <= limit), f"{what}: off by {off.max():.3e}, at most {float(np.max(limit)):.3e}"


SHAPES = [
    # kv_heads, heads, dim, bt, type, pad, shift
    (3, 9, 64, 16, F32, 0, 0),
    (1, 1, 64, 16, F32, 3, 1),
    (2, 16, 64, 32, BF16, 8, 0),
    (1, 12, 64, 64, F32, 0, 0),
    (2, 8, 128, 16, F16, 0, 1),
    (1, 16, 128, 128, F32, 4, 0),
    (1, 5, 256, 16, F32, 0, 0),
    (1, 11, 256, 64, BF16, 0, 0),
]
LENGTHS = [1, 2, 15, 16, 17, 31, 32, 33, 63, 65, 127, 128, 129, 300, 0, 511, -3, 777]


@FORMATS
@pytest.mark.parametrize("kv_heads, heads, dim, bt, kind, pad, shift", SHAPES)
def test_decode(torch_cuda, fmt, kv_heads, heads, dim, bt, kind, pad, shift):
    """Rows of every length at once, two layers, slots behind the last token holding anything (E4M3 NaN codes among
    them); then a few of them alone with a larger max_length, so that their tokens are split."""
    rng = np.random.default_rng(heads * dim + bt)
    cache = Cache(blocks_for(LENGTHS, bt), 2, kv_heads, bt, dim, fmt, rng)
    tables = tables_for(rng, cache.blocks, LENGTHS, bt)
    fill(cache, rng, tables, LENGTHS)
    device = Device(torch_cuda, cache)
    q = rounded(rng.standard_normal((len(LENGTHS), heads, dim)), kind)
    scale = 1.3 / dim ** 0.5
    v_max = max(np.nanmax(np.abs(cache.tokens(1, 1, t, max(n, 1)))) for t, n in zip(tables, LENGTHS) if n > 0)
    for pick, longest in ((range(len(LENGTHS)), 777), ((13, 17, 0), 5000), ((17,), 100000), ((12, 14), 129)):
        pick = list(pick)
        got = run_decode(device, 1, q[pick], kind, tables[pick], [LENGTHS[i] for i in pick], longest, scale, pad, shift)
        for j, i in enumerate(pick):
            want, err = cache.attention(1, q[i], tables[i], LENGTHS[i], scale)
            check_row(got[j], want, err, kind, v_max, False, f"length {LENGTHS[i]} of at most {longest}")


PREFILLS = [
    # used, counts: whole prompts, chunks behind a history, single tokens among them, sequences without rows
    ([0, 0, 0, 0], [1, 17, 100, 33]),
    ([300, 0, 47, 16, 5], [1, 0, 61, 16, 1]),
    ([900], [40]),
    ([0], [260]),
    ([31, 15, 2, 600], [1, 1, 1, 1]),
]


@FORMATS
@pytest.mark.parametrize("kv_heads, heads, dim, bt, kind, pad, shift", SHAPES)
def test_prefill(torch_cuda, fmt, kv_heads, heads, dim, bt, kind, pad, shift):
    for case, (used, counts) in enumerate(PREFILLS):
        rng = np.random.default_rng(heads + dim + bt + case)
        lengths = [u + c for u, c in zip(used, counts)]
        cache = Cache(blocks_for(lengths, bt), 2, kv_heads, bt, dim, fmt, rng)
        tables = tables_for(rng, cache.blocks, lengths, bt)
        fill(cache, rng, tables, lengths)
        device = Device(torch_cuda, cache)
        starts = starts_of(counts, first=1)
        rows = int(starts[-1]) + 2
        q = rounded(rng.standard_normal((rows, heads, dim)), kind)
        scale = 1 / dim ** 0.5
        for longest in (max(lengths), 40000):
            got = run_prefill(device, 1, q, kind, tables, starts, used, longest, scale, pad, shift)
            assert np.all(got[:1] == 7) and np.all(got[-2:] == 7)
            for s, u in enumerate(used):
                v_max = np.abs(cache.tokens(1, 1, tables[s], max(lengths[s], 1))).max()
                rows_of = range(counts[s]) if counts[s] <= 40 else sorted({0, 1, 15, 16, counts[s] // 2, counts[s] - 2, counts[s] - 1})
                for i in rows_of:
                    r = starts[s] + i
                    want, err = cache.attention(1, q[r], tables[s], u + i + 1, scale)
                    check_row(got[r], want, err, kind, v_max, True, f"case {case}, position {u + i} of {longest}")


def test_prefill_of_many_rows(torch_cuda):
    """Enough rows that every wavefront takes several column tiles: 70 sequences of 60 to 129 rows (many of them
    prompts), more sequences than a wavefront has lanes; sampled rows."""
    for dim, kind, fmt in ((64, F32, INT8), (128, BF16, E4M3), (128, F32, E4M3), (256, F16, INT8)):
        rng = np.random.default_rng(dim + kind)
        kv_heads, heads, bt = 2, 6, 16
        counts = [60 + s for s in range(70)]
        used = [0 if s % 3 else 2 * s + 1 for s in range(70)]
        lengths = [u + c for u, c in zip(used, counts)]
        cache = Cache(blocks_for(lengths, bt), 1, kv_heads, bt, dim, fmt, rng)
        # Random codes under the scales that are there: quicker than appending.
        if fmt == E4M3:
            for b in cache.bytes:
                b[(b & 127) == 127] = 0
        tables = tables_for(rng, cache.blocks, lengths, bt)
        device = Device(torch_cuda, cache)
        starts = starts_of(counts)
        q = rounded(rng.standard_normal((int(starts[-1]), heads, dim)) * 0.02, kind)
        for longest in (max(lengths), 20000):
            got = run_prefill(device, 0, q, kind, tables, starts, used, longest, 1 / dim ** 0.5)
            assert np.isfinite(got).all()
            for s in (0, 1, 2, 33, 63, 64, 65, 69):
                v_max = np.abs(cache.tokens(0, 1, tables[s], lengths[s])).max()
                for i in (0, 1, counts[s] // 2, counts[s] - 1):
                    r = starts[s] + i
                    want, err = cache.attention(0, q[r], tables[s], used[s] + i + 1, 1 / dim ** 0.5)
                    check_row(got[r], want, err, kind, v_max, True, f"dim {dim}, sequence {s}, row {i} of {longest}")


@FORMATS
def test_attention_closed_form(torch_cuda, fmt):
    """Scores of -1000 to 1001, and scales that differ by 2^40 between pages: exact powers, so the answer is known.
    Keys are 8 in one dim, queries pick the score; values are one number a page."""
    rng = np.random.default_rng(9)
    bt, dim, pages = 16, 64, 6
    cache = Cache(pages + 1, 1, 1, bt, dim, fmt, rng)
    tables = np.arange(pages, dtype=np.int32)[None]
    length = pages * bt
    for kind in range(2):
        cache.bytes[kind][:] = 128 if fmt == INT8 else 0
    one = {INT8: 129, E4M3: int(np.flatnonzero(VALUES[E4M3] == 1)[0])}[fmt]
    cache.bytes[0][:, :, :, cache.places[0][:, 0]] = one
    cache.bytes[1][:, :, :, cache.places[1][:, 5]] = one
    # Keys: page p scores 100 p (scale 1 after the softmax scale below), the last page the most.
    scores = np.array([1, 2, 4, 8, 16, 32], dtype=np.float32)
    cache.scales[:pages, 0, 0, 0] = scores
    cache.scales[:pages, 0, 0, 1] = 2.0 ** np.array([40, -3, 5, 0, 2, -6])
    device = Device(torch_cuda, cache)
    q = np.zeros((3, 1, dim), dtype=np.float32)
    q[:, 0, 0] = [1000, -1000, 1e-3]
    got = run_decode(device, 0, q, F32, np.repeat(tables, 3, 0), [length] * 3, length, 1.0)
    pre = run_prefill(device, 0, q[:1], F32, tables, [0, 1], [length - 1], length, 1.0)
    # Far apart: one page takes all.
    assert got[0, 0, 5] == 2.0 ** -6 and got[1, 0, 5] == 2.0 ** 40 and pre[0, 0, 5] == 2.0 ** -6
    want, err = cache.attention(0, q[2], tables[0], length, 1.0)
    assert np.all(np.abs(got[2] - want) <= err)
    assert np.all(np.delete(got, 5, axis=2) == 0)


def test_attention_beyond_what_is_there(torch_cuda):
    """Page ids outside the pool, a page past the table, a row longer than max_length, NaN in a page or in q: NaN in
    those rows and heads and nowhere else."""
    rng = np.random.default_rng(10)
    cache = Cache(12, 1, 2, 16, 64, INT8, rng)
    tables = np.array([[0, 1, 2], [3, -1, 4], [5, 12, 6], [7, 8, 9], [7, 8, 9], [10, 8, 9], [0, 1, 2]], dtype=np.int32)
    lengths = [48, 20, 33, 49, 48, 9, 48]
    cache.scales[10, 0, 1, 1] = np.nan
    q = rng.standard_normal((7, 4, 64)).astype(np.float32)
    q[6, 2, 7] = np.inf
    device = Device(torch_cuda, cache)
    lost = np.zeros((7, 4), dtype=bool)
    lost[[1, 2, 3]] = True
    lost[5, 2:] = True
    lost[6, 2] = True
    for longest in (64, 4000):
        got = run_decode(device, 0, q, F32, tables, lengths, longest, 0.1)
        assert np.array_equal(np.isnan(got).all(2), lost) and np.array_equal(np.isnan(got).any(2), lost)
        got = run_prefill(device, 0, q, F32, tables, range(8), [n - 1 for n in lengths], longest, 0.1)
        assert np.array_equal(np.isnan(got).all(2), lost) and np.array_equal(np.isnan(got).any(2), lost)
    lost[[0, 4, 6]] = True
    got = run_decode(device, 0, q, F32, tables, lengths, 47, 0.1)
    assert np.array_equal(np.isnan(got).all(2), lost)
    got = run_prefill(device, 0, q, F32, tables, range(8), [n - 1 for n in lengths], 47, 0.1)
    assert np.array_equal(np.isnan(got).all(2), lost)
    got = run_prefill(device, 0, q, F32, tables, range(8), [-1, -5, 2 ** 31 - 1, 2 ** 30, 47, 8, 47], 64, 0.1)
    lost[[0, 1, 2, 3]] = True
    lost[4] = lost[6] = False
    lost[6, 2] = True
    assert np.array_equal(np.isnan(got).all(2), lost)


@FORMATS
@pytest.mark.parametrize("dim, heads, kind", [(64, 3, F32), (128, 5, BF16), (256, 2, F32), (64, 2, F16)])
def test_prefill_rows_before_a_nan(torch_cuda, fmt, dim, heads, kind):
    """Rows of one work-group on both sides of a page of NaN keys, of NaN values, of no page at all, of the table's
    end and of max_length: those before are as without it, those after are NaN."""
    for case in ("keys", "values", "page", "table", "length"):
        rng = np.random.default_rng(15)
        cache = Cache(9, 1, 1, 16, dim, fmt, rng)
        tables = np.array([[3, 1, 4, 0, 5, 8]], dtype=np.int32)
        total, bad = 90, 48
        fill(cache, rng, tables, [total])
        q = rounded(rng.standard_normal((total, heads, dim)), kind)
        scale = 1 / dim ** 0.5
        clean = [cache.attention(0, q[i], tables[0], i + 1, scale) for i in range(total)]
        v_max = np.abs(cache.tokens(0, 1, tables[0], total)).max()
        longest, given = total, tables
        if case in ("keys", "values"):
            which = int(case == "values")
            cache.scales[0, 0, 0, which] = np.nan
            if fmt == E4M3:
                cache.bytes[which][0, 0, 0] = 0x7F  # what appending NaN leaves there
        elif case == "page":
            given = tables.copy()
            given[0, 3] = 9
        elif case == "table":
            given = np.ascontiguousarray(tables[:, :3])
        else:
            longest = bad
        device = Device(torch_cuda, cache)
        for many in (longest, 5000) if case != "length" else (longest,):
            got = run_prefill(device, 0, q, kind, given, [0, total], [0], many, scale)
            assert np.isnan(got[bad:]).all(), case
            for i in (0, 15, 16, 31, 40, 46, 47):
                check_row(got[i], *clean[i], kind, v_max, True, f"{case}, row {i}")


def test_out_over_q(torch_cuda):
    """The result in place of the queries, of one chunk and of several."""
    rng = np.random.default_rng(16)
    torch = torch_cuda
    cache = Cache(64, 1, 2, 16, 64, INT8, rng)
    tables = rng.integers(0, 64, (3, 300)).astype(np.int32)
    device = Device(torch, cache)
    q = (rng.standard_normal((3, 6, 64)) * 0.05).astype(np.float32)
    d_tables, d_lengths = device.ints(tables), device.ints([4800, 700, 33])
    starts, used = device.ints([0, 1, 2, 3]), device.ints([4799, 699, 32])
    for longest in (4800, 6000):
        want = run_decode(device, 0, q, F32, tables, [4800, 700, 33], longest, 0.125)
        space, size = workspace_for(device, 3, 3, 6, longest)
        x = torch.from_numpy(q.reshape(3, -1)).cuda()
        mp.kv8_attention_decode(device.view, 0, x.data_ptr(), 384, F32, d_tables.data_ptr(), 300, d_lengths.data_ptr(),
                                3, 6, longest, 0.125, x.data_ptr(), 384, space.data_ptr(), size)
        assert np.array_equal(device.back(x, 384).reshape(3, 6, 64), want)
        want = run_prefill(device, 0, q, F32, tables, [0, 1, 2, 3], [4799, 699, 32], longest, 0.125)
        x = torch.from_numpy(q.reshape(3, -1)).cuda()
        mp.kv8_attention_prefill(device.view, 0, x.data_ptr(), 384, F32, d_tables.data_ptr(), 300, starts.data_ptr(),
                                 used.data_ptr(), 3, 3, 6, longest, 0.125, x.data_ptr(), 384, space.data_ptr(), size)
        assert np.array_equal(device.back(x, 384).reshape(3, 6, 64), want)


def test_long_context(torch_cuda):
    """70,000 tokens of which the pool holds 128 pages again and again: splits of more than one batch, positions past
    16 bits; decode and a chunk of the last rows."""
    rng = np.random.default_rng(11)
    n, bt = 70001, 16
    cache = Cache(128, 1, 1, bt, 64, INT8, rng)
    tables = np.tile(np.arange(128, dtype=np.int32), -(-n // bt // 128) + 1)[None, :-(-n // bt)]
    device = Device(torch_cuda, cache)
    q = rng.standard_normal((3, 3, 64)).astype(np.float32) * 0.05
    got = run_decode(device, 0, q[2:], F32, tables, [n], n, 0.125)[0]
    pre = run_prefill(device, 0, q, F32, tables, [0, 3], [n - 3], n, 0.125)
    v_max = np.abs(cache.tokens(0, 1, tables[0], n)).max()
    for i in range(3):
        want, err = cache.attention(0, q[i], tables[0], n - 2 + i, 0.125)
        check_row(pre[i], want, err, F32, v_max, True, f"row {i}")
        if i == 2:
            check_row(got, want, err, F32, v_max, False, "decode")


# ---- together ----------------------------------------------------------------


def test_pool_past_four_gigabytes(torch_cuda):
    """A pool whose last pages lie past 2^32 bytes: append there, read and attend."""
    torch, blocks = torch_cuda, (1 << 32) // (16 * 64) + 40
    pools = [torch.full((blocks, 16 * 64), 128, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = torch.ones((blocks, 2), device="cuda")
    view = mp.Kv8Cache(pools[0].data_ptr(), pools[1].data_ptr(), scales.data_ptr(), blocks, 1, 16, 1, 64, INT8)
    rng = np.random.default_rng(12)
    small = Cache(4, 1, 1, 16, 64, INT8, rng)
    k, v = (rng.standard_normal((30, 1, 64)).astype(np.float32) for _ in range(2))
    small.append(0, k, v, np.array([[1, 3]]), [0, 30], [0])
    ints = [torch.tensor(a, dtype=torch.int32, device="cuda") for a in ([[blocks - 3, blocks - 1]], [0, 30], [0], [30])]
    rows = [torch.from_numpy(a.reshape(30, 64)).cuda() for a in (k, v)]
    mp.kv8_append(view, 0, rows[0].data_ptr(), 64, rows[1].data_ptr(), 64, F32, ints[0].data_ptr(), 2,
                  ints[1].data_ptr(), ints[2].data_ptr(), 1, 30)
    q = rng.standard_normal((1, 2, 64)).astype(np.float32)
    dq, out = torch.from_numpy(q.reshape(1, -1)).cuda(), torch.zeros((1, 128), device="cuda")
    mp.kv8_attention_decode(view, 0, dq.data_ptr(), 128, F32, ints[0].data_ptr(), 2, ints[3].data_ptr(), 1, 2, 32,
                            0.125, out.data_ptr(), 128)
    back = [torch.zeros((30, 64), device="cuda") for _ in range(2)]
    mp.kv8_read(view, 0, ints[0].data_ptr(), 2, ints[1].data_ptr(), ints[2].data_ptr(), 1, 30, F32,
                back[0].data_ptr(), 64, back[1].data_ptr(), 64)
    torch.cuda.synchronize()
    for kind in range(2):
        assert np.array_equal(back[kind].cpu().numpy(), small.tokens(0, kind, [1, 3], 30)[0].astype(np.float32))
        assert bool((pools[kind][:40] == 128).all())
    want, err = small.attention(0, q[0], [1, 3], 30, 0.125)
    check_row(out.cpu().numpy().reshape(2, 64), want, err, F32, 0, False, "decode")


class Service:
    """Three sequences over a two-layer cache: a prompt step, then decode steps, each layer an append and an
    attention, on a stream of its own."""

    def __init__(self, torch, fmt, kind):
        self.torch, self.kind, self.rng = torch, kind, np.random.default_rng(13 + fmt)
        self.kv_heads, self.heads, self.dim, self.bt, self.layers, self.most = 2, 6, 64, 16, 2, 400
        self.counts = [37, 150, 5]
        self.cache = Cache(3 * 25 + 1, 2, 2, 16, 64, fmt, self.rng)
        self.device = Device(torch, self.cache)
        self.tables = self.rng.permutation(75).astype(np.int32).reshape(3, 25)
        self.d_tables = self.device.ints(self.tables)
        self.cos, self.sin = angles(self.most, 64)
        self.angles = [torch.from_numpy(a).cuda() for a in (self.cos, self.sin)]
        self.rope = mp.Rope(self.angles[0].data_ptr(), self.angles[1].data_ptr(), self.most, 64, 0)
        self.space, self.size = workspace_for(self.device, 192, 3, 6, self.most)

    def rows(self, n):
        return [rounded(self.rng.standard_normal((n, 6 + 2 + 2, 64)), self.kind) for _ in range(self.layers)]

    def want(self, qkv, starts, used):
        """The reference's step: outputs and bounds of every row and layer."""
        from .kv8_reference import rotate
        out = []
        for layer in range(self.layers):
            x = qkv[layer]
            self.cache.append(layer, x[:, 6:8], x[:, 8:], self.tables, starts, used, (self.cos, self.sin, 64, False))
            rows = []
            for s in range(3):
                for i in range(starts[s + 1] - starts[s]):
                    p = used[s] + i
                    q = rounded(rotate(x[starts[s] + i, :6], self.cos[p], self.sin[p], 64, False), self.kind)
                    rows.append(self.cache.attention(layer, q, self.tables[s], p + 1, 0.125))
            out.append(rows)
        return out

    def launch(self, qkv, out, starts, used, lengths, n, stream):
        """qkv, out: per layer a device matrix; lengths: None for a prompt step."""
        for layer in range(self.layers):
            size = qkv[layer].element_size()
            at, width, o = qkv[layer].data_ptr(), 10 * 64, out[layer].data_ptr()
            mp.kv8_append(self.device.view, layer, at + 6 * 64 * size, width, at + 8 * 64 * size, width, self.kind,
                          self.d_tables.data_ptr(), 25, starts.data_ptr(), used.data_ptr(), 3, n, rope=self.rope, q=at,
                          q_stride=width, q_out=at, q_out_stride=width, heads=6, stream=stream)
            if lengths is None:
                mp.kv8_attention_prefill(self.device.view, layer, at, width, self.kind, self.d_tables.data_ptr(), 25,
                                         starts.data_ptr(), used.data_ptr(), 3, n, 6, self.most, 0.125, o, 384,
                                         self.space.data_ptr(), self.size, stream=stream)
            else:
                mp.kv8_attention_decode(self.device.view, layer, at, width, self.kind, self.d_tables.data_ptr(), 25,
                                        lengths.data_ptr(), n, 6, self.most, 0.125, o, 384, self.space.data_ptr(),
                                        self.size, stream=stream)

    def check(self, got, want, prefill, what):
        for layer in range(self.layers):
            x = got[layer].float().cpu().numpy().reshape(-1, 6, 64)
            v_max = max(np.nanmax(np.abs(self.cache.tokens(layer, 1, t, self.bt))) for t in self.tables) * 4
            for r, (w, err) in enumerate(want[layer]):
                check_row(x[r], w, err, self.kind, v_max, prefill, f"{what}, layer {layer}, row {r}")


@FORMATS
@pytest.mark.parametrize("kind", [F32, BF16], ids=["f32", "bf16"])
def test_serving_with_a_replayed_graph(torch_cuda, fmt, kind):
    """A prompt step, one direct decode step, then decode steps replayed from one graph of both layers' calls, whose
    positions and rows change in place, with other work between the replays."""
    torch = torch_cuda
    service = Service(torch, fmt, kind)
    dtype = getattr(torch, TYPES[kind])
    stream = torch.cuda.Stream()
    starts, used = starts_of(service.counts), np.zeros(3, dtype=np.int32)
    n = int(starts[-1])
    x = service.rows(n)
    d = [torch.from_numpy(a.reshape(n, -1)).to("cuda", dtype) for a in x]
    out = [torch.zeros((n, 384), dtype=dtype, device="cuda") for _ in range(2)]
    d_starts, d_used = service.device.ints(starts), service.device.ints(used)
    torch.cuda.synchronize()
    service.launch(d, out, d_starts, d_used, None, n, stream.cuda_stream)
    stream.synchronize()
    service.check(out, service.want(x, starts, used), True, "prompt")
    used = np.array(service.counts, dtype=np.int32)
    one = service.device.ints([0, 1, 2, 3])
    d_used, d_lengths = service.device.ints(used), service.device.ints(used + 1)
    step = [torch.zeros((3, 640), dtype=dtype, device="cuda") for _ in range(2)]
    result = [torch.zeros((3, 384), dtype=dtype, device="cuda") for _ in range(2)]
    graph = torch.cuda.CUDAGraph()
    for i in range(7):
        x = service.rows(3)
        for a, b in zip(step, x):
            a.copy_(torch.from_numpy(b.reshape(3, -1)))
        d_used.copy_(torch.from_numpy(used))
        d_lengths.copy_(torch.from_numpy(used + 1))
        torch.cuda.synchronize()
        if i == 0:
            service.launch(step, result, one, d_used, d_lengths, 3, stream.cuda_stream)
            stream.synchronize()
        else:
            if i == 1:
                with torch.cuda.graph(graph, stream=stream):
                    service.launch(step, result, one, d_used, d_lengths, 3, stream.cuda_stream)
                service.space.fill_(255)
            graph.replay()
            torch.cuda.synchronize()
        service.check(result, service.want(x, [0, 1, 2, 3], used), False, f"step {i}")
        service.device.check_bytes(service.cache)
        used = used + 1


def test_two_streams_with_workspaces_of_their_own(torch_cuda):
    """Two decode calls that may overlap give what each gives alone, bit for bit, again and again."""
    torch = torch_cuda
    rng = np.random.default_rng(14)
    cache = Cache(400, 1, 3, 16, 64, INT8, rng)
    device = Device(torch, cache)
    calls = []
    for i, longest in enumerate((3000, 2500)):
        tables = rng.integers(0, 400, (4, 188)).astype(np.int32)
        lengths = [longest, 1, longest // 2, 700]
        q = torch.from_numpy((rng.standard_normal((4, 576)) * 0.05).astype(np.float32)).cuda()
        space, size = workspace_for(device, 4, 4, 9, longest)
        calls.append((q, device.ints(tables), device.ints(lengths), longest, space, size,
                      torch.zeros((4, 576), device="cuda"), torch.cuda.Stream()))

    def launch(c, stream):
        q, tables, lengths, longest, space, size, out, _ = c
        mp.kv8_attention_decode(device.view, 0, q.data_ptr(), 576, F32, tables.data_ptr(), 188, lengths.data_ptr(), 4,
                                9, longest, 0.125, out.data_ptr(), 576, space.data_ptr(), size, stream=stream)

    torch.cuda.synchronize()
    alone = []
    for c in calls:
        launch(c, None)
        torch.cuda.synchronize()
        alone.append(c[6].clone())
        assert bool(c[6].isfinite().all())
    for _ in range(20):
        for c in calls:
            c[6].zero_()
        torch.cuda.synchronize()
        for c in calls:
            launch(c, c[7].cuda_stream)
        torch.cuda.synchronize()
        for c, want in zip(calls, alone):
            assert torch.equal(c[6], want)


def test_prefill_replayed_with_other_rows(torch_cuda):
    """One captured prompt step (append and prefill attention of two layers) replayed for other counts: more and fewer
    rows, sequences without any, single tokens, rows behind the last sequence left alone."""
    torch = torch_cuda
    service = Service(torch, INT8, F32)
    capacity = 60
    d = [torch.zeros((capacity, 640), device="cuda") for _ in range(2)]
    out = [torch.zeros((capacity, 384), device="cuda") for _ in range(2)]
    d_starts, d_used = service.device.ints([0, 0, 0, 0]), service.device.ints([0, 0, 0])
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    service.launch(d, out, d_starts, d_used, None, capacity, stream.cuda_stream)
    stream.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        service.launch(d, out, d_starts, d_used, None, capacity, stream.cuda_stream)
    used = np.zeros(3, dtype=np.int32)
    for counts in ([20, 33, 7], [1, 1, 1], [0, 50, 0], [17, 0, 30], [0, 0, 0], [40, 1, 2]):
        starts = starts_of(counts)
        x = service.rows(capacity)
        for a, b in zip(d, x):
            a.copy_(torch.from_numpy(b.reshape(capacity, -1)))
        for o in out:
            o.fill_(7.0)
        d_starts.copy_(torch.from_numpy(starts))
        d_used.copy_(torch.from_numpy(used))
        service.space.fill_(255)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        service.check(out, service.want(x, starts, used), True, f"counts {counts}")
        service.device.check_bytes(service.cache)
        for o in out:
            assert bool((o[int(starts[-1]):] == 7.0).all())
        used = used + np.array(counts, dtype=np.int32)


@pytest.mark.parametrize("seed", range(16))
def test_any_shape(torch_cuda, seed):
    """Everything drawn: heads, dims, pages, formats, types, paddings, alignments, rotations, counts and lengths; three
    steps of append and prefill, then decode, then reading back."""
    from .kv8_reference import rotate
    rng = np.random.default_rng(1000 + seed)
    pick = lambda *a: a[rng.integers(len(a))]
    kv_heads, group = int(pick(1, 2, 3, 5, 8)), int(pick(1, 2, 3, 4, 7, 8, 9, 16))
    heads, dim, bt = kv_heads * group, int(pick(64, 64, 128, 256)), int(pick(16, 32, 64, 128))
    fmt, kind = int(pick(INT8, E4M3)), int(pick(F32, BF16, F16))
    pad, shift = int(pick(0, 0, 1, 4, 8)), int(pick(0, 0, 1, 4))
    dims, interleaved = int(pick(0, dim, dim // 2, 2, 22)), bool(rng.integers(2))
    sequences, steps = int(pick(1, 2, 5)), 3
    counts = rng.integers(0, int(pick(2, 20, 90)), (steps, sequences)) + (rng.random((steps, sequences)) < 0.3)
    total = counts.sum(0) + 1
    cache = Cache(blocks_for(total, bt), 2, kv_heads, bt, dim, fmt, rng)
    tables = tables_for(rng, cache.blocks, total, bt)
    device = Device(torch_cuda, cache)
    cos, sin = angles(int(total.max()) + 1, dims)
    d_cos, d_sin = torch_cuda.from_numpy(cos).cuda(), torch_cuda.from_numpy(sin).cuda()
    rope = mp.Rope(d_cos.data_ptr(), d_sin.data_ptr(), len(cos), dims, int(interleaved))
    layer, scale = int(rng.integers(2)), float(rng.uniform(0.5, 1.5)) / dim ** 0.5
    used = np.zeros(sequences, dtype=np.int32)
    d_tables = device.ints(tables)
    what = f"{kv_heads}x{group} dim {dim} bt {bt} fmt {fmt} type {kind} pad {pad} shift {shift} rope {dims} {interleaved}"
    for step in range(steps + 1):
        new = counts[step] if step < steps else np.ones(sequences, dtype=np.int64)
        starts = starts_of(new)
        rows = int(starts[-1]) + 1
        q, k, v = (rounded(rng.standard_normal((rows, h, dim)) * 1.5 ** step, kind) for h in (heads, kv_heads, kv_heads))
        mq, q_at, q_stride = device.rows(q.reshape(rows, -1), kind, pad, shift)
        mk, k_at, k_stride = device.rows(k.reshape(rows, -1), kind, pad, shift)
        mv, v_at, v_stride = device.rows(v.reshape(rows, -1), kind, pad, shift)
        d_starts, d_used = device.ints(starts), device.ints(used)
        mp.kv8_append(device.view, layer, k_at, k_stride, v_at, v_stride, kind, d_tables.data_ptr(), tables.shape[1],
                      d_starts.data_ptr(), d_used.data_ptr(), sequences, rows, rope=rope, q=q_at, q_stride=q_stride,
                      q_out=q_at, q_out_stride=q_stride, heads=heads)
        cache.append(layer, k, v, tables, starts, used, (cos, sin, dims, interleaved))
        device.check_bytes(cache)
        turned = device.back(mq, heads * dim).reshape(rows, heads, dim)
        for s in range(sequences):
            for i in range(int(new[s])):
                r, p = starts[s] + i, used[s] + i
                want = rounded(rotate(q[r], cos[p], sin[p], dims, interleaved), kind) if dims else q[r]
                assert np.array_equal(turned[r], want), what
        longest = int((used + new).max()) + int(pick(0, 1, 5000))
        if step < steps:
            got = run_prefill(device, layer, turned, kind, tables, starts, used, longest, scale, pad, shift)
        else:
            got = run_decode(device, layer, turned[:sequences], kind, tables, used + 1, longest, scale, pad, shift)
        for s in range(sequences):
            if not new[s]:
                continue
            v_max = np.abs(cache.tokens(layer, 1, tables[s], int(used[s] + new[s]))).max()
            for i in sorted({0, int(new[s]) // 2, int(new[s]) - 1}):
                r = starts[s] + i
                want, err = cache.attention(layer, turned[r], tables[s], int(used[s]) + i + 1, scale)
                check_row(got[r], want, err, kind, v_max, step < steps, f"{what}: step {step}, sequence {s}, row {i}")
        used = used + new.astype(np.int32)
    starts = starts_of(used)
    rows = int(starts[-1])
    out = [device.rows(np.zeros((rows, kv_heads * dim)), kind, pad, shift) for _ in range(2)]
    d_starts, d_used = device.ints(starts), device.ints(np.zeros(sequences))
    mp.kv8_read(device.view, layer, d_tables.data_ptr(), tables.shape[1], d_starts.data_ptr(), d_used.data_ptr(),
                sequences, rows, kind, out[0][1], out[0][2], out[1][1], out[1][2])
    for which in range(2):
        want = np.concatenate([cache.tokens(layer, which, tables[s], int(used[s])).transpose(1, 0, 2) for s in range(sequences)])
        assert np.array_equal(device.back(out[which][0], kv_heads * dim), rounded(want.reshape(rows, -1), kind)), what


@FORMATS
@pytest.mark.parametrize("dim, heads, kind", [(64, 3, F32), (64, 2, BF16), (128, 5, BF16), (256, 2, F32), (256, 16, F32)])
def test_values_of_far_magnitudes(torch_cuda, fmt, dim, heads, kind):
    """Pages of values up to 2^200 apart: every row is right to the largest value that it sees, whatever the pages
    behind it hold, whether a page shares a pair of tiles with the larger one or comes pairs later."""
    rng = np.random.default_rng(20)
    total = 150
    for name, powers in (("up", [-60, -30, -14, 0, 9, 30, 60, 90, 100, 110]),
                         ("down", [100, 80, 60, 40, 20, 0, -20, -40, -60, -80]),
                         ("leaps", [-100, 100, -100, 90, 0, 20, 101, -126, 17, 110]),
                         ("zeros", [-200, 0, -200, -200, 7, 7, 30, -200, -200, 50])):
        cache = Cache(10, 1, 1, 16, dim, fmt, rng)
        tables = rng.permutation(10).astype(np.int32)[None]
        k, v = (rng.standard_normal((total, 1, dim)).astype(np.float32) for _ in range(2))
        for page, power in enumerate(powers):
            v[16 * page:16 * page + 16] *= np.float32(2.0 ** power if power > -200 else 0)
        cache.append(0, k, v, tables, [0, total], [0])
        q = rounded(rng.standard_normal((total, heads, dim)), kind)
        scale = 1 / dim ** 0.5
        device = Device(torch_cuda, cache)
        values = np.abs(cache.tokens(0, 1, tables[0], total)).max((0, 2))
        for many in (total, 600, 60000):
            got = run_prefill(device, 0, q, kind, tables, [0, total], [0], many, scale)
            for i in range(total):
                want, err = cache.attention(0, q[i], tables[0], i + 1, scale)
                check_row(got[i], want, err, kind, values[:i + 1].max(), True, f"{name}, at most {many}, row {i}")
        lengths = np.array([1, 15, 16, 17, 32, 40, 48, 64, 100, total], dtype=np.int32)
        got = run_decode(device, 0, q[lengths - 1], kind, np.repeat(tables, 10, 0), lengths, total, scale)
        for i, n in enumerate(lengths):
            want, err = cache.attention(0, q[n - 1], tables[0], int(n), scale)
            check_row(got[i], want, err, kind, values[:n].max(), False, f"{name}, decode of {n}")


@FORMATS
@pytest.mark.parametrize("dim, heads", [(64, 1), (64, 16), (128, 4), (256, 2)])
@pytest.mark.parametrize("kind", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_prefill_probabilities_are_not_rounded_to_16_bits(torch_cuda, fmt, dim, heads, kind):
    """Tokens in turn of probability 1 and value 1, and of probability (1 + 2^-11)/2 and value -2: after an even number
    of them the result is -2^-11 / 1.5 (to 2^-12), of which a probability rounded to FP16 leaves 0 or twice as much: off
    by 3.3e-4 where FP32 arithmetic is by 7e-5 at most (kv8_reference.bound) and the row type's half step is 1.3e-6."""
    total, rng = 64, np.random.default_rng(21)
    cache = Cache(5, 1, 1, 16, dim, fmt, rng)
    tables = np.array([[3, 0, 4, 1]], dtype=np.int32)
    code = {x: (128 + x if fmt == INT8 else int(np.flatnonzero(VALUES[E4M3] == x)[0])) for x in (0, 1, -2)}
    cache.scales[:] = 1
    for page in tables[0]:
        for which, even, odd in ((0, 0, 1), (1, 1, -2)):
            data = cache.bytes[which][page, 0, 0]
            data[:] = code[0]
            data[cache.places[which][0::2, 3]] = code[even]
            data[cache.places[which][1::2, 3]] = code[odd]
    q = np.zeros((total, heads, dim), dtype=np.float32)
    q[:, :, 3] = -1
    scale = float(np.float32(np.log(2) - np.log1p(2.0 ** -11)))
    device = Device(torch_cuda, cache)
    for longest in (total, 1 << 20):
        got = run_prefill(device, 0, q, kind, tables, [0, total], [0], longest, scale)
        for i in range(total):
            want, err = cache.attention(0, q[i], tables[0], i + 1, scale)
            assert i % 2 == 0 or abs(want[0, 3] + 2.0 ** -11 / 1.5) < 2.0 ** -12 and err.max() < 7e-5
            check_row(got[i], want, err, kind, 0, False, f"row {i} of {longest}")


@pytest.mark.parametrize("dim, heads, kind", [(64, 3, F32), (128, 5, BF16), (256, 2, F32), (64, 16, F16), (128, 16, F32)])
def test_nan_bytes_among_the_values(torch_cuda, dim, heads, kind):
    """Single E4M3 NaN bytes under finite scales, anywhere in a pair of tiles: a row that sees one is NaN in its dim and
    right in the others, one before it is right in all; alone, split, and in the batch that two column tiles take."""
    rng = np.random.default_rng(22)
    total, n = 90, 24
    cache = Cache(7, 1, 1, 16, dim, E4M3, rng)
    tables = np.array([[3, 1, 4, 0, 5, 6]], dtype=np.int32)
    fill(cache, rng, tables, [total])
    q = rounded(rng.standard_normal((total, heads, dim)), kind)
    scale = 1 / dim ** 0.5
    clean = [cache.attention(0, q[i], tables[0], i + 1, scale) for i in range(total)]
    bad = [(17, 5, 0x7F), (18, 5, 0xFF), (31, 16, 0x7F), (32, 63, 0xFF), (47, 0, 0x7F), (48, dim - 1, 0x7F), (77, 20, 0xFF), (89, 33, 0x7F)]
    for token, d, byte in bad:
        cache.bytes[1][tables[0, token // 16], 0, 0, cache.places[1][token % 16, d]] = byte
    lost = np.zeros((total, dim), dtype=bool)
    for token, d, _ in bad:
        lost[token:, d] = True
    device = Device(torch_cuda, cache)

    def check(got, what):
        for i in range(total):
            assert np.array_equal(np.isnan(got[i]), np.repeat(lost[i:i + 1], heads, 0)), f"{what}, row {i}"
            want, err = clean[i]
            check_row(got[i][:, ~lost[i]], want[:, ~lost[i]], err, kind, 0, False, f"{what}, row {i}")

    for longest in (total, 5000, 20000):
        check(run_prefill(device, 0, q, kind, tables, [0, total], [0], longest, scale), f"at most {longest}")
    # Chunks behind a history, so that other tokens are the first and the last of a work-group.
    for first in (16, 18, 47, 61):
        got = run_prefill(device, 0, q[first:], kind, tables, [0, total - first], [first], total, scale)
        check(np.concatenate((np.where(lost[:first, None], np.nan, [rounded(c[0], kind) for c in clean[:first]]), got)), f"from {first}")
    many = np.arange(n + 1) * total
    for longest in (total, 6000):
        got = run_prefill(device, 0, np.tile(q, (n, 1, 1)), kind, np.repeat(tables, n, 0), many, [0] * n, longest, scale)
        for s in (0, 13, n - 1):
            check(got[many[s]:many[s + 1]], f"sequence {s} of {n}, at most {longest}")
    lengths = np.array([17, 18, 31, 48, 77, 78, 90], dtype=np.int32)
    for longest in (total, 5000):
        got = run_decode(device, 0, q[lengths - 1], kind, np.repeat(tables, 7, 0), lengths, longest, scale)
        for i, m in enumerate(lengths):
            assert np.array_equal(np.isnan(got[i]), np.repeat(lost[m - 1:m], heads, 0))


@FORMATS
def test_prompt_past_the_rotation_tables(torch_cuda, fmt):
    """A prompt that runs past the rotation tables is appended without its last rows, whose slots keep what was there:
    the rows before them are right, those past the tables are NaN."""
    torch, rng = torch_cuda, np.random.default_rng(23)
    total, most, heads, dim = 60, 38, 3, 64
    cache = Cache(5, 1, 1, 16, dim, fmt, rng)
    if fmt == E4M3:
        for b in cache.bytes:
            b[rng.random(b.shape) < 0.1] = 0x7F
    tables = np.array([[2, 0, 4, 1]], dtype=np.int32)
    x = rng.standard_normal((total, heads + 2, dim)).astype(np.float32)
    cos, sin = angles(most, dim)
    device = Device(torch, cache)
    d = torch.from_numpy(x.reshape(total, -1)).cuda()
    d_angles = [torch.from_numpy(a).cuda() for a in (cos, sin)]
    rope = mp.Rope(d_angles[0].data_ptr(), d_angles[1].data_ptr(), most, dim, 0)
    ints = [device.ints(a) for a in (tables, [0, total], [0])]
    at, width = d.data_ptr(), x.shape[1] * dim
    mp.kv8_append(device.view, 0, at + 4 * heads * dim, width, at + 4 * (heads + 1) * dim, width, F32,
                  ints[0].data_ptr(), 4, ints[1].data_ptr(), ints[2].data_ptr(), 1, total, rope=rope, q=at,
                  q_stride=width, q_out=at, q_out_stride=width, heads=heads)
    cache.append(0, x[:, heads:heads + 1], x[:, heads + 1:], tables, [0, total], [0], (cos, sin, dim, False))
    device.check_bytes(cache)
    turned = device.back(d, heads * dim).reshape(total, heads, dim)
    for longest in (total, 5000):
        got = run_prefill(device, 0, turned, F32, tables, [0, total], [0], longest, 0.125)
        assert np.isnan(got[most:]).all()
        for i in range(most):
            want, err = cache.attention(0, turned[i], tables[0], i + 1, 0.125)
            check_row(got[i], want, err, F32, 0, False, f"row {i} of {longest}")


@FORMATS
@pytest.mark.parametrize("power", [-126, -115])
@pytest.mark.parametrize("dim, heads, kind", [(64, 3, F32), (128, 12, BF16), (256, 2, F32)])
def test_values_near_the_smallest(torch_cuda, fmt, power, dim, heads, kind):
    """Value scales of the smallest numbers over up to 20,000 tokens: the result is a normal float of the values' size,
    and as near as for any other scale; decode and prefill, alone and split."""
    rng = np.random.default_rng(24)
    cache = Cache(40, 1, 1, 16, dim, fmt, rng)
    for b in cache.bytes:  # keys of both signs, positive values
        b[:] = rng.integers(1, 256, b.shape) if fmt == INT8 else rng.integers(0, 0x7F, b.shape)
    cache.bytes[1][:] = rng.integers(130, 256, cache.bytes[1].shape) if fmt == INT8 else rng.integers(0x38, 0x7F, cache.bytes[1].shape)
    cache.scales[..., 0] = 2.0 ** -9
    cache.scales[..., 1] = 2.0 ** power
    tables = rng.integers(0, 40, (4, 1250)).astype(np.int32)
    lengths = [3, 64, 1000, 20000]
    q = rounded(rng.standard_normal((4, heads, dim)) * 0.1, kind)
    device = Device(torch_cuda, cache)
    want = [cache.attention(0, q[i], tables[i], lengths[i], 0.1) for i in range(4)]
    for pick, longest in (([0, 1], 64), ([0, 1, 2], 1000), ([0, 1, 2, 3], 20000)):
        got = run_decode(device, 0, q[pick], kind, tables[pick], [lengths[i] for i in pick], longest, 0.1)
        pre = run_prefill(device, 0, q[pick], kind, tables[pick], np.arange(len(pick) + 1), [lengths[i] - 1 for i in pick],
                          longest, 0.1)
        for i in pick:
            assert np.all(want[i][0] > 2.0 ** -126.01)  # no smaller than the smallest value
            check_row(got[i], *want[i], kind, 0, False, f"decode of {lengths[i]}, at most {longest}")
            check_row(pre[i], *want[i], kind, 0, False, f"prefill at {lengths[i]}, at most {longest}")


@pytest.mark.parametrize("dims", [0, 64])
def test_append_of_sequences_without_positions(torch_cuda, dims):
    """Sequences at positions below 0 or past 2^30 write no tokens; their queries pass, or are NaN where they turn. The
    others are as without them."""
    rng = np.random.default_rng(25)
    cache = Cache(4, 1, 1, 16, 64, INT8, rng)
    device = Device(torch_cuda, cache)
    tables = np.array([[0, 1], [2, 3], [0, 1], [2, 2], [3, 3]], dtype=np.int32)
    counts, used = [3, 20, 2, 2, 2], np.array([-1, 5, -2 ** 31, 2 ** 30 + 1, 2 ** 31 - 1], dtype=np.int32)
    starts = starts_of(counts)
    rows = int(starts[-1])
    k, v, q = (rng.standard_normal((rows, 1, 64)).astype(np.float32) for _ in range(3))
    cos, sin = angles(30, 64)
    d_angles = [torch_cuda.from_numpy(a).cuda() for a in (cos, sin)]
    rope = mp.Rope(d_angles[0].data_ptr(), d_angles[1].data_ptr(), 30, dims, 0)
    mk, mv, mq, mo = (device.rows(x.reshape(rows, -1), F32) for x in (k, v, q, np.zeros((rows, 64))))
    ints = [device.ints(a) for a in (tables, starts, used)]
    mp.kv8_append(device.view, 0, mk[1], 64, mv[1], 64, F32, ints[0].data_ptr(), 2, ints[1].data_ptr(),
                  ints[2].data_ptr(), 5, rows, rope=rope, q=mq[1], q_stride=64, q_out=mo[1], q_out_stride=64, heads=1)
    cache.append(0, k[3:23], v[3:23], tables[1:2], [0, 20], [5], (cos, sin, dims, False))
    device.check_bytes(cache)
    got, inside = device.back(mo[0], 64), (np.arange(rows) >= 3) & (np.arange(rows) < 23)
    if dims:
        assert np.isnan(got[~inside]).all() and np.isfinite(got[inside]).all()
    else:
        assert np.array_equal(got, q.reshape(rows, 64))


def check_close(got, want, err, kind, what):
    limit = err + HALF_STEP[kind] * np.abs(want)
    off = np.abs(got - want)
    assert np.all(off <= limit), f"{what}: off by {off.max():.3e}, {float((off / limit).max()):.2f} of what is allowed"


@FORMATS
@pytest.mark.parametrize("kv_heads, heads, dim, bt, kind, pad, shift", SHAPES)
def test_attention_is_close(torch_cuda, fmt, kv_heads, heads, dim, bt, kind, pad, shift):
    """Rows of ordinary data within what rounding to FP32 gives in earnest (kv8_reference.likely_bound), far below its
    worst case: a query or a probability held in a single 16-bit number is found out
    (test_kv8_rules.test_single_parts_are_too_far_off)."""
    rng = np.random.default_rng(heads * dim + bt + 7)
    lengths = [n for n in LENGTHS if n > 0]
    cache = Cache(blocks_for(lengths, bt), 1, kv_heads, bt, dim, fmt, rng)
    tables = tables_for(rng, cache.blocks, lengths, bt)
    fill(cache, rng, tables, lengths)
    device = Device(torch_cuda, cache)
    q = rounded(rng.standard_normal((len(lengths), heads, dim)), kind)
    scale = 1.3 / dim ** 0.5
    rows = np.arange(len(lengths) + 1)
    want = [attention_close(cache, 0, q[i], tables[i], n, scale) for i, n in enumerate(lengths)]
    for longest in (777, 5000, 100000):
        got = run_decode(device, 0, q, kind, tables, lengths, longest, scale, pad, shift)
        pre = run_prefill(device, 0, q, kind, tables, rows, [n - 1 for n in lengths], longest, scale, pad, shift)
        for i, n in enumerate(lengths):
            check_close(got[i], *want[i], kind, f"decode of {n} of at most {longest}")
            check_close(pre[i], *want[i], kind, f"prefill at {n} of at most {longest}")
    # A whole prompt.
    total = 129
    cache = Cache(blocks_for([total], bt), 1, kv_heads, bt, dim, fmt, rng)
    tables = tables_for(rng, cache.blocks, [total], bt)
    fill(cache, rng, tables, [total])
    device = Device(torch_cuda, cache)
    q = rounded(rng.standard_normal((total, heads, dim)), kind)
    for longest in (total, 100000):
        got = run_prefill(device, 0, q, kind, tables, [0, total], [0], longest, scale, pad, shift)
        for i in (0, 1, 2, 14, 15, 16, 17, 31, 32, 40, 63, 64, 100, 127, 128):
            want, err = attention_close(cache, 0, q[i], tables[0], i + 1, scale)
            check_close(got[i], want, err, kind, f"row {i} of at most {longest}")


@pytest.mark.parametrize("walk", WALKS, ids=[w.name for w in WALKS])
def test_wavefronts_that_walk_far(torch_cuda, walk):
    """Every page with scales of its own and nearly equal scores, so that a page or a scale taken from another place
    shows: calls beyond 32 and 64 steps of a wavefront, and of eight wavefronts. Lengths from half the longest on."""
    rng = np.random.default_rng(len(walk.name) + walk.dim)
    cache = Cache(300, 1, walk.kv_heads, walk.bt, walk.dim, walk.fmt, rng)
    if walk.fmt == E4M3:
        for b in cache.bytes:
            b[(b & 127) == 127] = 0
    for kind, low, high in ((0, -10, -7), (1, -3, 4)):
        cache.scales[..., kind] = 2.0 ** rng.integers(low, high, cache.scales.shape[:-1]).astype(np.float32)
    n, counts, heads = len(walk.counts), np.array(walk.counts), walk.kv_heads * walk.group
    lengths = np.linspace(walk.longest // 2, walk.longest, n).astype(np.int32)
    tables = rng.integers(0, 300, (n, -(-walk.longest // walk.bt))).astype(np.int32)
    device, scale = Device(torch_cuda, cache), 1 / walk.dim ** 0.5
    q = rounded(rng.standard_normal((int(counts.sum()), heads, walk.dim)) * 0.5, walk.kind)
    starts = starts_of(counts)
    if walk.decode:
        got = run_decode(device, 0, q, walk.kind, tables, lengths, walk.longest, scale)
    else:
        got = run_prefill(device, 0, q, walk.kind, tables, starts, lengths - counts, walk.longest, scale)
    assert np.isfinite(got).all()
    for s in sorted({0, n // 3, n - 2, n - 1}):
        for i in {0, int(counts[s]) - 1}:
            r = starts[s] + i
            want, err = attention_close(cache, 0, q[r], tables[s], int(lengths[s] - counts[s]) + i + 1, scale)
            check_close(got[r], want, err, walk.kind, f"sequence {s}, row {i}")


@pytest.mark.parametrize("walk", [w for w in WALKS if w.fmt == E4M3 and not w.decode and max(w.counts) > 1],
                         ids=lambda w: w.name)
def test_nan_bytes_at_the_end_of_a_far_walk(torch_cuda, walk):
    """NaN bytes among the values of each sequence's last page, which only some of its last rows see, behind walks whose
    tile places have been exchanged: NaN in those rows' dims and nowhere else."""
    rng = np.random.default_rng(26 + walk.dim)
    n, counts, heads = len(walk.counts), np.array(walk.counts), walk.kv_heads * walk.group
    cache = Cache(100 + n, 1, walk.kv_heads, walk.bt, walk.dim, E4M3, rng)
    for b in cache.bytes:
        b[(b & 127) == 127] = 0
    cache.scales[:] = 2.0 ** -9
    lengths = np.linspace(walk.longest - 40, walk.longest, n).astype(np.int32)
    tables = rng.integers(0, 100, (n, -(-walk.longest // walk.bt))).astype(np.int32)
    lost = np.zeros((int(counts.sum()), walk.kv_heads, walk.dim), dtype=bool)
    starts = starts_of(counts)
    for s in range(n):
        page = (lengths[s] - 1) // walk.bt
        tables[s, page] = 100 + s
        for _ in range(4):
            slot, head, d = rng.integers(lengths[s] - page * walk.bt), rng.integers(walk.kv_heads), rng.integers(walk.dim)
            cache.bytes[1][100 + s, 0, head, cache.places[1][slot, d]] = rng.choice([0x7F, 0xFF])
            first = max(page * walk.bt + slot - (lengths[s] - counts[s]), 0)  # row that is the first to see it
            lost[starts[s] + first:starts[s + 1], head, d] = True
    device = Device(torch_cuda, cache)
    q = rounded(rng.standard_normal((int(counts.sum()), heads, walk.dim)) * 0.5, walk.kind)
    got = run_prefill(device, 0, q, walk.kind, tables, starts, lengths - counts, walk.longest, 1 / walk.dim ** 0.5)
    assert lost.any() and not lost.all()
    assert np.array_equal(np.isnan(got), np.repeat(lost, walk.group, 1))
