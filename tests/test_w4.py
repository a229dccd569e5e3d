"""4-bit matrices, 8-bit rows, the norm and the products on the GPU, through their C entries, against their definition in
numpy (w4_reference.py): codes and scales bit for bit, the norm rounded once, products within the bound of their
arithmetic plus the rounding of the result's type."""
import math

import numpy as np
import pytest

from tinyinfer_amd import backend as mp

from . import w4_reference as ref
from .w4_reference import BF16, E2M1, F16, F32, HALF_STEP, I8, LEAST, TORCH, WHOLE
from .w4_sizes import CALLS, CALLS_EIGHT

pytestmark = pytest.mark.gpu

TYPES = pytest.mark.parametrize("kind", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
ANY = pytest.mark.parametrize("kind", [F32, BF16, F16, I8], ids=["f32", "bf16", "f16", "i8"])


class Floats:
    """Float rows on the GPU: `pad` elements behind every row, the first row `shift` elements into its buffer."""

    def __init__(self, torch, x, kind, pad=0, shift=0):
        n, width = x.shape
        self.buffer = torch.full((n * (width + pad) + shift,), 77.0, dtype=getattr(torch, TORCH[kind]), device="cuda")
        self.matrix = self.buffer[shift:].view(n, width + pad)
        self.matrix[:, :width] = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).cuda()
        self.width, self.torch = width, torch
        self.rows = mp.Rows(self.matrix.data_ptr(), width + pad, None, 0, kind)
        self.rows.owner = self.buffer  # the memory lives as long as the descriptor

    def back(self):
        self.torch.cuda.synchronize()
        return self.matrix[:, :self.width].double().cpu().numpy()

    def check_padding(self):
        assert bool((self.matrix[:, self.width:] == 77.0).all())


class Eight:
    """8-bit rows on the GPU, from values that 8 bits hold or empty; `pad` more bytes a row (multiples of 16)."""

    def __init__(self, torch, rows, width, x=None, pad=0):
        words = -(-width // 128) * 4 + pad // 4
        self.codes = torch.full((rows, width + pad), -128, dtype=torch.int8, device="cuda")
        self.scales = torch.full((rows, words), 255, dtype=torch.uint8, device="cuda")
        self.width, self.torch = width, torch
        if x is not None:
            code, sign, s = ref.split(x, WHOLE)
            self.codes[:, :width] = torch.from_numpy(np.where(sign, -code, code).astype(np.int8)).cuda()
            self.scales[:, :width // 32] = torch.from_numpy(s).cuda()
        self.rows = mp.Rows(self.codes.data_ptr(), width + pad, self.scales.data_ptr(), words, mp.TYPE_I8)
        self.rows.owner = (self.codes, self.scales)

    def bytes(self):
        self.torch.cuda.synchronize()
        return self.codes[:, :self.width].cpu().numpy(), self.scales[:, :self.width // 32].cpu().numpy()

    def back(self):
        codes, scales = self.bytes()
        return ref.values(np.minimum(np.abs(codes.astype(int)), 127), codes < 0, scales, WHOLE)

    def check_padding(self):
        assert bool((self.codes[:, self.width:] == -128).all()) and bool((self.scales[:, self.width // 32:] == 255).all())


class Matrix:
    """A 4-bit matrix on the GPU; from float values, packed here in numpy."""

    def __init__(self, torch, n, k, x=None):
        sizes = mp.w4_sizes(n, k)
        self.codes, self.scales = (torch.full((b,), 0xA5, dtype=torch.uint8, device="cuda") for b in sizes)
        self.view = mp.W4Matrix(self.codes.data_ptr(), self.scales.data_ptr(), n, k)
        self.torch = torch
        if x is not None:
            codes, scales = ref.pack(x)
            self.codes.copy_(torch.from_numpy(codes))
            self.scales.copy_(torch.from_numpy(scales))

    def bytes(self):
        self.torch.cuda.synchronize()
        return self.codes.cpu().numpy(), self.scales.cpu().numpy()


def rows_of(torch, x, kind, pad=0):
    return Eight(torch, *x.shape, x, pad) if kind == I8 else Floats(torch, x, kind, pad)


def empty(torch, rows, width, kind, pad=0):
    return Eight(torch, rows, width, None, pad) if kind == I8 else Floats(torch, np.zeros((rows, width)), kind, pad)


def in_type(x, kind):
    return ref.held(x, WHOLE) if kind == I8 else ref.rounded(x, kind)


def mixed(rng, rows, width, kind):
    """Groups of very different sizes, zeros, ties and powers of two among them, as numbers of a type."""
    x = rng.standard_normal((rows, width)) * np.exp(rng.standard_normal((rows, width)) * 2)
    spread = 12 if kind == F16 else 90
    x *= np.exp2(rng.integers(-spread, spread // 3, (rows, -(-width // 32))).repeat(32, 1)[:, :width])
    some = rng.random((rows, width))
    x[some < 0.1] = 0.0
    ties = rng.integers(-24, 25, (rows, width)) / 4 * np.exp2(rng.integers(-3, 3))
    x = np.where(some > 0.8, ties, x)
    x[0, :32] = 0.0
    if rows > 1:
        x[1, :32] = -0.0
    return ref.rounded(x, kind)


# ---- 4 bits ------------------------------------------------------------------------

SIZES = [(1, 32), (5, 96), (16, 128), (17, 160), (40, 512), (33, 544), (3, 1184), (130, 64)]


@TYPES
@pytest.mark.parametrize("n, k", SIZES)
def test_pack_and_read(torch_cuda, kind, n, k):
    rng = np.random.default_rng(n + k)
    x = mixed(rng, n, k, kind)
    for pad, shift in ((0, 0), (8, 8), (3, 1)):
        m = Matrix(torch_cuda, n, k)
        source = Floats(torch_cuda, x, kind, pad, shift)
        mp.w4_pack(m.view, 0, source.rows, n)
        want = ref.pack(x)
        got = m.bytes()
        for a, b, what in zip(got, want, ("codes", "scales")):
            # The sign of a zero is not told apart.
            if what == "codes":
                a, b = (np.where((c & 15) == 8, c & 0xF0, c) for c in (a, b))
                a, b = (np.where((c >> 4) == 8, c & 0x0F, c) for c in (a, b))
            assert np.array_equal(a, b), what
        ids = np.concatenate((rng.permutation(n), [0, n - 1, 0, -1, n, 1 << 30])).astype(np.int32)
        d_ids = torch_cuda.from_numpy(ids).cuda()
        out = Floats(torch_cuda, np.zeros((len(ids), k)), kind, pad, shift)
        mp.w4_read(m.view, d_ids.data_ptr(), len(ids), out.rows)
        back, held = out.back(), ref.held(x, E2M1)
        inside = (ids >= 0) & (ids < n)
        assert np.array_equal(back[inside], ref.rounded(held[ids[inside]], kind))
        assert np.isnan(back[~inside]).all()
        out.check_padding()


def test_pack_in_pieces_leaves_other_rows(torch_cuda):
    rng = np.random.default_rng(3)
    n, k = 53, 224
    x = mixed(rng, n, k, F32)
    m = Matrix(torch_cuda, n, k)
    for first, count in ((20, 1), (0, 20), (37, 16), (21, 16)):
        piece = Floats(torch_cuda, x[first:first + count], F32)
        mp.w4_pack(m.view, first, piece.rows, count)
    whole = Matrix(torch_cuda, n, k)
    mp.w4_pack(whole.view, 0, Floats(torch_cuda, x, F32).rows, n)
    for a, b in zip(m.bytes(), whole.bytes()):
        assert np.array_equal(a, b)
    before = [b.copy() for b in m.bytes()]
    mp.w4_pack(m.view, 18, Floats(torch_cuda, x[18:35], F32).rows, 17)  # the same rows again
    for a, b in zip(m.bytes(), before):
        assert np.array_equal(a, b)
    mp.w4_pack(m.view, 5, piece.rows, 0)
    mp.w4_pack(m.view, 7, Floats(torch_cuda, -x[7:8], F32).rows, 1)
    ids = torch_cuda.arange(n, dtype=torch_cuda.int32, device="cuda")
    out = Floats(torch_cuda, np.zeros((n, k)), F32)
    mp.w4_read(m.view, ids.data_ptr(), n, out.rows)
    want = ref.held(x, E2M1)
    want[7] = -want[7]
    assert np.array_equal(out.back(), want)


def test_groups_with_nan_or_infinity_are_nan(torch_cuda):
    x = np.random.default_rng(4).standard_normal((4, 128))
    x[0, 5], x[1, 40], x[2, 127], x[3, 70] = np.nan, np.inf, -np.inf, 3.3e38  # the last: past 6 and 127 times 2^120
    m = Matrix(torch_cuda, 4, 128)
    mp.w4_pack(m.view, 0, Floats(torch_cuda, x, F32).rows, 4)
    ids = torch_cuda.arange(4, dtype=torch_cuda.int32, device="cuda")
    out = Floats(torch_cuda, np.zeros((4, 128)), F32)
    mp.w4_read(m.view, ids.data_ptr(), 4, out.rows)
    want = np.zeros((4, 4), bool)
    want[0, 0] = want[1, 1] = want[2, 3] = want[3, 2] = True
    assert np.array_equal(np.isnan(out.back()), want.repeat(32, 1))
    eight = Eight(torch_cuda, 4, 128)
    mp.convert_rows(Floats(torch_cuda, x, F32).rows, 4, 128, eight.rows)
    assert np.array_equal(np.isnan(eight.back()), want.repeat(32, 1))


# ---- rows ------------------------------------------------------------------------------

@TYPES
@pytest.mark.parametrize("rows, width, pad, shift", [(1, 32, 0, 0), (7, 576, 0, 0), (5, 96, 16, 0), (3, 64, 1, 3),
                                                     (130, 160, 0, 0), (9, 2080, 3, 0)])
def test_rows_to_8_bits_and_back(torch_cuda, kind, rows, width, pad, shift):
    rng = np.random.default_rng(rows + width)
    x = mixed(rng, rows, width, kind)
    source = Floats(torch_cuda, x, kind, pad, shift)
    eight = Eight(torch_cuda, rows, width, None, 16 * (pad % 3))
    mp.convert_rows(source.rows, rows, width, eight.rows)
    code, sign, s = ref.split(x, WHOLE)
    codes, scales = eight.bytes()
    assert np.array_equal(scales, s)
    assert np.array_equal(codes, np.where(sign, -code, code))
    eight.check_padding()
    for to in (F32, BF16, F16):
        out = Floats(torch_cuda, np.zeros((rows, width)), to, pad, shift)
        mp.convert_rows(eight.rows, rows, width, out.rows)
        assert np.array_equal(out.back(), ref.rounded(ref.values(code, sign, s, WHOLE), to))
        out.check_padding()
    again = Eight(torch_cuda, rows, width)
    mp.convert_rows(eight.rows, rows, width, again.rows)
    assert np.array_equal(again.back(), eight.back())


@pytest.mark.parametrize("rows, width, pad, shift", [(3, 1, 0, 0), (4, 37, 0, 0), (2, 64, 0, 0), (5, 1001, 2, 1)])
def test_float_rows_to_float_rows(torch_cuda, rows, width, pad, shift):
    rng = np.random.default_rng(width)
    for kind in (F32, BF16, F16):
        x = ref.rounded(rng.standard_normal((rows, width)) * 100, kind)
        x[0, 0] = np.nan
        if width > 3:
            x[0, 1:3] = np.inf, -np.inf
        source = Floats(torch_cuda, x, kind, pad, shift)
        for to in (F32, BF16, F16):
            out = Floats(torch_cuda, np.zeros((rows, width)), to, pad, 0)
            mp.convert_rows(source.rows, rows, width, out.rows)
            assert np.array_equal(out.back(), ref.rounded(x, to), equal_nan=True)
            out.check_padding()
        mp.convert_rows(source.rows, rows, width, source.rows)
        assert np.array_equal(source.back(), x, equal_nan=True)


# ---- the norm ---------------------------------------------------------------------------

NORMS = [(1, 32), (3, 1), (2, 7), (5, 63), (4, 512), (6, 513), (1, 576), (7, 1024), (3, 1025), (5, 2047), (2, 4096), (3, 4100),
         (2, 16384), (2, 16416), (1, 40001), (1, 50016)]


@TYPES
@pytest.mark.parametrize("rows, width", NORMS)
def test_norm(torch_cuda, kind, rows, width):
    """Rounded once: the result is the neighbour of the exact value in its type, for any alignment, with and without a
    residual, and the 8-bit rows are those of the exact values."""
    rng = np.random.default_rng(rows * 100000 + width)
    x = ref.rounded(rng.standard_normal((rows, width)) * np.exp(rng.standard_normal(width)), kind)
    r = ref.rounded(3 * rng.standard_normal((rows, width)), kind)
    weight = (1 + 0.2 * rng.standard_normal(width)).astype(np.float32)
    d_weight = torch_cuda.from_numpy(weight).cuda()
    for residual, pad, shift in ((None, 0, 0), (r, 0, 0), (r, 3, 1), (None, 5, 2)):
        t, y = ref.norm(x, residual, weight, 1e-5)
        for to in (kind, (kind + 1) % 3) + ((I8,) if width % 32 == 0 else ()):
            source = Floats(torch_cuda, x, kind, pad, shift)
            out = Eight(torch_cuda, rows, width) if to == I8 else Floats(torch_cuda, np.zeros((rows, width)), to, pad)
            added = Floats(torch_cuda, residual, kind, pad, shift) if residual is not None else None
            total = Floats(torch_cuda, np.zeros((rows, width)), kind, pad, shift) if residual is not None else None
            mp.rms_norm(source.rows, d_weight.data_ptr(), 1e-5, rows, width, out.rows,
                        residual=added.rows if added else None, sum=total.rows if total else None)
            assert np.array_equal(out.back(), ref.held(y, WHOLE) if to == I8 else ref.rounded(y, to))
            out.check_padding()
            if total:
                assert np.array_equal(total.back(), ref.rounded(t, kind))
                total.check_padding()


@pytest.mark.parametrize("width", [576, 37, 20000])
def test_norm_in_place(torch_cuda, width):
    rng = np.random.default_rng(width)
    x, r = (ref.rounded(rng.standard_normal((5, width)), BF16) for _ in range(2))
    weight = np.ones(width, np.float32)
    d_weight = torch_cuda.from_numpy(weight).cuda()
    t, y = ref.norm(x, r, weight, 0.0)
    a, b = Floats(torch_cuda, x, BF16), Floats(torch_cuda, r, BF16)
    mp.rms_norm(a.rows, d_weight.data_ptr(), 0.0, 5, width, a.rows, residual=b.rows, sum=b.rows)
    assert np.array_equal(a.back(), ref.rounded(y, BF16)) and np.array_equal(b.back(), ref.rounded(t, BF16))
    a, b, out = Floats(torch_cuda, x, BF16), Floats(torch_cuda, r, BF16), Floats(torch_cuda, x, F32)
    mp.rms_norm(a.rows, d_weight.data_ptr(), 0.0, 5, width, out.rows, residual=b.rows, sum=a.rows)
    assert np.array_equal(a.back(), ref.rounded(t, BF16)) and np.array_equal(out.back(), ref.rounded(y, F32))
    a, out = Floats(torch_cuda, x, BF16), Floats(torch_cuda, x, F32)
    mp.rms_norm(a.rows, d_weight.data_ptr(), 0.0, 5, width, out.rows, residual=a.rows)  # x + x, the sum not wanted
    assert np.array_equal(out.back(), ref.rounded(ref.norm(x, x, weight, 0.0)[1], F32))


def test_norm_of_extremes(torch_cuda):
    """Squares past FP32, numbers near the smallest, zeros, infinities and NaN: rows apart."""
    width = 64
    rng = np.random.default_rng(9)
    x = rng.standard_normal((8, width))
    x[0] *= 1e37
    x[1] *= 1e-38
    x[2] = 0.0
    x[3, 5] = np.nan
    x[4, 63] = np.inf
    x[5] = 2.0 ** -149
    x[6, 0] = 3e38
    x = ref.rounded(x, F32)
    r = np.where(np.isfinite(x), x, 0.0)
    weight = np.ones(width, np.float32)
    d_weight = torch_cuda.from_numpy(weight).cuda()
    for epsilon in (0.0, 1e-5):
        for residual in (None, r):
            t, y = ref.norm(x, residual, weight, epsilon)
            for to in (F32, F16, I8):
                out = empty(torch_cuda, 8, width, to)
                mp.rms_norm(Floats(torch_cuda, x, F32).rows, d_weight.data_ptr(), epsilon, 8, width, out.rows,
                            residual=Floats(torch_cuda, residual, F32).rows if residual is not None else None)
                with np.errstate(invalid="ignore"):
                    want = ref.held(y, WHOLE) if to == I8 else ref.rounded(y, to)
                assert np.array_equal(out.back(), want, equal_nan=True)


# ---- products -----------------------------------------------------------------------------

def close(got, want, bound, to):
    """Within the bound and the rounding to a type."""
    if to == I8:
        # Half a step; the scale of a group whose largest element lies at a power's border may be twice.
        amax = np.abs(want).reshape(len(want), -1, 32).max(-1).repeat(32, 1)
        step = np.maximum(2 * amax / 127, 2.0 ** -100)
        bound = bound * (1 + 2.0 ** -3) + step
    else:
        bound = bound * (1 + HALF_STEP[to]) + HALF_STEP[to] * np.abs(want) + LEAST[to] / 2
    off = np.abs(got - want)
    assert (off <= bound).all(), f"off by up to {np.nanmax(off / bound)} of the bound, {np.isnan(got).sum()} NaN"


PARTS = {F32: 3, BF16: 1, F16: 2, I8: 1}


def check_product(torch, rng, rows, n, k, kind, to, gated, pad=0, scale=1.0):
    x = in_type(rng.standard_normal((rows, k)) * np.exp(rng.standard_normal(k)) * scale, kind)
    w = ref.held(rng.standard_normal((n, k)) * 0.05 * np.exp(rng.standard_normal((n, 1)) * 0.5), E2M1)
    g = ref.held(rng.standard_normal((n, k)) * 0.05, E2M1) if gated else None
    matrix, gate = Matrix(torch, n, k, w), Matrix(torch, n, k, g) if gated else None
    source, out = rows_of(torch, x, kind, pad), empty(torch, rows, n, to, pad)
    size = mp.w4_product_workspace(matrix.view, kind, rows, gated)
    workspace = torch.empty(size + 64, dtype=torch.uint8, device="cuda").fill_(0xFF)
    mp.w4_product(matrix.view, source.rows, rows, out.rows, gate=gate.view if gate else None,
                  workspace=workspace.data_ptr(), workspace_bytes=size)
    got = out.back()
    out.check_padding()
    assert bool((workspace[size:] == 0xFF).all())
    want = ref.product(x, w, g)
    bound = ref.gated_bound(x, w, g, PARTS[kind]) if gated else ref.product_bound(x, w, PARTS[kind])
    close(got, want, bound, to)
    if to == F32 and rows * n > 200:  # in earnest, as FP32 sums are
        off = np.linalg.norm(got - want) / np.linalg.norm(want)
        assert off < 1e-6, off
    return got


@ANY
@pytest.mark.parametrize("gated", [False, True], ids=["plain", "gated"])
@pytest.mark.parametrize("rows, n, k", [(1, 1, 32), (1, 16, 128), (1, 37, 576), (2, 100, 160), (3, 576, 1536), (5, 17, 96),
                                        (1, 960, 4128)])
def test_products_of_few_rows(torch_cuda, kind, gated, rows, n, k):
    check_product(torch_cuda, np.random.default_rng(rows + n + k), rows, n, k, kind, F32, gated)


@ANY
@pytest.mark.parametrize("gated", [False, True], ids=["plain", "gated"])
@pytest.mark.parametrize("rows, n, k", [(15, 64, 256), (16, 33, 576), (17, 130, 192), (33, 70, 640), (64, 200, 544), (65, 48, 64),
                                        (203, 96, 576), (130, 1100, 128)])
def test_products_of_rows(torch_cuda, kind, gated, rows, n, k):
    check_product(torch_cuda, np.random.default_rng(rows + n + k), rows, n, k, kind, F32, gated)


@ANY
@pytest.mark.parametrize("to", [F32, BF16, F16, I8], ids=["f32", "bf16", "f16", "i8"])
@pytest.mark.parametrize("rows, n, k, pad", [(1, 64, 96, 0), (19, 96, 160, 16), (70, 32, 288, 0), (5, 2080, 32, 48)])
def test_products_to_every_type(torch_cuda, kind, to, rows, n, k, pad):
    for gated in (False, True):
        check_product(torch_cuda, np.random.default_rng(n + k), rows, n, k, kind, to, gated, pad)


@TYPES
@pytest.mark.parametrize("pad, shift", [(1, 0), (0, 1), (5, 3), (2, 2)])
def test_products_of_any_alignment(torch_cuda, kind, pad, shift):
    rng = np.random.default_rng(pad + 10 * shift)
    for rows, n, k in ((1, 37, 96), (20, 51, 160), (70, 35, 64), (130, 16291, 96), (300, 22001, 64)):
        x = ref.rounded(rng.standard_normal((rows, k)), kind)
        w = ref.held(rng.standard_normal((n, k)), E2M1)
        matrix, source = Matrix(torch_cuda, n, k, w), Floats(torch_cuda, x, kind, pad, shift)
        out = Floats(torch_cuda, np.zeros((rows, n)), kind, pad, shift)
        size = mp.w4_product_workspace(matrix.view, kind, rows)
        workspace = torch_cuda.empty(size + 16, dtype=torch_cuda.uint8, device="cuda")
        mp.w4_product(matrix.view, source.rows, rows, out.rows, workspace=workspace.data_ptr(), workspace_bytes=size)
        close(out.back(), x @ w.T, ref.product_bound(x, w, PARTS[kind]), kind)
        out.check_padding()


@ANY
@pytest.mark.parametrize("rows, n", [(3, 50), (40, 50), (300, 50), (66, 16400), (2000, 4200)])
def test_nan_stays_in_its_row_and_column(torch_cuda, kind, rows, n):
    rng = np.random.default_rng(rows)
    k = 288
    x = in_type(rng.standard_normal((rows, k)), kind)
    w = ref.held(rng.standard_normal((n, k)), E2M1)
    want = x @ w.T
    bound = ref.product_bound(x, w, PARTS[kind])
    bad = x.copy()
    bad[1, 200] = np.nan
    if rows > 30:
        bad[30, 3] = np.nan if kind == I8 else np.inf
    source = rows_of(torch_cuda, bad, kind)
    matrix = Matrix(torch_cuda, n, k, w)
    scales = ref.pack(w)[1]
    scales[(2 * 1 + 0) * 256 + (1 * 16 + 3) * 4 + 1] = 255  # row 35, columns 160 ..+31
    matrix.scales.copy_(torch_cuda.from_numpy(scales))
    out = Floats(torch_cuda, np.zeros((rows, n)), F32)
    size = mp.w4_product_workspace(matrix.view, kind, rows)
    workspace = torch_cuda.empty(size + 16, dtype=torch_cuda.uint8, device="cuda")
    mp.w4_product(matrix.view, source.rows, rows, out.rows, workspace=workspace.data_ptr(), workspace_bytes=size)
    got = out.back()
    gone = np.zeros((rows, n), bool)
    gone[1] = gone[:, 35] = True
    if rows > 30:
        gone[30] = True
    assert not np.isfinite(got[gone]).any()
    close(got[~gone], want[~gone], bound[~gone], F32)


@TYPES
def test_far_smaller_elements_count(torch_cuda, kind):
    """Elements 2^20 below the largest of their group, which meets a weight of 0."""
    rng = np.random.default_rng(5)
    for rows in (1, 20, 300):
        k, n = 128, 48
        x = rng.standard_normal((rows, k)) * 2.0 ** -10
        x[:, ::32] = 2.0 ** 10 * (1 + rng.random((rows, 4)))
        x = ref.rounded(x, kind)
        w = rng.standard_normal((n, k))
        w[:, ::32] = 0
        w = ref.held(w, E2M1)
        matrix, source, out = Matrix(torch_cuda, n, k, w), Floats(torch_cuda, x, kind), Floats(torch_cuda, np.zeros((rows, n)), F32)
        size = mp.w4_product_workspace(matrix.view, kind, rows)
        workspace = torch_cuda.empty(size + 16, dtype=torch_cuda.uint8, device="cuda")
        mp.w4_product(matrix.view, source.rows, rows, out.rows, workspace=workspace.data_ptr(), workspace_bytes=size)
        close(out.back(), x @ w.T, ref.product_bound(x, w, PARTS[kind]), F32)


@pytest.mark.parametrize("rows, n", [(1, 480), (70, 480), (70, 16384), (2049, 2080)])
def test_calls_on_a_stream_and_replayed(torch_cuda, rows, n):
    """Norm, conversion and products captured on a stream of their own and replayed for other rows, with eager work
    between; every replay against eager calls."""
    torch = torch_cuda
    rng = np.random.default_rng(8)
    k = 576
    matrix = Matrix(torch, n, k, ref.held(rng.standard_normal((n, k)), E2M1))
    gate = Matrix(torch, n, k, ref.held(rng.standard_normal((n, k)), E2M1))
    weight = torch.ones(k, device="cuda")
    x = [Floats(torch, rng.standard_normal((rows, k)), F32) for _ in range(3)]
    still = Floats(torch, np.zeros((rows, k)), F32)
    normed, eight, out = Floats(torch, np.zeros((rows, k)), F32), Eight(torch, rows, k), Floats(torch, np.zeros((rows, n)), BF16)
    out8 = Eight(torch, rows, n)
    sizes = [mp.w4_product_workspace(matrix.view, t, rows, True) for t in (F32, I8)]
    spaces = [torch.empty(s + 16, dtype=torch.uint8, device="cuda") for s in sizes]

    def step(stream):
        mp.rms_norm(still.rows, weight.data_ptr(), 1e-5, rows, k, normed.rows, stream=stream)
        mp.w4_product(matrix.view, normed.rows, rows, out.rows, workspace=spaces[0].data_ptr(), workspace_bytes=sizes[0],
                      stream=stream)
        mp.convert_rows(normed.rows, rows, k, eight.rows, stream=stream)
        mp.w4_product(matrix.view, eight.rows, rows, out8.rows, gate=gate.view, workspace=spaces[1].data_ptr(),
                      workspace_bytes=sizes[1], stream=stream)

    want = []
    for source in x:
        still.matrix.copy_(source.matrix)
        step(None)
        want.append((out.back(), *out8.bytes()))
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step(torch.cuda.current_stream().cuda_stream)
    for i in (1, 0, 2, 2, 1):
        still.matrix.copy_(x[i].matrix)
        out.matrix.zero_()
        out8.codes.zero_()
        graph.replay()
        for got, there in zip((out.back(), *out8.bytes()), want[i]):
            assert np.array_equal(got, there)
        step(None)
        torch.cuda.synchronize()


def test_a_decode_step_of_a_layer(torch_cuda):
    """The operators as a model runs them, with the 8-bit cache between: embedding, norm, query/key/value projection,
    append, attention, output projection, norm with the residual, the gated pair, the last projection. Each against its
    definition on what the one before gave."""
    torch = torch_cuda
    rng = np.random.default_rng(21)
    hidden, heads, kv_heads, dim, inner, vocabulary, rows = 192, 3, 1, 64, 512, 300, 5
    width = (heads + 2 * kv_heads) * dim

    def matrix(n, k):
        m = Matrix(torch, n, k)
        w = rng.standard_normal((n, k)) / math.sqrt(k)
        mp.w4_pack(m.view, 0, Floats(torch, w, F32).rows, n)
        torch.cuda.synchronize()
        return m, ref.held(w.astype(np.float32).astype(np.float64), E2M1)

    table, table_w = matrix(vocabulary, hidden)
    qkv, qkv_w = matrix(width, hidden)
    o, o_w = matrix(hidden, heads * dim)
    gate, gate_w = matrix(inner, hidden)
    up, up_w = matrix(inner, hidden)
    down, down_w = matrix(hidden, inner)
    weight = torch.ones(hidden, device="cuda")
    ones = np.ones(hidden, np.float32)

    def zeros(n):
        return Floats(torch, np.zeros((rows, n)), F32)

    def check(got, x, w, g=None):
        close(got, ref.product(x, w, g), ref.product_bound(x, w, 3) if g is None else ref.gated_bound(x, w, g, 3), F32)

    ids = torch.tensor([7, 299, 0, 7, 150], dtype=torch.int32, device="cuda")
    x = zeros(hidden)
    mp.w4_read(table.view, ids.data_ptr(), rows, x.rows)
    assert np.array_equal(x.back(), table_w[ids.cpu().numpy()])
    h, projected = zeros(hidden), zeros(width)
    mp.rms_norm(x.rows, weight.data_ptr(), 1e-5, rows, hidden, h.rows)
    assert np.array_equal(h.back(), ref.rounded(ref.norm(x.back(), None, ones, 1e-5)[1], F32))
    mp.w4_product(qkv.view, h.rows, rows, projected.rows)
    check(projected.back(), h.back(), qkv_w)
    # Every row a sequence of its own, its first token: attention gives the value as the cache holds it.
    pools = [torch.zeros((rows, 1, kv_heads, 16 * dim), dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = torch.zeros((rows, 1, kv_heads, 2), device="cuda")
    cache = mp.Kv8Cache(pools[0].data_ptr(), pools[1].data_ptr(), scales.data_ptr(), rows, 1, 16, kv_heads, dim, mp.KV8_E4M3)
    tables = torch.arange(rows, dtype=torch.int32, device="cuda")
    starts = torch.arange(rows + 1, dtype=torch.int32, device="cuda")
    used = torch.zeros(rows, dtype=torch.int32, device="cuda")
    base = projected.matrix.data_ptr()
    mp.kv8_append(cache, 0, base + heads * dim * 4, width, base + (heads + kv_heads) * dim * 4, width, mp.TYPE_F32,
                  tables.data_ptr(), 1, starts.data_ptr(), used.data_ptr(), rows, rows)
    attended = zeros(heads * dim)
    lengths = used + 1
    mp.kv8_attention_decode(cache, 0, base, width, mp.TYPE_F32, tables.data_ptr(), 1, lengths.data_ptr(), rows, heads, 16,
                            1 / math.sqrt(dim), attended.matrix.data_ptr(), heads * dim)
    v = projected.back()[:, (heads + kv_heads) * dim:]
    assert np.abs(attended.back() - np.tile(v, (1, heads))).max() <= 2.0 ** -4 * np.abs(v).max() * (1 + 1e-5)
    mixed_in, total, h2 = zeros(hidden), zeros(hidden), zeros(hidden)
    mp.w4_product(o.view, attended.rows, rows, mixed_in.rows)
    check(mixed_in.back(), attended.back(), o_w)
    mp.rms_norm(mixed_in.rows, weight.data_ptr(), 1e-5, rows, hidden, h2.rows, residual=x.rows, sum=total.rows)
    t, y = ref.norm(mixed_in.back(), x.back(), ones, 1e-5)
    assert np.array_equal(total.back(), ref.rounded(t, F32)) and np.array_equal(h2.back(), ref.rounded(y, F32))
    inner_rows, last = zeros(inner), zeros(hidden)
    mp.w4_product(up.view, h2.rows, rows, inner_rows.rows, gate=gate.view)
    check(inner_rows.back(), h2.back(), up_w, gate_w)
    mp.w4_product(down.view, inner_rows.rows, rows, last.rows)
    check(last.back(), inner_rows.back(), down_w)


@ANY
@pytest.mark.parametrize("gated", [False, True], ids=["plain", "gated"])
@pytest.mark.parametrize("rows, n, k", [(129, 16500, 96), (640, 5000, 32), (1000, 4120, 192), (2049, 2000, 544), (130, 17000, 576),
                                        (2049, 4100, 160), (300, 21900, 64)])
def test_products_of_many_rows(torch_cuda, kind, gated, rows, n, k):
    check_product(torch_cuda, np.random.default_rng(rows + n + k), rows, n, k, kind, F32, gated)


@ANY
@pytest.mark.parametrize("to", [F32, BF16, F16, I8], ids=["f32", "bf16", "f16", "i8"])
@pytest.mark.parametrize("rows, n, k, pad", [(1025, 4128, 160, 16), (4097, 1056, 64, 0), (2050, 4128, 96, 0)])
def test_products_of_many_rows_to_every_type(torch_cuda, kind, to, rows, n, k, pad):
    for gated in (False, True):
        check_product(torch_cuda, np.random.default_rng(n + k), rows, n, k, kind, to, gated, pad)


def test_two_streams_at_once(torch_cuda):
    """Products of prompts on two streams, each with a workspace of its own, as one after the other."""
    torch = torch_cuda
    rng = np.random.default_rng(13)
    rows, n, k = 2049, 4160, 256
    matrix = Matrix(torch, n, k, ref.held(rng.standard_normal((n, k)), E2M1))
    x = [Eight(torch, rows, k, ref.held(rng.standard_normal((rows, k)), WHOLE)) for _ in range(2)]
    size = mp.w4_product_workspace(matrix.view, I8, rows)
    assert size > 0
    want = []
    for source in x:
        out, space = Floats(torch, np.zeros((rows, n)), BF16), torch.empty(size, dtype=torch.uint8, device="cuda")
        mp.w4_product(matrix.view, source.rows, rows, out.rows, workspace=space.data_ptr(), workspace_bytes=size)
        want.append(out.back())
    streams = [torch.cuda.Stream() for _ in x]
    outs = [Floats(torch, np.zeros((rows, n)), BF16) for _ in x]
    spaces = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in x]
    torch.cuda.synchronize()
    for _ in range(4):
        for source, out, space, stream in zip(x, outs, spaces, streams):
            mp.w4_product(matrix.view, source.rows, rows, out.rows, workspace=space.data_ptr(), workspace_bytes=size,
                          stream=stream.cuda_stream)
    for out, there in zip(outs, want):
        assert np.array_equal(out.back(), there)


def test_a_workspace_for_more_rows_is_enough(torch_cuda):
    rng = np.random.default_rng(14)
    n, k = 4160, 96
    w = ref.held(rng.standard_normal((n, k)), E2M1)
    matrix = Matrix(torch_cuda, n, k, w)
    size = mp.w4_product_workspace(matrix.view, I8, 2304)
    space = torch_cuda.empty(size, dtype=torch_cuda.uint8, device="cuda")
    for rows in (2304, 2200, 1950, 700, 3):
        assert mp.w4_product_workspace(matrix.view, I8, rows) <= size
        x = ref.held(rng.standard_normal((rows, k)), WHOLE)
        out = Floats(torch_cuda, np.zeros((rows, n)), F32)
        mp.w4_product(matrix.view, Eight(torch_cuda, rows, k, x).rows, rows, out.rows, workspace=space.data_ptr(),
                      workspace_bytes=size)
        close(out.back(), x @ w.T, ref.product_bound(x, w, 1), F32)
    x = Eight(torch_cuda, 2304, k, ref.held(rng.standard_normal((2304, k)), WHOLE))
    out = Floats(torch_cuda, np.zeros((2304, n)), F32)
    for bad in (dict(), dict(workspace=space.data_ptr(), workspace_bytes=size - 1),
                dict(workspace=space.data_ptr() + 8, workspace_bytes=size)):
        with pytest.raises(mp.BackendError, match="workspace"):
            mp.w4_product(matrix.view, x.rows, 2304, out.rows, **bad)


@pytest.mark.parametrize("rows, n", [(20, 96), (70, 16384)])
def test_rows_past_4_gib(torch_cuda, rows, n):
    """Rows 2^26 elements apart: norm, conversion and products find the last ones."""
    torch = torch_cuda
    rng = np.random.default_rng(rows)
    k, stride = 96, 1 << 26
    x = ref.rounded(rng.standard_normal((rows, k)), F32)
    w = ref.held(rng.standard_normal((n, k)), E2M1)
    buffer = torch.empty(rows * stride, device="cuda")
    far = buffer.view(rows, stride)[:, :k]
    far.copy_(torch.from_numpy(x.astype(np.float32)).cuda())
    source = mp.Rows(buffer.data_ptr(), stride, None, 0, F32)
    matrix, out = Matrix(torch, n, k, w), Floats(torch, np.zeros((rows, n)), F32)
    mp.w4_product(matrix.view, source, rows, out.rows)
    close(out.back(), x @ w.T, ref.product_bound(x, w, 3), F32)
    weight = torch.ones(k, device="cuda")
    near = Floats(torch, x, F32)
    mp.rms_norm(source, weight.data_ptr(), 1e-5, rows, k, near.rows)
    assert np.array_equal(near.back(), ref.rounded(ref.norm(x, None, np.ones(k, np.float32), 1e-5)[1], F32))
    mp.convert_rows(near.rows, rows, k, source)
    torch.cuda.synchronize()
    assert np.array_equal(far.double().cpu().numpy(), near.back())


def test_a_matrix_past_4_gib(torch_cuda):
    """Packing, reading and multiplying with the last rows of 2^24."""
    torch = torch_cuda
    n, k, last = 1 << 24, 576, 40
    rng = np.random.default_rng(15)
    sizes = mp.w4_sizes(n, k)
    assert sizes[0] > 1 << 32
    codes, scales = (torch.zeros(b, dtype=torch.uint8, device="cuda") for b in sizes)
    view = mp.W4Matrix(codes.data_ptr(), scales.data_ptr(), n, k)
    w = ref.rounded(rng.standard_normal((last, k)), F32)
    held = ref.held(w, E2M1)
    mp.w4_pack(view, n - last, Floats(torch, w, F32).rows, last)
    ids = torch.arange(n - last, n, dtype=torch.int32, device="cuda")
    back = Floats(torch, np.zeros((last, k)), F32)
    mp.w4_read(view, ids.data_ptr(), last, back.rows)
    assert np.array_equal(back.back(), held)
    for rows in (1, 33):
        x = ref.rounded(rng.standard_normal((rows, k)), BF16)
        source = Floats(torch, x, BF16)
        out = torch.empty((rows, n), dtype=torch.bfloat16, device="cuda")
        mp.w4_product(view, source.rows, rows, mp.Rows(out.data_ptr(), n, None, 0, BF16))
        got = out[:, -last:].double().cpu().numpy()
        close(got, x @ held.T, ref.product_bound(x, held, 1), BF16)
        assert bool((out[:, :-last] == 0).all())
        del out


@ANY
@pytest.mark.parametrize("rows, n", [(1, 96), (5, 96), (20, 96), (70, 16384), (300, 22016)])
def test_rows_behind_the_last_stay(torch_cuda, kind, rows, n):
    """Results of `rows` rows in a buffer of more, beside their inputs in one matrix: everything else stays."""
    torch = torch_cuda
    rng = np.random.default_rng(rows)
    k = 96
    w = ref.held(rng.standard_normal((n, k)), E2M1)
    matrix = Matrix(torch, n, k, w)
    x = in_type(rng.standard_normal((rows + 3, k)), kind)
    source = rows_of(torch, x, kind)
    size = mp.w4_product_workspace(matrix.view, kind, rows)
    space = torch.empty(size + 16, dtype=torch.uint8, device="cuda")
    out = torch.full((rows + 3, n + 8), 5.0, device="cuda")
    mp.w4_product(matrix.view, source.rows, rows, mp.Rows(out.data_ptr(), n + 8, None, 0, F32),
                  workspace=space.data_ptr(), workspace_bytes=size)
    got = out.double().cpu().numpy()
    close(got[:rows, :n], x[:rows] @ w.T, ref.product_bound(x[:rows], w, PARTS[kind]), F32)
    assert (got[rows:] == 5).all() and (got[:, n:] == 5).all()
    eight = Eight(torch, rows + 3, n)
    mp.w4_product(matrix.view, source.rows, rows, eight.rows, workspace=space.data_ptr(), workspace_bytes=size)
    codes, scales = eight.bytes()
    assert (codes[rows:] == -128).all() and (scales[rows:] == 255).all() and (scales[:rows] != 255).all()


def test_other_calls_leave_rows_behind_the_last(torch_cuda):
    torch = torch_cuda
    rng = np.random.default_rng(2)
    for rows, width in ((3, 64), (5, 37), (2, 9000)):
        x = rng.standard_normal((rows + 2, width))
        source, residual = Floats(torch, x, F32), Floats(torch, x, F32)
        out, total = Floats(torch, np.full((rows + 2, width), 5.0), F32), Floats(torch, np.full((rows + 2, width), 6.0), F32)
        weight = torch.ones(width, device="cuda")
        mp.rms_norm(source.rows, weight.data_ptr(), 1e-5, rows, width, out.rows, residual=residual.rows, sum=total.rows)
        assert (out.back()[rows:] == 5).all() and (total.back()[rows:] == 6).all() and (out.back()[:rows] != 5).any()
        mp.convert_rows(source.rows, rows, width, total.rows)
        assert (total.back()[rows:] == 6).all() and np.array_equal(total.back()[:rows], source.back()[:rows])
    m = Matrix(torch, 40, 64, ref.held(rng.standard_normal((40, 64)), E2M1))
    ids = torch.arange(6, dtype=torch.int32, device="cuda")
    out = Floats(torch, np.full((6, 64), 5.0), F32)
    mp.w4_read(m.view, ids.data_ptr(), 4, out.rows)
    assert (out.back()[4:] == 5).all() and (out.back()[:4] != 5).any()


@ANY
@pytest.mark.parametrize("rows, n", [(3, 250), (20, 250), (70, 16416), (300, 11008)])
def test_gates_far_below_zero(torch_cuda, kind, rows, n):
    """Gates down to -200, whose exp(-g) leaves FP32's range, with u up to 2^120: sums of one product each are exact, so
    that the result is off by silu's roundings alone. The gate's few exponentials (a unit in the last place each) and
    products are below 16 half steps."""
    rng = np.random.default_rng(rows)
    k = 64
    g = -np.concatenate((np.arange(60, 128), np.arange(128, 201, 2))).astype(np.float64)  # numbers of 8 bits
    x = np.zeros((rows, k))
    x[:, 0], x[:, 32] = rng.permutation(np.resize(g, max(rows, len(g))))[:rows], 1.0
    w, gate = np.zeros((n, k)), np.zeros((n, k))
    gate[:, 0] = 1.0
    w[:, 32] = np.exp2(120.0 - np.arange(n) % 221)
    x = in_type(x, kind)
    matrix, gates = Matrix(torch_cuda, n, k, w), Matrix(torch_cuda, n, k, gate)
    source, out = rows_of(torch_cuda, x, kind), Floats(torch_cuda, np.zeros((rows, n)), F32)
    size = mp.w4_product_workspace(matrix.view, kind, rows, True)
    workspace = torch_cuda.empty(size + 16, dtype=torch_cuda.uint8, device="cuda")
    mp.w4_product(matrix.view, source.rows, rows, out.rows, gate=gates.view, workspace=workspace.data_ptr(),
                  workspace_bytes=size)
    want = ref.product(x, w, gate)
    assert (np.abs(want) > 2.0 ** -126).any(1).sum() > rows // 2
    close(out.back(), want, 16 * 2.0 ** -24 * np.abs(want), F32)


@pytest.mark.parametrize("kind", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("width", [64, 4099])
def test_norm_below_the_normal_numbers(torch_cuda, kind, width):
    """Results of 2^-140 to 2^-120, most of them a little beside the border of two BF16 numbers, by less than FP32 has
    there: rounded once."""
    rng = np.random.default_rng(width)
    rows = 6
    x = np.ones((rows, width))
    x[1:, 0] = [1 + 2.0 ** -7, 0.5, 2.0, 0.75, 1.25]  # the row's root is a little more or less than 1
    x[4] *= 1 + 2.0 ** -7
    x = ref.rounded(x, kind)
    halves = (2 * rng.integers(0, 128, width) + 1) * 2.0 ** -134
    weight = np.where(rng.random(width) < 0.7, halves, np.exp2(rng.uniform(-140, -120, width))).astype(np.float32)
    weight *= np.where(rng.random(width) < 0.5, -1, 1).astype(np.float32)
    d_weight = torch_cuda.from_numpy(weight).cuda()
    for epsilon in (0.0, 2.0 ** -17, 2.0 ** -12):
        y = ref.norm(x, None, weight, epsilon)[1]
        for to in (BF16, F16, F32):
            out = Floats(torch_cuda, np.zeros((rows, width)), to)
            source = Floats(torch_cuda, x, kind)
            mp.rms_norm(source.rows, d_weight.data_ptr(), epsilon, rows, width, out.rows)
            assert np.array_equal(out.back(), ref.rounded(y, to))


# Rows and weights times these powers of two; 8-bit rows and weights have scales of 2^-100 to 2^120.
POWERS = [(-98, 0), (-108, 0), (-122, 0), (-130, 0), (-122, 60), (-130, 60), (-90, -36), (-90, -40), (-70, -70), (-98, -98),
          (-95, 115), (-90, 100), (5, 115), (100, -90), (117, -98), (117, -4), (3, 117)]


@ANY
@pytest.mark.parametrize("rows, n", [(1, 64), (20, 64), (70, 16416), (300, 22016)])
def test_products_over_all_magnitudes(torch_cuda, kind, rows, n):
    """Rows and weights near both ends of their ranges. Beside the ordinary bound: what of an FP32 element lies below
    2^-133 does not count, and products and sums are multiples of 2^-149 (one step lost for each of them at the most,
    and there are no more sums than products)."""
    rng = np.random.default_rng(rows)
    k = 96
    ways = [0] if kind == F16 else range(len(POWERS))  # FP16 has no such range
    x0, w0 = rng.standard_normal((rows, k)), ref.held(rng.standard_normal((n, k)), E2M1)
    for i in ways:
        a, b = (-13, 117) if kind == F16 else POWERS[i]
        x, w = in_type(x0 * 2.0 ** a, kind), ref.held(w0 * 2.0 ** b, E2M1)
        matrix, source = Matrix(torch_cuda, n, k, w), rows_of(torch_cuda, x, kind)
        size = mp.w4_product_workspace(matrix.view, kind, rows)
        workspace = torch_cuda.empty(size + 16, dtype=torch_cuda.uint8, device="cuda")
        bound = ref.product_bound(x, w, PARTS[kind]) + 2 * 128 * PARTS[kind] * 2.0 ** -149
        if kind == F32 and a < -105:  # else all elements but the smallest are exact, and those are lost in the bound
            bound += 2.0 ** -133 * np.abs(w).sum(1)
        for to in (F32, BF16):
            out = Floats(torch_cuda, np.zeros((rows, n)), to)
            mp.w4_product(matrix.view, source.rows, rows, out.rows, workspace=workspace.data_ptr(), workspace_bytes=size)
            close(out.back(), x @ w.T, bound, to)


@pytest.mark.parametrize("rows, n", [(1, 64), (20, 64), (70, 16416), (300, 22016)])
def test_fp32_elements_are_exact_from_2_to_the_minus_110_on(torch_cuda, rows, n):
    """One element a row, 24 bits long: its product with a power of two is the element, and below 2^-110 it is cut to a
    multiple of 2^-133."""
    rng = np.random.default_rng(rows)
    k = 64
    x = np.zeros((rows, k))
    one = 1 + rng.integers(0, 1 << 23, rows) * 2.0 ** -23
    x[:, 7] = one * np.exp2(-105.0 - np.arange(rows) % 30) * np.where(rng.random(rows) < 0.5, 1, -1)
    if rows == 1:
        x[0, 7] = 2.0 ** -110 * (2 - 2.0 ** -23)
    x = ref.rounded(x, F32)
    w = np.zeros((n, k))
    w[:, 7] = np.exp2(np.arange(n) % 90)
    matrix, source, out = Matrix(torch_cuda, n, k, w), Floats(torch_cuda, x, F32), Floats(torch_cuda, np.zeros((rows, n)), F32)
    mp.w4_product(matrix.view, source.rows, rows, out.rows)
    held = np.where(np.abs(x) < 2.0 ** -110, np.trunc(x * 2.0 ** 133) * 2.0 ** -133, x)
    assert np.array_equal(out.back(), held @ w.T)


@pytest.mark.filterwarnings("ignore:overflow encountered in exp")
@pytest.mark.parametrize("kind", [F32, BF16, I8], ids=["f32", "bf16", "i8"])
@pytest.mark.parametrize("scale", [2.0 ** -40, 2.0 ** 40])
@pytest.mark.parametrize("rows, n", [(1, 64), (20, 64), (70, 16416), (300, 11008)])
def test_gated_products_of_small_and_large_rows(torch_cuda, kind, rows, n, scale):
    check_product(torch_cuda, np.random.default_rng(rows), rows, n, 96, kind, F32, True, scale=scale)


def packed(torch, rng, n, k):
    """A matrix of every code and scales around 2^-5, packed on the GPU, and its values."""
    w = E2M1[rng.integers(0, 8, (n, k))] * np.exp2(rng.integers(-8, -3, (n, k // 32))).repeat(32, 1)
    w *= 1 - 2 * rng.integers(0, 2, (n, k))
    m = Matrix(torch, n, k)
    mp.w4_pack(m.view, 0, Floats(torch, w, F32).rows, n)
    torch.cuda.synchronize()
    return m, w


def product_of(torch, matrix, gate, source, rows, n, kind, out):
    size = mp.w4_product_workspace(matrix.view, kind, rows, gate is not None)
    workspace = torch.empty(size + 64, dtype=torch.uint8, device="cuda").fill_(0xFF)
    mp.w4_product(matrix.view, source.rows, rows, out.rows, gate=gate.view if gate else None,
                  workspace=workspace.data_ptr(), workspace_bytes=size)
    got = out.back()
    out.check_padding()
    assert bool((workspace[size:] == 0xFF).all())
    return got


@pytest.mark.parametrize("rows, n, k", [call[:3] for call in CALLS])
def test_every_way_of_a_product(torch_cuda, rows, n, k):
    """Every kernel that sizes can lead to (w4_sizes.py), for every type of rows, alone and gated, results of odd rows."""
    rng = np.random.default_rng(rows + n + k)
    (matrix, w), (gate, g) = packed(torch_cuda, rng, n, k), packed(torch_cuda, rng, n, k)
    for kind in (F32, BF16, F16, I8):
        x = in_type(rng.standard_normal((rows, k)) * np.exp(rng.standard_normal(k)), kind)
        source = rows_of(torch_cuda, x, kind, 16)
        for gates in (None, g):
            want = ref.product(x, w, gates)
            bound = ref.product_bound(x, w, PARTS[kind]) if gates is None else ref.gated_bound(x, w, g, PARTS[kind])
            for to, pad in ((F32, 3), (kind if kind != I8 else F16, 0)):
                out = Floats(torch_cuda, np.zeros((rows, n)), to, pad)
                got = product_of(torch_cuda, matrix, gate if gates is not None else None, source, rows, n, kind, out)
                close(got, want, bound, to)
                if to == F32:  # in earnest, as FP32 sums are
                    off = np.linalg.norm(got - want) / np.linalg.norm(want)
                    assert off < 1e-6, off


@pytest.mark.parametrize("rows, n, k", [call[:3] for call in CALLS_EIGHT])
def test_8_bit_results_of_every_way(torch_cuda, rows, n, k):
    """Results in 8 bits are those of the same sums in FP32, bit for bit: codes, scales, no code below -127."""
    rng = np.random.default_rng(rows + n + k)
    (matrix, w), (gate, g) = packed(torch_cuda, rng, n, k), packed(torch_cuda, rng, n, k)
    for kind in (F32, BF16, F16, I8):
        x = in_type(rng.standard_normal((rows, k)) * np.exp(rng.standard_normal(k)), kind)
        source = rows_of(torch_cuda, x, kind)
        for gates in (None, g):
            m = gate if gates is not None else None
            sums = product_of(torch_cuda, matrix, m, source, rows, n, kind, Floats(torch_cuda, np.zeros((rows, n)), F32))
            bound = ref.product_bound(x, w, PARTS[kind]) if gates is None else ref.gated_bound(x, w, g, PARTS[kind])
            close(sums, ref.product(x, w, gates), bound, F32)
            out = Eight(torch_cuda, rows, n, None, 16)
            product_of(torch_cuda, matrix, m, source, rows, n, kind, out)
            code, sign, s = ref.split(sums, WHOLE)
            codes, scales = out.bytes()
            assert np.array_equal(scales, s) and np.array_equal(codes, np.where(sign, -code, code))


@TYPES
@pytest.mark.parametrize("over, pad, shift", [(1, 0, 0), (7, 8, 8), (3, 3, 1)])
def test_reads_of_many_rows(torch_cuda, kind, over, pad, shift):
    """From 2^22 runs of 16 bytes on a thread has eight rows: counts that are no multiple of eight, ids that are no rows
    beside others, rows behind the last."""
    torch = torch_cuda
    rng = np.random.default_rng(over)
    n, k = 53, 544
    runs = k // (4 if kind == F32 else 8)
    count = -(-(1 << 22) // runs) // 8 * 8 + 8 + over
    matrix, w = packed(torch, rng, n, k)
    ids = rng.integers(0, n, count).astype(np.int32)
    ids[rng.random(count) < 0.05] = -1
    ids[rng.random(count) < 0.05] = n
    ids[rng.random(count) < 0.01] = -(1 << 31)
    ids[-1], ids[0] = n - 1, (1 << 31) - 1
    d_ids = torch.from_numpy(ids).cuda()
    width = k + pad
    buffer = torch.full(((count + 3) * width + shift,), 77.0, dtype=getattr(torch, TORCH[kind]), device="cuda")
    out = buffer[shift:].view(count + 3, width)
    mp.w4_read(matrix.view, d_ids.data_ptr(), count, mp.Rows(out.data_ptr(), width, None, 0, kind))
    there = torch.from_numpy((ids >= 0) & (ids < n)).cuda()
    table = torch.from_numpy(ref.rounded(w, kind)).cuda().to(buffer.dtype)
    want = table[d_ids.clamp(0, n - 1).long()]
    assert bool((out[:count, :k] == want)[there].all())
    assert bool(out[:count, :k][~there].isnan().all())
    assert bool((out[count:] == 77).all()) and bool((out[:, k:] == 77).all()) and bool((buffer[:shift] == 77).all())


@pytest.mark.parametrize("kind", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows, width, pad, shift", [(3, 64, 0, 0), (5, 576, 3, 1), (2, 16512, 0, 0), (2, 16512, 1, 1), (9, 120, 0, 0)])
def test_norm_from_every_type_to_every_type(torch_cuda, kind, rows, width, pad, shift):
    rng = np.random.default_rng(width + pad)
    x, r = (ref.rounded(rng.standard_normal((rows, width)), kind) for _ in range(2))
    weight = (1 + 0.2 * rng.standard_normal(width)).astype(np.float32)
    d_weight = torch_cuda.from_numpy(weight).cuda()
    for residual in (None, r):
        y = ref.norm(x, residual, weight, 1e-6)[1]
        for to in (F32, BF16, F16) + ((I8,) if width % 32 == 0 else ()):
            source = Floats(torch_cuda, x, kind, pad, shift)
            added = Floats(torch_cuda, residual, kind, pad, shift) if residual is not None else None
            out = empty(torch_cuda, rows, width, to, 16 * pad if to == I8 else pad)
            mp.rms_norm(source.rows, d_weight.data_ptr(), 1e-6, rows, width, out.rows, residual=added.rows if added else None)
            assert np.array_equal(out.back(), ref.held(y, WHOLE) if to == I8 else ref.rounded(y, to))
            out.check_padding()


@pytest.mark.parametrize("pad", [0, 1])
def test_conversion_of_extremes(torch_cuda, pad):
    """Numbers near the smallest and the largest of each type, ties among them, and 8-bit rows with the outermost scales."""
    rng = np.random.default_rng(pad)
    width = 256
    x = np.exp2(rng.uniform(-149, 128, (40, width))) * rng.choice([-1, 1], (40, width))
    x[0] = np.arange(width) * 2.0 ** -149
    x[1] = (2 * np.arange(width) + 1) * 2.0 ** -134  # between two BF16 numbers
    x[2] = (2 * np.arange(width) + 1) * 2.0 ** -25  # between two FP16 numbers
    x[3] = 65504 + np.arange(width) / 8  # up to and past the border to infinity
    x[4] = (2 - 2.0 ** -8 - np.arange(-128, 128) * 2.0 ** -23) * 2.0 ** 127
    for kind in (F32, BF16, F16):
        with np.errstate(over="ignore"):
            held = ref.rounded(x, kind)
        source = Floats(torch_cuda, held, kind, pad)
        for to in (F32, BF16, F16):
            out = Floats(torch_cuda, np.zeros(x.shape), to, pad)
            mp.convert_rows(source.rows, len(x), width, out.rows)
            assert np.array_equal(out.back(), ref.rounded(held, to))
        eight = Eight(torch_cuda, len(x), width)
        mp.convert_rows(source.rows, len(x), width, eight.rows)
        code, sign, s = ref.split(held, WHOLE)
        codes, scales = eight.bytes()
        fine = (s != 255).repeat(32, 1)
        assert np.array_equal(scales, s) and np.array_equal(codes[fine], np.where(sign, -code, code)[fine])
    codes, scales = rng.integers(-127, 128, (40, width)), rng.choice([27, 28, 100, 110, 127, 140, 246, 247], (40, 8))
    eight = Eight(torch_cuda, 40, width)
    eight.codes.copy_(torch_cuda.from_numpy(codes.astype(np.int8)))
    eight.scales[:, :8] = torch_cuda.from_numpy(scales.astype(np.uint8))
    for to in (F32, BF16, F16):
        out = Floats(torch_cuda, np.zeros((40, width)), to, pad)
        mp.convert_rows(eight.rows, 40, width, out.rows)
        assert np.array_equal(out.back(), ref.rounded(codes * np.exp2(scales - 127.0).repeat(32, 1), to))


@pytest.mark.parametrize("width, pad", [(64, 0), (544, 48)])
def test_8_bit_rows_in_place(torch_cuda, width, pad):
    """Rows whose scales are not the smallest get those, in their own memory; values stay."""
    rng = np.random.default_rng(width)
    rows = 37
    eight = Eight(torch_cuda, rows, width, None, pad)
    codes = rng.integers(-127, 128, (rows, width // 32, 32)) >> rng.integers(0, 8, (rows, width // 32, 1))
    codes[3, 1] = 0
    scales = rng.integers(40, 240, (rows, width // 32))
    scales[5, 0] = 255
    eight.codes[:, :width] = torch_cuda.from_numpy(codes.reshape(rows, width).astype(np.int8))
    eight.scales[:, :width // 32] = torch_cuda.from_numpy(scales.astype(np.uint8))
    before = eight.back()
    mp.convert_rows(eight.rows, rows, width, eight.rows)
    assert np.array_equal(eight.back(), before, equal_nan=True)
    code, sign, s = ref.split(before, WHOLE)
    got, got_scales = eight.bytes()
    fine = (s != 255).repeat(32, 1)
    assert np.array_equal(got_scales, s) and np.array_equal(got[fine], np.where(sign, -code, code)[fine])
    eight.check_padding()


@pytest.mark.parametrize("n, k", [(53, 96), (4000, 544)])
def test_packing_and_reading_replayed(torch_cuda, n, k):
    """Captured and replayed for other weights, with eager calls between; the same id twice and more."""
    torch = torch_cuda
    rng = np.random.default_rng(n)
    source = Floats(torch, np.zeros((n, k)), BF16)
    m, out = Matrix(torch, n, k), Floats(torch, np.zeros((n + 9, k)), F32)
    ids = torch.from_numpy(np.concatenate((rng.permutation(n), [0] * 5, [n - 1] * 4)).astype(np.int32)).cuda()

    def step(stream):
        mp.w4_pack(m.view, 0, source.rows, n, stream=stream)
        mp.w4_read(m.view, ids.data_ptr(), n + 9, out.rows, stream=stream)

    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        step(torch.cuda.current_stream().cuda_stream)
    for _ in range(4):
        x = ref.rounded(rng.standard_normal((n, k)), BF16)
        source.matrix.copy_(torch.from_numpy(x))
        graph.replay()
        assert np.array_equal(out.back(), ref.held(x, E2M1)[ids.cpu().numpy()])
        source.matrix.mul_(-1)
        step(None)
        assert np.array_equal(out.back(), ref.held(-x, E2M1)[ids.cpu().numpy()])


def test_parts_of_a_tile_packed_on_two_streams(torch_cuda):
    """Rows of one tile by calls that may overlap: each writes its own."""
    torch = torch_cuda
    rng = np.random.default_rng(6)
    n, k = 16 * 40, 544
    x = ref.rounded(rng.standard_normal((n, k)), F32)
    want = ref.pack(x)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        m, pieces = Matrix(torch, n, k), []
        torch.cuda.synchronize()
        for first in range(0, n, 5):
            count = min(5, n - first)
            pieces.append(Floats(torch, x[first:first + count], F32))
        torch.cuda.synchronize()
        for i, piece in enumerate(pieces):
            mp.w4_pack(m.view, 5 * i, piece.rows, piece.matrix.shape[0], stream=streams[i % 2].cuda_stream)
        codes, scales = m.bytes()
        signs = [np.where((c & 15) == 8, c & 0xF0, c) for c in (codes, want[0])]
        signs = [np.where((c >> 4) == 8, c & 0x0F, c) for c in signs]
        assert np.array_equal(*signs) and np.array_equal(scales, want[1])


@ANY
@pytest.mark.parametrize("rows", [1, 20])
def test_the_deepest_products(torch_cuda, kind, rows):
    rng = np.random.default_rng(rows)
    n, k = 33, 1 << 20
    matrix, w = packed(torch_cuda, rng, n, k)
    x = in_type(rng.standard_normal((rows, k)), kind)
    out = Floats(torch_cuda, np.zeros((rows, n)), F32)
    got = product_of(torch_cuda, matrix, None, rows_of(torch_cuda, x, kind), rows, n, kind, out)
    close(got, x @ w.T, ref.product_bound(x, w, PARTS[kind]), F32)


@pytest.mark.parametrize("width, pad", [(1 << 20, 0), ((1 << 20) - 1, 1)])
def test_the_widest_rows(torch_cuda, width, pad):
    rng = np.random.default_rng(pad)
    x = ref.rounded(rng.standard_normal((2, width)), BF16)
    weight = np.ones(width, np.float32)
    d_weight = torch_cuda.from_numpy(weight).cuda()
    source, out = Floats(torch_cuda, x, BF16, pad), Floats(torch_cuda, np.zeros((2, width)), F16, pad)
    mp.rms_norm(source.rows, d_weight.data_ptr(), 1e-5, 2, width, out.rows)
    assert np.array_equal(out.back(), ref.rounded(ref.norm(x, None, weight, 1e-5)[1], F16))
    mp.convert_rows(source.rows, 2, width, out.rows)
    assert np.array_equal(out.back(), ref.rounded(x, F16))
    out.check_padding()
