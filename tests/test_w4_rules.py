"""4-bit matrices and 8-bit rows without a GPU: how products are divided (tests/native/w4_rules_tests.cpp), sizes, and
what the C entries refuse before any launch."""
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

from tinyinfer_amd import backend as mp

from . import w4_reference as ref
from .w4_sizes import CALLS, CALLS_EIGHT

ROOT = Path(__file__).resolve().parent.parent
GXX = shutil.which("g++")
P = 4096  # an aligned address that is never read: a refused call launches nothing


@pytest.mark.skipif(GXX is None, reason="g++ not available")
def test_w4_rules(tmp_path):
    exe = tmp_path / "w4_rules_tests"
    subprocess.run([GXX, "-std=c++17", "-Wall", "-Werror", "-g", "-fsanitize=address,undefined",
                    "-fno-sanitize-recover=undefined", f"-I{ROOT / 'tinyinfer_amd' / 'csrc' / 'backend'}",
                    str(ROOT / "tests" / "native" / "w4_rules_tests.cpp"), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout == "ok\n", run.stderr


def rows(**changes):
    r = dict(data=P, stride=576, scales=None, scale_stride=0, type=mp.TYPE_F32)
    r.update(changes)
    return mp.Rows(*[r[n] for n, _ in mp.Rows._fields_])


def eight(**changes):
    return rows(**{**dict(scales=P, scale_stride=20, type=mp.TYPE_I8), **changes})


def matrix(**changes):
    m = dict(codes=P, scales=P, rows=960, depth=576)
    m.update(changes)
    return mp.W4Matrix(*[m[n] for n, _ in mp.W4Matrix._fields_])


def out(**changes):
    return rows(**{**dict(data=2 * P, stride=960), **changes})


def pack(m=None, first=0, x=None, rows_=960):
    mp.w4_pack(m or matrix(), first, x or rows(), rows_)


def read(m=None, ids=P, count=5, to=None):
    mp.w4_read(m or matrix(), ids, count, to or rows())


def convert(x=None, count=5, width=576, to=None):
    mp.convert_rows(x or rows(), count, width, to or rows(data=2 * P))


def norm(x=None, weight=P, epsilon=1e-5, count=5, width=576, to=None, residual=None, total=None):
    mp.rms_norm(x or rows(), weight, epsilon, count, width, to or rows(data=2 * P), residual=residual, sum=total)


def product(m=None, x=None, count=5, to=None, gate=None, **space):
    mp.w4_product(m or matrix(), x or rows(), count, to or out(), gate=gate, **space)


def refused(call, text):
    with pytest.raises(mp.BackendError, match=text) as e:
        call()
    assert e.value.status == mp.MP_INVALID_ARGUMENT


BAD_MATRICES = [dict(codes=None), dict(scales=None), dict(codes=P + 8), dict(scales=P + 8), dict(rows=0), dict(rows=-1),
                dict(rows=(1 << 24) + 1), dict(depth=0), dict(depth=-32), dict(depth=16), dict(depth=577), dict(depth=(1 << 20) + 32)]


@pytest.mark.parametrize("changes", BAD_MATRICES, ids=str)
def test_bad_matrices_are_refused(changes):
    for call in (pack, read, product):
        refused(lambda: call(matrix(**changes)), "4-bit matrix")
    refused(lambda: product(gate=matrix(**changes)), "4-bit")
    if "rows" in changes or "depth" in changes:
        m = matrix(**changes)
        refused(lambda: mp.w4_sizes(m.rows, m.depth), "4-bit matrix")
        refused(lambda: mp.w4_product_workspace(m, mp.TYPE_F32, 5), "4-bit matrix")


BAD_ROWS = [(rows(data=None), "missing"), (rows(data=P + 2), "misaligned"), (rows(stride=575), "stride"), (rows(stride=-576), "stride"),
            (rows(type=4), "type"), (rows(type=-1), "type"), (rows(data=P + 1, type=mp.TYPE_BF16), "misaligned"),
            (rows(stride=(1 << 40) + 1), "stride")]
BAD_EIGHT = [(eight(data=P + 8), "aligned"), (eight(stride=584), "aligned"), (eight(scales=None), "scales"),
             (eight(scales=P + 2), "scales"), (eight(scale_stride=16), "scales"), (eight(scale_stride=18), "scales")]


@pytest.mark.parametrize("bad, text", BAD_ROWS, ids=range(len(BAD_ROWS)))
def test_bad_rows_are_refused(bad, text):
    for call in (lambda: pack(x=bad), lambda: read(to=bad), lambda: convert(bad), lambda: convert(to=bad), lambda: norm(bad),
                 lambda: norm(to=bad), lambda: norm(residual=bad), lambda: product(x=bad)):
        refused(call, text)
    if "stride" not in text:
        bad.stride = 960
        refused(lambda: product(to=bad), text)


@pytest.mark.parametrize("bad, text", BAD_EIGHT, ids=range(len(BAD_EIGHT)))
def test_bad_8_bit_rows_are_refused(bad, text):
    for call in (lambda: convert(bad), lambda: convert(to=bad), lambda: norm(to=bad), lambda: product(x=bad)):
        refused(call, text)


@pytest.mark.parametrize("call, text", [
    (lambda: pack(x=eight()), "type"), (lambda: read(to=eight()), "type"), (lambda: norm(x=eight()), "type"),
    (lambda: norm(residual=eight()), "type"),
    (lambda: pack(first=-1), "no such rows"), (lambda: pack(first=1), "no such rows"), (lambda: pack(rows_=-1), "no such rows"),
    (lambda: pack(rows_=961), "no such rows"), (lambda: pack(first=(1 << 31) - 1, rows_=(1 << 31) - 1), "no such rows"),
    (lambda: read(ids=None), "ids"), (lambda: read(ids=P + 2), "ids"), (lambda: read(count=-1), "rows a call"),
    (lambda: read(count=(1 << 20) + 1), "rows a call"),
    (lambda: read(matrix(depth=16384), count=1 << 20, to=rows(stride=16384)), "too many"),
    (lambda: convert(count=-1), "rows a call"), (lambda: convert(count=(1 << 20) + 1), "rows a call"),
    (lambda: convert(width=0), "width"), (lambda: convert(width=-5), "width"),
    (lambda: convert(rows(stride=1 << 21), width=(1 << 20) + 1), "width"),
    (lambda: convert(rows(stride=16384), count=1 << 20, width=16384, to=rows(data=2 * P, stride=16384)), "too many"),
    (lambda: convert(to=eight(), width=570), "whole groups"), (lambda: convert(to=rows(stride=600)), "in place"),
    (lambda: convert(rows(data=P, type=mp.TYPE_BF16), to=rows()), "in place"),
    (lambda: convert(eight(), to=eight(scales=2 * P)), "in place"),
    (lambda: norm(weight=None), "weight"), (lambda: norm(weight=P + 2), "weight"), (lambda: norm(epsilon=-1.0), "epsilon"),
    (lambda: norm(epsilon=float("nan")), "epsilon"), (lambda: norm(epsilon=float("inf")), "epsilon"),
    (lambda: norm(total=rows(data=3 * P)), "without a residual"),
    (lambda: norm(residual=rows(data=3 * P, type=mp.TYPE_BF16)), "one type"),
    (lambda: norm(residual=rows(data=3 * P), total=rows(data=4 * P, type=mp.TYPE_F16)), "one type"),
    (lambda: norm(to=rows(stride=600)), "in place"), (lambda: norm(residual=rows(data=2 * P)), "in place"),
    (lambda: norm(residual=rows(data=3 * P), total=rows(data=2 * P)), "in place"),
    (lambda: norm(residual=rows(data=3 * P), total=rows(stride=600)), "in place"),
    (lambda: norm(residual=rows(data=3 * P), total=rows(data=3 * P, stride=600)), "in place"),
    (lambda: norm(to=eight(data=P)), "in place"), (lambda: norm(width=570, to=eight(data=2 * P)), "whole groups"),
    (lambda: product(count=-1), "rows a call"), (lambda: product(count=(1 << 20) + 1), "rows a call"),
    (lambda: product(to=out(stride=959)), "stride"), (lambda: product(gate=matrix(rows=950)), "gate"),
    (lambda: product(gate=matrix(depth=608)), "gate"), (lambda: product(to=out(data=P)), "in place"),
    (lambda: product(matrix(rows=950), to=eight(data=2 * P, stride=960, scale_stride=32)), "whole groups"),
    (lambda: mp.w4_product_workspace(matrix(), 4, 5), "type"), (lambda: mp.w4_product_workspace(matrix(), -1, 5), "type"),
    (lambda: mp.w4_product_workspace(matrix(), 0, -1), "rows a call"),
    (lambda: mp.w4_product_workspace(matrix(), 0, (1 << 20) + 1), "rows a call"),
])
def test_bad_arguments_are_refused(call, text):
    refused(call, text)


def test_nothing_to_do_launches_nothing():
    pack(rows_=0)
    pack(first=960, rows_=0)
    read(count=0)
    convert(count=0)
    norm(count=0)
    product(count=0)
    assert mp.w4_product_workspace(matrix(), mp.TYPE_F32, 0) == 0


@pytest.mark.parametrize("n, k", [(1, 32), (16, 128), (17, 160), (49152, 576), (33, 544)])
def test_sizes(n, k):
    codes, scales = mp.w4_sizes(n, k)
    assert codes == -(-n // 16) * -(-k // 128) * 1024 and scales == -(-n // 16) * -(-k // 512) * 256
    if n < 100:
        assert [len(b) for b in ref.pack(np.ones((n, k)))] == [codes, scales]


def test_the_reference_itself():
    """The grids, the ties and the scales that the definition names."""
    x = np.array([[6.0, 5.0, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25] + [0.0] * 24])
    assert ref.held(x, ref.E2M1).tolist() == [[6, 4, 4, 2, 2, 1, 1, 0] + [0] * 24]
    assert ref.held(-x, ref.E2M1).tolist() == (-ref.held(x, ref.E2M1)).tolist()
    assert ref.split(x * 1.0001, ref.E2M1)[2].tolist() == [[128]] and ref.split(x, ref.E2M1)[2].tolist() == [[127]]
    y = np.array([[127.0, 126.5, 0.5, 1.5] + [0.0] * 28])
    assert ref.held(y, ref.WHOLE).tolist() == [[127, 126, 0, 2] + [0] * 28]
    for grid, most in ((ref.E2M1, 6.0), (ref.WHOLE, 127.0)):
        for value, byte in ((most * 2.0 ** 120, 247), (most * 2.0 ** 120 * 1.001, 255), (np.inf, 255), (np.nan, 255), (0.0, 27),
                            (most * 2.0 ** -100, 27), (most * 2.0 ** -99, 28)):
            assert ref.split(np.full((1, 32), value), grid)[2].tolist() == [[byte]]


@pytest.mark.parametrize("count, n, depth, kind, gated", [
    (1 << 20, (1 << 17) + 1, 32, mp.TYPE_BF16, False), (1 << 20, (1 << 16) + 1, 32, mp.TYPE_F32, True),
    ((1 << 13) + 1, 1 << 24, 32, mp.TYPE_F16, False), (1 << 20, 4096, 32800, mp.TYPE_I8, False)])
def test_products_too_large_for_one_call_are_refused(count, n, depth, kind, gated):
    stride = -(-depth // 128) * 128
    x = rows(stride=stride, type=kind) if kind != mp.TYPE_I8 else eight(stride=stride, scale_stride=stride // 32)
    m = matrix(rows=n, depth=depth)
    size = mp.w4_product_workspace(m, kind, count, gated)
    refused(lambda: product(m, x, count, out(stride=n), gate=m if gated else None, workspace=P, workspace_bytes=size),
            "too large for one call")


@pytest.mark.skipif(GXX is None, reason="g++ not available")
def test_calls_take_every_way(tmp_path):
    """The calls of w4_sizes.py take the ways that they are there for, and leave none out that sizes can lead to."""
    exe = tmp_path / "w4_plan_of"
    subprocess.run([GXX, "-std=c++17", "-O2", "-Wall", "-Werror", f"-I{ROOT / 'tinyinfer_amd' / 'csrc' / 'backend'}",
                    str(ROOT / "tests" / "native" / "w4_plan_of.cpp"), "-o", str(exe)], check=True)

    def plan(*args):
        run = subprocess.run([str(exe), *map(str, args)], capture_output=True, text=True, check=True)
        return [tuple(map(int, line.split())) for line in run.stdout.splitlines()]

    taken = set()
    for eight, calls in ((0, CALLS), (1, CALLS_EIGHT)):
        for call in calls:
            for gated, want in ((0, call.plain), (1, call.gated)):
                for parts in (1, 2, 3):
                    got, = plan(call.rows, call.n, call.k, parts, gated, eight)
                    assert got[:3] == want, call
                    if eight and len(got) == 4:  # the same sums as with results in FP32
                        assert plan(call.rows, call.n, call.k, parts, gated, 0)[0][3] == got[3], call
                taken.add((gated, eight, *want))
    assert taken == set(plan())
