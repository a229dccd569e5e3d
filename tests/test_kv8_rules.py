"""The 8-bit K/V cache without a GPU: what its calls touch and how they are
divided (tests/native/kv8_rules_tests.cpp), and what the C entries refuse
before any launch."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

from tinyinfer_amd import backend as mp

from .kv8_reference import E4M3, INT8, Cache, likely_bound
from .kv8_sizes import WALKS

ROOT = Path(__file__).resolve().parent.parent
GXX = shutil.which("g++")
P = 4096  # an aligned address that is never read: a refused call launches nothing


@pytest.mark.skipif(GXX is None, reason="g++ not available")
def test_kv8_rules(tmp_path):
    exe = tmp_path / "kv8_rules_tests"
    subprocess.run([GXX, "-std=c++17", "-Wall", "-Werror", "-g", "-fsanitize=address,undefined",
                    "-fno-sanitize-recover=undefined", f"-I{ROOT / 'tinyinfer_amd' / 'csrc' / 'backend'}",
                    str(ROOT / "tests" / "native" / "kv8_rules_tests.cpp"), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout == "ok\n", run.stderr


def cache(**changes):
    c = dict(keys=P, values=P, scales=P, blocks=8, layers=2, block_tokens=16, kv_heads=3, dim=64, format=mp.KV8_INT8)
    c.update(changes)
    return mp.Kv8Cache(*[c[n] for n, _ in mp.Kv8Cache._fields_])


def append(c=None, layer=0, **changes):
    a = dict(k=P, k_stride=192, v=P, v_stride=192, type=mp.TYPE_F32, tables=P, table_stride=4, starts=P, used=P,
             sequences=2, rows=5, rope=None, q=P, q_stride=576, q_out=P, q_out_stride=576, heads=9)
    a.update(changes)
    mp.kv8_append(c or cache(), layer, **a)


def read(c=None, layer=0, **changes):
    a = dict(tables=P, table_stride=4, starts=P, used=P, sequences=2, rows=5, type=mp.TYPE_F32, k=P, k_stride=192,
             v=P, v_stride=192)
    a.update(changes)
    mp.kv8_read(c or cache(), layer, **a)


def decode(c=None, layer=0, **changes):
    a = dict(q=P, q_stride=576, type=mp.TYPE_F32, tables=P, table_stride=4, lengths=P, rows=5, heads=9, max_length=64,
             scale=0.125, out=P, out_stride=576)
    a.update(changes)
    mp.kv8_attention_decode(c or cache(), layer, **a)


def prefill(c=None, layer=0, **changes):
    a = dict(q=P, q_stride=576, type=mp.TYPE_F32, tables=P, table_stride=4, starts=P, used=P, sequences=2, rows=5,
             heads=9, max_length=64, scale=0.125, out=P, out_stride=576)
    a.update(changes)
    mp.kv8_attention_prefill(c or cache(), layer, **a)


def workspace(c=None, rows=5, sequences=2, heads=9, max_length=64):
    return mp.kv8_attention_workspace(c or cache(), rows, sequences, heads, max_length)


BAD_CACHES = [dict(keys=None), dict(values=None), dict(scales=None), dict(keys=P + 8), dict(values=P + 4),
              dict(scales=P + 4), dict(block_tokens=8), dict(block_tokens=24), dict(block_tokens=256),
              dict(block_tokens=0), dict(dim=32), dict(dim=96), dict(dim=512), dict(format=2), dict(format=-1),
              dict(blocks=0), dict(layers=0), dict(layers=1 << 20), dict(blocks=1 << 28), dict(kv_heads=0), dict(kv_heads=2000)]


def refused(call, text):
    with pytest.raises(mp.BackendError, match=text) as e:
        call()
    assert e.value.status == mp.MP_INVALID_ARGUMENT


@pytest.mark.parametrize("changes", BAD_CACHES, ids=str)
def test_bad_caches_are_refused(changes):
    for call in (append, read, decode, prefill):
        refused(lambda: call(cache(**changes)), "8-bit")
    if not {"keys", "values", "scales"} & set(changes):
        refused(lambda: workspace(cache(**changes)), "8-bit")


def test_bad_layers_are_refused():
    for call in (append, read, decode, prefill):
        for layer in (-1, 2):
            refused(lambda: call(layer=layer), "no such layer")


@pytest.mark.parametrize("call, changes, text", [
    (append, dict(k=None), "row matrix"), (append, dict(v=P + 2), "row matrix"), (append, dict(k_stride=191), "stride"),
    (append, dict(v_stride=-192), "stride"), (append, dict(type=3), "element type"), (append, dict(q_out=None), "row matrix"),
    (append, dict(q_stride=575), "stride"), (append, dict(q_out_stride=600), "in place"), (append, dict(heads=0), "heads"),
    (append, dict(tables=None), "tables"), (append, dict(table_stride=0), "table_stride"), (append, dict(starts=None), "starts"),
    (append, dict(used=P + 2), "starts or used"), (append, dict(rows=-1), "rows"), (append, dict(rows=(1 << 20) + 1), "rows"),
    (append, dict(sequences=-1), "sequences"),
    (append, dict(rope=mp.Rope(P, P, 10, 63, 0)), "rotated dims"), (append, dict(rope=mp.Rope(P, P, 10, 66, 0)), "rotated dims"),
    (append, dict(rope=mp.Rope(P, P, 10, -2, 0)), "rotated dims"), (append, dict(rope=mp.Rope(None, P, 10, 64, 0)), "tables"),
    (append, dict(rope=mp.Rope(P, P, 0, 64, 0)), "tables"),
    (append, dict(rows=1 << 20, k_stride=65536, v_stride=65536, c=cache(kv_heads=1024), q=None), "too many"),
    (read, dict(k=None), "row matrix"), (read, dict(v_stride=100), "stride"), (read, dict(starts=None), "starts"),
    (read, dict(type=-1), "element type"),
    (decode, dict(q=None), "row matrix"), (decode, dict(out=None), "row matrix"), (decode, dict(q_stride=64), "stride"),
    (decode, dict(lengths=None), "lengths"), (decode, dict(heads=10), "multiple of kv_heads"),
    (decode, dict(heads=51, q_stride=51 * 64, out_stride=51 * 64), "at most 16"), (decode, dict(heads=0), "heads"),
    (decode, dict(max_length=-1), "max_length"), (decode, dict(max_length=(1 << 30) + 1), "max_length"),
    (decode, dict(scale=float("nan")), "scale"), (decode, dict(scale=float("inf")), "scale"),
    (decode, dict(scale=-1.0), "scale"), (decode, dict(scale=3e38), "scale"),
    (decode, dict(rows=1 << 19), "too many"), (prefill, dict(rows=1 << 19), "too many"), (decode, dict(max_length=10000), "workspace"),
    (decode, dict(max_length=10000, workspace=P + 4, workspace_bytes=1 << 30), "aligned"),
    (decode, dict(max_length=10000, workspace=None, workspace_bytes=1 << 30), "workspace"),
    (prefill, dict(starts=None), "starts"), (prefill, dict(used=None), "used"), (prefill, dict(scale=float("nan")), "scale"),
    (prefill, dict(max_length=100000), "workspace"), (prefill, dict(out_stride=10), "stride"),
], ids=lambda v: getattr(v, "__name__", str(v)))
def test_bad_arguments_are_refused(call, changes, text):
    refused(lambda: call(**changes), text)


def test_nothing_to_do_launches_nothing():
    for call in (append, read, prefill):
        call(rows=0)
        call(sequences=0)
    decode(rows=0)
    assert workspace(rows=0) == 0 and workspace(max_length=0) == 0


def test_workspace_sizes():
    # One row needs none while one work-group's chunk holds it; long ones do.
    assert workspace(rows=1, sequences=1, max_length=128) == 0
    assert workspace(rows=1, sequences=1, max_length=16384) >= 9 * 66 * 4
    size = ctypes.c_size_t()
    assert mp.lib().mp_hip_kv8_attention_workspace(cache(), 1, 1, 9, 64, None) == mp.MP_INVALID_ARGUMENT
    assert mp.lib().mp_hip_kv8_attention_workspace(None, 1, 1, 9, 64, ctypes.byref(size)) == mp.MP_INVALID_ARGUMENT


@pytest.mark.parametrize("call", [decode, prefill])
def test_attention_over_its_queries_with_another_stride_is_refused(call):
    """A row's output would lie over the queries of others."""
    q = 1 << 16
    for strides in (dict(q_stride=576, out_stride=640), dict(q_stride=640, out_stride=576)):
        refused(lambda: call(q=q, out=q, **strides), "one stride")
    refused(lambda: call(q=q, out=q, q_stride=640, out_stride=576, rows=2, type=mp.TYPE_BF16), "one stride")
    call(q=q, out=q, q_stride=640, out_stride=576, rows=0)  # nothing to lie over


def evaluated(q, k, v, scale, q_parts, p_parts):
    """One row's attention as FP32 sums of products with FP16 numbers: q and p as the sum of one or two of them."""
    f = np.float32

    def parts(x, n):
        high = x.astype(np.float16).astype(f)
        return [high, (x - high).astype(np.float16).astype(f)][:n]

    up = f(2.0 ** (14 - np.floor(np.log2(np.abs(q).max()))))
    k, v, s = k.astype(f), v.astype(f), np.zeros(len(k), dtype=f)
    for d in range(0, len(q), 8):
        for part in parts(q * up, q_parts):
            s += k[:, d:d + 8] @ part[d:d + 8]
    s *= f(scale * 1.4426950408889634) / up
    out, total = np.zeros(v.shape[1], dtype=f), f(0)
    for part in parts(np.exp2(s - s.max() + f(11)), p_parts):
        for t in range(0, len(k), 32):
            out += part[t:t + 32] @ v[t:t + 32]
            total += part[t:t + 32].sum(dtype=f)
    return out / total


@pytest.mark.parametrize("fmt", [INT8, E4M3], ids=["int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_single_parts_are_too_far_off(dim, fmt):
    """The limit that attention is held to on the GPU (kv8_reference.likely_bound) finds out a query or a probability
    that has lost its low part, at every dim; with both parts arithmetic in FP32 is far inside of it."""
    rng = np.random.default_rng(dim + fmt)
    worst = {}
    for n in (1, 2, 15, 16, 17, 31, 32, 33, 63, 65, 127, 128, 129, 300, 777):
        pages = -(-n // 16)
        cache = Cache(pages, 1, 1, 16, dim, fmt, rng)
        table = np.arange(pages, dtype=np.int32)[None]
        k, v = (rng.standard_normal((n, 1, dim)).astype(np.float32) for _ in range(2))
        k *= np.exp(0.5 * rng.standard_normal(dim)).astype(np.float32)
        cache.append(0, k, v, table, [0, n], [0])
        k, v = (cache.tokens(0, kind, table[0], n)[0] for kind in range(2))
        for _ in range(3):
            q, scale = rng.standard_normal(dim).astype(np.float32), 1.3 / dim ** 0.5
            z = k @ q.astype(np.float64) * scale
            p = np.exp(z - z.max())
            p /= p.sum()
            for parts in ((2, 2), (1, 2), (2, 1)):
                off = np.abs(evaluated(q, k, v, scale, *parts) - p @ v).max() / likely_bound(p, z, q, k, v, scale)
                worst[parts] = max(worst.get(parts, 0.0), off)
    assert worst[2, 2] < 0.1 and worst[1, 2] > 1 and worst[2, 1] > 1, worst


@pytest.mark.skipif(GXX is None, reason="g++ not available")
def test_plans_of_the_far_walks(tmp_path):
    """The calls of kv8_sizes.py take the paths that they are there for."""
    exe = tmp_path / "kv8_plan_of"
    subprocess.run([GXX, "-std=c++17", "-Wall", "-Werror", f"-I{ROOT / 'tinyinfer_amd' / 'csrc' / 'backend'}",
                    str(ROOT / "tests" / "native" / "kv8_plan_of.cpp"), "-o", str(exe)], check=True)
    got = {}
    for w in WALKS:
        out = subprocess.run([str(exe), *(str(int(x)) for x in (w.decode, sum(w.counts), len(w.counts), w.kv_heads,
                                                                w.group, w.dim, w.longest))],
                             capture_output=True, text=True, check=True, timeout=60).stdout
        got[w.name] = tuple(int(x) for x in out.split()[:3])
    assert got == {w.name: w.plan for w in WALKS}
    steps = {(w.decode, w.plan[1], w.dim): 0 for w in WALKS}
    for w in WALKS:
        steps[w.decode, w.plan[1], w.dim] = max(steps[w.decode, w.plan[1], w.dim], w.steps)
    assert sum(n > 64 for n in steps.values()) >= 5 and sum(n > 32 for n in steps.values()) >= 8, steps
