"""Attention calls whose wavefronts walk far: the exchange of tile places beyond 32 steps, twice (beyond 64), and
work-groups of eight wavefronts. What plan each takes is held by test_kv8_rules.py, what it computes by test_kv8.py."""
from __future__ import annotations

from typing import NamedTuple

from .kv8_reference import BF16, E4M3, F16, F32, INT8


class Walk(NamedTuple):
    name: str
    decode: bool
    kind: int
    fmt: int
    kv_heads: int
    group: int
    dim: int
    bt: int
    counts: tuple   # rows of each sequence (decode: 1 each)
    longest: int    # max_length, the tokens that the longest sequence has
    plan: tuple     # column tiles, wavefronts, splits
    steps: int      # of 32 tokens, of one wavefront


def _steps(longest, waves):
    return -(-(-(-longest // 32)) // waves)


def _walk(name, decode, kind, fmt, kv_heads, group, dim, bt, counts, longest, tiles, waves):
    return Walk(name, decode, kind, fmt, kv_heads, group, dim, bt, tuple(counts), longest, (tiles, waves, 1),
                _steps(longest, waves))


WALKS = [
    # Eight wavefronts a work-group.
    _walk("decode_8_waves", True, F32, INT8, 3, 3, 64, 16, [1] * 64, 2175, 1, 8),
    _walk("decode_8_waves_far", True, F32, E4M3, 3, 3, 64, 16, [1] * 64, 8700, 1, 8),
    _walk("decode_8_waves_128", True, BF16, E4M3, 3, 4, 128, 64, [1] * 64, 4100, 1, 8),
    _walk("decode_8_waves_12_heads", True, F32, INT8, 3, 12, 128, 32, [1] * 60, 3000, 1, 8),
    _walk("decode_8_waves_256", True, F32, INT8, 3, 2, 256, 16, [1] * 64, 2500, 1, 8),
    _walk("prefill_8_waves", False, F32, INT8, 3, 3, 64, 16, [1] * 20 + [6] * 20, 4000, 1, 8),
    _walk("prefill_8_waves_two_tiles", False, F16, E4M3, 3, 3, 128, 32, [40] * 12, 6000, 2, 8),
    # Four, beyond 32 and 64 steps.
    _walk("decode_4_waves_far", True, F32, E4M3, 8, 1, 64, 16, [1] * 64, 8600, 1, 4),
    _walk("decode_4_waves_128", True, F16, INT8, 8, 4, 128, 128, [1] * 64, 4400, 1, 4),
    _walk("decode_4_waves_256", True, F32, E4M3, 8, 2, 256, 16, [1] * 64, 8400, 1, 4),
    _walk("prefill_4_waves_far", False, F32, INT8, 3, 3, 64, 16, [1] * 170 + [40] * 6, 8700, 2, 4),
    _walk("prefill_4_waves_far_e4m3", False, BF16, E4M3, 8, 4, 128, 64, [1] * 60 + [20] * 8, 8300, 2, 4),
    _walk("prefill_4_waves_256", False, F32, E4M3, 8, 2, 256, 16, [1] * 60 + [20] * 8, 4400, 1, 4),
    # One.
    _walk("prefill_1_wave_64", False, F32, E4M3, 8, 4, 64, 16, [250] * 18, 2200, 2, 1),
    _walk("prefill_1_wave_128", False, BF16, INT8, 8, 4, 128, 64, [250] * 18, 2100, 2, 1),
    _walk("prefill_1_wave_256", False, F16, E4M3, 8, 4, 256, 32, [150] * 18, 1500, 1, 1),
]
