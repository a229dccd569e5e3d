"""Products that take every way and every kernel that w4_rules.h can choose. Which one each takes is held by
test_w4_rules.py, what it computes by test_w4.py, for every type of rows and results."""
from __future__ import annotations

from typing import NamedTuple

FEW, SMALL, LARGE = range(3)


class Call(NamedTuple):
    rows: int
    n: int
    k: int
    plain: tuple  # way; for few rows also the side of a tile and a wavefront's tiles of columns
    gated: tuple


CALLS = [
    # A wavefront's tiles of 16 by 16: one, two (the last of them behind the end), four.
    Call(7, 333, 1184, (FEW, 16, 1), (FEW, 16, 1)),
    Call(1, 8221, 1056, (FEW, 16, 2), (FEW, 16, 2)),
    Call(9, 16301, 96, (FEW, 16, 2), (FEW, 16, 2)),
    Call(1, 16411, 1056, (FEW, 16, 4), (FEW, 16, 4)),
    Call(16, 16411, 160, (FEW, 16, 4), (FEW, 16, 4)),
    # Of 32 by 32: one, two.
    Call(203, 333, 544, (FEW, 32, 1), (FEW, 32, 1)),
    Call(20, 16411, 544, (FEW, 32, 2), (FEW, 32, 2)),
    Call(64, 8221, 544, (FEW, 32, 2), (FEW, 32, 2)),
    Call(96, 5461, 288, (FEW, 32, 2), (FEW, 32, 2)),
    # Tiles, small and large.
    Call(70, 8229, 160, (FEW, 32, 2), (SMALL,)),
    Call(40, 32771, 96, (SMALL,), (SMALL,)),
    Call(70, 16421, 160, (SMALL,), (SMALL,)),
    Call(300, 11001, 160, (SMALL,), (LARGE,)),
    Call(300, 21901, 96, (LARGE,), (LARGE,)),
]
# With results of 8 bits, whose groups of 32 need two tiles of 16 columns.
CALLS_EIGHT = [
    Call(7, 352, 1184, (FEW, 16, 2), (FEW, 16, 2)),
    Call(16, 8224, 1056, (FEW, 16, 2), (FEW, 16, 2)),
    Call(1, 16416, 1056, (FEW, 16, 4), (FEW, 16, 4)),
    Call(3, 16416, 160, (FEW, 16, 4), (FEW, 16, 4)),
    Call(203, 352, 544, (FEW, 32, 1), (FEW, 32, 1)),
    Call(20, 16416, 544, (FEW, 32, 2), (FEW, 32, 2)),
    Call(96, 5472, 288, (FEW, 32, 2), (FEW, 32, 2)),
    Call(70, 8224, 160, (FEW, 32, 2), (SMALL,)),
    Call(70, 16416, 160, (SMALL,), (SMALL,)),
    Call(300, 11008, 160, (SMALL,), (LARGE,)),
    Call(300, 21920, 96, (LARGE,), (LARGE,)),
]
