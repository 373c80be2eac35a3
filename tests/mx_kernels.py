"""Which kernel of csrc/mx_linear.hip serves a microscaled product, restated from plan_mx_linear, and product shapes that
together reach each of them, gated and not, dense and by expert, with K in whole windows of 512 columns and not."""

from __future__ import annotations

import re
from pathlib import Path

SOURCE = Path(__file__).resolve().parents[1] / "raon-npu_amd" / "csrc" / "mx_linear.hip"


def constants() -> dict[str, int]:
    text = SOURCE.read_text()
    names = ("kOneFragment", "kFewRows", "kFlat", "kFillSmall", "kFillLarge", "kFewEach", "kFillEach", "kStaying")
    return {n: int(re.search(rf"\b{n} = (\d+)", text).group(1)) for n in names}


def kernel_of(n: int, M: int, K: int, experts: int = 0, aligned: bool = True) -> tuple:
    """("few", NA, WR) or ("tiles", MA, NB, WA, WB, whole windows, stays) of n rows by M weight rows of K columns."""
    c = constants()

    def tiles(weights, rows):
        return -(-n // rows) * -(-M // weights)

    rows = M * (min(n, n // 16 + experts) if experts else -(-n // 16))
    if rows <= c["kOneFragment"]:
        return "few", 1, 1
    if rows <= c["kFewRows"]:
        return "few", 2, 1
    wide = K > 1 << 20 or M * (K // 32) >= 1 << 32
    whole = K % 512 == 0 and aligned

    def pick(*shape, stays=False):
        return ("tiles", *shape, whole, stays and whole)

    def large():
        return pick(4, 2, 2, 4, stays=tiles(256, 256) > c["kStaying"])

    if experts:
        if wide or n < c["kFewEach"] * experts:
            return "few", 2, 2
        if n >= c["kFillEach"] * experts and tiles(256, 256) >= c["kFillLarge"]:
            return large()
        return pick(2, 1, 2, 2)
    fill = tiles(64, 64) >= c["kFillSmall"]
    if wide or (n <= 2 and fill):
        return "few", 2, 4
    if n <= c["kFlat"]:
        return pick(2, 1, 2, 2) if fill else pick(1, 1, 2, 2)
    if tiles(256, 256) >= c["kFillLarge"]:
        return large()
    return pick(2, 2, 2, 2) if fill else pick(1, 1, 2, 2)


# (T, M, K) of dense products and (rows of each expert, M, K) of those by expert; each with and without a gate.
DENSE = [(5, 90, 160), (70, 42, 1024), (20, 4100, 544), (1, 8194, 1024),    # few rows: one fragment a wave, two
         (2, 64010, 96), (1, 64006, 512),                                  # without shared parts of K
         (70, 4100, 160), (300, 1030, 1056), (70, 4100, 512), (130, 3970, 1024),  # 64 x 64
         (3, 64010, 160), (40, 64006, 544), (3, 64010, 512), (4, 64010, 2560), (96, 33002, 1024),  # 128 x 64
         (1030, 4100, 992), (1030, 4100, 1024), (1030, 4098, 512),         # 128 x 128
         (1030, 9300, 96), (1030, 9300, 1056), (2100, 9300, 544), (1030, 9300, 1024), (1030, 9302, 512),  # 256 x 256
         (2100, 9300, 512), (2100, 9306, 1024)]                            # workgroups that take tile after tile
EXPERTS = [([1, 0, 3], 96, 160), ([5, 0, 1, 16, 17, 0], 130, 512), ([9, 0, 5, 30], 1604, 544),
           ([1, 3, 0, 2] * 10, 1030, 160), ([2] * 40, 1034, 1024),
           ([40, 0, 70, 55, 64, 1] * 3, 2050, 544), ([40, 70, 55, 64] * 3, 2050, 512), ([45, 3, 65, 64] * 3, 2050, 1024),
           ([1500, 0, 257, 2500], 3004, 352), ([1500, 0, 257, 2500], 3004, 1024), ([1000, 1, 256, 3000], 3002, 512),
           ([1500, 0, 257, 2500], 5004, 512), ([2600, 255, 1, 1500], 5006, 1024)]
