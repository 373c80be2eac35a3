"""CPU: the shapes of the GPU tests of microscaled products reach every kernel that a product can be served by."""

from __future__ import annotations

import re

from mx_kernels import DENSE, EXPERTS, SOURCE, constants, kernel_of


def _shapes(pattern: str, text: str) -> set:
    return {tuple(int(v) for v in re.findall(r"\d+", m)) for m in re.findall(pattern, text)}


def test_every_kernel_is_reached():
    rule = SOURCE.read_text()
    rule = rule[rule.index("Plan plan_mx_linear("):]
    few, tiles = _shapes(r"plan_few<([\d, ]+)>", rule), _shapes(r"pick_tiles<([\d, ]+?)(?:, (?:true|false))?>", rule)
    assert few == {(1, 1), (2, 1), (2, 2), (2, 4)} and tiles == {(1, 1, 2, 2), (2, 1, 2, 2), (2, 2, 2, 2), (4, 2, 2, 4)}
    dense = {kernel_of(*s) for s in DENSE}
    experts = {kernel_of(sum(counts), M, K, len(counts)) for counts, M, K in EXPERTS}
    every = {("tiles", *t, whole, False) for t in tiles for whole in (True, False)} | {("tiles", 4, 2, 2, 4, True, True)}
    # Few rows of each of several experts have two parts of K; dense calls that fill the card none.  By expert no tiles of
    # 64 x 64 or 128 x 128.
    assert dense == every | {("few", 1, 1), ("few", 2, 1), ("few", 2, 4)}
    assert experts == {k for k in every if k[1:5] in ((2, 1, 2, 2), (4, 2, 2, 4))} | {("few", *f) for f in few - {(2, 4)}}


def test_both_sides_of_a_launchs_tiles_without_whole_windows():
    """Tiles of 256 x 256 of a K that is not whole windows: more of them than workgroups that stay, and fewer."""
    most = constants()["kStaying"]
    sizes = [-(-T // 256) * -(-M // 256) for T, M, K in DENSE if kernel_of(T, M, K) == ("tiles", 4, 2, 2, 4, False, False)]
    assert min(sizes) <= most < max(sizes)


def test_even_rows_of_weights():
    assert all(M % 2 == 0 for _, M, _ in DENSE + EXPERTS)
