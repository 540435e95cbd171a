"""The sizes that the GPU tests take do reach every kernel that the launch rules can choose (no GPU needed: the rules
are asked)."""
import pytest

import pfa_native as P
from clear_shapes import PRODUCTS, TILES


def test_products_reach_every_tile_and_split():
    plans = {size: P.matmul_plan(*size) for size in PRODUCTS}
    assert {p for p in plans.values()} == {(*t, s) for t in TILES for s in (1, 2, 4, 8)}
    for tile in TILES:
        mine = [size for size, p in plans.items() if p == (*tile, 1)]
        whole = {k // 128 for _, _, k in mine}
        assert {0, 1, 2} <= whole and max(whole) >= 10, tile        # blocks of K before the rows' end
        assert {k % 128 == 0 for _, _, k in mine} == {True, False}, tile
        assert any(m % tile[0] and n % tile[1] for m, n, _ in mine), tile
        groups = 6 if tile[0] >= 256 else 8
        assert any(m > groups * tile[0] for (m, _, _), p in plans.items() if p[:2] == tile), tile


def test_plan_of_few_rows():
    assert P.matmul_plan(1, 4096, 4096) == (0, 16, 1) and P.matmul_plan(16, 16384, 100) == (0, 16, 1)
    assert P.matmul_plan(17, 4096, 4096)[0] > 0 and P.matmul_plan(1, 16385, 4096)[0] > 0
    with pytest.raises(ValueError, match="131071"):
        P.matmul_plan(1, 1, 131072)
