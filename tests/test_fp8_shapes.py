"""The sizes that the GPU tests take do reach every kernel that fp8_matmul's launch rules can choose (no GPU needed: the
rules are asked), and what the compiler made of those kernels."""
import re

import pytest

import pfa_native as P
from fp8_shapes import FEW, NARROW, NARROW_TILES, WIDE, WIDE_TILES
from test_clear_kernel_code import named
from test_kernel_code import kernels  # noqa: F401

F32, BF16, F16 = 0, 1, 2


@pytest.mark.parametrize("kind,sizes,tiles", [(F32, WIDE, WIDE_TILES), (BF16, NARROW, NARROW_TILES)])
def test_products_reach_every_tile(kind, sizes, tiles):
    plans = {size: P.fp8_plan(*size, kind) for size in sizes}
    splits = {t: {s for a, b, s in plans.values() if (a, b) == t} for t in tiles}
    assert {p[:2] for p in plans.values()} == set(tiles)
    for t in tiles:
        mine = [size for size, p in plans.items() if p == (*t, 1)]
        whole = {k // 128 for _, _, k in mine}
        if t == (256, 256):  # takes whole blocks of K only
            assert all(k % 128 == 0 for _, _, k in mine) and {1, 2, 3} <= whole and max(whole) >= 4
        elif kind == F32 and t[0] * t[1] > 128 * 128:  # for a block and more
            assert {1, 2, 3} <= whole and max(whole) >= 4 and {k % 128 == 0 for _, _, k in mine} == {True, False}
        elif t == (192, 128):  # for three blocks and more
            assert 3 in whole and max(whole) >= 4 and {k % 128 == 0 for _, _, k in mine} == {True, False}
        elif (kind, t) != (F32, (128, 128)):  # that one is for long sums only
            assert {0, 1, 2, 3} <= whole and max(whole) >= 4 and {k % 128 == 0 for _, _, k in mine} == {True, False}, t
        assert any(m % t[0] and n % t[1] for m, n, _ in mine), t
        assert any(m > (6 if t[0] >= 256 else 8) * t[0] for m, _, _ in mine), t
        for s in splits[t] - {1}:
            ends = {k % 128 == 0 for (_, _, k), p in plans.items() if p == (*t, s)}
            assert ends == ({True} if t == (256, 256) else {True, False}), (t, s)
    assert set().union(*splits.values()) == {1, 2, 4, 8}


def test_plan():
    for kind in (F32, BF16, F16):
        assert P.fp8_plan(1, 4096, 4096, kind) == (0, 16, 1) and P.fp8_plan(16, 8192, 100, kind) == (0, 16, 1)
        assert {P.fp8_plan(*size, kind) for size in FEW} == {(0, 16, 1)}
        assert P.fp8_plan(1, (1 << 26) - 1, 128, kind) == (0, 16, 1) and P.fp8_plan(1, 1 << 26, 128, kind)[0] > 0  # a grid's end
        assert P.fp8_plan(17, 16384, 4096, kind)[0] > 0 and P.fp8_plan(1, 4096, 24577, kind)[0] > 0
    assert P.fp8_plan(333, 777, 999, BF16) == P.fp8_plan(333, 777, 999, F16)
    for m, n, k in WIDE + NARROW:
        for kind in (F32, BF16):
            tile_rows, _, splits = P.fp8_plan(m, n, k, kind)
            assert P.fp8_workspace(m, n, k, kind) == (4 * splits * m * n if tile_rows and splits > 1 else 0)


def test_nothing_is_spilled(kernels):
    """Operands and sums stay in registers; the tiles of 256 x 256 give up a few numbers outside of their loop."""
    for name in ("k_fp8_rows", "k_fp8_squares", "k_fp8_norm", "k_fp8_few", "k_fp8_far", "k_fp8_tiles", "k_fp8_join", "k_log_rows",
                 "k_log_parts", "k_log_join"):
        found = named(kernels, name)
        assert found, name
        for full, k in found.items():
            most = 32 if re.search(r"k_fp8_tiles.*Li256ELi256E", full) else 0
            assert int(k[".private_segment_fixed_size"]) <= most, full


@pytest.mark.parametrize("shape,groups,types", [("32, 64, 2, 2, 6", 2, 3), ("64, 64, 2, 2, 4", 2, 3), ("64, 128, 2, 2, 3", 2, 3),
                                                ("128, 128, 2, 4, 4", 1, 3), ("192, 128, 4, 2, 3", 1, 3), ("128, 256, 2, 4, 3", 1, 3),
                                                ("256, 128, 4, 2, 3", 1, 3), ("256, 256, 4, 2, 2", 1, 2)])
def test_tiles_fit(kernels, shape, groups, types):
    """As many workgroups as the costs of the shapes were measured with: 160 KiB of LDS a CU, 512 registers a lane of a
    SIMD.  The ring is part of the kernel."""
    found = named(kernels, "k_fp8_tiles", shape)
    assert len(found) == types
    bm, bn, wm, wn, stages = (int(v) for v in shape.split(","))
    for n, k in found.items():
        held = int(k[".group_segment_fixed_size"])
        assert ((bm + bn) * 128 + wm * wn * 256) * stages <= held <= 160 * 1024 // groups, n
        assert int(k[".vgpr_count"]) * wm * wn * groups / 4 <= 512, n
