"""The LDS of the product's tiles is part of the kernels.  A kernel that takes more than 64 KiB at its launch needs its limit
raised on every device that runs it; one that holds it does not."""
import pytest

from test_clear_kernel_code import named
from test_kernel_code import kernels  # noqa: F401

# (matrix instruction, rows, columns, waves down, waves across, blocks in the ring)
SHAPES = ["16, 32, 64, 2, 2, 6", "16, 64, 64, 2, 2, 4", "16, 64, 128, 1, 4, 3", "32, 128, 128, 2, 2, 3",
          "16, 128, 192, 2, 4, 3", "16, 128, 256, 2, 4, 3", "16, 256, 128, 4, 2, 3"]


@pytest.mark.parametrize("shape", SHAPES)
def test_tiles_hold_their_lds(kernels, shape):
    found = named(kernels, "k_tiles", shape)
    assert len(found) == 3  # the three types of outputs
    mf, bm, bn, wm, wn, stages = (int(v) for v in shape.split(","))
    ring = (bm + bn) * 128 * stages
    for name, k in found.items():
        # the ring, and in the same place afterwards scales, offsets and a line of outputs a wave
        lines = (2 * bn + bm) * 4 + wm * wn * mf * (bn // wn * 4 + 16)
        held = int(k[".group_segment_fixed_size"])
        assert max(ring, lines) <= held <= 160 * 1024, name


def test_every_tile_is_looked_at(kernels):
    assert len(named(kernels, "k_tiles")) == 3 * len(SHAPES)
