"""What the compiler made of the clear operators' kernels: rows and tiles of sums stay in registers, and as many
workgroups fit a CU as their launch rules count on (512 registers a lane of a SIMD, 160 KiB of LDS a CU)."""
import re

import pytest

from test_kernel_code import kernels  # noqa: F401

CLEAR = ("k_quantize_rows", "k_prob_rows", "k_prob_parts", "k_prob_write", "k_prob_short", "k_verify", "k_tiles",
         "k_few_rows", "k_join")


def named(kernels, name, values=""):
    """Kernels of this name, by their mangled names (the demangler here does not know the 16-bit types)."""
    tail = "".join("L[ib]%sE" % v.strip() for v in values.split(",")) if values else ""
    return {k[".name"]: k for k in kernels.values() if re.search(r"\d%s(I|E).*%s" % (name, tail), k[".name"])}


def test_every_kernel_is_there(kernels):
    for name in CLEAR:
        assert named(kernels, name), name


def test_nothing_is_spilled(kernels):
    """The widest rows of 1024 threads give up a few registers for a second workgroup on the CU."""
    for name in CLEAR:
        for full, k in named(kernels, name).items():
            most = 32 if re.search(r"k_prob_rows.*Li1024E", full) else 0
            assert int(k[".private_segment_fixed_size"]) <= most, full


@pytest.mark.parametrize("shape,groups", [("16, 32, 64, 2, 2, 6", 2), ("16, 64, 64, 2, 2, 4", 2),
                                          ("16, 64, 128, 1, 4, 3", 2), ("32, 128, 128, 2, 2, 3", 1),
                                          ("16, 128, 192, 2, 4, 3", 1), ("16, 128, 256, 2, 4, 3", 1),
                                          ("16, 256, 128, 4, 2, 3", 1)])
def test_tiles_fit(kernels, shape, groups):
    found = named(kernels, "k_tiles", shape)
    assert len(found) == 3  # the three types of outputs
    _, bm, bn, wm, wn, stages = (int(v) for v in shape.split(","))
    assert (bm + bn) * 128 * stages * groups <= 160 * 1024
    for n, k in found.items():
        waves = wm * wn * groups / 4  # a SIMD's
        assert int(k[".vgpr_count"]) * waves <= 512, n


def test_two_workgroups_of_wide_rows(kernels):
    for n, k in named(kernels, "k_prob_rows").items():
        if re.search(r"Li1024ELi[24]E", n):
            assert int(k[".vgpr_count"]) <= 64, n
