"""The choice of a microscaled product's kernel (csrc/nc_rules.h), compiled on the host (no GPU)."""

from __future__ import annotations

import pytest

from tests import test_mx_gpu
from tests.test_rules import run  # noqa: F401 (the fixture)

ROW, LONG_ROW, WIDE_ROW, SPLIT, JOINED, SMALL, DEEP, MEDIUM, MEDIUM_DEEP, LARGE = range(10)
MISSING = {(4, 1): {WIDE_ROW, MEDIUM}, (8, 1): set(), (4, 2): {WIDE_ROW, MEDIUM, MEDIUM_DEEP},
           (8, 2): {WIDE_ROW, MEDIUM_DEEP}}


def kinds(run, cases):
    body = "".join(f'printf("%d ", (int)nc::mx_tile({m}ll, {n}ll, {(k + 127) // 128}ll, {bits}, {weights}));'
                   for bits, weights, m, n, k in cases)
    return [int(kind) for kind in run(body).split()]


def test_where_each_measured_quicker(run):  # noqa: F811
    cases = [(4, 1, 2, 4864, 896, ROW), (4, 1, 3, 726, 6801, LONG_ROW), (8, 1, 13, 4096, 4096, LONG_ROW), (8, 1, 8, 8192, 8192, WIDE_ROW),
             (8, 1, 163, 896, 4864, ROW),
             (4, 1, 76, 1152, 896, ROW), (4, 1, 199, 918, 287, SPLIT), (4, 1, 2021, 161, 1104, SPLIT),
             (4, 1, 146, 896, 4864, JOINED), (8, 2, 53, 3195, 5597, JOINED), (4, 2, 190, 3139, 2592, DEEP),
             (4, 1, 2162, 896, 4864, DEEP), (4, 2, 465, 4864, 896, SMALL), (4, 1, 923, 8192, 2048, MEDIUM_DEEP),
             (8, 1, 789, 4096, 4096, MEDIUM_DEEP), (4, 1, 1960, 8192, 2048, LARGE), (8, 2, 1867, 8192, 8192, MEDIUM),
             (8, 2, 48, 32000, 2048, SMALL), (8, 1, 2000, 4864, 896, MEDIUM), (8, 2, 1000, 4864, 896, MEDIUM),
             (8, 2, 640, 4864, 896, LARGE), (4, 1, 1, 151936, 896, ROW), (4, 1, 1, 1, 1, ROW)]
    assert kinds(run, [c[:-1] for c in cases]) == [c[-1] for c in cases]


@pytest.mark.parametrize("weights", [1, 2])
@pytest.mark.parametrize("bits", [4, 8])
def test_the_products_tests_reach_every_kind(run, bits, weights):  # noqa: F811
    shapes = test_mx_gpu.SHAPES + test_mx_gpu.WIDE + test_mx_gpu.LONG + test_mx_gpu.SHORT + test_mx_gpu.TILES
    reached = set(kinds(run, [(bits, weights, *shape) for shape in shapes]))
    assert reached == set(range(10)) - MISSING[bits, weights]


@pytest.mark.parametrize("weights", [1, 2])
@pytest.mark.parametrize("bits", [4, 8])
def test_one_shape_of_each_kind(run, bits, weights):  # noqa: F811
    reached = set(kinds(run, [(bits, weights, *shape) for shape in test_mx_gpu.KINDS]))
    assert reached == set(range(JOINED, 10)) - MISSING[bits, weights]


def test_what_the_kernels_need(run):  # noqa: F811
    """Four steps for the kernels of whole tiles, twelve for the one that splits them; never a missing kind;
    the largest shapes without overflow."""
    assert run("""
    long bad = 0;
    for (int bits : {4, 8})
        for (int weights : {1, 2})
            for (int64_t m : {1, 16, 17, 100, 400, 1000, 5000, 1 << 20, (1 << 26) - 1})
                for (int64_t n : {1, 64, 896, 4864, 32000, 1 << 20, (1 << 26) - 1})
                    for (int64_t steps : {1, 2, 3, 4, 7, 8, 11, 12, 20, 64, 1 << 17}) {
                        const nc::MxTile t = nc::mx_tile(m, n, steps, bits, weights);
                        bad += steps < 4 && t > nc::MxTile::kSplit;
                        bad += steps < 12 && t == nc::MxTile::kJoined;
                        bad += weights == 2 && t == nc::MxTile::kMediumDeep;
                        bad += bits == 4 && t == nc::MxTile::kMedium;
                        bad += m >= 5000 && n >= 4864 && steps >= 8 && t < (bits == 4 ? nc::MxTile::kMediumDeep : nc::MxTile::kMedium);
                    }
    printf("%ld", bad);
    """) == "0"
