"""The histogram's bins that the beam selection finds its bound with
(rank_bins.hpp), compiled for the CPU: every rank above -inf has a bin of the
array, the bins follow the ranks' order, and the highest rank is in the last."""
from __future__ import annotations

import os
import subprocess

import numpy as np
import pytest

from conftest import ROOT

BINS = 256
MOST = np.finfo(float).max


@pytest.fixture(scope="module")
def bins_of(tmp_path_factory):
    exe = os.path.join(tmp_path_factory.mktemp("bins"), "rank_bins")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-I", os.path.join(ROOT, "rustcrates_amd", "csrc"),
                    os.path.join(ROOT, "tests", "c", "rank_bins.cpp"), "-o", exe], check=True)

    def of(low, high, ranks):
        text = "".join(f"{float(low).hex()} {float(high).hex()} {float(x).hex()}\n" for x in ranks)
        return np.array(subprocess.run([exe], input=text, capture_output=True, text=True, check=True).stdout.split(), int)

    return of


@pytest.mark.parametrize("low", [-10.0, -1e9, -1e30, -3.4e38, -1e39, -1e40, -1e300, -MOST])
@pytest.mark.parametrize("high", [-9.5, 0.0, 1e300, MOST, np.inf])
def test_a_rank_within_the_range_has_a_bin(bins_of, low, high):
    r = np.random.default_rng(1)
    top = min(high, MOST)
    ranks = np.sort(np.concatenate([[low, top], 2.0 * (0.5 * low + (0.5 * top - 0.5 * low) * r.random(400))]))
    ranks = np.clip(ranks, low, top)
    b = bins_of(low, high, ranks)
    assert b.min() >= 0 and b.max() == BINS - 1 and b[0] == 0
    assert (np.diff(b) >= 0).all()
    if high == np.inf:
        assert bins_of(low, high, [high])[0] == BINS - 1


@pytest.mark.parametrize("low", [-1e300, -MOST])
def test_a_mask_of_the_lowest_value_leaves_the_best_ranks_in_the_highest_bin(bins_of, low):
    assert bins_of(low, -9.5, [low, low * 0.75, -1e100, -700.0, -9.6, -9.5]).tolist() == [0, 64, 255, 255, 255, 255]


def test_ranks_of_minus_1e40_and_minus_1e120_part(bins_of):
    for size in (1e40, 1e120):
        b = bins_of(-4.0 * size, -1.0 * size, np.linspace(-4.0, -1.0, 60) * size)
        assert len(set(b.tolist())) == 60


def test_below_the_range_and_ranges_of_nothing(bins_of):
    assert bins_of(-2.0, -1.0, [-3.0, -1e300, -2.002]).tolist() == [-1, -1, 0]
    assert bins_of(-2.0, -2.0, [-2.0]).tolist() == [0]  # one rank: no steps
    assert bins_of(5e-324, 1e-323, [5e-324, 1e-323]).tolist() == [0, 0]  # too close for steps
