"""The paths of the feed-forward block's products, planned without a GPU: which
tile, whole or split or only the last round's tiles split, alone or in a pair,
rows left over by themselves.  Every path that sizes up to 8192 tokens x 4096 x
14336 take has to be one that the GPU tests' sizes take too."""

from __future__ import annotations

import ctypes
import math
import os
import random
import shutil
import subprocess

import numpy as np
import pytest

from scao_amd import _lib as L
from scao_amd.build import HIPCC, ROOT
from tests.ffn_paths import PATHS_16, PATHS_32
from tests.test_gpu_ffn import SIZES

KINDS = ("gate_up", "down", "dh", "dx", "dw")
TILES = ("256x256", "256x128", "128x128", "64x128", "32x128")


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """plan(tokens, d, f, dtype code, train): the launches' rows as an array"""
    if shutil.which(HIPCC) is None:
        pytest.skip("no hipcc")
    so = str(tmp_path_factory.mktemp("plan") / "ffn_plan.so")
    subprocess.run([HIPCC, "--offload-host-only", "--offload-arch=gfx950", "-std=c++17", "-O1",
                    "-fPIC", "-shared", "-o", so, os.path.join(ROOT, "tests", "ffn_plan.hip")],
                   check=True)
    lib = ctypes.CDLL(so)
    lib.ffn_plan.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_void_p,
                             ctypes.c_int]
    lib.ffn_choose.restype = ctypes.c_double
    lib.ffn_choose.argtypes = [ctypes.c_int] + 3 * [ctypes.c_int64] + [ctypes.c_void_p]
    desc = np.zeros(1, dtype=L.FFN_DESC)
    for k in ("x", "w_gate", "w_up", "w_down"):
        desc[k] = 4096
    out = np.zeros((64, 8), dtype=np.int32)

    def call(tokens, d, f, dtype, train):
        for k, v in dict(ldx=d, ld_gate=d, ld_up=d, ld_down=f, tokens=tokens, d=d, f=f,
                         dtype=dtype).items():
            desc[k] = v
        n = lib.ffn_plan(desc.ctypes.data, int(train), d, out.ctypes.data, len(out))
        assert 0 < n <= len(out)
        return out[:n].tolist()

    call.lib = lib
    return call


def _paths(plan, size, dtype):
    paths = set()
    for train in (False, True):
        for kind, tile, type_, whole, tiles, splits, row0, paired in plan(*size, dtype, train):
            assert type_ == dtype
            if kind < 0:   # few tokens: (tokens, columns) in the places of tiles and splits
                halves = tiles <= 8 and splits < 4096
                paths.add(("few", kind == -1, 0 if halves else max(16, 1 << (tiles - 1).bit_length())))
                continue
            mode = "whole" if whole == tiles else "split" if whole == 0 else "last round split"
            assert 0 <= whole <= tiles and (splits > 1) == (whole < tiles)
            paths.add((KINDS[kind], TILES[tile], mode, row0 > 0, bool(paired)))
    return paths


def _any_size(rng, dtype):
    """Sizes spread over their logarithms, half of them multiples of 64"""
    size = [math.exp(rng.uniform(math.log(lo), math.log(hi)))
            for lo, hi in ((1, 2048 if dtype == 0 else 8192), (64, 4096), (128, 14336))]
    return [max(1, int(s) // 64 * 64) if rng.random() < 0.5 else int(s) for s in size]


@pytest.mark.parametrize("dtype,more", [(1, PATHS_16), (0, PATHS_32)])
def test_the_tests_take_every_path(plan, dtype, more):
    tested = set().union(*(_paths(plan, s, dtype) for s in SIZES + more))
    rng = random.Random(11)
    for _ in range(30000):
        size = _any_size(rng, dtype)
        left = _paths(plan, size, dtype) - tested
        assert not left, (size, left)


def test_both_16_bit_types_take_the_same_paths(plan):
    for size in SIZES + PATHS_16:
        a, b = (plan(*size, dtype, True) for dtype in (1, 2))
        assert [row[:2] + row[3:] for row in a] == [row[:2] + row[3:] for row in b]


def test_choice_of_tiles_against_measured_products(plan):
    """perf/ffn_fit.py's model is the one that chooses (a last round split alone
    aside, which it does not know), and stays near the best of what was measured."""
    import importlib.util
    spec = importlib.util.spec_from_file_location("ffn_fit", os.path.join(ROOT, "perf", "ffn_fit.py"))
    fit = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(fit)
    forms = fit.Forms(fit.read(os.path.join(ROOT, "profiles", "ffn_tiles.csv")))
    slots, c = fit.constants()
    out = (ctypes.c_int32 * 4)()
    alone = 0
    for (kind, *size), at in zip(forms.products, forms.chosen(slots, c)):
        plan.lib.ffn_choose(KINDS.index(kind), *size, out)
        tile, whole, parts, tiles = out
        if 0 < whole < tiles:
            alone += 1
        else:
            assert (tile, parts) == (forms.tile[at], forms.parts[at]), (kind, size)
    assert alone < 10 and len(forms.products) == 225
    assert np.exp(np.log(forms.behind(slots, c)).mean()) < 1.04
