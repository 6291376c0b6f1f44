"""How the orthogonalisation of updates cuts its products, planned without a GPU."""

from __future__ import annotations

import csv
import ctypes
import math
import os
import random
import shutil
import subprocess

import numpy as np
import pytest

from scao_amd import _lib as L
from scao_amd.build import FLAGS, HIPCC, ROOT
from tests.ortho_paths import LISTS, matrices

GRAM = 0   # the first phase of a pass's rows


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """plan([(rows, cols, precision)]): a dict for every phase of every pass"""
    if shutil.which(HIPCC) is None:
        pytest.skip("no hipcc")
    so = str(tmp_path_factory.mktemp("plan") / "ortho_plan.so")
    subprocess.run([HIPCC, *FLAGS, "-O1", "-shared", "-o", so,
                    os.path.join(ROOT, "tests", "ortho_plan.hip")], check=True)
    lib = ctypes.CDLL(so)
    lib.ortho_plan.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_int, ctypes.c_void_p,
                               ctypes.c_void_p, ctypes.c_int]
    out, us = np.zeros((256, 8), dtype=np.int32), np.zeros(256)

    def call(shapes, steps=5):
        t = np.zeros(len(shapes), dtype=L.ORTHO_DESC)
        for i, (rows, cols, precision) in enumerate(shapes):
            t[i]["rows"], t[i]["cols"], t[i]["precision"] = rows, cols, precision
        n = lib.ortho_plan(t.ctypes.data, len(t), steps, out.ctypes.data, us.ctypes.data, len(out))
        assert 0 <= n <= len(out)
        names = ("run", "phase", "side", "tiles", "whole", "parts", "matrices", "panels")
        return [dict(zip(names, row.tolist()), us=float(t)) for row, t in zip(out[:n], us)]

    return call


def _sum(phase, rows, cols, words):
    """k steps of a tile: 64 k, or 32 of two words"""
    k = max(rows, cols) if phase == GRAM else min(rows, cols)
    return -(-k * words // 64)


def _words(rows, cols, precision):
    return 2 if precision == L.ORTHO_FP32 or min(rows, cols) <= 128 else 1


def _lists(seed, many):
    """lists of up to three shapes, one to 24 matrices of each, in one pass"""
    rng = random.Random(seed)
    for _ in range(many):
        shapes = []
        for _ in range(rng.randint(1, 3)):
            m, n = (max(1, int(math.exp(rng.uniform(math.log(16), math.log(16384)))))
                    for _ in range(2))
            m, n = (v // 64 * 64 if rng.random() < 0.5 and v >= 64 else v for v in (m, n))
            shapes += [(m, n, rng.randint(0, 1))] * rng.choice([1, 1, 2, 4, 8, 24])
        yield shapes


def test_long_sums_of_two_words_are_not_left_to_the_matrix_cores(plan):
    """Tiles of 256 x 256 add up to 64 steps of two words each."""
    fixed = [[(4096, 14336, 1)] * 2, [(2048, 8192, 1)] * 8, [(4096, 4096, 1)] * 4,
             [(512, 65536, 1)] * 64, [(4096, 14336, 1), (4096, 14336, 0)], [(120, 1 << 19, 0)] * 9,
             [(32768, 32768, 1)]]
    large = 0
    for shapes in fixed + list(_lists(5, 400)):
        left = sorted(shapes, key=lambda s: (-min(s[:2]), -s[0], -s[1], -_words(*s)))
        for row in plan(shapes):
            if row["phase"] == GRAM:
                mine, left = left[:row["matrices"]], left[row["matrices"]:]
            if row["side"] == 128:
                continue
            sums = [_sum(row["phase"], m, n, 2) for m, n, p in mine if _words(m, n, p) == 2]
            if not sums:
                continue
            large += 1
            parts = 1 if row["whole"] else row["parts"]
            assert -(-max(sums) // parts) <= 64, (shapes, row)
        assert not left or not plan(shapes)
    assert large > 20


def _paths(plan, shapes):
    """of a list: panels, or what each phase does with every kind of matrix"""
    paths = set()
    left = sorted(shapes, key=lambda s: (-min(s[:2]), -s[0], -s[1], -_words(*s)))
    for row in plan(shapes):
        if row["phase"] == GRAM:
            mine, left = left[:row["matrices"]], left[row["matrices"]:]
        if row["panels"]:
            paths.add("panels")
            continue
        assert 0 <= row["whole"] <= row["tiles"]
        assert (row["parts"] > 1) == (row["whole"] < row["tiles"])
        mode = ("whole" if row["whole"] == row["tiles"] else
                "split" if row["whole"] == 0 else "last round split")
        for m, n, p in mine:
            paths.add((row["phase"], row["side"], mode, _words(m, n, p), m <= n))
    return paths


def test_the_tests_take_every_path(plan):
    tested = set()
    for precision, shapes in LISTS:
        p = L.ORTHO_FP32 if precision == "fp32" else L.ORTHO_FAST
        tested |= _paths(plan, [(*s, p) for s in matrices(shapes)])
    assert len(tested) > 60
    rng = random.Random(3)
    for _ in range(8000):
        shapes, p = [], rng.randint(0, 1)
        for _ in range(rng.randint(1, 3)):
            m, n = (max(1, int(math.exp(rng.uniform(math.log(16), math.log(6000)))))
                    for _ in range(2))
            m, n = (v // 64 * 64 if rng.random() < 0.4 and v >= 64 else v for v in (m, n))
            shapes += [(m, n, p)] * rng.choice([1, 1, 2, 4, 8, 24])
        left = _paths(plan, shapes) - tested
        assert not left, (shapes, left)


def _matrices(text, words):
    return [(*map(int, shape.split("x")), words - 1) for shape, many in
            (part.split("*") for part in text.split(",")) for _ in range(int(many))]


def test_choice_against_measured_products(plan):
    """Tiles, parts and panels as they are chosen, against the best of what
    perf/ortho_tiles.hip measured."""
    tiles, panels = {}, {}
    with open(os.path.join(ROOT, "profiles", "ortho_tiles.csv")) as fh:
        for r in csv.DictReader(fh):
            key = r["list"], int(r["words"])
            if r["phase"] == "panels":
                panels[key] = float(r["us"])
            else:
                forms = tiles.setdefault(key, {}).setdefault(int(r["phase"]), {})
                forms[int(r["side"]), int(r["parts"]), int(r["whole"])] = float(r["us"])
    behind, steps = [], []
    for (text, words), phases in tiles.items():
        shapes = _matrices(text, words)
        rows = plan(shapes)
        assert len(rows) == 3
        took = 0.0
        for row in rows:
            forms = phases[row["phase"]]
            chosen = forms[row["side"], row["parts"], row["whole"]]
            long = max((_sum(row["phase"], m, n, 2) for m, n, p in shapes
                        if _words(m, n, p) == 2), default=0)
            allowed = [us for (side, parts, whole), us in forms.items()
                       if side == 128 or (long if whole else -(-long // parts)) <= 64]
            behind.append(chosen / min(allowed))
            took += chosen
        if (text, words) in panels:
            by = panels[text, words]
            steps.append((by if rows[0]["panels"] else took) / min(by, took))
    print(f"{len(behind)} launches: {np.exp(np.log(behind).mean()):.4f}, {max(behind):.3f}; "
          f"{len(steps)} steps: {np.exp(np.log(steps).mean()):.4f}, {max(steps):.3f}")
    assert len(behind) == 222 and np.exp(np.log(behind).mean()) < 1.03 and max(behind) < 1.3
    assert len(steps) == 33 and np.exp(np.log(steps).mean()) < 1.05 and max(steps) < 1.3
