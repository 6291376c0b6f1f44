"""The feed-forward block's choice of tile and parts against measured products.

    python perf/ffn_fit.py [profiles/ffn_tiles.csv] [--fit STEPS]

Reads what perf/ffn_tiles.hip printed and the constants of csrc/ffn.hip's Cost
table, and says how far behind the best measured form the chosen one is, on the
geometric average and by product.  With --fit the constants are changed at
random, a change being kept where the average falls.  (Only forms that were
measured: all tiles split alike.  The choice may also split the last round alone.)
"""

from __future__ import annotations

import argparse
import collections
import csv
import math
import os
import random
import re

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TILES = {"256x256": (256, 256), "256x128": (256, 128), "128x128": (128, 128),
         "64x128": (64, 128), "32x128": (32, 128)}
NAMES = list(TILES)


def read(path):
    """{(product, tokens, d, f): {(tile, parts): us}}"""
    out = collections.defaultdict(dict)
    with open(path) as fh:
        for r in csv.DictReader(fh):
            key = r["product"], int(r["tokens"]), int(r["d"]), int(r["f"])
            out[key][NAMES.index(r["tile"]), int(r["parts"])] = float(r["us"])
    return out


def constants():
    """slots, and (lone, full, ends) of each tile as an array"""
    with open(os.path.join(ROOT, "scao_amd", "csrc", "ffn.hip")) as fh:
        table = re.search(r"costs\[FFN_TILES\] = \{(.*?)\};", fh.read(), re.S)[1]
    rows = np.array([[float(x) for x in r.split(",")] for r in re.findall(r"\{([^{}]*)\}", table)])
    return rows[:, 0], rows[:, 1:]


class Forms:
    """Every measured form of every product, as arrays"""

    def __init__(self, data):
        rows, self.products = [], list(data)
        for i, (key, forms) in enumerate(data.items()):
            kind, tokens, d, f = key
            gated = kind == "gate_up"
            m = 2 * f if kind == "dw" else tokens
            n = f if kind in ("gate_up", "dh") else d
            k = tokens if kind == "dw" else f if kind in ("down", "dx") else d
            steps = -(-k // 64) * (2 if kind == "dx" else 1)
            moved = 8 if gated else 10 if kind == "dh" else 0
            for (tile, parts), us in forms.items():
                bm, bn = TILES[NAMES[tile]]
                groups = -(-m // bm) * -(-n // (bn // 2 if gated else bn)) * parts
                join = (2 + (8 / 7.4e6 * parts * (2 if gated else 1) + moved / 5e6) * m * n
                        if parts > 1 else 0.0)
                epilogue = 2.5 if gated and tile >= NAMES.index("64x128") and parts == 1 else 0.0
                rows.append((i, tile, parts, us, groups, -(-steps // parts), join, epilogue))
        a = np.array(rows)
        self.product, self.tile, self.parts = (a[:, j].astype(int) for j in range(3))
        self.us, self.groups, self.steps, self.join, self.epilogue = (a[:, j] for j in range(3, 8))
        self.first = np.searchsorted(self.product, np.arange(len(self.products) + 1))
        self.best = np.minimum.reduceat(self.us, self.first[:-1])

    def chosen(self, slots, c):
        """the form of the least estimate, for each product"""
        s, lone, full = slots[self.tile], c[self.tile, 0], c[self.tile, 1]
        ends = c[self.tile, 2] + self.epilogue
        rounds, last = self.groups // s, self.groups % s
        crowd = np.where(s == 256, last / 256,
                         np.clip((last - 256) / np.where(s == 256, 1, s - 256), 0, 1))
        us = rounds * (self.steps * full + ends) + self.join
        us += np.where(last > 0, self.steps * (lone + (full - lone) * crowd) + ends, 0)
        return [a + int(np.argmin(us[a:b])) for a, b in zip(self.first, self.first[1:])]

    def behind(self, slots, c):
        """us of the chosen over us of the best, for each product"""
        return self.us[self.chosen(slots, c)] / self.best


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("csv", nargs="?", default=os.path.join(ROOT, "profiles", "ffn_tiles.csv"))
    ap.add_argument("--fit", type=int, default=0)
    a = ap.parse_args()
    forms, (slots, c) = Forms(read(a.csv)), constants()
    mean = lambda c: float(np.exp(np.log(forms.behind(slots, c)).mean()))   # noqa: E731
    rng, now = random.Random(0), mean(c)
    for _ in range(a.fit):
        other = c.copy()
        other[rng.randrange(len(c)), rng.randrange(3)] *= math.exp(rng.gauss(0, 0.12))
        if mean(other) < now:
            c, now = other, mean(other)
    behind, chosen = forms.behind(slots, c), forms.chosen(slots, c)
    print(f"{len(behind)} products: {100 * (now - 1):.1f}% behind the best on average, "
          f"{100 * (behind.max() - 1):.0f}% at most")
    if a.fit:
        print("lone, full, ends:", np.round(c, 2).tolist())
    for i in np.argsort(-behind)[:10]:
        at = chosen[i]
        print(*forms.products[i], f"{NAMES[forms.tile[at]]} in {forms.parts[at]}: "
              f"{forms.us[at]:.1f} us, best {forms.best[i]:.1f}")


if __name__ == "__main__":
    main()
