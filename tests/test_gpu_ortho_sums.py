"""Long sums of two-word products, which the matrix cores do not add up alone: results in
float32 are as exact in company, which decides the tiles, as by themselves."""

from __future__ import annotations

import pytest
import torch

import scao_amd
from tests.ortho_reference import orthogonalize
from tests.ortho_words import PUBLISHED, relative
from tests.test_gpu_ortho import _update

pytestmark = pytest.mark.gpu


def _plain(x):
    x = x / (x.norm() + 1e-7)
    for a, b, c in PUBLISHED:
        gram = x @ x.t()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x


@pytest.mark.parametrize("shapes", [[(2048, 8192)] * 8, [(4096, 4096)] * 4, [(1024, 14336)] * 16,
                                    [(4096, 14336)] * 2,
                                    [(2048, 2048)] * 3 + [(512, 4096)] * 30])
def test_published_steps_in_company(hip_device, shapes):
    """A sum of 64 products of 32 terms each is 2.4e-7 off in the matrix cores (root mean
    square; of 448, 6.3e-7), so that one of 64 steps, three products each, is 4.2e-7 off.
    Three such sums a step, independent of one another: 1.6e-6 after five steps.  Words and
    sums that are put aside leave 1.5e-6 by themselves: together 2.2e-6.  And no further off
    than a plain form in float32, all of whose sums are of full length."""
    mats = [_update(hip_device, i, m, n, torch.float32) for i, (m, n) in enumerate(shapes)]
    got = scao_amd.orthogonalize(mats)
    for i in {0, len(mats) // 2, len(mats) - 1}:
        want = orthogonalize(mats[i], PUBLISHED)
        own, other = relative(got[i], want), relative(_plain(mats[i]), want)
        alone = relative(scao_amd.orthogonalize(mats[i]), want)
        print(f"{shapes[i]}: {own:.2e}, alone {alone:.2e}, plain {other:.2e}", flush=True)
        assert own <= 2.2e-6 and own <= other
