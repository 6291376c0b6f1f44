"""The products' accuracy by the caller's choice, whatever the results' type is."""

from __future__ import annotations

import pytest
import torch

import scao_amd
from tests.ortho_reference import orthogonalize
from tests.ortho_words import PUBLISHED, allowed, relative
from tests.test_gpu_ortho import _update

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n", [(256, 300), (700, 1030), (2048, 640)])
def test_products_of_either_kind(hip_device, m, n):
    for dtype in (torch.bfloat16, torch.float32, torch.float16):
        g = _update(hip_device, 1, m, n, dtype)
        want = orthogonalize(g, PUBLISHED)
        # exact products, rounded once to the result's type
        full = scao_amd.orthogonalize(g, dtype=torch.float32, ns_dtype=torch.float32)
        for out in (torch.bfloat16, torch.float16, torch.float32):
            got = scao_amd.orthogonalize(g, dtype=out, ns_dtype=torch.float32)
            assert torch.equal(got, full.to(out))
        # products of one word
        got = scao_amd.orthogonalize(g, dtype=torch.float32, ns_dtype=torch.bfloat16)
        assert relative(full, want) < 1e-5 < relative(got, want) <= allowed(
            g, PUBLISHED, torch.float32)[1]
        # and what None is
        kind = torch.bfloat16 if dtype == torch.bfloat16 else torch.float32
        assert torch.equal(scao_amd.orthogonalize(g), scao_amd.orthogonalize(g, ns_dtype=kind))


def test_refused(hip_device):
    g = torch.randn(8, 8, device=hip_device)
    for bad in (torch.float16, torch.float64):
        with pytest.raises(ValueError):
            scao_amd.orthogonalize(g, ns_dtype=bad)
        with pytest.raises(RuntimeError):
            torch.ops.scao_amd.orthogonalize([g], [1.0, 0.0, 0.0], 1e-7, None, bad)
