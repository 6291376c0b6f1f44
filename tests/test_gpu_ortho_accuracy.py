"""The published five steps against their definition in 64 bits, as exactly as is said of
them; bounds: tests/ortho_words.py."""

from __future__ import annotations

import pytest
import torch

import scao_amd
from scao_amd import _lib as L
from tests.ortho_reference import orthogonalize
from tests.ortho_words import PUBLISHED, allowed, relative
from tests.test_gpu_ortho import _call, _update

pytestmark = pytest.mark.gpu

# by panels for themselves (up to 512 x 1024); by tiles; 256 x 256 tiles
SIZES = [(160, 160), (256, 256), (1024, 256), (256, 512), (384, 384), (300, 200), (160, 900),
         (512, 512), (512, 1024),
         (640, 640), (1001, 333), (2048, 512), (700, 1030), (150, 3000), (2049, 2000), (4096, 1024)]


@pytest.mark.parametrize("m,n", SIZES)
def test_one_word(hip_device, m, n):
    g = _update(hip_device, m + n, m, n, torch.bfloat16)
    want, room = allowed(g, PUBLISHED, torch.bfloat16)
    err = relative(scao_amd.orthogonalize(g), want)
    # and in float32, where nothing but the words' roundings is left
    full = torch.empty(m, n, device=hip_device)
    _call([g], [full], L.ORTHO_FAST, PUBLISHED)
    _, room32 = allowed(g, PUBLISHED, torch.float32)
    err32 = relative(full, want)
    print(f"{m}x{n}: {err:.2e} of {room:.2e}, in float32 {err32:.2e} of {room32:.2e}", flush=True)
    assert err <= room and err32 <= room32


def test_one_word_in_company(hip_device):
    """Whatever shares the call, which decides between panels and tiles."""
    shapes = [(256, 1024), (160, 900), (256, 256), (300, 200)]
    mats = [_update(hip_device, i, *s, torch.bfloat16) for i, s in enumerate(shapes)]
    for more in ([], [(640, 640)], [(2048, 2048)], [(256, 1024)] * 20):
        others = [_update(hip_device, 50 + i, *s, torch.bfloat16) for i, s in enumerate(more)]
        full = [torch.empty(t.shape, device=hip_device) for t in mats + others]
        _call(mats + others, full, L.ORTHO_FAST, PUBLISHED)
        for g, got in zip(mats, full):
            want, room = allowed(g, PUBLISHED, torch.float32)
            err = relative(got, want)
            print(f"{tuple(g.shape)} beside {len(more)}: {err:.2e} of {room:.2e}", flush=True)
            assert err <= room


@pytest.mark.parametrize("m,n", [(64, 64), (96, 160), (128, 128), (100, 700), (2000, 128)])
def test_up_to_128_rows_have_two_words(hip_device, m, n):
    """results in bfloat16 are off by their own rounding, and 1% for the rest"""
    g = _update(hip_device, m + n, m, n, torch.bfloat16)
    want = orthogonalize(g, PUBLISHED)
    assert relative(scao_amd.orthogonalize(g), want) <= 1.01 * relative(want.bfloat16(), want)


@pytest.mark.parametrize("m,n", [(256, 256), (300, 160), (640, 700)])
def test_one_word_with_strong_growth(hip_device, m, n):
    """Singular values that the first step takes far up and the second far down."""
    g = _update(hip_device, 9, m, n, torch.float32)
    co = [(30.0, 0.0, 0.0), (1.0 / 16, 2.0 ** -14, 2.0 ** -24), (0.5, 0.125, 0.0)]
    full = torch.empty(m, n, device=hip_device)
    _call([g], [full], L.ORTHO_FAST, co)
    want, room = allowed(g, co, torch.float32)
    err = relative(full, want)
    print(f"{m}x{n}: {err:.2e} of {room:.2e}", flush=True)
    assert err <= room <= 2e-3
