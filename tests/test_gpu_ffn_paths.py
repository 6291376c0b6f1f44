"""The feed-forward block on every path of its products, and how near its
outputs are in the 2-norm (tests/ffn_bounds.py)."""

from __future__ import annotations

import pytest
import torch

import scao_amd
from tests.ffn_bounds import norm_bound
from tests.ffn_paths import PATHS_16, PATHS_32
from tests.ffn_reference import reference
from tests.test_gpu_ffn import ACTS, SIZES, TYPES, _inputs, _run

pytestmark = pytest.mark.gpu


def _check(dev, tokens, d, f, dtype, name, elements):
    print(f"tokens {tokens} d {d} f {f} {dtype} {name}", flush=True)
    ins = _inputs(dev, tokens, d, f, dtype)
    want = reference(*ins, name)
    got = _run(*ins, name)
    got["forward"] = scao_amd.gated_ffn(*ins[:4], activation=name)
    for k, v in got.items():
        value, bound = want["y" if k == "forward" else k]
        err = v.double() - value
        rel = (err.norm() / value.norm()).item()
        most = norm_bound(dtype, "y" if k == "forward" else k, tokens, d, f)
        print(f"{k}: {rel / most:.3f} of the norm's bound, {rel:.2e}", flush=True)
        if v.numel() >= 1000:
            assert rel <= most, (k, rel, most)
        if elements:
            assert bool((err.abs() <= bound).all()), (k, (err.abs() / bound).max().item())


@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize("size", PATHS_16)
def test_every_path_of_16_bit_products(hip_device, dtype, size):
    _check(hip_device, *size, dtype, "silu", True)


@pytest.mark.parametrize("size", PATHS_32)
def test_every_path_of_fp32_products(hip_device, size):
    _check(hip_device, *size, torch.float32, "silu", True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("size", [s for s in SIZES if s[0] >= 17 and s[0] * s[1] * s[2] > 1e5])
def test_norms_of_the_errors(hip_device, dtype, name, size):
    _check(hip_device, *size, dtype, name, False)
