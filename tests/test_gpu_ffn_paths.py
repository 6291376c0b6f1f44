"""The feed-forward block on every path of its products; bounds:
tests/ffn_reference.py."""

from __future__ import annotations

import pytest
import torch

import scao_amd
from tests.ffn_paths import PATHS_16, PATHS_32
from tests.ffn_reference import reference
from tests.test_gpu_ffn import TYPES, _compare, _inputs, _run

pytestmark = pytest.mark.gpu


def _check(dev, tokens, d, f, dtype):
    print(f"tokens {tokens} d {d} f {f} {dtype}", flush=True)
    ins = _inputs(dev, tokens, d, f, dtype)
    want = reference(*ins, "silu")
    _compare(_run(*ins, "silu"), want, dtype, "training")
    _compare(dict(y=scao_amd.gated_ffn(*ins[:4])), want, dtype, "forward")


@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize("size", PATHS_16)
def test_every_path_of_16_bit_products(hip_device, dtype, size):
    _check(hip_device, *size, dtype)


@pytest.mark.parametrize("size", PATHS_32)
def test_every_path_of_fp32_products(hip_device, size):
    _check(hip_device, *size, torch.float32)
