"""Every path of the orthogonalisation's products (tests/ortho_paths.py), as
``orthogonalize`` and as Muon's step take it, against the definitions in 64 bits.

Results of one word: tests/ortho_words.py's bound.  Of two: tests/ortho_reference.py's.
A step's parameter is p' = decay p - rate O: what is rounded to its type is off by that
rounding (which is computed from the exact p'; 5% for those that fall the other way), by
rate times O's own error, and by two roundings of 2^-24 of both terms; the update u, whose
O is taken, by three."""

from __future__ import annotations

import math

import pytest
import torch

import scao_amd
from scao_amd import _lib as L
from tests.ortho_paths import LISTS
from tests.ortho_reference import QUINTIC, ULP, bound, orthogonalize, triples
from tests.ortho_words import PUBLISHED, allowed, emulate, relative
from tests.test_gpu_ortho import _call, _update

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float32, torch.float16]


@pytest.mark.parametrize("which", range(len(LISTS)))
def test_orthogonalize(hip_device, which):
    precision, shapes = LISTS[which]
    mats, dst = [], []
    for k, (m, n, many) in enumerate(shapes):
        for i in range(many):
            mats.append(_update(hip_device, 10 * k + i, m, n, TYPES[(which + i) % 3], i % 3, i % 2))
            dst.append(torch.full((m, n + i % 2 * 3), 7.0, device=hip_device,
                                  dtype=TYPES[(which + k) % 3])[:, :n])
    fast = precision == "fast"
    co = PUBLISHED if fast else triples(QUINTIC, 2)
    _call(mats, dst, L.ORTHO_FAST if fast else L.ORTHO_FP32, co)
    at = 0
    for m, n, many in shapes:
        for i in {at, at + many - 1}:
            if fast:
                want, room = allowed(mats[i], co, dst[i].dtype)
            else:
                want = orthogonalize(mats[i], co)
                room = bound(mats[i], co, "fp32") / float(want.norm()) + ULP[dst[i].dtype]
            err = relative(dst[i], want)
            print(f"{m}x{n} {dst[i].dtype}: {err:.2e} of {room:.2e}", flush=True)
            assert err <= room
            if dst[i].stride(0) > n:
                beside = dst[i].as_strided((m, 3), (dst[i].stride(0), 1), n)
                assert bool((beside == 7.0).all())
        at += many


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("which", range(len(LISTS)))
def test_muon(hip_device, which, nesterov):
    precision, shapes = LISTS[which]
    fast = precision == "fast"
    co = PUBLISHED if fast else triples(QUINTIC, 2)
    rate, decay, mu = 0.5, 0.9, 0.9
    g = torch.Generator(device=hip_device).manual_seed(which)
    params, grads, momenta = [], [], []
    for k, (m, n, many) in enumerate(shapes):
        # the types of a model's: 16-bit ones, or float32; gradients of any
        dtype = TYPES[(which + k) % 2 * 2] if fast else torch.float32
        params.append((torch.randn(many, m, n, generator=g, device=hip_device) * 0.05).to(dtype))
        grads.append(_stack(hip_device, which, many, m, n).to(TYPES[(which + k + nesterov) % 3]))
        momenta.append(_stack(hip_device, which + 100, many, m, n))
    before = [p.clone() for p in params]
    old = [b.clone() for b in momenta]
    count = len(params)
    L.torch_host().muon_step(params, grads, momenta, [rate] * count, [decay] * count, mu, nesterov,
                             [x for t in co for x in t], 1e-7,
                             [L.ORTHO_FAST if fast else L.ORTHO_FP32] * count)
    for k, (m, n, many) in enumerate(shapes):
        for i in {0, many - 1}:
            grad = grads[k][i].double()
            buf = mu * old[k][i].double() + (1 - mu) * grad
            assert torch.allclose(momenta[k][i].double(), buf, rtol=0,
                                  atol=4 * 2.0 ** -24 * float(buf.abs().max()))
            u = mu * buf + (1 - mu) * grad if nesterov else buf
            o = orthogonalize(u, co)
            new = decay * before[k][i].double() - rate * o
            if fast:
                own = 1.15 * float((emulate(u, co) - o).norm())
            else:
                own = bound(u, co, "fp32") + 4e-7 * min(m, n) ** 0.5 * 16
            room = (1.05 * float((new.to(params[k].dtype).double() - new).norm()) + rate * own
                    + 2.0 ** -22 * (float(before[k][i].double().norm()) + rate * float(o.norm())))
            err = float((params[k][i].double() - new).norm())
            print(f"{m}x{n} {params[k].dtype}: {err:.2e} of {room:.2e}, the update's "
                  f"{rate * float(o.norm()):.2e}", flush=True)
            # a bound that tells a lost update, and one that is a hundredth off
            assert err <= room <= 0.02 * rate * float(o.norm())


def _stack(dev, seed, many, m, n):
    g = torch.Generator(device=dev).manual_seed(seed)
    t = torch.randn(many, m, n, generator=g, device=dev)
    strong = torch.randn(many, m, 2, generator=g, device=dev) @ torch.randn(
        many, 2, n, generator=g, device=dev)
    return (t + strong * ((m + n) / (m * n)) ** 0.5) * 1e-3
