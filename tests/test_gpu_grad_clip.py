"""Gradient norm and clipping (scao_grad_norm, scao_grad_clip) against their
definition in 64 bits.

Tolerances.  The norm is summed in double from exact terms and rounded once to
float32: half an ulp, 6e-8, and as much again for the double sum's rounding of
up to 1e7 terms.  The factor is formed in double and rounded once to float32
(6e-8 relative), the product once to the gradient's type: 2^-24, 2^-11 or 2^-8
relative, half an ulp, plus the factor's."""

from __future__ import annotations

import math

import pytest
import torch

import scao_amd

pytestmark = pytest.mark.gpu

ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 1e-44, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-40}


def _params(grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.zeros(g.shape, dtype=g.dtype, device=g.device))
        p.grad = g
        out.append(p)
    return out


def _want(grads, max_norm, p, scale):
    flat = torch.cat([g.detach().double().cpu().reshape(-1) for g in grads])
    norm = torch.linalg.vector_norm(flat, p).item() * scale if flat.numel() else 0.0
    f = scale * min(1.0, max_norm / (norm + 1e-6))
    return norm, [g.detach().double().cpu() * f for g in grads]


def _check(grads, max_norm, p=2.0, scale=1.0):
    norm, want = _want(grads, max_norm, p, scale)
    got = scao_amd.clip_grad_norm_(_params(grads), max_norm, norm_type=p, scale=scale)
    assert got.shape == () and got.dtype == torch.float32
    assert abs(got.item() - norm) <= 1.2e-7 * norm
    for g, w in zip(grads, want):
        err = (g.double().cpu() - w).abs()
        assert bool((err <= w.abs() * (ULP[g.dtype] + 1.3e-7) + TINY[g.dtype]).all())


def _normal(dev, seed, *shape, dtype=torch.float32, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(dev)


@pytest.mark.parametrize("dtype", list(ULP))
@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("sizes", [(1,), (7, 0, 3), (8191, 8192, 8193), (16384, 1, 16385, 70001)])
def test_types_norms_and_sizes(hip_device, dtype, p, sizes):
    grads = [_normal(hip_device, i, n, dtype=dtype) for i, n in enumerate(sizes)]
    _check(grads, 0.5, p)


@pytest.mark.parametrize("dtype", list(ULP))
@pytest.mark.parametrize("start", [0, 1, 2, 3, 5, 7, 9])
def test_views_at_any_start_leave_their_neighbours(hip_device, dtype, start):
    """Tensors one after the other in one buffer, at every alignment of a
    16-byte vector: all are scaled, the buffer's other elements are not."""
    sizes = [1, 2, 8, 16389, 3, 33, 8192]
    total = start + sum(sizes) + 5
    buf = _normal(hip_device, start, total, dtype=dtype)
    before = buf.clone()
    grads, at = [], start
    for n in sizes:
        grads.append(buf[at:at + n])
        at += n
    _check(grads, 0.25, scale=0.5)
    assert torch.equal(buf[:start], before[:start]) and torch.equal(buf[at:], before[at:])


def test_many_tensors_of_mixed_types(hip_device):
    """More tensors than one launch's table holds (336), empty ones among them."""
    types = list(ULP)
    grads = [_normal(hip_device, i, (i * 37) % 501, dtype=types[i % 3]) for i in range(431)]
    _check(grads, 1.0)
    _check(grads, 0.01, math.inf, 0.5)


def test_a_large_tensor_in_two_tables(hip_device):
    """More than 2^31 elements, which take two entries of a table: the first in
    one launch's last place, the second in the next launch."""
    small = [_normal(hip_device, i, i % 50 + 1, dtype=torch.bfloat16) for i in range(340)]
    n = (1 << 31) + 9
    big = torch.zeros(n, dtype=torch.bfloat16, device=hip_device)
    big[::1 << 20] = 2.0
    big[-1] = 4.0
    count = (n + (1 << 20) - 1) >> 20
    kept = [g.double() for g in small]
    norm = (sum(g.square().sum().item() for g in kept) + 4.0 * count + 16.0) ** 0.5
    got = scao_amd.clip_grad_norm_(_params(small[:335] + [big] + small[335:]), 1.0)
    assert abs(got.item() - norm) <= 1.2e-7 * norm
    for g, k in zip(small, kept):
        assert bool(((g.double() - k / norm).abs()
                     <= k.abs() / norm * (ULP[torch.bfloat16] + 1.3e-7) + TINY[torch.bfloat16]).all())
    for i, v in ((0, 2.0), (1 << 31, 2.0), (n - 1, 4.0)):
        assert abs(big[i].item() - v / norm) <= 2.0 ** -8 * v / norm
    assert int((big != 0).sum()) == count + 1


def test_strides(hip_device):
    """Dense gradients in another order are scaled in place; slices of larger
    tensors are scaled, the rest of their storage is not."""
    a = _normal(hip_device, 0, 40, 30)
    b = _normal(hip_device, 1, 40, 30)
    c = _normal(hip_device, 2, 2, 3, 8, 8).to(memory_format=torch.channels_last)
    kept = b.clone()
    _check([a.t(), b[:, 3:20], c, b[:, 25:]], 0.5)
    assert torch.equal(b[:, :3], kept[:, :3]) and torch.equal(b[:, 20:25], kept[:, 20:25])


def test_nothing_is_written_under_the_norm(hip_device):
    g = _normal(hip_device, 3, 5000, dtype=torch.bfloat16)
    kept = g.clone()
    norm = scao_amd.clip_grad_norm_(_params([g]), 1e4)
    assert torch.equal(g, kept)
    assert abs(norm.item() - kept.double().norm().item()) <= 1.2e-7 * norm.item()


def test_squares_outside_fp32(hip_device):
    """Values whose squares overflow or vanish in 32 bits."""
    _check([torch.full((300,), 1e30, device=hip_device), torch.ones(5, device=hip_device)], 2.0)
    _check([torch.full((300,), 1e-30, device=hip_device)], 1e-35)
    zero = [torch.zeros(300, device=hip_device)]
    assert scao_amd.clip_grad_norm_(_params(zero), 1.0).item() == 0.0


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("dtype", list(ULP))
def test_nan_and_infinity(hip_device, dtype, p):
    for bad in (math.nan, math.inf, -math.inf):
        g, h = _normal(hip_device, 4, 20000, dtype=dtype), _normal(hip_device, 5, 7, dtype=dtype)
        g[12345] = bad
        kept = g.clone()
        with pytest.raises(RuntimeError, match="cannot be clipped"):
            scao_amd.clip_grad_norm_(_params([g, h]), 1.0, norm_type=p, error_if_nonfinite=True)
        assert torch.equal(g.view(torch.uint8), kept.view(torch.uint8))
        norm = scao_amd.clip_grad_norm_(_params([g, h]), 1.0, norm_type=p)
        if math.isnan(bad):
            assert math.isnan(norm.item()) and bool(g.isnan().all()) and bool(h.isnan().all())
        else:
            assert norm.item() == math.inf and bool(h.eq(0).all())
            assert bool(g[12345].isnan()) and int(g.isnan().sum()) == 1


def test_norm_alone(hip_device):
    grads = [_normal(hip_device, 6, 333, 77), _normal(hip_device, 7, 4096, dtype=torch.float16)]
    for p in (1.0, 2.0, math.inf):
        norm, _ = _want(grads, 1.0, p, 3.0)
        kept = [g.clone() for g in grads]
        got = scao_amd.global_grad_norm(_params(grads), p, scale=3.0).item()
        assert abs(got - norm) <= 1.2e-7 * norm
        assert all(torch.equal(a, b) for a, b in zip(grads, kept))
    wide = torch.ones(1, device=hip_device).expand(100)   # allowed where nothing is written
    p = torch.nn.Parameter(torch.zeros(100, device=hip_device))
    p.grad = wide
    assert scao_amd.global_grad_norm([p]).item() == 10.0


def test_same_bits_every_time_and_on_another_stream(hip_device):
    grads = [_normal(hip_device, 8, 1 << 20), _normal(hip_device, 9, 999, dtype=torch.bfloat16)]
    first = None
    side = torch.cuda.Stream()
    for i in range(4):
        work = [g.clone() for g in grads]
        torch.cuda.synchronize()
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            norm = scao_amd.clip_grad_norm_(_params(work), 0.125)
        torch.cuda.synchronize()
        now = [norm.view(1), *work]
        first = first or now
        assert all(torch.equal(a, b) for a, b in zip(first, now))


def test_graph_replays(hip_device):
    """Captured once, replayed on other gradients."""
    g = _normal(hip_device, 10, 100003)
    params = _params([g])
    scao_amd.clip_grad_norm_(params, 1.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = scao_amd.clip_grad_norm_(params, 1.0)
    for i in range(3):
        new = _normal(hip_device, 20 + i, 100003, std=10.0 ** (i - 1))
        g.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        n, want = _want([new], 1.0, 2.0, 1.0)
        assert abs(norm.item() - n) <= 1.2e-7 * n
        assert bool(((g.double().cpu() - want[0]).abs() <= want[0].abs() * 2e-7).all())


def test_refusals(hip_device):
    g = _normal(hip_device, 11, 100)
    kept = g.clone()
    clip = scao_amd.clip_grad_norm_
    for kw in (dict(max_norm=-1.0), dict(max_norm=math.nan), dict(max_norm=1.0, norm_type=3.0),
               dict(max_norm=1.0, scale=0.0), dict(max_norm=1.0, scale=math.inf),
               dict(max_norm=1.0, scale=math.nan)):
        with pytest.raises(ValueError):
            clip(_params([g]), **kw)
    with pytest.raises(ValueError, match="share memory"):
        clip(_params([g[:60], g[59:]]), 0.1)
    with pytest.raises(ValueError, match="share memory"):
        clip(_params([g, g]), 0.1)
    p = torch.nn.Parameter(torch.zeros(100, device=hip_device))
    p.grad = torch.ones(1, device=hip_device).expand(100)
    with pytest.raises(ValueError, match="expanded"):
        clip([p], 0.1)
    with pytest.raises(TypeError):
        clip(_params([g.double()]), 0.1)
    with pytest.raises(RuntimeError, match="gradient is on 'cpu'"):
        clip(_params([g.cpu()]), 0.1)
    assert torch.equal(g, kept)
    assert clip([], 1.0).item() == 0.0
    assert clip([torch.nn.Parameter(torch.zeros(3, device=hip_device))], 1.0).item() == 0.0
    assert clip(_params([g[:0]]), 1.0).item() == 0.0


@pytest.mark.parametrize("dtype", list(ULP))
def test_more_than_the_caches_hold(hip_device, dtype):
    """Over 512 MiB, in tensors of odd sizes, one past 2^27 elements."""
    size = torch.finfo(dtype).bits // 8
    sizes = [1, 70001, (1 << 27) + 12345, 3, (400 << 20) // size + 1]
    flat = torch.empty(sum(sizes), dtype=dtype, device=hip_device)
    period = _normal(hip_device, 0, 100003, dtype=dtype)
    for at in range(0, flat.numel(), 100003):
        n = min(100003, flat.numel() - at)
        flat[at:at + n] = period[:n]
    norm = flat.double().norm().item() if size == 2 else sum(
        c.double().square().sum().item() for c in flat.split(1 << 26)) ** 0.5
    want = (period.double() * min(1.0, 0.5 / (norm + 1e-6)))
    got = scao_amd.clip_grad_norm_(_params(list(flat.split(sizes))), 0.5)
    assert abs(got.item() - norm) <= 2e-7 * norm
    for at in range(0, flat.numel(), 100003):
        n = min(100003, flat.numel() - at)
        err = (flat[at:at + n].double() - want[:n]).abs()
        assert bool((err <= want[:n].abs() * (ULP[dtype] + 1.3e-7) + TINY[dtype]).all())


def test_a_tensor_past_2_31_elements(hip_device):
    n = (1 << 31) + 70_003
    g = torch.zeros(n, dtype=torch.bfloat16, device=hip_device)
    g[::1 << 16] = 3.0
    g[-1] = 4.0
    count = (n + (1 << 16) - 1) >> 16
    norm = (9.0 * count + 16.0) ** 0.5
    got = scao_amd.clip_grad_norm_(_params([g]), 1.0)
    assert abs(got.item() - norm) <= 1.2e-7 * norm
    for i, v in ((0, 3.0), (((n - 2) >> 16) << 16, 3.0), (n - 1, 4.0)):
        assert abs(g[i].item() - v / norm) <= 2.0 ** -8 * v / norm
    assert int((g != 0).sum()) == count + 1
