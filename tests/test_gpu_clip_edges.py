"""Gradient norm and clipping at the ends of what they take: gradients that
only an iterator holds, versions, bounds of infinity, shared memory, tracing.

The norm of small whole numbers is exact; scaled values are compared with the
product in 64 bits, rounded once."""

from __future__ import annotations

import math

import pytest
import torch

import scao_amd

pytestmark = pytest.mark.gpu


def _params(grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.zeros(g.shape, dtype=g.dtype, device=g.device))
        p.grad = g
        out.append(p)
    return out


def _normal(dev, seed, *shape, dtype=torch.float32, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(dev)


def test_gradients_that_only_an_iterator_holds(hip_device):
    """They live until the kernels are queued: in several tables, the memory of
    the last ones freed first would hold the first table's sums."""
    torch.cuda.empty_cache()
    for entry in (scao_amd.global_grad_norm, lambda p: scao_amd.clip_grad_norm_(p, 1.0)):
        params = _params([torch.ones(4000, device=hip_device) for _ in range(1000)])

        def temporaries():
            while params:
                yield params.pop()

        torch.cuda.synchronize()
        assert entry(temporaries()).item() == 2000.0


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("scale", [1.0, 0.5])
def test_a_bound_of_infinity_clips_nothing(hip_device, p, scale):
    """max_norm = inf measures: the factor is `scale`, with an infinite norm too."""
    for bad in (None, math.inf, -math.inf):
        g, h = _normal(hip_device, 4, 20000), _normal(hip_device, 5, 7, dtype=torch.bfloat16)
        if bad is not None:
            g[12345] = bad
        want = [t * scale for t in (g, h)]
        norm = scao_amd.clip_grad_norm_(_params([g, h]), math.inf, norm_type=p, scale=scale)
        assert norm.item() == math.inf if bad is not None else math.isfinite(norm.item())
        assert torch.equal(g, want[0]) and torch.equal(h, want[1])
    g[3] = math.nan
    norm = scao_amd.clip_grad_norm_(_params([g, h]), math.inf, norm_type=p)
    assert math.isnan(norm.item()) and bool(g.isnan().all()) and bool(h.isnan().all())


def test_traces_hold_the_clipping(hip_device):
    from torch.fx.experimental.proxy_tensor import make_fx
    params = _params([_normal(hip_device, 8, 33), _normal(hip_device, 9, 5, 7)])

    def clip(a, b):
        params[0].grad, params[1].grad = a * 2, b * 2
        norm = scao_amd.clip_grad_norm_(params, 0.5)
        return norm, scao_amd.global_grad_norm(params), params[0].grad, params[1].grad

    first = [p.grad for p in params]
    new = [_normal(hip_device, 10, 33), _normal(hip_device, 11, 5, 7)]
    want = [t.clone() for t in clip(*new)]
    assert abs(want[1].item() - 0.5) < 1e-5
    for traced in (torch.jit.trace(clip, first), make_fx(clip)(*first)):
        for got, w in zip(traced(*new), want):
            assert torch.equal(got, w)


def test_dispatch_modes_see_the_clipping(hip_device):
    from torch.utils._python_dispatch import TorchDispatchMode
    seen = []

    class Log(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    g = torch.ones(100, device=hip_device)
    with Log():
        assert scao_amd.global_grad_norm(_params([g])).item() == 10.0
        assert scao_amd.clip_grad_norm_(_params([g]), 20.0).item() == 10.0
    assert {s.split(".")[1] for s in seen if s.startswith("scao_amd.")} == {"grad_norm",
                                                                          "grad_clip_"}


def test_operators_check_their_arguments(hip_device):
    """Called by their names, past the Python functions' own checks."""
    g = torch.ones(100, device=hip_device)
    scao_amd.global_grad_norm(_params([g]))
    norm, clip = torch.ops.scao_amd.grad_norm, torch.ops.scao_amd.grad_clip_
    assert norm([g, g], 1, 1.0).item() == 200.0
    for grads in ([g.double()], [g, g.cpu()], [g.to_sparse()]):
        with pytest.raises((RuntimeError, NotImplementedError)):
            norm(grads, 2, 1.0)
        with pytest.raises((RuntimeError, NotImplementedError)):
            clip(grads, 2, 1.0, 0.1)
    with pytest.raises(ValueError, match="share memory"):
        clip([g, g], 2, 1.0, 0.1)
    with pytest.raises(RuntimeError):
        clip([g], 3, 1.0, 0.1)
    assert bool(g.eq(1).all())


def test_negated_views(hip_device):
    """A gradient that holds its values negated is scaled in place all the same."""
    g = _normal(hip_device, 12, 500)
    want = g.double() * 0.25
    neg = torch._neg_view(-g)
    assert neg.is_neg()
    scao_amd.clip_grad_norm_(_params([neg]), math.inf, scale=0.25)
    assert torch.equal(neg.double(), want)


def test_versions_count_the_clipping(hip_device):
    buf = _normal(hip_device, 0, 40, 30)
    grads = [_normal(hip_device, 1, 100), buf[:, 3:20], _normal(hip_device, 2, 7, 5).t()]
    params = _params(grads)
    before = [g._version for g in grads]
    scao_amd.global_grad_norm(params)
    assert [g._version for g in grads] == before
    scao_amd.clip_grad_norm_(params, 0.1)
    assert all(g._version > v for g, v in zip(grads, before))
    with torch.inference_mode():
        g = torch.ones(10, device=hip_device)
        scao_amd.clip_grad_norm_(_params([g]), 1.0)
    assert abs(g[0].item() - 10 ** -0.5) < 1e-6


def test_a_clipped_gradient_that_a_graph_holds(hip_device):
    """Its later backward pass must not use the scaled values."""
    p = torch.nn.Parameter(_normal(hip_device, 3, 50))
    (p ** 3).sum().backward(create_graph=True)
    again = (p.grad ** 2).sum()
    scao_amd.clip_grad_norm_([p], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        again.backward()


def _shared():
    """names of layouts of two gradients in one buffer of 40 x 30 that share an element"""
    return {
        "columns": lambda b: (b[:, 0:10], b[:, 9:20]),
        "columns of another order": lambda b: (b[:, 9:20], b[:, 0:10]),
        "one twice": lambda b: (b[:, 0:10], b[:, 0:10]),
        "a row and columns": lambda b: (b[7], b[:, 29:]),
        "every second and every third": lambda b: (b.view(-1)[::2], b.view(-1)[1::3]),
        "a corner": lambda b: (b[:20, :16], b[19:, 15:]),
        "the buffer's last element": lambda b: (b[:, 20:], b[39, 29:]),
        "another type's bytes": lambda b: (b[:, :4], b.view(torch.bfloat16)[:, 7:9]),
        "a window on itself": lambda b: (b.as_strided((30, 9), (4, 1)),),
        "two dimensions of one stride": lambda b: (b.as_strided((4, 4), (2, 2)),),
    }


@pytest.mark.parametrize("name", _shared())
def test_gradients_with_gaps_that_share_memory(hip_device, name):
    b = _normal(hip_device, 6, 40, 30)
    kept = b.clone()
    with pytest.raises(ValueError, match="share memory"):
        scao_amd.clip_grad_norm_(_params(_shared()[name](b)), 0.1)
    assert torch.equal(b, kept)


APART = {
    "columns": lambda b: (b[:, 0:10], b[:, 10:20], b[:, 25:]),
    "every second": lambda b: (b[:, ::2], b[:, 1::2]),
    "rows between columns": lambda b: (b[::2, :], b[1::2, :7], b[1::2, 7:]),
    "corners": lambda b: (b[:20, :16], b[:20, 16:], b[20:, :9], b[20:, 9:]),
    "a block and its frame": lambda b: (b[10:20, 10:20], b[:10], b[20:], b[10:20, :10],
                                       b[10:20, 20:]),
    "another type's bytes": lambda b: (b[:, :4], b.view(torch.bfloat16)[:, 8:11]),
    "transposed": lambda b: (b[:, :10].t(), b[:, 10:20].t()),
    "strides of 3 and 2": lambda b: (b.as_strided((2, 3), (3, 2)), b[1:]),
}


@pytest.mark.parametrize("name", APART)
def test_gradients_with_gaps_beside_each_other(hip_device, name):
    """Those that only lie between each other's elements are scaled once each."""
    b = _normal(hip_device, 7, 40, 30)
    if "type" in name:
        b.view(torch.bfloat16)[:, 8:11] = 1.0
    grads = APART[name](b)
    wide = [g.double() for g in grads]
    norm = math.sqrt(sum(w.square().sum().item() for w in wide))
    got = scao_amd.clip_grad_norm_(_params(grads), 0.25)
    assert abs(got.item() - norm) <= 1.2e-7 * norm
    for g, w in zip(grads, wide):
        want = w * (0.25 / (norm + 1e-6))
        ulp = 2.0 ** -24 if g.dtype == torch.float32 else 2.0 ** -8
        assert bool(((g.double() - want).abs() <= want.abs() * (ulp + 1.3e-7)).all())


def test_forward_mode_is_refused(hip_device):
    import torch.autograd.forward_ad as fwd
    g = _normal(hip_device, 13, 50)
    kept = g.clone()
    p = torch.nn.Parameter(torch.zeros(50, device=hip_device))
    with fwd.dual_level():
        p.grad = fwd.make_dual(g, torch.ones_like(g))
        with pytest.raises(RuntimeError, match="forward"):
            scao_amd.clip_grad_norm_([p], 0.1)
        with pytest.raises(RuntimeError, match="forward"):
            scao_amd.global_grad_norm([p])
    assert torch.equal(g, kept)
