"""Norms and rotation of queries and keys (scao_qk_rope_forward, _backward) against
their definition in 64 bits; bounds: tests/rope_reference.py."""

from __future__ import annotations

import pytest
import torch

import scao_amd
from tests.rope_reference import reference

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _normal(dev, seed, *shape, dtype=torch.float32, std=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * std).to(dtype)


def _inputs(dev, batch, tokens, hq, hk, dim, dtype, layout="plain", seed=0):
    """plain: dense; packed: slices of rows that hold values too, at any element;
    turned: heads before tokens"""
    if layout == "packed":
        rows = _normal(dev, seed, batch, tokens, (hq + 2 * hk) * dim + 3, dtype=dtype, std=1.5)
        q = rows[..., 1:1 + hq * dim].unflatten(-1, (hq, dim))
        k = rows[..., 1 + hq * dim:1 + (hq + hk) * dim].unflatten(-1, (hk, dim))
        return q, k
    shape = (batch, hq, tokens, dim), (batch, hk, tokens, dim)
    if layout == "turned":
        return tuple(_normal(dev, seed + i, *s, dtype=dtype, std=1.5).transpose(1, 2)
                     for i, s in enumerate(shape))
    return tuple(_normal(dev, seed + i, batch, tokens, h, dim, dtype=dtype, std=1.5)
                 for i, h in enumerate((hq, hk)))


def _check(dev, batch, tokens, hq, hk, dim, rot, dtype, layout="plain", interleaved=False,
           weights="same", far=50, wide=True, eps=1e-6):
    print(f"{batch}x{tokens} heads {hq}/{hk} dim {dim}/{rot} {dtype} {layout} {interleaved} "
          f"{weights}", flush=True)
    q, k = _inputs(dev, batch, tokens, hq, hk, dim, dtype, layout)
    wt = {"same": dtype, "fp32": torch.float32, "bf16": torch.bfloat16}.get(weights)
    wq, wk = (None if wt is None else (1 + _normal(dev, 7 + i, dim, std=0.3)).to(wt)
              for i in range(2))
    cos, sin = scao_amd.rotary_table(tokens + far, rot, 10000.0, dev)
    first = torch.randint(0, far + 1, (batch, 1), device=dev)
    positions = (first + torch.arange(tokens, device=dev)).to(torch.int64 if wide else torch.int32)
    if far == 0:
        assert int(positions.max()) == tokens - 1
    dq, dk = _normal(dev, 11, *q.shape, dtype=dtype), _normal(dev, 12, *k.shape, dtype=dtype)
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk) if t is not None]
    lq, lk, lwq, lwk = leaves if wt is not None else (*leaves, None, None)
    y = scao_amd.qk_norm_rope(lq, lk, lwq, lwk, cos, sin, None if far == 0 else positions, eps,
                              interleaved)
    grads = torch.autograd.grad(y, leaves, (dq, dk))
    alone = scao_amd.qk_norm_rope(q, k, wq, wk, cos, sin, positions, eps, interleaved)
    assert all(torch.equal(a, b) for a, b in zip(alone, y))
    for i, (x, w, d) in enumerate(((q, wq, dq), (k, wk, dk))):
        got = dict(y=y[i].detach(), dx=grads[i])
        if wt is not None:
            got["dw"] = grads[2 + i]
        want = reference(x, w, cos, sin, positions.long(), d, eps, interleaved)
        for name, (value, bound) in want.items():
            assert got[name].shape == value.shape
            assert got[name].dtype == (x.dtype if name != "dw" else wt)
            worst = ((got[name].double() - value).abs() / bound).max().item()
            assert worst <= 1.0, (name, i, worst)


DIMS = [(1, 0), (2, 2), (3, 2), (6, 4), (8, 8), (20, 12), (64, 64), (72, 36), (80, 80), (96, 48),
        (90, 34), (128, 128), (128, 64), (130, 130), (192, 64), (256, 256), (258, 10), (511, 510),
        (512, 512), (512, 0)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,rot", DIMS)
def test_head_sizes(hip_device, dim, rot, dtype, interleaved):
    _check(hip_device, 2, 5, 5, 2, dim, rot, dtype, interleaved=interleaved)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,tokens,hq,hk", [(1, 1, 1, 1), (1, 1, 32, 8), (96, 1, 32, 8),
                                                (1, 777, 16, 2), (3, 501, 5, 3), (2, 300, 9, 9),
                                                (1, 4099, 4, 1), (7, 2, 70, 1)])
def test_tokens_and_heads(hip_device, batch, tokens, hq, hk, dtype):
    _check(hip_device, batch, tokens, hq, hk, 64, 64, dtype)


@pytest.mark.parametrize("layout", ["packed", "turned"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,rot", [(128, 128), (40, 20), (33, 10)])
def test_layouts(hip_device, layout, dtype, dim, rot):
    _check(hip_device, 3, 50, 8, 3, dim, rot, dtype, layout)


@pytest.mark.parametrize("weights", ["fp32", "bf16", "none"])
@pytest.mark.parametrize("dtype", TYPES)
def test_weights(hip_device, weights, dtype):
    _check(hip_device, 2, 40, 6, 2, 96, 96, dtype, weights=weights, wide=False)


def test_default_positions_and_leading_dimensions(hip_device):
    cos, sin = scao_amd.rotary_table(64, 32, device=hip_device)
    w = torch.ones(32, device=hip_device)
    q, k = (_normal(hip_device, i, 2, 3, 20, h, 32) for i, h in enumerate((4, 2)))
    at = torch.arange(20, device=hip_device).expand(2, 3, 20)
    want = scao_amd.qk_norm_rope(q, k, w, w, cos, sin, at)
    got = scao_amd.qk_norm_rope(q, k, w, w, cos, sin)
    assert all(torch.equal(a, b) and a.shape == t.shape for a, b, t in zip(got, want, (q, k)))
    one = scao_amd.qk_norm_rope(q[1, 2], k[1, 2], w, w, cos, sin)
    assert all(torch.equal(a, b[1, 2]) for a, b in zip(one, want))
    tok = scao_amd.qk_norm_rope(q[1, 2, 7], k[1, 2, 7], w, w, cos, sin, at[1, 2, 7])
    assert all(torch.equal(a, b[1, 2, 7]) for a, b in zip(tok, want))


def test_positions_outside_of_the_table(hip_device):
    cos, sin = scao_amd.rotary_table(10, 16, device=hip_device)
    q, k = (_normal(hip_device, i, 1, 4, h, 32) for i, h in enumerate((3, 1)))
    at = torch.tensor([[3, 10, -1, 1 << 40]], device=hip_device)
    for i, y in enumerate(scao_amd.qk_norm_rope(q, k, None, None, cos, sin, at)):
        assert bool(y[:, 1:, :, :16].isnan().all()) and not bool(y[:, 1:, :, 16:].isnan().any())
        assert not bool(y[:, 0].isnan().any())


def test_nan_stays_in_its_head(hip_device):
    cos, sin = scao_amd.rotary_table(8, 64, device=hip_device)
    q, k = (_normal(hip_device, i, 2, 8, h, 64, dtype=torch.bfloat16) for i, h in enumerate((4, 2)))
    clean = scao_amd.qk_norm_rope(q, k, None, None, cos, sin)
    q[1, 3, 2, 5] = float("nan")
    q[0, 0, 1, 63] = float("inf")
    leaf = q.detach().requires_grad_()
    y, yk = scao_amd.qk_norm_rope(leaf, k, None, None, cos, sin)
    bad = torch.zeros(2, 8, 4, dtype=torch.bool, device=hip_device)
    bad[1, 3, 2] = bad[0, 0, 1] = True
    assert bool(y[1, 3, 2].isnan().all()) and bool(y[0, 0, 1].isnan().any())
    assert torch.equal(y[~bad], clean[0][~bad]) and torch.equal(yk, clean[1])
    (dx,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
    assert bool(dx[bad].isnan().any()) and not bool(dx[~bad].isnan().any())


def test_gradients_against_differences(hip_device):
    """in fp32, along random directions: central differences are off by h^2 times a
    third derivative (1e-4 of the values here) and by 2^-24 / h of them (1e-4)"""
    dev = hip_device
    cos, sin = scao_amd.rotary_table(40, 12, 100.0, dev)
    q, k = (_normal(dev, i, 2, 5, h, 20) for i, h in enumerate((3, 2)))
    wq, wk = (1 + _normal(dev, 5 + i, 20, std=0.3) for i in range(2))
    dq, dk = _normal(dev, 8, *q.shape), _normal(dev, 9, *k.shape)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    grads = torch.autograd.grad(scao_amd.qk_norm_rope(*leaves, cos, sin), leaves, (dq, dk))

    def loss(*args):
        with torch.no_grad():
            y = scao_amd.qk_norm_rope(*args, cos, sin)
            return float((y[0].double() * dq).sum() + (y[1].double() * dk).sum())

    for i, g in enumerate(grads):
        way, h = _normal(dev, 20 + i, *g.shape), 1e-2
        moved = [[t.detach() + (s * h * way if i == j else 0) for j, t in enumerate(leaves)]
                 for s in (1, -1)]
        slope = (loss(*moved[0]) - loss(*moved[1])) / (2 * h)
        want = float((g.double() * way).sum())
        scale = float(g.double().norm() * way.double().norm())
        assert abs(slope - want) <= 2e-3 * scale


def test_partial_gradients(hip_device):
    cos, sin = scao_amd.rotary_table(16, 32, device=hip_device)
    q, k = (_normal(hip_device, i, 2, 16, h, 32) for i, h in enumerate((4, 2)))
    w = [1 + _normal(hip_device, 5 + i, 32, std=0.1) for i in range(2)]
    d = _normal(hip_device, 9, *q.shape), _normal(hip_device, 10, *k.shape)
    every = [t.clone().requires_grad_() for t in (q, k, *w)]
    all_grads = torch.autograd.grad(scao_amd.qk_norm_rope(*every, cos, sin), every, d)
    for mask in range(1, 16):
        leaves = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((q, k, *w))]
        y = scao_amd.qk_norm_rope(*leaves, cos, sin)
        wanted = [t for t in leaves if t.requires_grad]
        outs = [(a, b) for a, b in zip(y, d) if a.requires_grad]
        got = torch.autograd.grad([a for a, _ in outs], wanted, [b for _, b in outs])
        for g, want in zip(got, [g for i, g in enumerate(all_grads) if mask >> i & 1]):
            assert torch.equal(g, want)
    # one of the weights alone
    for i in range(2):
        leaves = [t.clone().requires_grad_() for t in (q, k, w[i])]
        pair = [None, None]
        pair[i] = leaves[2]
        y = scao_amd.qk_norm_rope(leaves[0], leaves[1], *pair, cos, sin)
        got = torch.autograd.grad(y, leaves, d)
        assert torch.equal(got[2], all_grads[2 + i]) and torch.equal(got[i], all_grads[i])
        ones = [t.clone().requires_grad_() for t in (q, k)]
        y = scao_amd.qk_norm_rope(*ones, None, None, cos, sin)
        assert torch.equal(got[1 - i], torch.autograd.grad(y, ones, d)[1 - i])
    # one output alone
    leaves = [t.clone().requires_grad_() for t in (q, k, *w)]
    got = torch.autograd.grad(scao_amd.qk_norm_rope(*leaves, cos, sin)[0], leaves, d[0])
    assert torch.equal(got[0], all_grads[0]) and bool((got[1] == 0).all())


def test_empty(hip_device):
    cos, sin = scao_amd.rotary_table(16, 32, device=hip_device)
    w = torch.ones(32, device=hip_device, requires_grad=True)
    q = torch.empty(2, 0, 4, 32, device=hip_device, requires_grad=True)
    y = scao_amd.qk_norm_rope(q, q, w, None, cos, sin)
    assert y[0].shape == q.shape
    dq, dw = torch.autograd.grad(y, (q, w), (torch.empty_like(q), torch.empty_like(q)))
    assert dq.shape == q.shape and bool((dw == 0).all())


def test_captured_with_its_backward_pass(hip_device):
    cos, sin = scao_amd.rotary_table(64, 64, device=hip_device)
    m = scao_amd.QKNormRope(64, 64, device=hip_device, dtype=torch.bfloat16)
    q, k = (_normal(hip_device, i, 2, 64, h, 64, dtype=torch.bfloat16).requires_grad_()
            for i, h in enumerate((8, 2)))
    d = [torch.empty_like(q), torch.empty_like(k)]

    def go():
        return torch.autograd.grad(m(q, k), (q, k, m.q, m.k), d)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = go()
    for i in range(3):
        with torch.no_grad():
            for t in (q, k, *d):
                t.copy_(_normal(hip_device, 30 + i, *t.shape))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, go()))


def test_another_stream_and_the_same_bits(hip_device):
    cos, sin = scao_amd.rotary_table(700, 128, device=hip_device)
    q, k = (_normal(hip_device, i, 3, 700, h, 128, dtype=torch.bfloat16).requires_grad_()
            for i, h in enumerate((8, 2)))
    w = torch.ones(128, device=hip_device, dtype=torch.bfloat16, requires_grad=True)

    def go():
        y = scao_amd.qk_norm_rope(q, k, w, w, cos, sin)
        return *y, *torch.autograd.grad(y, (q, k, w), y)

    want = go()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = go()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_offsets_past_32_bits(hip_device):
    """tokens more than 2^31 elements apart"""
    row = (1 << 31) + 24
    buf = torch.empty(row + 4 * 64, device=hip_device, dtype=torch.bfloat16)
    x = buf.as_strided((1, 2, 4, 64), (0, row, 64, 1))
    x.copy_(_normal(hip_device, 1, 1, 2, 4, 64))
    cos, sin = scao_amd.rotary_table(2, 64, device=hip_device)
    got = scao_amd.qk_norm_rope(x, x[:, :, :1], None, None, cos, sin)
    y = x.contiguous()
    want = scao_amd.qk_norm_rope(y, y[:, :, :1], None, None, cos, sin)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(hip_device):
    cos, sin = scao_amd.rotary_table(16, 32, device=hip_device)
    q, k = (_normal(hip_device, i, 2, 8, h, 32) for i, h in enumerate((4, 2)))
    w = torch.ones(32, device=hip_device)
    for bad, error in (((q.double(), k.double(), w, w, cos, sin), TypeError),
                       ((q, k.half(), w, w, cos, sin), TypeError),
                       ((q, k[..., :30], w, w, cos, sin), ValueError),
                       ((q, k[:1], w, w, cos, sin), ValueError),
                       ((q, k, w[:5], w, cos, sin), ValueError),
                       ((q, k, w, w, cos.double(), sin.double()), TypeError),
                       ((q, k, w, w, cos, sin[:3]), ValueError),
                       ((q, k, w, w, cos[:7], sin[:7]), ValueError),
                       ((q[..., :20], k[..., :20], None, None, cos, sin), ValueError),
                       ((q, k, w, w, cos, sin, torch.zeros(2, 8, device=hip_device)), TypeError),
                       ((q, k, w, w, cos, sin, torch.zeros(2, 7, device=hip_device,
                                                           dtype=torch.int64)), ValueError),
                       ((q, k, w, w, cos, sin, None, -1.0), ValueError)):
        with pytest.raises(error):
            scao_amd.qk_norm_rope(*bad)
    with pytest.raises(NotImplementedError):
        scao_amd.qk_norm_rope(q, k, w, w, cos.clone().requires_grad_(), sin)
    leaf = q.clone().requires_grad_()
    y = scao_amd.qk_norm_rope(leaf, k, w, w, cos, sin)[0]
    (g,) = torch.autograd.grad(y.square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(NotImplementedError):
            scao_amd.qk_norm_rope(dual, k, w, w, cos, sin)


def test_module_keeps_its_tables(hip_device):
    m = scao_amd.QKNormRope(64, 100, rotary_dim=32, base=1e4)
    cos = m.cos.clone()
    m = m.to(hip_device, torch.bfloat16)
    assert m.q.dtype == torch.bfloat16 and m.cos.dtype == torch.float32
    assert torch.equal(m.cos.cpu(), cos) and m.sin.device == m.q.device
    assert list(m.state_dict()) == ["q", "k"]
    assert m.half().cos.dtype == torch.float32
