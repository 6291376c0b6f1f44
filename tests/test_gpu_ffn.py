"""The gated feed-forward block (scao_ffn_forward, scao_ffn_backward) against
its definition in 64 bits; bounds: tests/ffn_reference.py."""

from __future__ import annotations

import math

import pytest
import torch

import scao_amd
from tests.ffn_reference import norm_bound, reference

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
ACTS = ["silu", "gelu", "gelu_tanh", "relu", "sigmoid"]


def _normal(dev, seed, rows, cols, dtype, std=1.0, pad=0, skip=0):
    """rows x cols inside rows of cols + pad, the first at element skip"""
    g = torch.Generator(device=dev).manual_seed(seed)
    t = torch.randn(rows * (cols + pad) + skip, generator=g, device=dev) * std
    return t.to(dtype)[skip:].view(rows, cols + pad)[:, :cols]


def _inputs(dev, tokens, d, f, dtype, seed=0, pad=0, skip=0, packed=False):
    if packed:
        gate, up = _normal(dev, seed + 1, 2 * f, d, dtype, d ** -0.5, pad, skip).split(f)
    else:
        gate = _normal(dev, seed + 1, f, d, dtype, d ** -0.5, pad, skip)
        up = _normal(dev, seed + 2, f, d, dtype, d ** -0.5, pad, skip)
    return (_normal(dev, seed, tokens, d, dtype, 1.0, pad, skip), gate, up,
            _normal(dev, seed + 3, d, f, dtype, f ** -0.5, pad, skip),
            _normal(dev, seed + 4, tokens, d, dtype, 0.5, pad, skip))


def _run(x, gate, up, down, dy, name):
    leaves = [t.detach().requires_grad_() for t in (x, gate, up, down)]
    y = scao_amd.gated_ffn(*leaves, activation=name)
    grads = torch.autograd.grad(y, leaves, dy)
    return dict(y=y.detach(), **dict(zip(("dx", "dgate", "dup", "ddown"), grads)))


def _compare(got, want, dtype, what=""):
    for k, (v, bound) in want.items():
        if k not in got:
            continue
        assert got[k].dtype == dtype and got[k].shape == v.shape
        err = (got[k].double() - v).abs()
        worst = (err / bound).max().item()
        rel = (err.norm() / v.norm().clamp_min(1e-300)).item()
        print(f"{what} {k}: {worst:.3f} of the bound, rel {rel:.2e}", flush=True)
        assert worst <= 1.0, (what, k, worst)
        if v.numel() >= 1000:
            assert rel <= norm_bound(dtype), (what, k, rel)


def _check(dev, tokens, d, f, dtype, name="silu", **kw):
    print(f"tokens {tokens} d {d} f {f} {dtype} {name} {kw}", flush=True)
    ins = _inputs(dev, tokens, d, f, dtype, **kw)
    want = reference(*ins, name)
    _compare(_run(*ins, name), want, dtype, "training")
    y = scao_amd.gated_ffn(*ins[:4], activation=name)
    _compare(dict(y=y), want, dtype, "forward")


SIZES = [(1, 1, 1), (1, 64, 128), (2, 8, 8), (3, 7, 5), (17, 40, 24), (64, 64, 64), (65, 63, 129),
         (130, 72, 200), (129, 257, 131), (256, 256, 256), (257, 264, 520), (33, 1001, 67),
         (700, 96, 1000), (257, 512, 384), (300, 520, 1030), (521, 264, 2056), (777, 256, 512),
         (1030, 2048, 8192)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,d,f", SIZES)
def test_sizes(hip_device, dtype, tokens, d, f):
    _check(hip_device, tokens, d, f, dtype, ACTS[(tokens + d + f) % 5])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ACTS)
def test_activations(hip_device, dtype, name):
    _check(hip_device, 150, 136, 264, dtype, name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,d,f", [(1, 2048, 640), (5, 4096, 64), (24, 512, 1376),
                                        (128, 2048, 256), (16, 64, 4096)])
def test_few_tokens(hip_device, dtype, tokens, d, f):
    """Weights' rows and k, cut into parts that are joined."""
    _check(hip_device, tokens, d, f, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 15, 16, 17, 32, 33, 48, 63, 64, 65])
@pytest.mark.parametrize("d,f,skip", [(32, 33, 0), (31, 100, 1), (520, 264, 0), (2050, 70, 3)])
def test_serving_sizes(hip_device, dtype, tokens, d, f, skip):
    """The forward pass alone around the sizes where its kernels change, with
    rows that start and end anywhere."""
    ins = _inputs(hip_device, tokens, d, f, dtype, seed=tokens, skip=skip)
    y = scao_amd.gated_ffn(*ins[:4], activation=ACTS[tokens % 5])
    _compare(dict(y=y), reference(*ins, ACTS[tokens % 5]), dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_tiles(hip_device, dtype):
    _check(hip_device, 2050, 1032, 2056, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,d,f", [(1000, 129, 4099), (1023, 777, 2049), (1490, 1537, 4097)])
def test_down_projections_between(hip_device, dtype, tokens, d, f):
    """Too few columns for 256 x 256 tiles, rows enough for 256 x 128, in parts."""
    _check(hip_device, tokens, d, f, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kw", [dict(pad=8), dict(pad=3), dict(skip=1), dict(pad=64, skip=8),
                                dict(packed=True), dict(packed=True, pad=5, skip=3)])
@pytest.mark.parametrize("d,f", [(96, 144), (97, 141)])
def test_strides_and_starts(hip_device, dtype, kw, d, f):
    _check(hip_device, 70, d, f, dtype, **kw)


def test_gate_and_up_of_different_strides(hip_device):
    ins = list(_inputs(hip_device, 40, 64, 48, torch.bfloat16))
    ins[2] = _normal(hip_device, 9, 48, 64, torch.bfloat16, 0.125, pad=24)
    _compare(_run(*ins, "silu"), reference(*ins, "silu"), torch.bfloat16)
    ins[1], ins[2] = ins[2], ins[1]
    _compare(_run(*ins, "silu"), reference(*ins, "silu"), torch.bfloat16)


@pytest.mark.parametrize("dtype", TYPES)
def test_each_gradient_alone(hip_device, dtype):
    x, gate, up, down, dy = _inputs(hip_device, 50, 72, 90, dtype)
    want = reference(x, gate, up, down, dy, "silu")
    for mask in range(1, 16):
        leaves = [t.detach().requires_grad_(bool(mask >> i & 1))
                  for i, t in enumerate((x, gate, up, down))]
        y = scao_amd.gated_ffn(*leaves)
        y.backward(dy)
        for t, k in zip(leaves, ("dx", "dgate", "dup", "ddown")):
            assert (t.grad is not None) == t.requires_grad
            if t.grad is not None:
                _compare({k: t.grad}, want, dtype, f"mask {mask}")


def test_gradients_against_differences(hip_device):
    """Central differences of sum(y * dy) along random directions, fp32.  With
    steps of 1e-2 the difference is off by about its third derivative's 1e-4
    and by the sums' rounding, 1e-6 of sum |y dy| / 1e-2."""
    for name in ACTS:
        if name == "relu":   # its jumps have no third derivative
            continue
        ins = _inputs(hip_device, 40, 24, 56, torch.float32, seed=3)
        got = _run(*ins, name)
        dy = ins[4].double()
        scale = (scao_amd.gated_ffn(*ins[:4], activation=name).double() * dy).abs().sum().item()
        for i, k in enumerate(("dx", "dgate", "dup", "ddown")):
            v = _normal(hip_device, 50 + i, *ins[i].shape, torch.float32)
            v = v / v.norm()
            both = []
            for s in (1e-2, -1e-2):
                moved = list(ins[:4])
                moved[i] = moved[i] + s * v
                y = scao_amd.gated_ffn(*moved, activation=name)
                both.append((y.double() * dy).sum().item())
            num = (both[0] - both[1]) / 2e-2
            ana = (got[k].double() * v.double()).sum().item()
            assert abs(num - ana) <= 1e-3 * got[k].double().norm().item() + 1e-4 * scale, (name, k)


def test_offsets_past_32_bits(hip_device):
    """More than 2^31 elements of h: the last tokens' outputs and gradients are
    those of the last tokens alone, the weights' gradients the sums over pieces
    (fp32 sums of bf16 results: the pieces' roundings, 2^-8 of each)."""
    tokens, d, f = 270_001, 64, 8192
    x, gate, up, down, dy = _inputs(hip_device, tokens, d, f, torch.bfloat16)
    got = _run(x, gate, up, down, dy, "silu")
    tail = slice(tokens - 999, tokens)
    part = _run(x[tail], gate, up, down, dy[tail], "silu")
    want = reference(x[tail], gate, up, down, dy[tail], "silu")
    for k in ("y", "dx"):
        _compare({k: got[k][tail]}, want, torch.bfloat16, "tail")
        _compare({k: part[k]}, want, torch.bfloat16, "alone")
    for k in ("dgate", "dup", "ddown"):
        total, size = 0.0, 0.0
        for at in range(0, tokens, 54_001):
            piece = _run(x[at:at + 54_001], gate, up, down, dy[at:at + 54_001], "silu")[k].float()
            total, size = total + piece, size + piece.abs()
        err = (got[k].float() - total).abs()
        assert bool((err <= 2.0 ** -8 * (size + total.abs()) + 1e-3).all()), k


def test_shapes_of_x_and_views(hip_device):
    x, gate, up, down, dy = _inputs(hip_device, 60, 32, 48, torch.bfloat16)
    flat = scao_amd.gated_ffn(x, gate, up, down)
    for shape in ((60, 32), (3, 20, 32), (2, 3, 10, 32)):
        y = scao_amd.gated_ffn(x.reshape(shape), gate, up, down)
        assert y.shape == shape and torch.equal(y.reshape(60, 32), flat)
    assert torch.equal(scao_amd.gated_ffn(x[7], gate, up, down), scao_amd.gated_ffn(x[7:8], gate, up, down)[0])
    # columns of another stride, and a transposed batch
    xt = x.t().contiguous().t()
    assert torch.equal(scao_amd.gated_ffn(xt, gate, up, down), flat)
    assert torch.equal(scao_amd.gated_ffn(x, gate.t().contiguous().t(), up, down), flat)
    x3 = x.reshape(3, 20, 32).transpose(0, 1).detach().requires_grad_()
    y = scao_amd.gated_ffn(x3, gate, up, down)
    kept = scao_amd.gated_ffn(x.detach().requires_grad_(), gate, up, down)   # as for training
    assert torch.equal(y, kept.reshape(3, 20, 32).transpose(0, 1))
    y.sum().backward()   # an expanded gradient of the output
    assert x3.grad.shape == x3.shape and bool(x3.grad.isfinite().all())
    one = torch.ones(60, 32, dtype=torch.bfloat16, device=hip_device)
    want = reference(x, gate, up, down, one, "silu")
    _compare(dict(dx=x3.grad.transpose(0, 1).reshape(60, 32)), want, torch.bfloat16)


def test_saved_tensors_that_moved(hip_device):
    """Hooks that keep what the backward pass needs somewhere else."""
    x, gate, up, down, dy = _inputs(hip_device, 33, 40, 56, torch.bfloat16, packed=True, pad=8)
    want = _run(x, gate, up, down, dy, "silu")
    leaves = [t.detach().requires_grad_() for t in (x, gate, up, down)]
    with torch.autograd.graph.save_on_cpu():
        y = scao_amd.gated_ffn(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    for k, g in zip(("dx", "dgate", "dup", "ddown"), grads):
        assert torch.equal(g, want[k])


def test_nothing_to_do(hip_device):
    for t, d, f in ((0, 8, 16), (3, 8, 0), (3, 0, 16)):
        leaves = [torch.zeros(s, device=hip_device, requires_grad=True)
                  for s in ((t, d), (f, d), (f, d), (d, f))]
        y = scao_amd.gated_ffn(*leaves)
        assert y.shape == (t, d) and not y.any()
        y.sum().backward()
        assert all(p.grad.shape == p.shape and not p.grad.any() for p in leaves)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_bad_token_stays_alone(hip_device, dtype):
    """NaN and infinity in one token's input reach that token's output and
    gradient and no other's; operands' padding never reaches a result."""
    x, gate, up, down, dy = _inputs(hip_device, 37, 41, 53, dtype)
    clean = _run(x, gate, up, down, dy, "silu")
    for bad in (math.nan, math.inf):
        x2 = x.clone()
        x2[11, 3] = bad
        got = _run(x2, gate, up, down, dy, "silu")
        others = [i for i in range(37) if i != 11]
        assert torch.equal(got["y"][others], clean["y"][others])
        assert torch.equal(got["dx"][others], clean["dx"][others])
        assert not bool(got["y"][11].isfinite().any())


def test_large_pre_activations(hip_device):
    """f at both of its ends: no overflow inside where the result is finite."""
    for dtype in TYPES:
        for name in ACTS:
            x = torch.tensor([[-300.0], [-30.0], [30.0], [300.0], [0.0]], dtype=dtype,
                             device=hip_device)
            one = torch.ones(1, 1, dtype=dtype, device=hip_device)
            got = _run(x, one, one, one, torch.ones_like(x), name)
            want = reference(x, one, one, one, torch.ones_like(x), name)
            for k in ("y", "dx"):
                fits = want[k][0].to(dtype).isfinite()   # 300^2 is too large for fp16
                assert torch.equal(got[k].isfinite(), fits), (dtype, name, k)
                err = (got[k].double() - want[k][0]).abs()[fits]
                assert bool((err <= want[k][0][fits].abs() * 2.0 ** -7 + 1e-3).all()), (dtype, name)


def test_same_bits_every_time_and_on_another_stream(hip_device):
    ins = _inputs(hip_device, 300, 264, 520, torch.bfloat16)
    first, side = None, torch.cuda.Stream()
    for i in range(4):
        torch.cuda.synchronize()
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            got = _run(*ins, "silu")
        torch.cuda.synchronize()
        first = first or got
        assert all(torch.equal(got[k], first[k]) for k in first)


@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_graph_replays(hip_device, tokens):
    x, gate, up, down, _ = _inputs(hip_device, tokens, 264, 520, torch.bfloat16)
    scao_amd.gated_ffn(x, gate, up, down)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = scao_amd.gated_ffn(x, gate, up, down)
    for i in range(3):
        x.copy_(_normal(hip_device, 90 + i, tokens, 264, torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, scao_amd.gated_ffn(x, gate, up, down))


def test_module(hip_device):
    for packed in (False, True):
        m = scao_amd.GatedFFN(64, 96, "gelu", packed, device=hip_device, dtype=torch.bfloat16)
        x = _normal(hip_device, 1, 20, 64, torch.bfloat16)
        gate, up = m.gate_up.split(96) if packed else (m.gate, m.up)
        y = m(x)
        assert torch.equal(y, scao_amd.gated_ffn(x, gate, up, m.down, "gelu"))
        y.float().sum().backward()
        assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in m.parameters())
        assert sorted(m.state_dict()) == (["down", "gate_up"] if packed else ["down", "gate", "up"])
        assert len(set(map(tuple, [p.shape for p in m.parameters()]))) == 2


def test_refusals(hip_device):
    x, gate, up, down, _ = _inputs(hip_device, 4, 16, 24, torch.bfloat16)
    ffn = scao_amd.gated_ffn
    with pytest.raises(ValueError, match="activation"):
        ffn(x, gate, up, down, "tanh")
    with pytest.raises(ValueError, match="shape mismatch"):
        ffn(x, gate, up[:-1], down)
    with pytest.raises(ValueError, match="shape mismatch"):
        ffn(x[:, :-1], gate, up, down)
    with pytest.raises(ValueError, match="shape mismatch"):
        ffn(x, gate, up, down.t())
    with pytest.raises(ValueError):
        ffn(x, gate[0], up, down)
    with pytest.raises(TypeError):
        ffn(x.float(), gate, up, down)
    with pytest.raises(TypeError):
        ffn(x.double(), gate.double(), up.double(), down.double())
    with pytest.raises(RuntimeError, match="x is on 'cpu'"):
        ffn(x.cpu(), gate.cpu(), up.cpu(), down.cpu())
    with pytest.raises(RuntimeError):   # differentiable once
        leaf = x.detach().requires_grad_()
        (g,) = torch.autograd.grad(ffn(leaf, gate, up, down).float().sum(), leaf,
                                   create_graph=True)
        g.float().sum().backward()
