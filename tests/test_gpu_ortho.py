"""Orthogonalised updates (scao_orthogonalize) against their definition in 64
bits; bounds: tests/ortho_reference.py.  The classical coefficients (cubic and
quintic) enlarge errors little, so that their bounds are near the roundings; the
default ones are tested by the wider bound that their slopes give."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import scao_amd
from scao_amd import _lib as L
from tests.ortho_reference import CUBIC, QUINTIC, ULP, bound, orthogonalize, triples

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _update(dev, seed, m, n, dtype, pad=0, skip=0):
    """noise and a few strong directions, in rows of n + pad from element skip on"""
    g = torch.Generator(device=dev).manual_seed(seed)
    t = torch.randn(m, n, generator=g, device=dev)
    t += torch.randn(m, 2, generator=g, device=dev) @ torch.randn(2, n, generator=g, device=dev) * (
        (m + n) / (m * n)) ** 0.5
    flat = torch.zeros(m * (n + pad) + skip, device=dev)
    rows = flat[skip:].view(m, n + pad)
    rows[:, :n] = t * 1e-3
    if pad:
        rows[:, n:] = 1e4   # not to be read
    return flat.to(dtype)[skip:].view(m, n + pad)[:, :n]


def _check(got, g, coefficients, precision, what):
    want = orthogonalize(g, coefficients)
    room = bound(g, coefficients, precision) + ULP[got.dtype] * float(want.norm()) + 1e-30
    err = float((got.double() - want).norm())
    print(f"{what} {tuple(g.shape)} {g.dtype}: {err / room:.3f} of the bound, "
          f"rel {err / max(float(want.norm()), 1e-30):.2e}", flush=True)
    assert got.shape == g.shape and err <= room, (what, err, room)


SIZES = [(1, 1), (1, 7), (5, 1), (2, 2), (7, 5), (8, 8), (16, 64), (33, 31), (64, 64), (63, 257),
         (129, 65), (128, 128), (130, 500), (256, 256), (257, 264), (333, 1001), (1001, 333),
         (512, 2048), (700, 520), (1025, 129), (2049, 77)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", SIZES)
def test_sizes(hip_device, m, n, dtype):
    g = _update(hip_device, m + n, m, n, dtype)
    co = triples(QUINTIC, 2)
    _check(scao_amd.orthogonalize(g, steps=2, coefficients=QUINTIC), g, co,
           "fast" if dtype == torch.bfloat16 else "fp32", "quintic")
    got = scao_amd.orthogonalize(g, steps=1, coefficients=CUBIC, dtype=torch.bfloat16)
    assert got.dtype == torch.bfloat16
    _check(got, g, triples(CUBIC, 1), "fast", "cubic")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", [(96, 160), (300, 200), (512, 1024)])
def test_default_coefficients(hip_device, m, n, dtype):
    g = _update(hip_device, 3, m, n, dtype)
    co = triples(scao_amd.ortho.NS_COEFFICIENTS, 5)
    got = scao_amd.orthogonalize(g)
    _check(got, g, co, "fast" if dtype == torch.bfloat16 else "fp32", "default")
    if dtype != torch.bfloat16:   # to within a few roundings of a plain form in 32 bits
        plain = g.float()
        plain = plain / (plain.norm() + 1e-7)
        for a, b, c in co:
            gram = plain @ plain.t() if m <= n else plain.t() @ plain
            f = b * gram + c * (gram @ gram)
            plain = a * plain + (f @ plain if m <= n else plain @ f)
        want = orthogonalize(g, co)
        own, other = (float((t.double() - want).norm() / want.norm()) for t in (got, plain))
        print(f"error {own:.2e}, plain form's {other:.2e}", flush=True)
        # (fp16 results: half an ulp evenly spread)
        assert own <= 4 * other + (2.0 ** -11 / 3 ** 0.5 if dtype == torch.float16 else 0)


def _hadamard(k, dev):
    h = torch.ones(1, 1, device=dev)
    for _ in range(k):
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)])
    return h


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [64, 256, 1024])
def test_exact_where_every_word_is(hip_device, rows, dtype):
    """Rows of a Hadamard matrix in any order: X = G / (32 sqrt(rows)) is a power of
    two everywhere, A = 1 / rows on the diagonal and zero beside it, and B = 1.5 -
    0.5 / rows needs 8, 10 or 12 bits.  So with one step every element is exact, at
    its place, but for 12 bits in words of 11."""
    g = torch.Generator().manual_seed(rows)
    h = _hadamard(10, hip_device)[torch.randperm(1024, generator=g)[:rows].to(hip_device)]
    s = rows ** -0.5   # every singular value
    want = 1.5 * s - 0.5 * s ** 3
    for update in (h, h.t().contiguous()):
        got = scao_amd.orthogonalize(update.to(dtype), steps=1, coefficients=CUBIC, eps=1e-30)
        if rows < 1024 or dtype != torch.bfloat16:
            assert torch.equal(got, (update * (want / 32)).to(dtype))
        # A second step of other coefficients.  Its A is s1^2 with up to 30 bits, so it,
        # B and the result are rounded: A and B to words of 11 or 22 bits, w = 2^-11 or
        # 2^-22 of each, A's error entering B = 1.5 - 0.5 A times 0.5 A / B < 1; X1 and
        # the first step's B likewise, w each; the result to its type.
        co = [(2.0, -1.0, 0.5), (1.5, -0.5, 0.0)]
        s2 = s
        for a, b, c in co:
            s2 = a * s2 + b * s2 ** 3 + c * s2 ** 5
        got = scao_amd.orthogonalize(update.to(dtype), steps=2, coefficients=co, eps=1e-30)
        w = 2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -22
        exact = update.double() * (s2 / 32)
        assert bool(((got.double() - exact).abs() <= exact.abs() * (4 * w + ULP[dtype])).all())


def _call(mats, dst, precision, coefficients, eps=1e-7):
    table = np.zeros(len(mats), dtype=L.ORTHO_DESC)
    for i, (s, d) in enumerate(zip(mats, dst)):
        table[i] = (s.data_ptr(), d.data_ptr(), *s.shape, s.stride(0), d.stride(0),
                    L.DTYPE_CODE[s.dtype], L.DTYPE_CODE[d.dtype], precision, 0)
    co = np.array(coefficients, dtype=np.float64).reshape(-1)
    steps, at = len(coefficients), table.ctypes.data
    ws = torch.empty(L.lib().scao_orthogonalize_workspace(at, len(mats), steps),
                     dtype=torch.uint8, device=mats[0].device)
    ws.fill_(0xff)   # NaN in any word
    L.call("scao_orthogonalize", at, len(mats), co.ctypes.data, steps, ctypes.c_double(eps),
           ws.data_ptr(), L.stream_ptr(mats[0].device))


@pytest.mark.parametrize("precision", ["fast", "fp32"])
def test_many_shapes_types_and_strides_in_one_call(hip_device, precision):
    """More shapes than a launch holds, more matrices than a pass holds; results
    in wider rows keep what is beside them."""
    shapes = [(3 + 5 * i, 200 - 9 * i) for i in range(20)] + [(40, 72)] * 70 + [(300, 40)] * 3
    mats, dst = [], []
    for i, (m, n) in enumerate(shapes):
        pad, skip = (0, 3, 8)[i % 3], (0, 1, 5, 8)[i % 4]
        mats.append(_update(hip_device, i, m, n, TYPES[i % 3], pad, skip))
        dst.append(torch.full((m, n + i % 2 * 5), 7.0, device=hip_device)[:, :n])
    co = triples(QUINTIC, 2)
    _call(mats, dst, L.ORTHO_FAST if precision == "fast" else L.ORTHO_FP32, co)
    for i, (g, d) in enumerate(zip(mats, dst)):
        if i < 24 or i % 13 == 0:
            _check(d, g, co, precision, f"matrix {i}")
        if d.stride(0) > d.shape[1]:
            whole = d.as_strided((d.shape[0], d.stride(0)), (d.stride(0), 1))
            assert bool((whole[:, d.shape[1]:] == 7.0).all())
    single = torch.empty_like(dst[0])
    _call(mats[:1], [single], L.ORTHO_FAST if precision == "fast" else L.ORTHO_FP32, co)
    # company may cut a matrix's sums differently, which changes their rounding alone
    assert float((single - dst[0]).norm()) <= 2 * bound(mats[0], co, precision)


# Sizes whose steps go by panels: sides just behind a multiple of 16 and 32, one to
# four blocks of columns a wave, all pieces kept or not, and several shapes at once.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shapes", [
    [(129, 129)], [(256, 256)], [(241, 255)], [(257, 225)], [(160, 900)], [(1000, 145)],
    [(384, 384)], [(256, 512)], [(513, 256)], [(512, 512)], [(300, 449)] * 3,
    [(200, 256)] * 17, [(384, 300), (150, 150), (150, 150), (100, 400), (401, 140)]])
def test_panels(hip_device, shapes, dtype):
    mats = [_update(hip_device, i, m, n, dtype, i % 3, i % 2) for i, (m, n) in enumerate(shapes)]
    precision = "fast" if dtype == torch.bfloat16 else "fp32"
    for co in (triples(QUINTIC, 3), triples((3.4445, -4.7750, 2.0315), 2), triples(CUBIC, 1)):
        dst = [torch.full((m, n + 3), 7.0, device=hip_device)[:, :n] for m, n in shapes]
        _call(mats, dst, L.ORTHO_FAST if precision == "fast" else L.ORTHO_FP32, co)
        for i in {0, len(mats) // 2, len(mats) - 1}:
            _check(dst[i], mats[i], co, precision, f"matrix {i}")
        assert all(bool((d.as_strided((d.shape[0], 3), (d.stride(0), 1), d.shape[1]) == 7.0).all())
                   for d in dst)


def test_many_of_128_rows(hip_device):
    """17 of them are a workgroup's each, 16 go by panels."""
    for dtype, precision in ((torch.float32, "fp32"), (torch.bfloat16, "fast")):
        mats = [_update(hip_device, i, *((128, 128), (100, 120), (121, 97))[i % 3], dtype)
                for i in range(17)]
        for n in (17, 16):
            got = scao_amd.orthogonalize(mats[:n], steps=3, coefficients=QUINTIC)
            for i in range(5):
                _check(got[i], mats[i], triples(QUINTIC, 3), precision, f"{n} of")


def test_panels_of_nan_and_zeros(hip_device):
    for dtype in TYPES:
        mats = [_update(hip_device, i, 300, 200, dtype) for i in range(4)]
        alone = scao_amd.orthogonalize(mats)
        bad = [t.clone() for t in mats]
        bad[1][299, 199] = float("nan")
        bad[2].zero_()
        got = scao_amd.orthogonalize(bad)
        assert torch.equal(got[0], alone[0]) and torch.equal(got[3], alone[3])
        assert bool(got[1].isnan().all()) and bool((got[2] == 0).all())


@pytest.mark.parametrize("m,n", [(256, 256), (300, 160)])
def test_panels_with_strong_growth(hip_device, m, n):
    """Singular values that the first step takes far up and the second far down."""
    g = _update(hip_device, 9, m, n, torch.float32)
    co = [(30.0, 0.0, 0.0), (1.0 / 16, 2.0 ** -14, 2.0 ** -24), (0.5, 0.125, 0.0)]
    for dtype, precision in ((torch.float32, "fp32"), (torch.bfloat16, "fast")):
        got = scao_amd.orthogonalize(g, steps=3, coefficients=co, dtype=dtype)
        _check(got, g, co, precision, "growth")


# sizes whose products take 256 x 256 tiles, tiles in parts, and both
@pytest.mark.parametrize("m,n,many", [(2048, 2048, 1), (2048, 2048, 3), (4096, 512, 2),
                                      (1030, 4100, 2), (4100, 1030, 2), (640, 640, 30)])
def test_large(hip_device, m, n, many):
    g = torch.stack([_update(hip_device, i, m, n, torch.bfloat16) for i in range(many)])
    co = triples(QUINTIC, 2)
    for dtype, precision in ((torch.bfloat16, "fast"), (torch.float32, "fp32")):
        got = scao_amd.orthogonalize(g, steps=2, coefficients=QUINTIC, dtype=dtype)
        for i in {0, many - 1}:
            _check(got[i], g[i], co, precision, f"{many} of")


def test_the_same_call_gives_the_same_bits(hip_device):
    mats = [_update(hip_device, i, m, n, torch.float32) for i, (m, n) in
            enumerate([(300, 500), (1000, 700), (64, 2000)])]
    first = scao_amd.orthogonalize(mats)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, scao_amd.orthogonalize(mats)))


@pytest.mark.parametrize("dtype", TYPES)
def test_nan_infinity_zeros_and_extremes(hip_device, dtype):
    good = [_update(hip_device, i, 70, 130, dtype) for i in range(5)]
    alone = scao_amd.orthogonalize(good)
    bad = [t.clone() for t in good]
    bad[1][69, 129] = float("nan")
    bad[2][0, 0] = float("inf")
    bad[3].zero_()
    got = scao_amd.orthogonalize(bad)
    assert torch.equal(got[0], alone[0]) and torch.equal(got[4], alone[4])
    assert bool(got[1].isnan().all()) and bool(got[2].isnan().all()) and bool((got[3] == 0).all())
    # sums of squares beyond float32's range, both ways
    big, small = (torch.finfo(dtype).max / 8, 1e-20 if dtype != torch.float16 else 1e-6)
    for scale in (big, small):
        unit = torch.randn(70, 130, device=hip_device).clamp_(-4, 4).to(dtype)
        g = (unit.double() * (scale / 4)).to(dtype)
        got = scao_amd.orthogonalize(g, steps=2, coefficients=QUINTIC, eps=1e-30)
        want = orthogonalize(g, triples(QUINTIC, 2), eps=1e-30)
        rel = float((got.double() - want).norm() / want.norm())
        assert rel <= 2 * ULP[dtype] if dtype != torch.float32 else rel <= 1e-5


def test_the_smallest_and_a_large_eps(hip_device):
    z = torch.zeros(300, 200, device=hip_device)
    for dtype in (torch.bfloat16, torch.float32):
        assert bool((scao_amd.orthogonalize(z, eps=1e-300, dtype=dtype) == 0).all())
    assert bool((scao_amd.orthogonalize(z[:30, :40], eps=1e-300) == 0).all())
    # a norm of 3 beside an eps of 200
    g = _update(hip_device, 4, 300, 200, torch.float32)
    g = g * (3.0 / g.norm())
    co = triples(QUINTIC, 2)
    want = orthogonalize(g, co, eps=200.0)
    got = scao_amd.orthogonalize(g, steps=2, coefficients=QUINTIC, eps=200.0)
    # X to 2^-39 an element, times 1.875 a step
    room = bound(g, co, "fp32", eps=200.0) + 4 * 2.0 ** -39 * g.numel() ** 0.5
    assert float((got.double() - want).norm()) <= room


def test_low_rank_and_a_single_direction(hip_device):
    """A rank-one update: one singular value, the others zero throughout."""
    u = torch.randn(200, 1, device=hip_device)
    v = torch.randn(1, 300, device=hip_device)
    g = u @ v
    for dtype, tol in ((torch.float32, 1e-5), (torch.bfloat16, 2.0 ** -7)):
        got = scao_amd.orthogonalize(g, steps=3, coefficients=QUINTIC, dtype=dtype).double()
        want = (u / u.norm()).double() @ (v / v.norm()).double()   # p(1) = 1
        assert float((got - want).norm()) <= tol


def test_layouts(hip_device):
    """Stacks with gaps, a transposed matrix, an expanded one, a single column."""
    g = _update(hip_device, 5, 6 * 40, 90, torch.float32).reshape(2, 3, 40, 90)
    got = scao_amd.orthogonalize(g.transpose(0, 1)[1:, :, 3:, 5:])
    assert got.is_contiguous()
    want = scao_amd.orthogonalize([g[j, i, 3:, 5:].contiguous() for i in (1, 2) for j in (0, 1)])
    assert torch.equal(got.flatten(0, 1), torch.stack(want))
    t = g[0, 0].t()
    assert torch.equal(scao_amd.orthogonalize(t), scao_amd.orthogonalize(t.contiguous()))
    e = g[0, 0, :1].expand(50, 90)
    assert torch.equal(scao_amd.orthogonalize(e), scao_amd.orthogonalize(e.contiguous()))
    c = g[0, 0, :, 4:5]
    assert torch.equal(scao_amd.orthogonalize(c), scao_amd.orthogonalize(c.contiguous()))
    neg = torch._neg_view(g[0, 0])
    assert torch.equal(scao_amd.orthogonalize(neg), scao_amd.orthogonalize(-g[0, 0]))


def test_empty(hip_device):
    z = scao_amd.orthogonalize([torch.empty(0, 5, device=hip_device),
                                torch.empty(3, 0, 4, device=hip_device),
                                torch.eye(4, device=hip_device)])
    assert z[0].shape == (0, 5) and z[1].shape == (3, 0, 4) and z[2].shape == (4, 4)
    assert scao_amd.orthogonalize([]) == []
    assert scao_amd.orthogonalize(torch.empty(0, 8, 8, device=hip_device)).shape == (0, 8, 8)


def test_captured_and_on_another_stream(hip_device):
    mats = [_update(hip_device, i, 200, 300, torch.bfloat16) for i in range(3)]
    want = scao_amd.orthogonalize(mats)
    side = torch.cuda.Stream(hip_device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = scao_amd.orthogonalize(mats)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = scao_amd.orthogonalize(mats)
    for k in range(3):
        for i, t in enumerate(mats):
            t.copy_(_update(hip_device, 10 * k + i, 200, 300, torch.bfloat16))
        graph.replay()
        eager = scao_amd.orthogonalize(mats)
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_refusals(hip_device):
    g = torch.randn(8, 8, device=hip_device)
    with pytest.raises(NotImplementedError):
        scao_amd.orthogonalize(g.clone().requires_grad_())
    with torch.no_grad():
        scao_amd.orthogonalize(g.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="1024"):
        scao_amd.orthogonalize(g, coefficients=(40.0, 0.0, 0.0))
    with pytest.raises(TypeError):
        scao_amd.orthogonalize(g.double())
    with pytest.raises(TypeError):
        scao_amd.orthogonalize(g, dtype=torch.float64)
    with pytest.raises(ValueError):
        scao_amd.orthogonalize(g[0])
