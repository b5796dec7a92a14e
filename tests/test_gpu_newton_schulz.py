"""ops.newton_schulz against the iteration in 64 bits.

Bound.  Matrices are held within 2^-23 of a value plus half of 2^-35, products lose 2^-21 of the terms'
magnitudes (the pairs, the product left out, fp32 sums of up to K terms in random order:
sqrt(K) 2^-24), so a step leaves an error of at most u = (2^-21 + sqrt(K) 2^-23) |q| |X| in the Frobenius
norm, |X|_F <= 1.2 sqrt(S), |q| <= a + |b| + |c| in the 2-norm.  The next steps multiply it by at most the
iteration's slope, a = 3.4445 (its largest, at 0).  Summed over five steps: u (1 + 3.4445 + ... + 3.4445^4)
< 200 u in the Frobenius norm; X's own norm then is about sqrt(S), so relative to it 200 * 1.2 * 10.3 * (2^-21 +
sqrt(K) 2^-23).  That worst case is far from what happens (slope a only for vanishing singular values, whose
errors are as small); the tests hold the kernels to a tenth of it.  Half types add half a step of the value.
"""
import pytest
import torch

from igr import ops
from igr._lib import IgrError

pytestmark = pytest.mark.gpu
DEV = 'cuda'
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
COEFFS = (3.4445, -4.7750, 2.0315)


def formula(g, steps=5, coeffs=COEFFS, eps=1e-7):
    a, b, c = coeffs
    x = g.double()
    x = x / (x.square().sum().sqrt() + eps)
    flip = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if flip else x
    for _ in range(steps):
        y = x.matmul(x.t())
        x = a * x + (b * y + c * y.matmul(y)).matmul(x)
    return x.t() if flip else x


def check(g, **kw):
    y = ops.newton_schulz(g, **kw)
    assert y.dtype == g.dtype and y.shape == g.shape and y.is_contiguous()
    for yy, gg in zip(y if g.dim() == 3 else [y], g if g.dim() == 3 else [g]):
        ref = formula(gg, **kw)
        k = max(gg.shape)
        u = 0.1 * 200 * 1.2 * 10.3 * (2.0 ** -21 + k ** 0.5 * 2.0 ** -23)
        norm = float(ref.square().sum().sqrt())
        err = float((yy.double() - ref).square().sum().sqrt())
        assert err <= (u + HALF[g.dtype]) * norm + 1e-12, (err / norm, u)
    return y


def weight(b, r, c, seed=0, scale=1e-3):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    k = min(8, r, c)
    n = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    return scale * (n(b, r, c) + 0.3 * torch.bmm(n(b, r, k), n(b, k, c)))


SHAPES = [(1, 1, 1), (2, 1, 9), (1, 7, 3), (6, 64, 64), (3, 64, 33), (2, 5, 128), (1, 64, 129), (2, 256, 64), (1, 33, 256),
          (1, 64, 257), (2, 65, 64), (1, 65, 65), (2, 200, 520), (1, 520, 200), (1, 16, 4000), (1, 1000, 130),
          (1, 1100, 1030), (3, 700, 900), (1, 1030, 3001), (2, 1500, 1100), (1, 2304, 2304), (9, 300, 700), (1, 40981, 64),
          (2, 33, 9000), (1, 20000, 100), (1, 300000, 8)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('b,r,c', SHAPES)
def test_matches_the_iteration(b, r, c, dtype):
    check(weight(b, r, c, seed=r + c).to(dtype))


def test_two_dimensional_and_other_settings():
    g = weight(1, 96, 160)[0]
    check(g)
    check(g, steps=1)
    check(g, steps=9)
    check(g, coeffs=(1.5, -0.5, 0.0))       # the cubic iteration
    check(g, coeffs=(1.875, -1.25, 0.375))  # the quintic that converges to 1
    check(g, eps=1e-3)
    check(weight(2, 40, 50), steps=2, coeffs=(1.5, -0.5, 0.0))


def test_converged_iteration_is_orthogonal():
    g = torch.randn(300, 400, device=DEV)
    y = ops.newton_schulz(g, steps=40, coeffs=(1.875, -1.25, 0.375)).double()
    assert (y.matmul(y.t()) - torch.eye(300, device=DEV, dtype=torch.float64)).abs().max() < 1e-4


@pytest.mark.parametrize('r,c', [(64, 64), (200, 300)])
def test_scales_of_the_input(r, c):
    """Normalised first: any power of two that fp32 holds, and far apart entries."""
    g = weight(1, r, c, scale=1.0)[0]
    base = check(g, eps=0.0)
    for e in (-120, -40, 40, 120):
        v = g * 2.0 ** e
        y = check(v, eps=0.0)
        # entries below 2^-6 lose bits to fp32's subnormals at 2^-120; where none did, the same bits
        if torch.equal(v * 2.0 ** -e, g):
            assert torch.equal(y, base)
        else:
            assert e == -120
    g[0] *= 1e6
    check(g)


@pytest.mark.parametrize('r,c', [(60, 100), (150, 90)])
def test_zero_and_non_finite_matrices_of_a_batch(r, c):
    g = weight(4, r, c)
    g[1] = 0
    g[2, 3, 4] = float('nan')
    g[3, 0, 0] = float('inf')
    y = ops.newton_schulz(g)
    assert not y[1].any() and torch.isnan(y[2]).all() and torch.isnan(y[3]).any()
    assert torch.equal(y[0], ops.newton_schulz(g[0]))


@pytest.mark.parametrize('dtype', TYPES)
def test_strides(dtype):
    base = weight(3, 170, 190).to(dtype)
    for v in (base[:, 1:60, 3:120], base[:, ::2, 5:100], base.transpose(1, 2), base[:, :, ::3], base[0], base[:1].expand(3, 170, 190),
              base[0, :100, :64], base[::2]):
        assert torch.equal(ops.newton_schulz(v), ops.newton_schulz(v.contiguous()))
    check(base[:, 1:60, 3:120])


def test_transposed_input_gives_the_transposed_result():
    for r, c in ((48, 200), (130, 300)):
        g = weight(1, r, c)[0]
        assert torch.equal(ops.newton_schulz(g.t().contiguous()).t(), ops.newton_schulz(g))


def test_empty():
    assert ops.newton_schulz(torch.zeros(0, 5, 6, device=DEV)).shape == (0, 5, 6)
    assert ops.newton_schulz(torch.zeros(0, 6, device=DEV)).shape == (0, 6)


@pytest.mark.parametrize('b,r,c', [(6, 64, 64), (1, 200, 300)])
def test_captured_and_on_another_stream(b, r, c):
    g = weight(b, r, c)
    ref = ops.newton_schulz(g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(ops.newton_schulz(g), ref)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.newton_schulz(g)
    for _ in range(3):
        g.add_(torch.randn_like(g) * 1e-3)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.newton_schulz(g))


def test_refusals():
    g = torch.zeros(3, 4, device=DEV)
    with pytest.raises(IgrError, match='float32'):
        ops.newton_schulz(g.double())
    with pytest.raises(IgrError, match='batch'):
        ops.newton_schulz(g[0])
    with pytest.raises(IgrError, match='steps'):
        ops.newton_schulz(g, steps=0)
    with pytest.raises(IgrError, match='coefficients'):
        ops.newton_schulz(g, coeffs=(3.0, 1.0, 1.0))
    with pytest.raises(IgrError, match='three'):
        ops.newton_schulz(g, coeffs=(3.0, 1.0))
    with pytest.raises(IgrError, match='eps'):
        ops.newton_schulz(g, eps=-1.0)
