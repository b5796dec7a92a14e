"""ops.newton_schulz at inputs where its normalisation or its products could go wrong."""
import pytest
import torch

from igr import ops
from test_pair_products import FLOOR, TIMES, iterate, momentum, near_enough, off_by

pytestmark = pytest.mark.gpu
DEV = 'cuda'


@pytest.mark.parametrize('r,c', [(3, 4), (60, 100), (150, 90), (600, 800)])
@pytest.mark.parametrize('eps', [0.0, 5e-324, 1e-310])
def test_zeros_stay_zeros_whatever_eps_is(r, c, eps):
    g = torch.zeros(3, r, c, device=DEV)
    g[1] = torch.randn(r, c, device=DEV)
    y = ops.newton_schulz(g, eps=eps)
    assert not y[0].any() and not y[2].any()
    # tiles, and with them the order of sums, go by the whole batch: alone the matrix may come out with other bits, each
    # within u of the iteration's in the Frobenius norm (the bound of the tests against 64 bits)
    u = 0.1 * 200 * 1.2 * 10.3 * (2.0 ** -21 + max(r, c) ** 0.5 * 2.0 ** -23)
    alone = ops.newton_schulz(g[1], eps=eps)
    assert torch.isfinite(y[1]).all() and (y[1] - alone).norm() <= 2 * u * alone.norm()
    g[1] = 0
    g[1, 2, 3] = 1e-45   # the smallest there is
    y = ops.newton_schulz(g, eps=eps)
    assert not y[0].any() and torch.isfinite(y[1]).all() and 0.6 < float(y[1, 2, 3]) < 1.3


SHAPES = [(1, 1), (1, 9), (7, 3), (64, 64), (64, 33), (5, 128), (64, 129), (256, 64), (33, 256), (64, 257), (65, 64), (65, 65),
          (200, 520), (520, 200), (16, 4000), (1000, 130), (1100, 1030), (700, 900), (1030, 3001), (1500, 1100), (2304, 2304),
          (300, 700), (40981, 64), (33, 9000), (20000, 100), (300000, 8)]


@pytest.mark.parametrize('r,c', SHAPES)
def test_as_near_as_pairs_of_halves_come(r, c):
    """Within the bound that tells them from less (test_pair_products)."""
    g = momentum(r, c).to(DEV)
    y = ops.newton_schulz(g)
    plain, exact = iterate(g, torch.float32), iterate(g, torch.float64)
    assert near_enough(y, plain, exact), (off_by(y, exact), off_by(plain, exact))
    print('off by %.3g, plain %.3g' % (off_by(y, exact), off_by(plain, exact)))


@pytest.mark.parametrize('r,c', [(64, 64), (1, 300), (5, 128), (200, 520), (1030, 300), (1500, 1600)])
@pytest.mark.parametrize('size', [1e-3, 1e-7, 1e-12, 1e-20, 1e-32])
def test_matrices_far_below_eps_keep_their_digits(r, c, size):
    """|G| below eps: X starts small and stays so for some steps.  The plain fp32 form holds it relative to itself."""
    g = momentum(r, c).to(DEV)
    g = g * (size * 1e-7 / g.norm())
    for steps in (1, 5, 12):
        y = ops.newton_schulz(g, steps=steps)
        plain, exact = iterate(g, torch.float32, steps=steps), iterate(g, torch.float64, steps=steps)
        if float(exact.abs().max()) < 1e-30:   # near fp32's own subnormals: in steps of these
            assert (y.double() - exact).abs().max() <= 2.0 ** -149 + 1e-5 * float(exact.abs().max())
        else:
            # one row has one singular value, whose errors no others average: three products a step, each off by up to
            # 2^-21, are 2^-20 in the 5 steps that the bound is made for if half of them cancel, 12 / 5 of it in 12
            assert off_by(y, exact) <= TIMES * off_by(plain, exact) + FLOOR * max(steps, 5) / 5, (steps, off_by(y, exact))


@pytest.mark.parametrize('coeffs', [(1.5, -0.5, 0.0), (1.875, -1.25, 0.375), (0.5, 0.2, 0.1), (2.0, -1.5, 0.5)])
def test_small_matrices_under_other_coefficients(coeffs):
    for r, c in ((40, 50), (130, 300)):
        g = momentum(r, c).to(DEV)
        for size in (1.0, 1e-9, 1e-17):
            v = g * (size / g.norm())
            for steps in (1, 9, 60):
                y = ops.newton_schulz(v, steps=steps, coeffs=coeffs)
                plain, exact = (iterate(v, t, steps=steps, coeffs=coeffs) for t in (torch.float32, torch.float64))
                if float(exact.abs().max()) > 1e-30:
                    assert near_enough(y, plain, exact), (r, size, steps, off_by(y, exact), off_by(plain, exact))


def test_a_batch_of_sizes_far_apart():
    """Each matrix by its own power, in one launch."""
    for r, c in ((60, 90), (130, 200), (520, 300)):
        g = torch.stack([momentum(r, c).to(DEV) * f for f in (1.0, 1e-14, 1e12, 0.0, 1e-25, 1e-5)])
        y = ops.newton_schulz(g)
        for k in range(len(g)):
            exact = iterate(g[k], torch.float64)
            if k == 3:
                assert not y[k].any()
            else:
                assert near_enough(y[k], iterate(g[k], torch.float32), exact), (r, k)
