"""ops.newton_schulz at inputs where its normalisation or its products could go wrong."""
import pytest
import torch

from igr import ops
from test_pair_products import iterate, momentum, near_enough, off_by

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
