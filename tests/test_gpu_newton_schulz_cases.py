"""ops.newton_schulz at inputs where its normalisation or its products could go wrong."""
import pytest
import torch

from igr import ops

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
