"""ops.quantize_rows and ops.gemm_int8 at the ends of what a launch holds."""
import pytest
import torch

from igr import ops

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def test_more_rows_than_a_dimension_of_a_launch_has_threads():
    """A wave a row and 2^26 rows: 2^32 threads and more (17 GB of rows)."""
    n, k = (1 << 26) + 9, 129
    x = torch.zeros(n, k, dtype=torch.bfloat16, device=DEV)
    x[-5:] = torch.randn(5, k, device=DEV).to(torch.bfloat16)
    q, s = ops.quantize_rows(x)
    a = x[-5:].float().abs().amax(1)
    assert torch.equal(s[-5:], a / 127)
    assert torch.equal(q[-5:], torch.round(x[-5:].float() / a[:, None] * 127).to(torch.int8))
    assert not s[:-5].any() and not q[:1000].any() and not q[-1000:-5].any()
