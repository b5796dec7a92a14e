"""What ops.softmax_loss holds its sums and weights in, where a plain 32-bit form would keep its digits.

The bounds are those of the formula in 64 bits with each rounding counted: a logit of half-type tables is a sum
of exact products in fp32, off by at most (d + 16) 2^-24 of its terms' magnitudes A_b (d additions, the scale, the
exponent's own fma); a weight is then off by e = 2 (that) + 2^-20 (exp2) + n 2^-24 relative, n the longest chain
of additions.
"""
import pytest
import torch

from igr import ops

pytestmark = pytest.mark.gpu
DEV = 'cuda'
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def reference(x, w, t):
    """(loss per row, dx, dw of their sum, magnitudes of dx's and dw's terms, A) in 64 bits."""
    X, W = x.detach().double(), w.detach().double()
    s = X.matmul(W.t())
    lse = torch.logsumexp(s, 1, keepdim=True)
    p = (s - lse).exp()
    hot = torch.zeros_like(p)
    hot[torch.arange(len(t), device=x.device), t] = 1.0
    a = X.abs().matmul(W.abs().t()).amax(1)
    g = (p - hot)
    return (lse[:, 0] - s.gather(1, t[:, None])[:, 0], g.matmul(W), g.t().contiguous().matmul(X), (p + hot).matmul(W.abs()),
            (p + hot).t().contiguous().matmul(X.abs()), a)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('B,V,d', [(64, 40, 16), (200, 300, 16), (40, 50, 200), (300, 90, 100)])
def test_half_type_gradients_are_rounded_once(B, V, d, dtype):
    """The gradients of half types are sums of weights held to twice the type's digits (a pair: half a step of
    the rest, 2^-16 for bf16, 2^-22 for fp16), rounded once at the end.  Few items share a row's weight
    here, so a weight rounded to the type itself would show in the small entries of the gradient."""
    gen = torch.Generator(device=DEV).manual_seed(B + V + d)
    std = (2.0 / d ** 0.5) ** 0.5
    x = (std * torch.randn(B, d, generator=gen, device=DEV)).to(dtype).requires_grad_()
    w = (std * torch.randn(V, d, generator=gen, device=DEV)).to(dtype).requires_grad_()
    t = torch.randint(0, V, (B,), generator=gen, device=DEV)
    dx, dw = torch.autograd.grad(ops.softmax_loss(x, w, t, reduction='sum'), (x, w))
    _, rx, rw, mx, mw, a = reference(x, w, t)
    half = HALF[dtype]
    e = 2 * (d + 16) * 2.0 ** -24 * a + 2.0 ** -20 + (65 + max(B, V) // 32) * 2.0 ** -24 + half * half
    floor = 2.0 ** -37 * max(V, B) * float(torch.maximum(x.detach().abs().max(), w.detach().abs().max()))
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-37
    assert ((dx.double() - rx).abs() <= e[:, None] * mx + half * rx.abs() + floor + tiny).all()
    assert ((dw.double() - rw).abs() <= e.max() * mw + half * rw.abs() + floor + tiny).all()
