"""How near fp32 products from pairs of halves have to come, and that less than the pairs does not (CPU).

The bound: against 64 bits a result is at most 4 times as far off as the plain fp32 form on the same input, in
the 2-norm, and 2^-20.  A pair holds 2^-23 of a value where fp32 holds 2^-24, twice as far for each of two operands,
and the product left out, 2^-22, is as much again as both together; sums are fp32's own.  The 2^-20 is for inputs of few
terms, where the plain form's roundings may be next to none, and for logarithms of up to 24 in
fp32 (a loss's exponents).

The mistakes that a kernel could make without its worst-case bounds noticing - halves without their rests, one
of the three products missing - are planted in a simulation of the products here: each is far outside."""
import pytest
import torch

TIMES, FLOOR = 4.0, 2.0 ** -20
COEFFS = (3.4445, -4.7750, 2.0315)
KINDS = ['halves alone', 'a product missing']


def off_by(y, exact):
    return float((y.double() - exact).norm() / exact.norm().clamp(min=1e-300))


def near_enough(y, plain, exact):
    return off_by(y, exact) <= TIMES * off_by(plain, exact) + FLOOR


def as_pair(x, rows=32):
    """hi and lo of x under a power of two for each `rows` rows (0: the fixed 2^11), in 64 bits."""
    if rows:
        pad = -x.shape[0] % rows
        y = torch.nn.functional.pad(x, (0, 0, 0, pad)).view(-1, rows * x.shape[1])
        s = torch.exp2(14 - y.abs().amax(1, keepdim=True).clamp(min=1e-30).log2().floor())
        s = s.expand(-1, rows).reshape(-1, 1)[:x.shape[0]].double()
    else:
        s = 2.0 ** 11
    hi = (x.double() * s).half().double()
    lo = (x.double() * s - hi).half().double()
    return hi / s, lo / s


def product(a, b, kind):
    """a b^T of two pairs."""
    (ah, al), (bh, bl) = a, b
    r = ah.matmul(bh.t())
    if kind != 'halves alone':
        r = r + al.matmul(bh.t())
    if kind == 'pairs':
        r = r + ah.matmul(bl.t())
    return r.float()


# ------------------------------------------------------------------ Newton-Schulz

def momentum(r, c):
    gen = torch.Generator().manual_seed(r + c)
    k = min(8, r, c)
    n = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return 1e-3 * (n(r, c) + 0.3 * n(r, k).matmul(n(k, c)))


def iterate(g, dtype, mul=None, steps=5, coeffs=COEFFS, eps=1e-7):
    a, b, c = coeffs
    mul = mul or (lambda p, q: p.matmul(q.t()))
    x = (g.double() / (g.double().square().sum().sqrt() + eps)).to(dtype)
    flip = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if flip else x
    for _ in range(steps):
        y = mul(x, x)
        x = a * x + mul(b * y + c * mul(y, y), x.t())
    return x.t() if flip else x


@pytest.mark.parametrize('r,c', [(64, 64), (5, 128), (64, 129), (256, 64), (200, 520), (1000, 130), (700, 900), (20000, 100)])
def test_orthogonalised_matrices_tell_pairs_from_less(r, c):
    g = momentum(r, c)
    exact, plain = iterate(g, torch.float64), iterate(g, torch.float32)
    by = lambda kind: iterate(g, torch.float32, lambda p, q: product(as_pair(p, 0), as_pair(q, 0), kind))  # noqa: E731
    assert near_enough(by('pairs'), plain, exact)
    for kind in KINDS:
        assert off_by(by(kind), exact) > 10 * (TIMES * off_by(plain, exact) + FLOOR), kind


# ------------------------------------------------------------------ softmax loss

def tables(B, V, d):
    gen = torch.Generator().manual_seed(B + V + d)
    std = (2.0 / d ** 0.5) ** 0.5
    r = lambda n: torch.randn(n, d, generator=gen) * std * torch.exp(0.3 * torch.randn(n, 1, generator=gen))  # noqa: E731
    return r(B), r(V), torch.randint(0, V, (B,), generator=gen)


def loss_and_gradients(x, w, t, dtype):
    """The rows' losses and the gradients of their sum in the plain form."""
    x, w = x.detach().to(dtype).requires_grad_(), w.detach().to(dtype).requires_grad_()
    loss = torch.nn.functional.cross_entropy(x.matmul(w.t().contiguous()), t, reduction='none')
    return (loss.detach(),) + torch.autograd.grad(loss.sum(), (x, w))


def simulated(x, w, t, logits='pairs', weights='pairs', sums='pairs'):
    """The same from products of pairs: of the logits, of the weights with the tables' rows."""
    X, W = as_pair(x), as_pair(w)
    s = product(X, W, logits).double()
    lse = torch.logsumexp(s, 1)
    at = torch.arange(len(t))
    p = (s - lse[:, None]).exp()
    p[at, t] = 0.0
    rest = p.sum(1)
    most = p.amax(1, keepdim=True).clamp(min=1e-300)

    def halves(v):
        hi, lo = as_pair((v * 2.0 ** 3).float(), 0)   # weights up to 1 times 2^14
        return hi / 8, (lo * 0 if weights == 'halves alone' else lo) / 8
    wt = tuple(v.t().contiguous() for v in W)
    dx = product(halves(p / most), wt, sums).double() * most - rest[:, None] * w.double()[t]
    p[at, t] = -rest
    dw = product(tuple(v.t() for v in halves(p)), tuple(v.t().contiguous() for v in X), sums)
    return (lse - s[at, t]).float(), dx.float(), dw


@pytest.mark.parametrize('B,V,d', [(3, 5, 7), (33, 31, 64), (129, 1000, 100), (256, 1682, 64), (700, 333, 200), (64, 4097, 256),
                                   (2050, 300, 33), (1, 5000, 129)])
def test_losses_and_gradients_tell_pairs_from_less(B, V, d):
    x, w, t = tables(B, V, d)
    exact, plain = loss_and_gradients(x, w, t, torch.float64), loss_and_gradients(x, w, t, torch.float32)
    for y, p, e in zip(simulated(x, w, t), plain, exact):
        assert near_enough(y, p, e)
    # which of (loss, dx, dw) show a mistake
    for what, shown in ((dict(logits=KINDS[0]), (0, 1, 2)), (dict(logits=KINDS[1]), (0, 1, 2)),
                        (dict(weights=KINDS[0]), (1, 2)), (dict(sums=KINDS[0]), (1, 2)), (dict(sums=KINDS[1]), (1, 2))):
        y = simulated(x, w, t, **what)
        for i in shown:
            assert off_by(y[i], exact[i]) > 2 * (TIMES * off_by(plain[i], exact[i]) + FLOOR), (what, i)
