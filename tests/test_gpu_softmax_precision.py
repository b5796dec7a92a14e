"""What ops.softmax_loss holds its sums and weights in, where a plain 32-bit form would keep its digits.

The bounds are those of the formula in 64 bits with each rounding counted: a logit of half-type tables is a sum
of exact products in fp32, off by at most (d + 16) 2^-24 of its terms' magnitudes A_b (d additions, the scale, the
exponent's own fma); a weight is then off by e = 2 (that) + 2^-20 (exp2) + n 2^-24 relative, n the longest chain
of additions.
"""
import pytest
import torch

from igr import ops
from test_pair_products import loss_and_gradients, near_enough, off_by, tables

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


def pairwise(x, w, t, scale=1.0):
    """As `reference` for fp32 tables, with the errors of each logit by its own terms: (loss, its bound, dx, its bound,
    dw, its bound).  A logit is off by at most d_bv = (3 d + 16) 2^-24 sum_k |x_bk w_vk| (three products a term,
    their rows held to 2^-23 whatever their neighbours are), a weight relative by d_bv, the row's mean of
    these (its log-sum), 2^-20 and n 2^-24.  Below that there is a floor for each term of a gradient: a weight
    times the power of two of its row is held to 2^-37 of the largest of these (of the row's in dx, where a
    block's rows may share an exponent 2^8 above theirs; of the batch's in dw)."""
    X, W = x.detach().double(), w.detach().double()
    s = scale * X.matmul(W.t())
    lse = torch.logsumexp(s, 1, keepdim=True)
    p = (s - lse).exp()
    at = torch.arange(len(t), device=x.device)
    hot = torch.zeros_like(p)
    hot[at, t] = 1.0
    err = (3 * x.shape[1] + 16) * 2.0 ** -24 * scale * X.abs().matmul(W.abs().t())
    mean = torch.where(p > 0, p * err, torch.zeros_like(p)).sum(1, keepdim=True)
    n = 65 + max(x.shape[0], w.shape[0]) // 32
    rel = err + mean + 2.0 ** -20 + n * 2.0 ** -24
    loss = lse[:, 0] - s[at, t]
    el = mean[:, 0] + err[at, t] + n * 2.0 ** -24 + 2.0 ** -22 * (loss.abs() + lse[:, 0].abs() + s[at, t].abs())
    we = torch.where(p > 0, p * rel, torch.zeros_like(p)) + hot * (mean + 2.0 ** -20 + n * 2.0 ** -24)
    top = (p * W.abs().amax(1)).amax(1, keepdim=True)
    dx, dw = scale * (p - hot).matmul(W), scale * (p - hot).t().contiguous().matmul(X)
    ex = scale * (we.matmul(W.abs()) + 2.0 ** -29 * w.shape[0] * top) + 2.0 ** -23 * dx.abs()
    ew = scale * (we.t().contiguous().matmul(X.abs()) + 2.0 ** -37 * len(t) * X.abs().max()) + 2.0 ** -23 * dw.abs()
    return loss, el, dx, ex, dw, ew


def check_rows(x, w, t, scale=1.0, dx_columns=slice(None)):
    x.requires_grad_()
    w.requires_grad_()
    loss = ops.softmax_loss(x, w, t, scale=scale, reduction='none')
    dx, dw = torch.autograd.grad(loss.sum(), (x, w))
    rl, el, rx, ex, rw, ew = pairwise(x, w, t, scale)
    assert ((loss.double() - rl).abs() <= el).all()
    assert ((dx.double() - rx).abs() <= ex + 1e-37)[:, dx_columns].all()
    assert ((dw.double() - rw).abs() <= ew + 1e-37).all()
    with torch.no_grad():
        assert torch.equal(loss, ops.softmax_loss(x, w, t, scale=scale, reduction='none'))


def normal_tables(B, V, d, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    std = (2.0 / d ** 0.5) ** 0.5
    r = lambda n: std * torch.randn(n, d, generator=gen, device=DEV)  # noqa: E731
    return r(B), r(V), torch.randint(0, V, (B,), generator=gen, device=DEV)


@pytest.mark.parametrize('B,V,d', [(70, 300, 33), (200, 1000, 64), (40, 500, 100), (300, 260, 250)])
@pytest.mark.parametrize('low', [-1e4, -1e9, torch.finfo(torch.float32).min])
def test_items_masked_by_a_bias_column_leave_the_others_their_digits(B, V, d, low):
    """A table with a bias column whose masked items hold a very low value, down to the type's lowest: they weigh
    nothing, and the items that lie next to them are scored as if they were not there."""
    x, w, t = normal_tables(B, V, d, B + d)
    x[:, -1] = 1.0
    w[:, -1] = 0.1
    masked = torch.arange(0, V, 7, device=DEV)
    w[masked, -1] = low
    t = torch.where(t % 7 == 0, t + 1, t).clamp_(max=V - 1)
    t[t % 7 == 0] = 1
    check_rows(x, w, t)


@pytest.mark.parametrize('B,V,d', [(70, 300, 33), (200, 1000, 64), (40, 500, 100)])
@pytest.mark.parametrize('up', [9, 15, 25, 40, 100])
def test_large_items_that_weigh_nothing_leave_the_others_their_digits(B, V, d, up):
    """Items 2^up times the others' size in a direction that every batch row points away from: their weight
    is nothing, and the weighted sums of the others hold their digits."""
    x, w, t = normal_tables(B, V, d, B + up)
    x[:, 0] = 1.5
    w[:, 0] = 0.0
    w[5::40] = 0.0
    w[5::40, 0] = -2.0 ** up
    w[6::80, 1] = 2.0 ** (up - 20)     # and some of another size
    w[6::80, 0] = -2.0 ** up
    t[(t % 40 == 5) | (t % 80 == 6)] = 0
    check_rows(x, w, t)


@pytest.mark.parametrize('up', [9, 15, 25])
def test_large_batch_rows_leave_the_others_their_digits(up):
    """Batch rows 2^up times the size of those beside them (at a scale that keeps their logits in range)."""
    x, w, t = normal_tables(150, 400, 48, up)
    x[::13] *= 2.0 ** up
    check_rows(x, w, t, scale=2.0 ** (3 - up) if up > 12 else 1.0)
    x, w, t = normal_tables(150, 400, 48, up + 1)
    x[::13] *= 2.0 ** -up
    w[::11] *= 2.0 ** -up
    check_rows(x, w, t)


def test_items_of_sizes_from_2_to_the_minus_60_to_2_to_the_60():
    """Each row a size of its own, the large ones out of the batch rows' way."""
    x, w, t = normal_tables(90, 640, 40, 3)
    x[:, 0], w[:, 0] = 1.0, 0.0
    e = (torch.arange(640, device=DEV) * 37 % 121 - 60).float()
    w *= torch.exp2(e.clamp(max=0.0))[:, None]
    w[:, 0] = -torch.exp2(e) * (e > 3)
    t = torch.where(e[t] > 3, torch.zeros_like(t), t)
    w[0] = 0.25
    check_rows(x, w, t)


def test_rows_of_their_own_size_in_a_long_table():
    """Enough items for two blocks of them a wave in the backward, both tables with rows far from their neighbours."""
    x, w, t = normal_tables(40, 140_000, 8, 5)
    x[:, -1], w[:, -1] = 1.0, 0.0
    x[::9] *= 2.0 ** -12
    w[17::1000, -1] = -1e9
    t = torch.where(t % 1000 == 17, t + 1, t)
    check_rows(x, w, t)


def test_ignored_rows_and_outside_targets_beside_masked_items():
    x, w, t = normal_tables(100, 200, 24, 6)
    x[:, -1], w[:, -1] = 1.0, 0.0
    w[::5, -1] = -1e9
    t = torch.where(t % 5 == 0, t + 1, t)
    x.requires_grad_()
    w.requires_grad_()
    keep = torch.arange(100, device=DEV) % 3 != 0
    ignored = torch.where(keep, t, torch.full_like(t, -100))
    loss = ops.softmax_loss(x, w, ignored, reduction='none')
    dx, dw = torch.autograd.grad(loss.sum(), (x, w))
    xs, ts = x.detach()[keep], t[keep]
    rl, el, rx, ex, rw, ew = pairwise(xs, w, ts)
    assert ((loss[keep].double() - rl).abs() <= el).all() and not loss[~keep].any()
    assert ((dx[keep].double() - rx).abs() <= ex).all() and not dx[~keep].any()
    assert ((dw.double() - rw).abs() <= ew).all()
    out = t.clone()
    out[7], out[50] = 200, -3
    rows = ops.softmax_loss(x, w, out, reduction='none')
    assert torch.isnan(rows[[7, 50]]).all() and int(torch.isnan(rows).sum()) == 2


def test_blocks_of_zeros_are_even_with_any():
    """Items of zeros (a padding row, a fresh table) have no size that others could differ from."""
    x, w, t = normal_tables(150, 400, 40, 8)
    w[32:96] = 0.0
    w[100] = 0.0
    x[64:96] = 0.0
    check_rows(x, w, t)
    check_rows(torch.zeros_like(x), w.detach().clone(), t)
    check_rows(x.detach().clone(), torch.zeros_like(w), t)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('B', [8192, 8193, 70_000])
def test_gradients_of_long_batches_with_one_for_each_row(B, dtype):
    """The largest coefficient of the batch, which all rows' weights are held against, at any place of a batch that is
    long enough for a pass of its own over them."""
    gen = torch.Generator(device=DEV).manual_seed(B)
    x = (0.5 * torch.randn(B, 16, generator=gen, device=DEV)).to(dtype).requires_grad_()
    w = (0.5 * torch.randn(40, 16, generator=gen, device=DEV)).to(dtype).requires_grad_()
    t = torch.randint(0, 40, (B,), generator=gen, device=DEV)
    X, W = x.detach().double(), w.detach().double()
    p = X.matmul(W.t()).softmax(1)
    p[torch.arange(B, device=DEV), t] -= 1.0
    loss = ops.softmax_loss(x, w, t, reduction='none')
    for at in (0, B // 2, B - 1):
        g = torch.randn(B, generator=gen, device=DEV)
        g[at] = -2.0 ** 20
        dx, dw = torch.autograd.grad(loss, (x, w), g, retain_graph=True)
        c = p * g.double()[:, None]
        rx, rw = c.matmul(W), c.t().contiguous().matmul(X)
        half = HALF[dtype]
        # 2^-15 stands for the sums' and weights' errors as in `reference`, relative to the terms' magnitudes
        assert ((dx.double() - rx).abs() <= 2.0 ** -15 * c.abs().matmul(W.abs()) + half * rx.abs()).all()
        assert ((dw.double() - rw).abs() <= 2.0 ** -15 * c.abs().t().contiguous().matmul(X.abs()) + half * rw.abs()).all()


def test_the_backward_of_a_long_batch_takes_time_in_proportion():
    """A gradient for each of 2^19 rows: a few hundred microseconds of work on 64 items.  (With every workgroup going through
    the whole batch it took over ten times the backward of one gradient for all.)"""
    B = 1 << 19
    x, w = (torch.randn(n, 16, device=DEV, requires_grad=True) for n in (B, 64))
    t = torch.randint(0, 64, (B,), device=DEV)
    took = {}
    for reduction in ('sum', 'none'):
        loss = ops.softmax_loss(x, w, t, reduction=reduction)
        g = torch.ones_like(loss)
        for _ in range(3):
            torch.autograd.grad(loss, (x, w), g, retain_graph=True)
        times = []
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            torch.autograd.grad(loss, (x, w), g, retain_graph=True)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        took[reduction] = sorted(times)[2]
    assert took['none'] < 3 * took['sum'] + 0.2, took


def test_more_batch_rows_than_a_dimension_of_a_launch_has_workgroups():
    """2^24 rows and more (a workgroup of 256 threads a row would pass 2^32 of them): the last ones are there."""
    B, V, d = (1 << 24) + 77, 5, 4
    gen = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(B, d, generator=gen, device=DEV, dtype=torch.bfloat16).requires_grad_()
    w = torch.randn(V, d, generator=gen, device=DEV, dtype=torch.bfloat16).requires_grad_()
    t = torch.randint(0, V, (B,), generator=gen, device=DEV)
    loss = ops.softmax_loss(x, w, t, reduction='none')
    g = torch.zeros(B, device=DEV)
    some = torch.cat([torch.arange(100, device=DEV), torch.arange(B - 200, B, device=DEV)])
    g[some] = 1.0
    dx, dw = torch.autograd.grad(loss, (x, w), g)
    X, W, T = x.detach()[some].double(), w.detach().double(), t[some]
    p = X.matmul(W.t()).log_softmax(1)
    at = torch.arange(len(some), device=DEV)
    assert (loss.detach()[some].double() + p[at, T]).abs().max() < 1e-5
    p = p.exp()
    p[at, T] -= 1.0
    rx, rw = p.matmul(W), p.t().contiguous().matmul(X)
    assert ((dx[some].double() - rx).abs() <= 2.0 ** -8 * rx.abs() + 1e-4 * W.abs().max()).all()
    assert ((dw.double() - rw).abs() <= 2.0 ** -8 * rw.abs() + 1e-4 * p.abs().t().contiguous().matmul(X.abs())).all()
    assert not dx[100:B - 200].any()


@pytest.mark.parametrize('B,V,d', [(3, 5, 7), (32, 32, 32), (33, 31, 64), (31, 33, 65), (129, 1000, 100), (256, 1682, 64),
                                   (100, 70001, 32), (700, 333, 200), (64, 4097, 256), (300, 20000, 256), (2050, 300, 33),
                                   (1, 5000, 129), (5000, 2, 16), (300, 140000, 24)])
def test_as_near_as_pairs_of_halves_come(B, V, d):
    """Losses row by row and both gradients, within the bound that tells pairs from less (test_pair_products)."""
    x, w, t = (v.to(DEV) for v in tables(B, V, d))
    x.requires_grad_()
    w.requires_grad_()
    loss = ops.softmax_loss(x, w, t, reduction='none')
    got = (loss.detach(),) + torch.autograd.grad(loss.sum(), (x, w))
    plain, exact = loss_and_gradients(x, w, t, torch.float32), loss_and_gradients(x, w, t, torch.float64)
    for y, p, e in zip(got, plain, exact):
        print('off by %.3g, plain %.3g' % (off_by(y, e), off_by(p, e)))
        assert near_enough(y, p, e), (off_by(y, e), off_by(p, e))


LOWS = {torch.float32: [-1e5, -1e9, -1e15, -3e38], torch.bfloat16: [-1e5, -1e9, -1e15, -3e38], torch.float16: [-6e4]}


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('B,V,d,lo,hi', [(2, 34, 2, 32, 34), (40, 5000, 24, 1000, 3300), (200, 3000, 64, 64, 2990),
                                         (60, 900, 130, 5, 870)])
def test_a_range_of_masked_items(B, V, d, lo, hi, dtype):
    """Whole stretches of the catalogue masked by a bias column, all that some workgroups see: logits of
    down to -3e38, whose fp32 steps are far above 1."""
    for low in LOWS[dtype]:
        for scale in (0.3, 1.0, 2.0):
            x, w, t = normal_tables(B, V, d, B + V)
            x[:, -1], w[:, -1] = 1.0, 0.0
            w[lo:hi, -1] = low
            t = torch.where((t >= lo) & (t < hi), t % lo, t)
            if dtype == torch.float32:
                check_rows(x, w, t, scale=scale)
                continue
            x, w = x.to(dtype).requires_grad_(), w.to(dtype).requires_grad_()
            loss = ops.softmax_loss(x, w, t, scale=scale, reduction='none')
            dx, dw = torch.autograd.grad(loss.sum(), (x, w))
            rl, el, rx, ex, rw, ew = pairwise(x.detach().float(), w.detach().float(), t, scale)
            half, tiny = HALF[dtype], 2.0 ** -25 if dtype == torch.float16 else 1e-37
            assert ((loss.double() - rl).abs() <= el).all()
            weights = half * half   # as pairs: twice the type's digits, of the terms' magnitudes
            p = (scale * x.detach().double().matmul(w.detach().double().t())).softmax(1)
            p[torch.arange(B, device=DEV), t] += 1.0
            mx, mw = scale * p.matmul(w.detach().double().abs()), scale * p.t().contiguous().matmul(x.detach().double().abs())
            assert ((dx.double() - rx).abs() <= ex + weights * mx + half * rx.abs() + tiny).all()
            assert ((dw.double() - rw).abs() <= ew + weights * mw + half * rw.abs() + tiny).all()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('size', [2.0 ** 12, 2.0 ** 20, 2.0 ** 40, 2.0 ** 80])
def test_losses_of_large_logits(size, dtype):
    """Logits that fp32 holds exactly, in steps of their own size: equal ones share the weight, others have none."""
    B, V, d = 50, 300, 6
    gen = torch.Generator(device=DEV).manual_seed(9)
    w = torch.zeros(V, d, device=DEV)
    w[:, 0] = torch.randint(-3, 3, (V,), generator=gen, device=DEV).float()
    w[:, 1] = torch.randn(V, generator=gen, device=DEV)
    x = torch.zeros(B, d, device=DEV)
    x[:, 0] = size
    x[25:, 0] = -size
    x, w = x.to(dtype).requires_grad_(), w.to(dtype).requires_grad_()
    t = torch.randint(0, V, (B,), generator=gen, device=DEV)
    loss = ops.softmax_loss(x, w, t, reduction='none')
    dx, = torch.autograd.grad(loss.sum(), x, retain_graph=True)
    X, W = x.detach().double(), w.detach().double()
    s = X.matmul(W.t())
    top = s.amax(1, keepdim=True)   # (a log-sum of 2^42 has steps of 2^-11 in 64 bits too)
    ref = (s - top).exp().sum(1).log() + (top - s.gather(1, t[:, None]))[:, 0]
    assert ((loss.double() - ref).abs() <= 2.0 ** -20 * ref.abs() + 2.0 ** -20 * 8).all()
    p = s.softmax(1)
    p[torch.arange(B, device=DEV), t] -= 1.0
    rx = p.matmul(W)
    assert ((dx.double() - rx).abs() <= HALF[dtype] * rx.abs() + 2.0 ** -16 * p.abs().matmul(W.abs()) + 1e-6).all()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('size', [2.0 ** 7, 2.0 ** 9, 2.0 ** 12, 2.0 ** 17, 2.0 ** 23, 2.0 ** 40, 2.0 ** 80])
@pytest.mark.parametrize('reduction', ['sum', 'none'])
def test_items_gradients_of_large_logits(size, dtype, reduction):
    """As above, beside rows of small logits in the same blocks.  The log-sum of such a row is kept to 2^-16 of half its
    fp32 step, or of 32 where that is less (steps from 2^6 on): a weight is off by 2^-11 at most for that, 2^-16 for
    the rest."""
    B, V, d = 90, 300, 6
    gen = torch.Generator(device=DEV).manual_seed(9)
    w = torch.zeros(V, d, device=DEV)
    w[:, 0] = torch.randint(-3, 3, (V,), generator=gen, device=DEV).float()
    w[:, 1] = torch.randn(V, generator=gen, device=DEV)
    x = torch.zeros(B, d, device=DEV)
    x[:, 0] = size
    x[30:, 0] = -size
    x[::3, 0], x[::3, 1] = 0.0, 1.0
    x, w = x.to(dtype).requires_grad_(), w.to(dtype).requires_grad_()
    t = torch.randint(0, V, (B,), generator=gen, device=DEV)
    loss = ops.softmax_loss(x, w, t, reduction=reduction)
    g = torch.ones_like(loss) if reduction == 'sum' else torch.randn(B, generator=gen, device=DEV)
    dw, = torch.autograd.grad(loss, w, g)
    X, W = x.detach().double(), w.detach().double()
    s = X.matmul(W.t())
    p = (s - s.amax(1, keepdim=True)).softmax(1)
    p[torch.arange(B, device=DEV), t] -= 1.0
    p = p * (g.double()[:, None] if reduction == 'none' else 1.0)
    rw = p.t().contiguous().matmul(X)
    terms = p.abs().t().contiguous().matmul(X.abs())
    floor = 2.0 ** -37 * B * float(X.abs().max()) * float(g.abs().max())
    off = (2.0 ** -11 if size >= 2.0 ** 17 else 0.0) + 2.0 ** -16
    assert ((dw.double() - rw).abs() <= off * terms + HALF[dtype] * rw.abs() + floor).all()
