"""ops.softmax_loss: the catalogue softmax cross entropy and its gradients against the formula in
64 bits.

Bounds.  With A_b = max_v scale sum_k |x_bk w_vk|, a logit is off by at most (3 d + 16) 2^-24 A_b:
three fp32-accumulated products a term (3 d roundings), 2^-21 from the operands' pairs and the product
left out, and the exponent's own fma.  A softmax weight is then off by e = 2 (that) + 2^-20 (exp2,
the weight's pair) + n 2^-24 relative, n the longest chain of fp32 additions (at most 1 + V / 32 + 64
blocks and joins, likewise B).  A gradient is a sum of weights times rows, so its error is at most
e times the sum of the terms' magnitudes.  For fp32 and fp16 there is a floor: a weight |c_b| p is
held as 2^14 at the largest product of a |c_b| and a block's entry (powers of two at most twice
either), so half of the smallest half's step, 2^-25, stands for 2^(-25 - 14 + 2) of that
product, for each term.  Half types add 2^-8 (bf16) or 2^-11 (fp16), half a step, of the terms'
magnitudes for the rounded weights and of the value for the rounded result (fp16 also its
subnormal step).
"""
import pytest
import torch

from igr import ops
from igr._lib import IgrError

pytestmark = pytest.mark.gpu
DEV = 'cuda'
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def formula(x, w, t, scale, ignore, g):
    """(per-row loss, dx, dw, sum of |terms| of dx, of dw, e) in 64 bits; g: gradient per row."""
    live = (t != ignore).nonzero()[:, 0]
    X, W, T = x.detach().double()[live], w.detach().double(), t[live]
    s = scale * X.matmul(W.t())
    a = (scale * X.abs().matmul(W.abs().t())).amax(1) if len(live) else s.new_zeros(0)
    lse = torch.logsumexp(s, 1)
    at = torch.arange(len(live), device=x.device)
    loss = x.new_zeros(len(t), dtype=torch.float64)
    loss[live] = lse - s[at, T]
    p = (s - lse[:, None]).exp()
    hot = torch.zeros_like(p)
    hot[at, T] = 1.0
    c = (g.double()[live] * scale)[:, None]
    dx, mx = torch.zeros_like(x, dtype=torch.float64), torch.zeros_like(x, dtype=torch.float64)
    dx[live] = c * (p - hot).matmul(W)
    mx[live] = c.abs() * (p + hot).matmul(W.abs())
    dw = ((p - hot) * c).t().contiguous().matmul(X)
    n = 65 + max(len(t), W.shape[0]) // 32
    e_row = x.new_zeros(len(t), dtype=torch.float64)
    e_row[live] = 2 * (3 * x.shape[1] + 16) * 2.0 ** -24 * a + 2.0 ** -20 + n * 2.0 ** -24
    mw = ((p + hot) * c.abs() * e_row[live][:, None]).t().contiguous().matmul(X.abs())
    if x.dtype != torch.bfloat16 and len(live):
        floor = 2.0 ** -37 * c.abs().max()
        mw = mw + floor * len(live) * X.abs().max()
        e_floor = floor * W.shape[0] * W.abs().max()
    else:
        e_floor = 0.0
    mw1 = ((p + hot) * c.abs()).t().contiguous().matmul(X.abs())
    return loss, dx, dw, mx, mw, mw1, e_row, e_floor


def check(x, w, t, scale=1.0, ignore=-100, reduction='mean', g=None):
    x.requires_grad_()
    w.requires_grad_()
    loss = ops.softmax_loss(x, w, t, scale=scale, ignore_index=ignore, reduction=reduction)
    n = max(int((t != ignore).sum()), 1)
    if reduction == 'none':
        gr = torch.ones(len(t), device=DEV) if g is None else g
        dx, dw = torch.autograd.grad(loss, (x, w), gr)
    else:
        g0 = torch.tensor(1.0 if g is None else g, device=DEV)
        gr = g0.expand(len(t)) / (n if reduction == 'mean' else 1)
        dx, dw = torch.autograd.grad(loss, (x, w), g0)
    rl, rx, rw, mx, mw, mw1, e, e_floor = formula(x, w, t, scale, ignore, gr)
    el = e + 2.0 ** -23 * rl.abs()
    if reduction == 'none':
        assert loss.dtype == torch.float32 and loss.shape == t.shape
        assert ((loss.double() - rl).abs() <= el).all()
    else:
        div = n if reduction == 'mean' else 1
        loss = loss.detach()
        assert abs(float(loss) - float(rl.sum()) / div) <= float(el.sum()) / div + 2.0 ** -23 * abs(float(loss))
    half = HALF[x.dtype]
    w_round = 0.0 if x.dtype == torch.float32 else half
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 1e-37
    assert dx.dtype == x.dtype and dw.dtype == w.dtype
    assert ((dx.double() - rx).abs() <= (e[:, None] + w_round) * mx + e_floor + half * rx.abs() + tiny).all()
    assert ((dw.double() - rw).abs() <= mw + w_round * mw1 + half * rw.abs() + tiny).all()
    return loss, dx, dw


def tables(B, V, d, dtype, seed=0, std=None, spread=0.3):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    std = (2.0 / d ** 0.5) ** 0.5 if std is None else std
    r = lambda n: torch.randn(n, d, generator=gen, device=DEV) * std * torch.exp(  # noqa: E731
        spread * torch.randn(n, 1, generator=gen, device=DEV))
    x, w = r(B).to(dtype), r(V).to(dtype)
    return x, w, torch.randint(0, V, (B,), generator=gen, device=DEV)


SHAPES = [(1, 1, 1), (1, 2, 8), (3, 5, 7), (32, 32, 32), (33, 31, 64), (31, 33, 65), (129, 1000, 100), (256, 1682, 64),
          (100, 70001, 32), (700, 333, 200), (64, 4097, 256), (2050, 300, 33), (1, 5000, 129), (5000, 1, 16)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('B,V,d', SHAPES)
def test_loss_and_gradients(B, V, d, dtype):
    x, w, t = tables(B, V, d, dtype, seed=B + V + d)
    check(x, w, t)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
def test_reductions_scale_and_incoming_gradients(reduction, dtype):
    x, w, t = tables(300, 777, 48, dtype, seed=3)
    g = -2.5
    if reduction == 'none':  # signs, zeros and sizes that differ from row to row
        g = torch.randn(300, device=DEV) * torch.exp2(torch.randint(-12, 3, (300,), device=DEV).float())
        g[::7] = 0.0
    check(x, w, t, scale=0.37, reduction=reduction, g=g)


@pytest.mark.parametrize('dtype', TYPES)
def test_sharp_and_large_logits(dtype):
    x, w, t = tables(200, 900, 64, dtype, seed=4)
    check(x, w, t, scale=40.0)   # one item takes all
    x, w, t = tables(200, 900, 64, dtype, seed=5, std=1e-3)
    check(x, w, t)               # nearly uniform
    x, w, t = tables(64, 500, 64, dtype, seed=6, std=8.0)
    check(x, w, w.float().matmul(x.float()[0]).argmax().expand(64).contiguous())  # one item is every row's target


@pytest.mark.parametrize('dtype', TYPES)
def test_rows_that_are_sure_of_their_target_keep_their_digits(dtype):
    """With p_t = 1 - r and r from 3e-1 down to 1e-7, the loss log(1 + r / p_t) and dx = c (sum_{v != t} p_v w_v -
    r w_t) are as small as r.  Both are sums without the target, so their error is e (as above, of the
    terms of these sums), not the fp32 step of 1: relative to r."""
    gen = torch.Generator(device=DEV).manual_seed(21)
    V, d, B = 300, 64, 64
    w = torch.randn(V, d, generator=gen, device=DEV) * 0.3
    t = torch.randint(0, V, (B,), generator=gen, device=DEV)
    x = w[t] / w[t].square().sum(1, keepdim=True) * torch.linspace(7, 26, B, device=DEV)[:, None]
    x, w = x.to(dtype).requires_grad_(), w.to(dtype).requires_grad_()
    loss = ops.softmax_loss(x, w, t, reduction='none')
    dx, dw = torch.autograd.grad(loss.sum(), (x, w))
    X, W = x.detach().double(), w.detach().double()
    s = X.matmul(W.t())
    at = torch.arange(B, device=DEV)
    rel = (s - s[at, t][:, None]).exp()
    rel[at, t] = 0.0
    ref = torch.log1p(rel.sum(1))
    p = rel / (1.0 + rel.sum(1, keepdim=True))
    r = p.sum(1, keepdim=True)
    assert float(ref.min()) < 1e-6 and float(ref.max()) > 1e-2
    a = X.abs().matmul(W.abs().t()).amax(1)
    e = 2 * (3 * d + 16) * 2.0 ** -24 * a + 2.0 ** -20 + 75 * 2.0 ** -24
    assert ((loss.double() - ref).abs() <= 2 * e * ref + 1e-30).all()
    half = HALF[dtype]
    w_round = 0.0 if dtype == torch.float32 else half
    gx = p.matmul(W) - r * W[t]
    mx = p.matmul(W.abs()) + r * W[t].abs()
    # the forward's weights are held from 2^14 at the largest logit, here another item's or the target's
    floor = (V * 2.0 ** -37 if dtype != torch.bfloat16 else 0.0) * p.amax(1, keepdim=True) * W.abs().max()
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-37
    assert ((dx.double() - gx).abs() <= (2 * e[:, None] + w_round) * mx + floor + half * gx.abs() + tiny).all()


def test_rows_of_very_different_size():
    """Block scales: whole blocks of the tables 2^10 apart, single large rows among small ones."""
    x, w, t = tables(320, 1000, 64, torch.float32, seed=7)
    x[:64] *= 2.0 ** -10
    w[96:160] *= 2.0 ** -10
    w[500] *= 32.0
    check(x, w, t)


@pytest.mark.parametrize('dtype', TYPES)
def test_ignored_rows_count_for_nothing(dtype):
    x, w, t = tables(200, 321, 72, dtype, seed=8)
    t[::3] = -100
    a = check(x, w, t)
    y = x.detach().clone()
    y[::3] = float('nan')
    y[3] = float('inf')
    y.requires_grad_()
    loss = ops.softmax_loss(y, w, t)
    dx, dw = torch.autograd.grad(loss, (y, w))
    assert torch.equal(loss, a[0]) and torch.equal(dw, a[2]) and torch.equal(dx, a[1])
    assert not dx[::3].any()
    t[:] = 7
    out = [ops.softmax_loss(x, w, t, ignore_index=7, reduction=r) for r in ('mean', 'sum', 'none')]
    for o in out:
        assert not o.any()
        for gr in torch.autograd.grad(o.sum(), (x, w)):
            assert not gr.any()
    check(x, w, torch.full_like(t, 5), ignore=-1)


def test_empty_batch():
    x, w = torch.zeros(0, 16, device=DEV, requires_grad=True), torch.randn(9, 16, device=DEV, requires_grad=True)
    t = torch.zeros(0, dtype=torch.int64, device=DEV)
    loss = ops.softmax_loss(x, w, t)
    assert float(loss.detach()) == 0.0
    dx, dw = torch.autograd.grad(loss, (x, w))
    assert dx.shape == (0, 16) and not dw.any()
    assert ops.softmax_loss(x, w, t, reduction='none').shape == (0,)


def test_target_outside_the_table_is_nan_not_a_read():
    x, w, t = tables(70, 50, 24, torch.float32, seed=9)
    t[5], t[40] = 50, -7
    x.requires_grad_()
    w.requires_grad_()
    rows = ops.softmax_loss(x, w, t, reduction='none')
    assert torch.isnan(rows[[5, 40]]).all() and int(torch.isnan(rows).sum()) == 2
    dx, dw = torch.autograd.grad(rows.sum(), (x, w))
    assert torch.isnan(dx[[5, 40]]).all() and int(torch.isnan(dx).any(1).sum()) == 2
    assert torch.isnan(dw).all()
    assert torch.isnan(ops.softmax_loss(x, w, t))


def test_non_finite_inputs_show():
    x, w, t = tables(40, 60, 32, torch.float32, seed=10)
    x[3, 4] = float('nan')
    x[9, 0] = float('inf')
    rows = ops.softmax_loss(x, w, t, reduction='none')
    assert not torch.isfinite(rows[[3, 9]]).any() and int(torch.isfinite(rows).sum()) == 38


@pytest.mark.parametrize('dtype', TYPES)
def test_strided_and_unaligned_tables(dtype):
    gen = torch.Generator(device=DEV).manual_seed(11)
    base = torch.randn(500, 150, generator=gen, device=DEV).to(dtype) * 0.3
    t = torch.randint(0, 333, (100,), generator=gen, device=DEV)
    views = [(base[:100, 1:65], base[100:433, 3:67]),           # rows not 16-byte aligned
             (base[:200:2, :64], base[100:433, 64:128]),        # every other row, a column block
             (base[:100, ::2][:, :64], base[67:400].flip(0)[:, :64]),  # inner stride 2, a copy
             (base[:1].expand(100, 150)[:, :64], base[100:433, :64])]  # one row broadcast
    for xv, wv in views:
        got = ops.softmax_loss(xv, wv, t)
        assert torch.equal(got, ops.softmax_loss(xv.contiguous(), wv.contiguous(), t))
        x, w = xv.detach(), wv.detach()
        check(x, w, t.int().long())
    # a leaf read through views: the gradients land in the leaf, the shared rows' summed
    leaf = base.clone().requires_grad_()
    ops.softmax_loss(leaf[:1].expand(100, 150)[:, :64], leaf[100:433, :64], t).backward()
    x, w = base[:1].expand(100, 150)[:, :64].contiguous(), base[100:433, :64].contiguous()
    _, dx, dw = check(x, w, t)
    assert torch.equal(leaf.grad[100:433, :64], dw) and not leaf.grad[1:100].any() and not leaf.grad[:, 64:].any()
    assert torch.allclose(leaf.grad[0, :64].float(), dx.float().sum(0), rtol=0.02, atol=1e-3)


def test_gradient_against_differences():
    x, w, t = tables(5, 40, 12, torch.float32, seed=12)
    _, dx, dw = check(x, w, t)
    f = lambda a, b: torch.nn.functional.cross_entropy(a.matmul(b.t()), t)  # noqa: E731
    h = 1e-5
    for leaf, grad, which in ((x, dx, 0), (w, dw, 1)):
        d = torch.randn(leaf.shape, device=DEV, dtype=torch.float64)
        args = [x.detach().double(), w.detach().double()]
        lo, hi = list(args), list(args)
        lo[which], hi[which] = args[which] - h * d, args[which] + h * d
        num = float(f(*hi) - f(*lo)) / (2 * h)
        assert abs(num - float((grad.double() * d).sum())) <= 1e-5 * float((grad.double() * d).abs().sum()) + 1e-7


def test_one_sided_gradients_and_no_grad():
    x, w, t = tables(90, 210, 40, torch.float32, seed=13)
    both = check(x, w, t)
    xo, wo = x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    l1 = ops.softmax_loss(xo, w.detach(), t)
    l2 = ops.softmax_loss(x.detach(), wo, t)
    assert torch.equal(torch.autograd.grad(l1, xo)[0], both[1])
    assert torch.equal(torch.autograd.grad(l2, wo)[0], both[2])
    with torch.no_grad():
        l3 = ops.softmax_loss(x, w, t)
    assert not l3.requires_grad and torch.equal(l1, l3) and torch.equal(l2, l3)


def test_no_grad_keeps_nothing_for_a_backward(monkeypatch):
    x, w, t = tables(90, 210, 40, torch.float32, seed=13)
    x.requires_grad_()
    w.requires_grad_()
    asked = []
    layout = ops._softmax_layout
    monkeypatch.setattr(ops, '_softmax_layout', lambda *a: asked.append(a[4:]) or layout(*a))
    with torch.no_grad():
        quiet = ops.softmax_loss(x, w, t)
    assert torch.equal(quiet, ops.softmax_loss(x, w, t)) and asked == [(False, False), (True, True)]


def test_same_bits_again_and_on_another_stream():
    x, w, t = tables(513, 3333, 64, torch.float32, seed=14)
    a = check(x, w, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = check(x, w, t)
    torch.cuda.current_stream().wait_stream(side)
    for p, q in zip(a, b):
        assert torch.equal(p, q)


def test_captured_forward_and_backward_replay():
    x, w, t = tables(300, 1000, 64, torch.float32, seed=15)
    x.requires_grad_()
    w.requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(ops.softmax_loss(x, w, t), (x, w))
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    outs = []
    for g in (g1, g2):
        with torch.cuda.graph(g):
            loss = ops.softmax_loss(x, w, t)
            outs.append((loss.detach(),) + torch.autograd.grad(loss, (x, w)))
    for rep in range(3):
        with torch.no_grad():
            x.mul_(0.9)
            t.copy_(t.roll(1))
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        loss = ops.softmax_loss(x, w, t)
        ref = (loss.detach(),) + torch.autograd.grad(loss, (x, w))
        for o in outs:
            for p, q in zip(o, ref):
                assert torch.equal(p, q), rep


def test_changed_tables_between_forward_and_backward_are_refused():
    x, w, t = tables(20, 30, 16, torch.float32, seed=16)
    x.requires_grad_()
    w.requires_grad_()
    loss = ops.softmax_loss(x, w, t)
    with torch.no_grad():
        w.add_(1.0)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()


def test_table_past_32_bits():
    """2^31 + bytes of item rows (and twice that packed): the last rows are read and their gradients written
    where they are.  Sixteen rows at the end carry all of the softmax's weight but 1e-6."""
    V, d, B = 9_000_000, 64, 8
    gen = torch.Generator(device=DEV).manual_seed(31)
    w = torch.zeros(V, d, device=DEV)
    w[-16:] = torch.randn(16, d, generator=gen, device=DEV)
    w[:, 0] = -1.0
    w[-16:, 0] = 0.0
    x = torch.randn(B, d, generator=gen, device=DEV)
    x[:, 0] = 32.0   # the other nine million: logits of -32
    t = V - 1 - torch.randint(0, 16, (B,), generator=gen, device=DEV)
    x.requires_grad_()
    w.requires_grad_()
    loss = ops.softmax_loss(x, w, t)
    dx, dw = torch.autograd.grad(loss, (x, w))
    X, W = x.detach().double(), w.detach()[-16:].double()
    s = torch.cat([X.matmul(W.t()), torch.full((B, 1), -32.0, device=DEV, dtype=torch.float64)
                   + torch.log(torch.tensor(float(V - 16), device=DEV, dtype=torch.float64))], 1)
    p = s.softmax(1)[:, :16]
    at = t - (V - 16)
    assert abs(float(loss.detach()) - float(torch.nn.functional.cross_entropy(s, at))) < 1e-5
    p[torch.arange(B, device=DEV), at] -= 1.0
    assert (dw[-16:].double() - p.t().contiguous().matmul(X) / B).abs().max() < 1e-5 * 32
    assert dw[:-16].abs().max() < 1e-9 and (dx[:, 1:].double() - p.matmul(W)[:, 1:] / B).abs().max() < 1e-6


def test_second_derivatives_are_refused():
    x, w, t = tables(20, 30, 16, torch.float32, seed=17)
    x.requires_grad_()
    loss = ops.softmax_loss(x, w, t)
    with pytest.raises(IgrError, match='second derivative'):
        torch.autograd.grad(loss, x, create_graph=True)


def test_backward_twice_gives_the_same_bits_in_new_tensors():
    x, w, t = tables(70, 90, 24, torch.float32, seed=18)
    x.requires_grad_()
    w.requires_grad_()
    loss = ops.softmax_loss(x, w, t)
    a = torch.autograd.grad(loss, (x, w), retain_graph=True)
    kept = [g.clone() for g in a]
    b = torch.autograd.grad(loss, (x, w), torch.tensor(1.0, device=DEV))
    for g, k, h in zip(a, kept, b):
        assert torch.equal(g, k) and torch.equal(g, h) and g.data_ptr() != h.data_ptr()


def test_refusals_on_the_device():
    x, w, t = tables(4, 6, 8, torch.float32)
    with pytest.raises(IgrError, match='share'):
        ops.softmax_loss(x, w.half(), t)
    with pytest.raises(IgrError, match='share'):
        ops.softmax_loss(x.double(), w.double(), t)
    with pytest.raises(IgrError, match='shapes'):
        ops.softmax_loss(x, w[:, :7], t)
    with pytest.raises(IgrError, match='shapes'):
        ops.softmax_loss(x, w, t[:3])
    with pytest.raises(IgrError, match='int64'):
        ops.softmax_loss(x, w, t.float())
    with pytest.raises(IgrError, match='width'):
        ops.softmax_loss(torch.zeros(4, 257, device=DEV), torch.zeros(6, 257, device=DEV), t)
    with pytest.raises(IgrError, match='no items'):
        ops.softmax_loss(x, w[:0], t)
    for s in (0.0, -1.0, float('nan'), float('inf')):
        with pytest.raises(IgrError, match='scale'):
            ops.softmax_loss(x, w, t, scale=s)
    with pytest.raises(IgrError, match='reduction'):
        ops.softmax_loss(x, w, t, reduction='max')
