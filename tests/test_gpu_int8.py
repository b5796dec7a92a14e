"""ops.quantize_rows and ops.gemm_int8 against the definitions.

The quantiser's whole numbers are defined in 32-bit arithmetic and have to be equal; its scale is one
correctly rounded division.  The product's sums are exact, so a result is off by the roundings of the sum
to fp32, of two products with the scales (3 * 2^-24) and of the output type (half a step).
"""
import pytest
import torch

from igr import ops
from igr._lib import IgrError

pytestmark = pytest.mark.gpu
DEV = 'cuda'
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def ref_quantize(x):
    x = x.detach().float().cpu()
    a = x.abs().amax(1)
    live = torch.isfinite(a) & (a > 0)
    q = torch.round(x / torch.where(live, a, torch.ones_like(a))[:, None] * 127)
    q = torch.where(live[:, None], q, torch.zeros_like(q)).to(torch.int8)
    return q, torch.where(torch.isfinite(a), a / 127, torch.full_like(a, float('nan')))


def check_quantize(x):
    q, s = ops.quantize_rows(x)
    rq, rs = ref_quantize(x)
    assert q.dtype == torch.int8 and s.dtype == torch.float32 and q.shape == x.shape
    assert torch.equal(q.cpu(), rq)
    assert torch.equal(s.cpu().nan_to_num(nan=-1.0), rs.nan_to_num(nan=-1.0))
    return q, s


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n,k', [(1, 1), (3, 7), (65, 15), (100, 16), (33, 64), (257, 100), (5, 200), (1000, 128), (2, 2048),
                                 (3, 2049), (2, 5000), (7, 4104), (0, 8)])
def test_quantize(n, k, dtype):
    gen = torch.Generator(device=DEV).manual_seed(n + k)
    x = (torch.randn(n, k, generator=gen, device=DEV) * torch.exp(3 * torch.randn(n, 1, generator=gen, device=DEV)))
    check_quantize(x.to(dtype))


def test_quantize_special_rows():
    x = torch.randn(12, 40, device=DEV)
    x[0] = 0
    x[1] = -0.0
    x[2, 3] = float('nan')
    x[3, 39] = float('inf')
    x[4, 0] = -float('inf')
    x[5] = 3e38
    x[6] = 1e-45           # a subnormal
    x[7] = torch.linspace(-1e-40, 1e-40, 40, device=DEV)
    x[8] = 63.5 / 127      # with the row's 1.0: on a tie
    x[8, 0] = 1.0
    x[9, 1] = torch.finfo(torch.float32).min
    check_quantize(x)


@pytest.mark.parametrize('dtype', TYPES)
def test_quantize_strides(dtype):
    base = torch.randn(90, 200, device=DEV).to(dtype)
    for v in (base[:, 1:65], base[::3, 8:72], base[:, ::2], base[:1].expand(9, 200), base.t()[:60], base[5:6, 3:4]):
        check_quantize(v)


def test_padding_columns_are_zero_and_rows_aligned():
    q, _ = ops.quantize_rows(torch.randn(50, 100, device=DEV) + 3.0)
    assert q.stride() == (112, 1) and q.data_ptr() % 16 == 0
    whole = torch.as_strided(q, (50, 112), (112, 1))
    assert not whole[:, 100:].any()


def check_product(a, sa, b, sb, out):
    y = ops.gemm_int8(a, sa, b, sb, out_dtype=out)
    ref = a.double().matmul(b.double().t()) * sa.double()[:, None] * sb.double()[None, :]
    assert y.dtype == out and y.shape == ref.shape
    tiny = 2.0 ** -25 if out == torch.float16 else 2.0 ** -140
    assert ((y.double() - ref).abs() <= (3 * 2.0 ** -24 + HALF[out]) * ref.abs() + tiny).all()
    return y


def tables(m, n, k, seed=0, pad=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda p: torch.randint(-128, 128, (p, k + pad), generator=gen, device=DEV, dtype=torch.int8)[:, :k]  # noqa: E731
    s = lambda p: torch.rand(p, generator=gen, device=DEV) * 0.01 + 1e-4  # noqa: E731
    return r(m), s(m), r(n), s(n)


SHAPES = [(1, 1, 1), (1, 1000, 64), (1, 33, 7), (2, 3, 16), (5, 257, 15), (32, 300, 48), (33, 129, 64), (31, 4000, 300),
          (130, 131, 17), (64, 64, 256), (300, 200, 257), (129, 127, 1000), (257, 260, 128), (40, 50, 2048), (100, 500, 513),
          (3, 2, 40000)]


@pytest.mark.parametrize('out', TYPES)
@pytest.mark.parametrize('m,n,k', SHAPES)
def test_product(m, n, k, out):
    check_product(*tables(m, n, k, seed=m + n + k), out)


@pytest.mark.parametrize('k,pad', [(64, 1), (100, 12), (65, 3), (1000, 8), (300, 1)])
def test_product_of_strided_and_unaligned_tables(k, pad):
    a, sa, b, sb = tables(70, 90, k, seed=k, pad=pad)
    y = check_product(a, sa, b, sb, torch.float32)
    assert torch.equal(y, ops.gemm_int8(a.contiguous(), sa, b.contiguous(), sb))
    assert torch.equal(y[::2], ops.gemm_int8(a[::2], sa[::2], b, sb))           # every other row, strided scales
    assert torch.equal(y[:1].expand(9, 90), ops.gemm_int8(a[:1].expand(9, k), sa[:1].expand(9), b, sb))
    t = b.t().contiguous().t()                                                  # column-major items
    assert torch.equal(y, ops.gemm_int8(a, sa, t, sb))


def test_both_scales_strided():
    """Each side's packed copy of its scales outlives the launch, not only the other copy's allocation."""
    a, sa, b, sb = tables(40, 50, 64, seed=3)
    wide_a, wide_b = sa.repeat_interleave(2), sb.repeat_interleave(3)
    assert torch.equal(ops.gemm_int8(a, wide_a[::2], b, wide_b[::3]), check_product(a, sa, b, sb, torch.float32))


def test_extreme_sums_and_scales():
    a = torch.full((40, 131071), -128, dtype=torch.int8, device=DEV)  # the largest sum that is allowed
    one = torch.ones(40, device=DEV)
    y = check_product(a, one, a[:33], one[:33], torch.float32)
    assert float(y[0, 0]) == float(torch.tensor(16384.0 * 131071).float())
    a, sa, b, sb = tables(5, 6, 32)
    sa[1], sa[2], sb[3] = float('nan'), 0.0, float('inf')
    y = ops.gemm_int8(a, sa, b, sb)
    assert torch.isnan(y[1]).all() and torch.isnan(y[2, 3]) and torch.isinf(y[0, 3])
    assert not y[2, [0, 1, 2, 4, 5]].any()


def test_empty_sides():
    a, sa, b, sb = tables(4, 6, 32)
    assert ops.gemm_int8(a[:0], sa[:0], b, sb).shape == (0, 6)
    assert ops.gemm_int8(a, sa, b[:0], sb[:0]).shape == (4, 0)


def test_nothing_past_the_result_is_written():
    """Through the C entry: a strided result, its other columns and rows left as they were."""
    from igr import _lib as L
    a, sa, b, sb = tables(70, 75, 40)
    for out in TYPES:
        c = torch.full((90, 200), 7.0, device=DEV, dtype=out)
        L.call('igr_gemm_int8', 70, 75, 40, ops._p(a), 40, ops._p(sa), ops._p(b), 40, ops._p(sb), ops._DTYPES[out],
               ops._p(c[:, 3:]), 200, ops._stream())
        assert torch.equal(c[:70, 3:78], ops.gemm_int8(a, sa, b, sb, out_dtype=out))
        rest = c.clone()
        rest[:70, 3:78] = 7.0
        assert (rest == 7.0).all()


def test_offsets_past_32_bits():
    """An item table of 2^31 + bytes: its last rows are read where they are."""
    n, k = 2_200_000, 1024
    b = torch.zeros(n, k, dtype=torch.int8, device=DEV)
    b[-3:] = torch.randint(-128, 128, (3, k), device=DEV, dtype=torch.int8)
    a, sa = torch.randint(-128, 128, (2, k), device=DEV, dtype=torch.int8), torch.ones(2, device=DEV)
    y = ops.gemm_int8(a, sa, b, torch.ones(n, device=DEV))
    ref = a.double().matmul(b[-3:].double().t())
    assert torch.equal(y[:, -3:].double(), ref) and not y[:, :-3].any()
    big = torch.zeros(2_200_000, 256, device=DEV)   # 2^31 + bytes of fp32 rows
    big[-2:] = torch.randn(2, 256, device=DEV)
    q, s = ops.quantize_rows(big)
    rq, rs = ref_quantize(big[-2:])
    assert torch.equal(q[-2:].cpu(), rq) and torch.equal(s[-2:].cpu(), rs) and not q[:-2].any() and not s[:-2].any()


def test_quantise_then_score_is_close_to_the_float_product():
    """The run as it is used: half a quantisation step for each operand, elementwise."""
    gen = torch.Generator(device=DEV).manual_seed(5)
    u, w = torch.randn(50, 64, generator=gen, device=DEV), torch.randn(700, 64, generator=gen, device=DEV)
    (qu, su), (qw, sw) = ops.quantize_rows(u), ops.quantize_rows(w)
    y = ops.gemm_int8(qu, su, qw, sw).double()
    ref = u.double().matmul(w.double().t())
    eu, ew = 0.5 * su.double()[:, None], 0.5 * sw.double()[None, :]   # |x - q s| <= s / 2, up to fp32 roundings
    bound = (eu * w.abs().double().sum(1)[None, :] + ew * u.abs().double().sum(1)[:, None] + 64 * eu * ew) * (1 + 1e-4)
    assert ((y - ref).abs() <= bound + 1e-6 * ref.abs()).all()


def test_captured_and_on_another_stream():
    u, w = torch.randn(200, 100, device=DEV), torch.randn(300, 100, device=DEV)

    def go():
        q, s = ops.quantize_rows(u)
        qw, sw = ops.quantize_rows(w)
        return ops.gemm_int8(q, s, qw, sw)
    ref = go()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(go(), ref)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = go()
    for _ in range(3):
        u.mul_(1.3).add_(0.1)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, go())


def test_refusals():
    a, sa, b, sb = tables(4, 6, 32)
    with pytest.raises(IgrError, match='int8'):
        ops.gemm_int8(a.int(), sa, b, sb)
    with pytest.raises(IgrError, match='shapes'):
        ops.gemm_int8(a, sa, b[:, :31], sb)
    with pytest.raises(IgrError, match='scales'):
        ops.gemm_int8(a, sa[:3], b, sb)
    with pytest.raises(IgrError, match='float32'):
        ops.gemm_int8(a, sa.half(), b, sb)
    with pytest.raises(IgrError, match='out_dtype'):
        ops.gemm_int8(a, sa, b, sb, out_dtype=torch.int32)
    with pytest.raises(IgrError, match='131071'):
        z = torch.zeros(2, 131072, dtype=torch.int8, device=DEV)
        ops.gemm_int8(z, sa[:2], z, sa[:2])
    with pytest.raises(IgrError, match='2-D'):
        ops.quantize_rows(sa)
    with pytest.raises(IgrError, match='float32, bfloat16'):
        ops.quantize_rows(a)
