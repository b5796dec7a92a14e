"""Argument checks of the catalogue operators that are made before any GPU work (CPU)."""
import ctypes

import pytest
import torch

from igr import _lib as L
from igr import ops


def test_softmax_loss_refuses_cpu_tensors():
    with pytest.raises(L.IgrError, match='no CPU fallback'):
        ops.softmax_loss(torch.zeros(2, 4), torch.zeros(3, 4), torch.zeros(2, dtype=torch.int64))


def test_softmax_loss_c_arguments():
    lib = L.lib()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 255) & ~255

    def fwd(dtype=0, b=4, v=6, d=8, ldx=8, ldw=8, scale=1.0, x=p, ws=p, wsb=1 << 40, total=p, count=p):
        return lib.igr_softmax_loss_fwd(dtype, b, v, d, x, ldx, p, ldw, p, -100, scale, 1, p, p, p, p, total, count, None,
                                        ws, wsb, None)

    for kw, msg in ((dict(dtype=3), 'dtype'), (dict(b=-1), 'sizes'), (dict(v=0), 'sizes'), (dict(d=0), 'sizes'),
                    (dict(v=1 << 31), 'rows'), (dict(ldx=7), 'leading'), (dict(ldw=7), 'leading'),
                    (dict(scale=0.0), 'scale'), (dict(scale=float('nan')), 'scale'), (dict(x=None), 'null'),
                    (dict(ws=None), 'workspace'), (dict(wsb=16), 'workspace'), (dict(ws=p + 4), 'workspace'),
                    (dict(count=None), 'together')):
        assert fwd(**kw) == 1, kw  # IGR_ERR_ARG
        assert msg in lib.igr_last_error().decode(), (kw, lib.igr_last_error())
    assert fwd(d=257, ldx=257, ldw=257) == 3  # IGR_ERR_UNSUPPORTED

    def bwd(dtype=0, d=8, ldw=8, scale=1.0, grad=p, ws=p, wsb=1 << 40, count=p, pack=p):
        return lib.igr_softmax_loss_bwd(dtype, 4, 6, d, p, ldw, p, -100, scale, 1, 0, grad, pack, p, p, count, p, p, p, ws, wsb,
                                        None)

    for kw, msg in ((dict(dtype=-1), 'dtype'), (dict(ldw=7), 'leading'), (dict(scale=-1.0), 'scale'),
                    (dict(grad=None), 'null'), (dict(count=None), 'null'), (dict(pack=None), 'null'), (dict(ws=None), 'workspace'),
                    (dict(wsb=16), 'workspace')):
        assert bwd(**kw) == 1, kw
        assert msg in lib.igr_last_error().decode(), (kw, lib.igr_last_error())


def test_softmax_loss_sizes():
    lib = L.lib()
    # two 16-bit planes in two layouts for fp32, one plane for half types, an exponent a block of 32
    assert lib.igr_softmax_loss_pack_size(64, 64, 0) == 2 * (2 * 2 * 32 * 64 * 2) + 256
    assert lib.igr_softmax_loss_pack_size(33, 33, 1) == 2 * (2 * 32 * 64 * 2) + 256
    assert lib.igr_softmax_loss_pack_size(0, 64, 0) == 0 and lib.igr_softmax_loss_pack_size(4, 300, 0) == 0
    for b, v, d in ((1, 1, 1), (2048, 1000000, 64), (1, 1000000, 256), (100000, 7, 128)):
        for back in (0, 1):
            ws = lib.igr_softmax_loss_workspace_size(b, v, d, back, 1)
            # partials of at most 512 workgroups of 256 rows, rounded up, and the rows' own data
            assert 0 < ws <= 4 * (512 + 256) * 256 * (256 + 4) + 16 * (b + 512 * 32) + 4096 + 8 * 256 * min(b, v), (b, v, ws)


def test_int8_refuses_cpu_tensors():
    with pytest.raises(L.IgrError, match='no CPU fallback'):
        ops.quantize_rows(torch.zeros(2, 4))
    q, s = torch.zeros(2, 4, dtype=torch.int8), torch.ones(2)
    with pytest.raises(L.IgrError, match='no CPU fallback'):
        ops.gemm_int8(q, s, q, s)


def test_int8_c_arguments():
    lib = L.lib()

    def quant(dtype=0, n=2, k=8, x=4096, ldx=8, q=4096, ldq=16, s=4096):
        return lib.igr_quantize_rows(dtype, n, k, x, ldx, q, ldq, s, None)

    def mul(m=2, n=3, k=8, a=4096, lda=8, sa=4096, ldb=8, out=0, c=4096, ldc=3):
        return lib.igr_gemm_int8(m, n, k, a, lda, sa, 4096, ldb, 4096, out, c, ldc, None)

    for f, kw, msg in ((quant, dict(dtype=7), 'dtype'), (quant, dict(n=-1), 'sizes'), (quant, dict(k=0), 'sizes'),
                       (quant, dict(ldx=7), 'leading'), (quant, dict(ldq=7), 'leading'), (quant, dict(x=None), 'null'),
                       (quant, dict(q=None), 'null'), (quant, dict(s=None), 'null'), (mul, dict(out=3), 'dtype'),
                       (mul, dict(m=-1), 'sizes'), (mul, dict(k=0), 'sizes'), (mul, dict(k=131072, lda=1 << 20), '131071'),
                       (mul, dict(lda=7), 'leading'), (mul, dict(ldb=7), 'leading'), (mul, dict(ldc=2), 'leading'),
                       (mul, dict(a=None), 'null'), (mul, dict(sa=None), 'null'), (mul, dict(c=None), 'null')):
        assert f(**kw) == 1, kw
        assert msg in lib.igr_last_error().decode(), (kw, lib.igr_last_error())
    assert quant(n=0) == 0 and mul(m=0) == 0 and mul(n=0, ldc=0) == 0  # nothing to do, no launch


def test_newton_schulz_refuses_cpu_tensors():
    with pytest.raises(L.IgrError, match='no CPU fallback'):
        ops.newton_schulz(torch.zeros(2, 4))


def test_newton_schulz_c_arguments():
    lib = L.lib()

    def ns(dtype=0, batch=1, rows=100, cols=300, ldg=300, sg=0, steps=5, a=3.4445, b=-4.775, c=2.0315, eps=1e-7, g=4096,
           ws=4096, wsb=1 << 40):
        return lib.igr_newton_schulz(dtype, batch, rows, cols, g, ldg, sg, steps, a, b, c, eps, 4096, ws, wsb, None)

    nan = float('nan')
    for kw, msg in ((dict(dtype=3), 'dtype'), (dict(batch=-1), 'size'), (dict(ldg=299), 'leading'),
                    (dict(batch=2, sg=-1), 'leading'), (dict(steps=0), 'steps'), (dict(steps=101), 'steps'),
                    (dict(eps=-1.0), 'eps'), (dict(eps=nan), 'eps'), (dict(a=nan), 'coefficients'),
                    (dict(a=5.0, b=0.0, c=0.0), 'coefficients'), (dict(batch=65536), 'large'),
                    (dict(rows=40000, cols=40000, ldg=40000), 'large'), (dict(g=None), 'null'),
                    (dict(ws=None), 'workspace'), (dict(wsb=16), 'workspace'), (dict(ws=4100), 'workspace')):
        assert ns(**kw) == 1, kw
        assert msg in lib.igr_last_error().decode(), (kw, lib.igr_last_error())
    assert ns(batch=0) == 0 and ns(rows=0) == 0
    assert lib.igr_newton_schulz_workspace_size(6, 64, 64) == 0  # one workgroup a matrix
    assert lib.igr_newton_schulz_workspace_size(1, 128, 512) == (3 * 128 * 512 + 2 * 128 * 128) * 4 + 256 * 8


def test_muon_c_arguments():
    lib = L.lib()
    s = (L.IgrMuonSlot * 17)()
    at = ctypes.addressof(s)
    for f, tail in ((lib.igr_muon_direction_f32, (0.9, 1)), (lib.igr_muon_apply_f32, (0.1, 0.0, 1.0))):
        for n, p, msg in ((-1, at, 'n_slots'), (17, at, 'n_slots'), (1, None, 'NULL slots'), (1, at, 'size')):
            assert f(n, p, *tail, None) == 1 and msg in lib.igr_last_error().decode()
        s[0].n = 4
        assert f(1, at, *tail, None) == 1 and 'NULL pointer' in lib.igr_last_error().decode()
        s[0].n = 0
        assert f(0, None, *tail, None) == 0
