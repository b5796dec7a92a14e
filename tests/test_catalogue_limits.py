"""Sizes of the catalogue operators that no launch holds are refused before any GPU work (CPU)."""
import ctypes

from igr import _lib as L


def test_more_result_tiles_than_a_launch_holds_are_refused():
    lib = L.lib()
    # 2^32 threads along a dimension and more: 2^24 tiles of 32 x 256
    rc = lib.igr_gemm_int8(1, 1 << 33, 1, 4096, 1, 4096, 4096, 1, 4096, 0, 4096, 1 << 33, None)
    assert rc == 1 and 'tiles' in lib.igr_last_error().decode()
    rc = lib.igr_gemm_int8(1 << 20, 1 << 20, 64, 4096, 64, 4096, 4096, 64, 4096, 0, 4096, 1 << 20, None)
    assert rc == 1 and 'tiles' in lib.igr_last_error().decode()


def test_more_batch_rows_than_a_launch_holds_are_refused():
    lib = L.lib()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 255) & ~255
    rc = lib.igr_softmax_loss_fwd(1, (1 << 31) - 100, 6, 8, p, 8, p, 8, p, -100, 1.0, 1, p, p, p, p, p, p, None, p, 1 << 50, None)
    assert rc == 1 and 'rows' in lib.igr_last_error().decode()
