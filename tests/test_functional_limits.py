"""The sizes at which the float operators' launches end, at the C entries and without a device: what would need 2^32 threads
or more is refused before anything is launched, and sums over many rows get the partial sums that keep them short."""
import ctypes

import pytest


def call(name, *args):
    from qnn import _lib
    return getattr(_lib.load(), name)(*args), _lib.load().qnn_last_error()


P = ctypes.c_void_p(4096)  # an address that no check reads
SIZES = {0: 4, 1: 2, 2: 2}  # QNN_F32, QNN_BF16, QNN_F16


@pytest.mark.parametrize("code", SIZES)
def test_layer_norm_rows_longer_than_registers(code):
    dim = 4096 * 16 // SIZES[code] + 1
    for rows in (1 << 22, (1 << 31) - 1):
        rc, msg = call("qnn_layer_norm_fwd", P, dim, None, None, P, None, None, rows, dim, 1e-5, code, code, None)
        assert rc == 1 and b"too many rows" in msg
        rc, msg = call("qnn_layer_norm_bwd", P, dim, P, dim, None, P, P, P, P, P, rows, dim, code, code, P, 1 << 62, None)
        assert rc == 1 and b"too many rows" in msg


@pytest.mark.parametrize("code", SIZES)
@pytest.mark.parametrize("dim", [1, 3, 8, 16, 100, 1000, 8192, 70000])
def test_layer_norm_partial_rows(code, dim):
    """At least one for each 512 rows that a lane adds (256 rows side by side where a row is a thread's, 16 where 16 lanes
    have it), few of them where rows are few, and never more than rows."""
    n = ctypes.c_int64(-1)
    group = 16 // SIZES[code]
    side = 256 if dim < group else 16 if dim <= 16 * group else 4 if dim <= 128 * group else 1
    for rows in (0, 1, 500, 100000, 1 << 22, (1 << 31) - 1):
        assert call("qnn_layer_norm_bwd_work", rows, dim, code, ctypes.byref(n))[0] == 0
        parts, rest = divmod(n.value, 8 * dim)
        assert rest == 0 and rows <= 512 * side * parts and parts <= rows
        assert parts <= max(512, -(-rows // (512 * side)))
    assert call("qnn_layer_norm_bwd_work", 5, dim, 3, ctypes.byref(n))[0] == 1


@pytest.mark.parametrize("code", SIZES)
@pytest.mark.parametrize("n,k", [(1, 1), (64, 64), (4096, 8192), (4099, 8191), (1 << 21, 1 << 21)])
def test_linear_act_work_of_no_rows(code, n, k):
    """None; for a large weight of a 16-bit type the plan of no tiles divided by their number, which ended the process."""
    size = ctypes.c_int64(-1)
    for name in ("qnn_linear_act_fwd_work", "qnn_linear_act_bwd_work"):
        assert call(name, 0, n, k, code, ctypes.byref(size))[0] == 0 and size.value == 0
        size.value = -1


THREADS = {(256, 256): 512, (128, 128): 512, (128, 64): 256, (64, 64): 256, (32, 64): 128}


@pytest.mark.parametrize("code", SIZES)
@pytest.mark.parametrize("n,k", [(8, 8), (1, 8), (8, 1), (64, 64), (65, 24), (7, 3), (31, 31)])
def test_linear_act_tiles_fit_a_launch(code, n, k):
    """To two thousand million rows the plan takes tiles whose launch can be made."""
    tm, tn, sp = ctypes.c_int(), ctypes.c_int(), (ctypes.c_int * 2)()
    for m in (1 << 29, (1 << 30) - 1, 1 << 30, 2_000_000_000):
        if m * (n + k) * SIZES[code] > 1 << 38:  # what no card holds
            continue
        for grads in (0, 1):
            assert call("qnn_linear_act_plan", m, n, k, code, grads, ctypes.byref(tm), ctypes.byref(tn), sp)[0] == 0
            tiles = lambda rows, cols: -(-rows // tm.value) * -(-cols // tn.value)
            blocks = tiles(m, k) * sp[0] + tiles(n, k) * sp[1] if grads else tiles(m, n) * sp[0]
            assert blocks * THREADS[tm.value, tn.value] < 1 << 32, (m, grads, tm.value, tn.value)


@pytest.mark.parametrize("code", SIZES)
@pytest.mark.parametrize("n,k", [(2048, 8), (8, 2048), (2048, 2048), (2047, 31)])
def test_linear_act_tiles_past_a_launch(code, n, k):
    m = (1 << 31) - 1
    if n > 8:
        rc, msg = call("qnn_linear_act_fwd", P, k, P, k, None, None, 0, P, None, m, n, k, code, 0, P, 1 << 62, None)
        assert rc == 1 and b"too many rows" in msg
    if k > 8:
        for act in (0, 2):  # (GELU: before its dz is launched)
            rc, msg = call("qnn_linear_act_bwd", P, n, P, P, k, P, k, P, P, P, P, m, n, k, code, act, P, 1 << 62, None)
            assert rc == 1 and b"too many rows" in msg


@pytest.mark.parametrize("code", [1, 2])
def test_linear_act_padding_past_a_launch(code):
    """Rows that are padded: 2^32 groups of 16 bytes are too many."""
    n, k = 64, 1031
    rc, msg = call("qnn_linear_act_bwd", P, n, None, P, k, P, k, None, None, P, None, 1 << 25, n, k, code, 0, P, 1 << 62, None)
    assert rc == 1 and b"too many rows" in msg


@pytest.mark.parametrize("code", SIZES)
@pytest.mark.parametrize("n", [1, 8, 600, 100000])
def test_linear_act_strips_of_rows(code, n):
    """The bias's gradient has a partial row for each 2048 rows at least: 512 that a lane adds."""
    size = ctypes.c_int64(-1)
    for m in (1000, 3_000_000, 1 << 26, (1 << 31) - 1):
        if m * n > 1 << 37:
            continue
        assert call("qnn_linear_act_bwd_work", m, n, 8, code, ctypes.byref(size))[0] == 0
        assert size.value >= -(-m // 2048) * n * 4 * (m > 256)
