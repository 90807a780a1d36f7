"""How long rows may be: a tile's rows are addressed by 32-bit offsets from its first, so tiles of long
rows are lower, and what 64 rows cannot reach is refused.  The plan answers without a GPU."""
import ctypes

import pytest

from rocm_qlora import _native as nat
from rocm_qlora import ops

UNSUPPORTED = 5
FAR = 1 << 32


def reached(rows, pitch):
    """The last row's last 128 bytes of a step from the first row's."""
    return (rows - 1) * pitch * 2 + 128 <= FAR


def tiles(M, K, N, dx=0, dtype=nat.DTYPE_BF16, E=1, grouped=0, bits=16, shared=1):
    """Rows of a tile, splits, whether the rows are copied; None where the call is refused."""
    out = (ctypes.c_int32 * 3)()
    status = nat.load().rq_mx4_tile_plan(dtype, M, K, N, E, shared, grouped, bits, dx, N if dx else K, 1, out)
    if status == UNSUPPORTED:
        return None
    assert status == 0, status
    return tuple(out)


# (8421504 is the longest row of which 256 are reached)
@pytest.mark.parametrize("dtype", [nat.DTYPE_BF16, nat.DTYPE_F16, nat.DTYPE_F32])
@pytest.mark.parametrize("M,K,N", [(512, 1 << 24, 2048), (2048, 9_000_000, 1024), (512, 8421504, 2048), (512, 8421505, 2048), (1024, 8388609, 2048),
                                   (2048, 1 << 24, 2048), (1024, 8388608, 1024)])
def test_rows_of_a_tile_lie_within_4_gib(M, K, N, dtype):
    bm, splits, copied = tiles(M, K, N, dtype=dtype)
    assert copied and bm >= 64 and splits >= 1
    assert reached(min(bm, M), ops.mx4_pad(K))


@pytest.mark.parametrize("M,K,N", [(256, 1024, 1 << 24), (2048, 1920, (1 << 24) + 64), (300, 700, (1 << 25) - 70), (4096, 2048, 1 << 24)])
def test_rows_of_a_gradient_tile_lie_within_4_gib(M, K, N):
    bm, _, copied = tiles(M, K, N, dx=1)
    assert copied and reached(min(bm, M), -(-N // 64) * 64)


def test_experts_tiles_of_copied_slots():
    """Rows that 32-bit offsets do not reach are copied in the plan's order, and the copy's tiles keep the bound."""
    for M, K, N, E in ((2048, 1 << 24, 2048, 2), (4096, 9_000_000, 1024, 3)):
        bm, _, copied = tiles(M, K, N, E=E, grouped=1)
        assert copied and reached(bm, ops.mx4_pad(K))


def test_what_64_rows_cannot_reach_is_refused():
    for M, K, N in ((64, 128, 40_000_000), (64, 128, 34_087_041), (4096, 100, 1 << 26), (17, 64, 1 << 27)):
        assert tiles(M, K, N, dx=1) is None, (M, K, N)
        n = ctypes.c_int64(-1)
        assert nat.load().rq_mx4_linear_scratch_size(1, M, K, N, 1, 1, 0, 16, 1, N, 1, ctypes.byref(n)) == UNSUPPORTED
        a = 4096  # an address that is never read
        assert nat.load().rq_mx4_linear_dx(a, 1, M, N, N, None, 0, a, a, 1, K, 1, a, K, None, 0, None) == UNSUPPORTED
    assert tiles(64, 128, 40_000_000, dx=1, E=2, grouped=1) is None
    # the largest that are reached, and fewer rows than a tile
    for M, K, N in ((64, 128, 34_087_040), (63, 128, 34_000_000), (16, 64, 1 << 27), (1, 64, 1 << 28)):
        assert tiles(M, K, N, dx=1) is not None, (M, K, N)


def test_sizes_that_were_in_reach_keep_their_tiles():
    assert tiles(4096, 4096, 14336)[0] == 256 and tiles(4096, 4096, 14336, dx=1)[0] == 128
    assert tiles(2048, 8388608, 1024)[0] == 256 and tiles(512, 8421504, 2048)[0] == 256
    assert tiles(512, 8421505, 2048)[0] == 128
    assert tiles(1, 4096, 4096) == (0, 0, 0)
    assert tiles(4096, 4096, 14336, bits=4)[0] == 256


def test_arguments():
    out = (ctypes.c_int32 * 3)()
    f = nat.load().rq_mx4_tile_plan
    assert f(1, 8, 64, 16, 1, 1, 0, 16, 0, 64, 1, None) == 1
    assert f(9, 8, 64, 16, 1, 1, 0, 16, 0, 64, 1, out) == 2
    assert f(1, 0, 64, 16, 1, 1, 0, 16, 0, 64, 1, out) == 3 and f(1, 8, 64, 16, 1, 1, 0, 16, 0, 63, 1, out) == 3
