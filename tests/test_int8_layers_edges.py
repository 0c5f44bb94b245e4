"""Operators of layers in 8-bit integers on the CPU: sizes at the ends of what the library takes."""
import ctypes

import pytest

MOST = 0x7fff0000                       # rows and channels that the library takes


def _plan(T, N, K, sms=148, clusters=(74, 33, 22, 15)):
    """(the library's answer, (pairs, tokens a tile, parts, stages))"""
    from lorax_b200.ops import native
    out = (ctypes.c_int * 4)()
    return native.load().lx_gemm_int8_plan(T, N, K, sms, (ctypes.c_int * 4)(*clusters), out), tuple(out)


@pytest.mark.parametrize("clusters", [(74, 33, 22, 15), (0, 0, 0, 0)])
@pytest.mark.parametrize("T,N,K", [(MOST, 1, 16), (2139128000, 128, 4096), (2139127700, 1, 16), (MOST, 4096, 128), (1, MOST, 16), (33, MOST, 4096), (2000, 2139128000, 128)])
def test_plans_of_rows_and_channels_near_the_most_that_are_taken(T, N, K, clusters):
    """Rows evened out over millions of tiles: no sum on the way passes 31 bits."""
    rc, (pairs, bn, parts, stages) = _plan(T, N, K, clusters=clusters)
    assert rc == 0 and 16 <= bn <= 256 and bn % (32 if pairs else 16) == 0 and 1 <= parts <= -(-K // 128)
    assert pairs >= 0 and (pairs > 0 or 4 <= stages <= 16)


def test_tiles_whose_number_passes_31_bits_are_refused():
    """The kernels count a product's tiles in 32 bits."""
    for T, N in ((MOST, MOST), (1 << 30, 1 << 28)):
        assert _plan(T, N, 16)[0] == -1001
    assert _plan(1 << 20, 1 << 20, 16)[0] == 0                   # 2^16 tiles of 16 rows by 2^13 of channels at most
