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


def test_rows_that_a_product_left_apart_are_summed_over_ranks_as_one_block():
    """Results of a number of features that is no multiple of eight lie in wider rows, which a collective does not take."""
    import torch

    from lorax_b200.models.decoder import DecoderModel, Int8Weight
    from lorax_b200.ops import reference as ref
    taken = []

    class Ops:
        quant_rows_int8 = staticmethod(ref.quant_rows_int8)

        @staticmethod
        def gemm_int8(x, w, w_scale, bias=None, dtype=None, w_const=False):
            T, N = x.q.shape[0], w.shape[0]
            return ref.gemm_int8(x, w, w_scale, bias, out=torch.empty(T, (N + 7) // 8 * 8)[:, :N], dtype=dtype)

    class Ranks:
        world_size, fused = 2, None

        @staticmethod
        def all_reduce(x):
            taken.append(x.is_contiguous())
            return 2 * x
    m = DecoderModel.__new__(DecoderModel)
    m.ops, m.tp, m.adapters, m.dtype = Ops, Ranks, None, torch.float32
    w, ws = ref.quantize_weight_int8(torch.randn(13, 32))
    x = torch.randn(3, 32)
    y = m._row_parallel(x, Int8Weight(w, ws), None, "o", 0, type("Step", (), dict(tok_slot=None, lora_tiles=None))())
    assert taken == [True]
    torch.testing.assert_close(y, 2 * ref.gemm_int8(ref.quant_rows_int8(x), w, ws, dtype=torch.float32))
