"""Sizes past what a call can launch or count: refused with RLXQ_E_SHAPE before
anything is queued, whatever the pointers hold (none is read)."""
import ctypes as C

import pytest

from conftest import announce

pytestmark = pytest.mark.gpu

GGUF_Q4_1, F32 = 3, 0


@pytest.fixture
def buf():
    import torch

    return torch.full((1 << 16,), 7, dtype=torch.uint8, device="cuda")


def _unchanged(buf):
    import torch

    torch.cuda.synchronize()
    assert bool((buf == 7).all())


# rows x top_k in 64 bits is 0, 4, too large, -2, or just too large
PAIRS = [(2 ** 62, 4), (2 ** 62 + 1, 4), (2 ** 61 + 3, 3), (2 ** 63 - 1, 2), (2 ** 28 + 1, 1), (2 ** 26 + 1, 4)]


@pytest.mark.parametrize("rows,top_k", PAIRS)
def test_rows_times_top_k(ctx, buf, rows, top_k):
    import rlxq

    announce(f"rows {rows} top_k {top_k}")
    L, p = rlxq.lib(), C.c_void_p(buf.data_ptr())
    for logits, router in ((p, None), (None, p)):
        assert L.rlxq_moe_layer(ctx.h, p, F32, router, F32, logits, GGUF_Q4_1, p, None, GGUF_Q4_1, p, None, rows, 32, 32, 8,
                                top_k, 1, None, None, p, F32, None) == rlxq.E_SHAPE
        assert b"2^28" in L.rlxq_last_error(ctx.h)
    for mode in (rlxq.MOE_EXPAND, rlxq.MOE_COMBINE, rlxq.MOE_EXPAND_SWIGLU):
        assert L.rlxq_moe_grouped(ctx.h, GGUF_Q4_1, mode, p, F32, p, p, p, rows, top_k, 32, 32, 8, p, F32,
                                  None) == rlxq.E_SHAPE
        assert b"2^28" in L.rlxq_last_error(ctx.h)
    _unchanged(buf)


def test_layer_rows(ctx, buf):
    """A wave a row: 2^26 rows are 2^32 work-items."""
    import rlxq

    L, p = rlxq.lib(), C.c_void_p(buf.data_ptr())
    announce("moe_layer 2^26 rows")
    assert L.rlxq_moe_layer(ctx.h, p, F32, None, F32, p, GGUF_Q4_1, p, None, GGUF_Q4_1, p, None, 2 ** 26, 32, 32, 8, 1, 1, p, p,
                            p, F32, None) == rlxq.E_SHAPE
    assert b"2^26" in L.rlxq_last_error(ctx.h)
    announce("moe_layer 2^20 rows of 4096 columns")   # (the weighted sum: a work-item an output)
    assert L.rlxq_moe_layer(ctx.h, p, F32, None, F32, p, GGUF_Q4_1, p, None, GGUF_Q4_1, p, None, 2 ** 20, 4096, 32, 8, 1, 1, p,
                            p, p, F32, None) == rlxq.E_SHAPE
    assert b"2^32 work-items" in L.rlxq_last_error(ctx.h)
    _unchanged(buf)


def test_layer_rows_beyond_lds(ctx, buf):
    """Rows of f32 activations whose records do not fit LDS, where no other
    kernel takes them: nothing of the layer is queued, the ids stay as they are."""
    import rlxq

    L, p = rlxq.lib(), C.c_void_p(buf.data_ptr())
    announce("moe_layer 40 rows of 32768")
    assert L.rlxq_moe_layer(ctx.h, p, F32, p, F32, None, GGUF_Q4_1, p, None, GGUF_Q4_1, p, None, 40, 32768, 32, 64, 1, 1, p, p,
                            p, F32, None) == rlxq.E_SHAPE
    assert b"LDS" in L.rlxq_last_error(ctx.h)
    _unchanged(buf)


def test_mxfp4_launches(ctx, buf):
    import rlxq

    L, p = rlxq.lib(), C.c_void_p(buf.data_ptr())
    announce("quantize_mxfp4 2^37 elements")
    assert L.rlxq_quantize_mxfp4(ctx.h, p, F32, 2 ** 26, 2 ** 11, p, p, None) == rlxq.E_SHAPE
    assert b"2^37" in L.rlxq_last_error(ctx.h)
    announce("dequantize 2^36 weights")
    assert L.rlxq_dequantize(ctx.h, rlxq.MLX_MXFP4, 32, p, p, None, rlxq.U8, 2 ** 26, 2 ** 10, p, None) == rlxq.E_SHAPE
    assert b"2^36" in L.rlxq_last_error(ctx.h)
    # rows and columns whose launches are too large: decode, its preparation
    # (fewer rows of more elements), the tiles' preparation, the tiles
    for m, k, n in ((1, 32, 2 ** 30), (33, 32, 2 ** 29), (2 ** 29, 32, 64), (2 ** 22, 64, 2 ** 22)):
        announce(f"mxfp4_gemm {m} x {k} x {n}")
        assert L.rlxq_mxfp4_gemm(ctx.h, p, F32, p, p, m, k, n, p, F32, None) == rlxq.E_SHAPE
        assert b"2^32 work-items" in L.rlxq_last_error(ctx.h)
    _unchanged(buf)
