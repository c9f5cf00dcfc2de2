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
