"""The expert layer on MXFP4 scales far from one: scale bytes up to 255 and down
to 0 against activations whose products with them are ordinary, or zero because
the codes are.  Bounds as in test_moe_layer_gpu.py."""
import numpy as np
import pytest

from conftest import announce
from test_moe_layer_gpu import Layer, _as, _t

pytestmark = pytest.mark.gpu


def _values(orc, codes, scales):
    return orc.mxfp4_dequantize(codes, scales, codes.shape[0], codes.shape[1] * 2).astype(np.float64)


@pytest.mark.parametrize("xdt", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 3, 14, 40])
def test_far_scales(ctx, orc, rows, xdt):
    """gate|up: block 1 has byte 254 or 255 over zero codes, on rows of 2^20;
    block 2 2^105 on rows of 2^-104; block 3 byte 0 on rows of 2^30; block 4
    2^-100 on rows of 2^99.  down: block 1 255 over zero codes, on activations
    beyond 2^15."""
    import torch

    announce(f"moe_layer far scales rows={rows} x={xdt}")
    H, I, E, K = 256, 128, 4, 2
    rng = np.random.default_rng(rows)
    L = Layer(orc, rng, rows, H, I, E, K, "mxfp4", "mxfp4", xdt=xdt)
    x = rng.standard_normal((rows, H)).astype(np.float32)
    for b, e in ((1, 20), (2, -104), (3, 30), (4, 99)):
        x[:, 32 * b:32 * b + 32] *= np.float32(2.0 ** e)
    L.x, xv = _as(x, xdt)
    L.xv = xv.astype(np.float64)
    g, gs = rng.integers(0, 256, (E * 2 * I, H // 2), dtype=np.uint8), rng.integers(119, 123, (E * 2 * I, H // 32), dtype=np.uint8)
    g[:, 16:32] &= 0x88   # (zeros of both signs)
    gs[:, 1] = np.resize(np.array([254, 255], np.uint8), len(gs))
    gs[:, 2], gs[:, 3], gs[:, 4] = 127 + 105, 0, 127 - 100
    gs[:, 5] = 127 + 7    # (activations of some 2^20)
    d, ds = rng.integers(0, 256, (E * H, I // 2), dtype=np.uint8), rng.integers(119, 123, (E * H, I // 32), dtype=np.uint8)
    d[:, 16:32] &= 0x88
    ds[:, 1] = 255
    L.g, L.gs, L.d, L.ds = _t(g), _t(gs), _t(d), _t(ds)
    L.gv, L.dv = _values(orc, g, gs).reshape(E, 2 * I, H), _values(orc, d, ds).reshape(E, H, I)
    logits = rng.standard_normal((rows, E)).astype(np.float32)
    ids, p, gap, big = L.route(True, logits)
    a = np.abs(np.stack([L.gv[e] @ L.xv[0] for e in ids[0]]))
    assert gap > 1e-6 and (a[:, :I] * a[:, I:])[:, 32:64].max() > 2 ** 16
    y = L.call(ctx, router=None, logits=_t(logits))
    torch.cuda.synchronize()
    assert torch.isfinite(y).all()
    L.check(y, ids, p, big)
