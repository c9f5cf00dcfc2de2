"""The MXFP4 x MXFP4 matmul where no sum rounds: the outputs bit for bit.

x holds E2M1 values times 1 or 2 with a 6 in every block, so that the quantiser
keeps them; the weights' scales are 1/2, 1 or 2.  Products are multiples of
1/2 * 1/2 * 1/2 of at most 6 * 6 * 4, so a sum of K of them is a multiple of 2^-3
below 2^7.2 K, which f32 holds for K up to 2^13.8 whatever the order.  A block, a
column of K or a split left out, taken twice or misplaced changes it; the bounds
of test_mxfp4_gemm_gpu.py, relative to sums of magnitudes, need not see that."""
import numpy as np
import pytest

from conftest import announce
from test_mxfp4_gemm_gpu import SHAPES, _as, _t

pytestmark = pytest.mark.gpu

E2M1 = np.array([0, .5, 1, 1.5, 2, 3, 4, 6], np.float32)


def _inputs(orc, m, k, n):
    rng = np.random.default_rng(m + k + n)
    x = E2M1[rng.integers(0, 8, (m, k))] * rng.choice(np.float32([-1, 1]), (m, k))
    b = x.reshape(m, k // 32, 32)
    np.put_along_axis(b, rng.integers(0, 32, (m, k // 32, 1)), np.float32(6.0), 2)
    x = (b * rng.choice(np.float32([1, 2]), (m, k // 32, 1))).reshape(m, k)
    codes, eb = rng.integers(0, 256, (n, k // 2), dtype=np.uint8), rng.integers(126, 129, (n, k // 32), dtype=np.uint8)
    return x, codes, eb, x.astype(np.float64) @ orc.mxfp4_dequantize(codes, eb, n, k).astype(np.float64).T


def _check(ctx, orc, shape, xdt, ydt):
    import torch

    m, k, n = shape
    x, codes, eb, want = _inputs(orc, m, k, n)
    assert np.array_equal(want, want.astype(np.float32))
    y = ctx.mxfp4_gemm(_as(x, xdt)[0], _t(codes), _t(eb), n, y_dtype=torch.bfloat16 if ydt == "bf16" else torch.float32)
    torch.cuda.synchronize()
    w = torch.from_numpy(want.astype(np.float32))
    assert torch.equal(y.cpu(), w.to(torch.bfloat16) if ydt == "bf16" else w)


@pytest.mark.parametrize("xdt,ydt", [("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_shapes(ctx, orc, shape, xdt, ydt):
    announce(f"mxfp4_gemm exact {shape} x={xdt} y={ydt}")
    _check(ctx, orc, shape, xdt, ydt)


@pytest.mark.parametrize("cfg", ["m256n256", "m256n256,3", "m128n128", "m128n128,2", "m128n64", "m128n64,4", "m64n64",
                                 "m64n64,2"])
@pytest.mark.parametrize("shape", [(70, 2336, 264), (130, 800, 301), (512, 1152, 520), (197, 4096, 384)],
                         ids=lambda s: "x".join(map(str, s)))
def test_every_tiling(ctx, orc, monkeypatch, shape, cfg):
    announce(f"mxfp4_gemm exact {cfg} {shape}")
    monkeypatch.setenv("RLXQ_MX_CFG", cfg)
    _check(ctx, orc, shape, "f32", "f32")
