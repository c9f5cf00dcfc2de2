"""Accuracy of the whole expert layer beside its worst-case bounds: the RMS error
over the RMS of y against float64, which a rounding or an element too many
cannot hide in.

Bound of the grouped products (f32 between them): a factor held as a high and a
low part is off by at most 2^-16 of itself, evenly spread and of either sign: 2^-16
/ sqrt(3) / 1.4 = 6.3e-6 RMS over a binade.  Unsigned 4-bit codes carry it ahead of
their minimum: their RMS is sqrt(77.5) = 8.8 where the centred weight's is 4.6, so
1.9 times of it reaches a dot product, 1.2e-5 of its RMS; f32 sums of some 100
additions add 1e-6.  silu(g) u holds two such errors (a slope of 1.1 at most), down
one more: sqrt(1 + 1.1^2 + 1) 1.2e-5 = 2.1e-5.  GROUPED takes 2^-15 = 3.1e-5, for
the formats tested here (the minima of the generated Q5_K and Q2_K banks are
further from their codes' mean).
Activations rounded to bf16 (at most 2^-8, 2^-8 / sqrt(3) / 1.4 RMS over
a binade) are 1.6e-3 off.

Bound of the few-token kernels: f32 rows and the gated activations as two f16
planes (off by at most 2^-22), codes exact, so what is left is f32 sums: at most
64 additions of a block's products, K / 32 / 8 of its lane's blocks and 4 across
lanes, each off by 2^-24 / sqrt(3) RMS of a partial sum that stays below 4 times
the RMS of the dot product (unsigned codes ahead of their minimum): sqrt(64 + 16
+ 4) 4 2^-24 / sqrt(3) = 1.3e-6 for K up to 4096, over the products as above
sqrt(1 + 1.1^2 + 1) 1.3e-6 = 2.3e-6.  FEW takes 2^-18 = 3.8e-6."""
import numpy as np
import pytest

from conftest import announce
from test_moe_layer_gpu import GGUF, Layer, _bank, _t

GROUPED, FEW = 2.0 ** -15, 2.0 ** -18


def _bf16(v):
    import torch

    return torch.from_numpy(np.ascontiguousarray(v, np.float32)).to(torch.bfloat16).float().numpy().astype(np.float64)


class Values:
    """A layer's inputs as float64 (and packed), with logits of the caller's that
    give every slot weight."""

    def __init__(self, orc, rows, hidden, inter, experts, top_k, gu, down, xdt, seed=0):
        rng = np.random.default_rng(seed + rows + hidden + inter)
        self.shape, self.names, self.xdt = (rows, hidden, inter, experts, top_k), (gu, down), xdt
        self.g, self.gs, gv = _bank(orc, gu, rng, experts * 2 * inter, hidden)
        self.d, self.ds, dv = _bank(orc, down, rng, experts * hidden, inter)
        self.gv, self.dv = gv.reshape(experts, 2 * inter, hidden), dv.reshape(experts, hidden, inter)
        x = rng.standard_normal((rows, hidden)) / max(1.0, float(np.std(self.gv)) * hidden ** 0.5 / 2)
        self.x = _bf16(x) if xdt == "bf16" else x.astype(np.float32).astype(np.float64)
        self.logits = (rng.standard_normal((rows, experts)) * 0.1).astype(np.float32)
        l = self.logits.astype(np.float64)
        self.ids = np.argsort(-l, axis=1, kind="stable")[:, :top_k]
        p = np.exp(np.take_along_axis(l, self.ids, 1))
        self.p = p / p.sum(1, keepdims=True)

    def forward(self, x=lambda v: v, a=lambda v: v, slots=None):
        """y in float64, with x and the gated activations passed through the
        functions given, over the first `slots` slots."""
        rows, hidden, inter, _, top_k = self.shape
        y = np.zeros((rows, hidden))
        for r in range(rows):
            v = x(self.x[r])
            for j in range(slots or top_k):
                e = self.ids[r, j]
                gu = self.gv[e] @ v
                y[r] += self.p[r, j] * (self.dv[e] @ a(gu[:inter] / (1 + np.exp(-gu[:inter])) * gu[inter:]))
        return y

    def call(self, ctx, y_dtype):
        import rlxq
        import torch

        rows, hidden, inter, experts, top_k = self.shape
        x = torch.from_numpy(self.x.astype(np.float32)).to(torch.bfloat16 if self.xdt == "bf16" else torch.float32).cuda()
        sch = [rlxq.MLX_MXFP4 if n == "mxfp4" else GGUF[n] for n in self.names]
        gs, ds = (None if s is None else _t(s) for s in (self.gs, self.ds))
        y = ctx.moe_layer(x, None, _t(self.g), _t(self.d), sch[0], sch[1], top_k, inter, experts, logits=_t(self.logits),
                          gate_up_scales=gs, down_scales=ds, y_dtype=y_dtype)
        torch.cuda.synchronize()
        return y.double().cpu().numpy()


def _rms(v):
    return float(np.sqrt(np.mean(v * v)))


# (rows, hidden, inter, experts, top_k): experts too wide for the few-token
# kernels, few and many entries an expert
GROUPED_SHAPES = [(1, 256, 5632, 8, 7), (40, 512, 256, 24, 4), (70, 256, 256, 9, 3), (200, 512, 256, 4, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("xdt", ["bf16", "f32"])
@pytest.mark.parametrize("name", ["mxfp4", "q4_1", "q8_0", "q4_k"])
@pytest.mark.parametrize("shape", GROUPED_SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_grouped_products_keep_f32_between_them(ctx, orc, shape, name, xdt):
    import torch

    announce(f"moe_layer accuracy {shape} {name} x={xdt}")
    v = Values(orc, *shape, name, name, xdt)
    want = v.forward()
    err = _rms(v.call(ctx, torch.float32) - want) / _rms(want)
    assert "moefew" not in ctx.last_kernel
    assert err <= GROUPED, f"{err:.2e}"


@pytest.mark.gpu
def test_wide_down_rows_are_served(ctx, orc):
    """inter past what LDS holds of an f32 row: bf16 x still gives f32 y, each
    activation off by at most 2^-8 of itself.  How far that moves y depends on how
    its terms cancel: the bound is the element-wise one of test_moe_layer_gpu.py,
    with 2^-8 |a| among the errors of an activation."""
    import rlxq
    import torch

    announce("moe_layer inter 20480")
    v = Values(orc, 2, 32, 20480, 3, 2, "q4_1", "q4_1", "bf16")
    L = Layer.__new__(Layer)
    L.shape, L.xdt, L.xv, L.gv, L.dv = v.shape, v.xdt, v.x, v.gv, v.dv
    L.check(torch.from_numpy(v.call(ctx, torch.float32)), v.ids, v.p, float(np.abs(v.logits).max()), act_eps=2.0 ** -8)
    assert rlxq.lib().rlxq_last_error(ctx.h) == b""


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["mxfp4", "q4_1"])
def test_more_f32_activations_than_the_matrix_kernels_hold(ctx, orc, name):
    """bf16 x, f32 y and more than 1 GiB of gathered f32 activations: down runs in
    pieces of rows (the last one shorter), each row as in a call of its own size."""
    import torch

    rows, times = 37, 541   # 20017 rows of 14336 activations
    announce(f"moe_layer {rows * times} rows of inter 14336 {name}")
    v = Values(orc, rows, 32, 14336, 2, 1, name, name, "bf16")
    want = v.forward()
    v.x, v.logits = np.tile(v.x, (times, 1)), np.tile(v.logits, (times, 1))
    v.shape = (rows * times,) + v.shape[1:]
    y = v.call(ctx, torch.float32).reshape(times, rows, 32)
    assert _rms(y - want) <= GROUPED * _rms(want)
    assert max(_rms(t - want) for t in y) <= GROUPED * _rms(want)


def test_the_bound_sees_bf16_activations(orc):
    """On the CPU: a forward that rounds the activations between the products to
    bf16 is far outside the bound."""
    v = Values(orc, 3, 512, 256, 6, 2, "q4_1", "q4_1", "bf16")
    want = v.forward()
    assert _rms(v.forward(a=_bf16) - want) > 16 * GROUPED * _rms(want)


# every format, wide and narrow layers, up to 64 slots of nearly even weight, one
# and four entries a pass
FEW_CASES = [((3, 512, 256, 6, 2), n, n) for n in ("mxfp4", *GGUF)] + [
    ((1, 4096, 1536, 4, 3), "mxfp4", "q4_k"), ((7, 2048, 768, 9, 8), "mxfp4", "mxfp4"), ((7, 2048, 768, 9, 8), "q4_1", "q4_1"),
    ((16, 1024, 512, 12, 4), "q4_k", "q6_k"), ((32, 512, 256, 40, 8), "q8_0", "mxfp4"), ((4, 256, 64, 65, 64), "q8_0", "q4_0"),
    ((1, 128, 96, 70, 64), "mxfp4", "q4_1"), ((24, 1056, 160, 12, 3), "q4_1", "mxfp4")]


def _few_id(c):
    return "-".join(["x".join(map(str, c[0])), *c[1:]])


@pytest.mark.gpu
@pytest.mark.parametrize("xdt", ["bf16", "f32"])
@pytest.mark.parametrize("case", FEW_CASES, ids=_few_id)
def test_few_tokens(ctx, orc, case, xdt):
    import torch

    announce(f"moe_layer accuracy {case} x={xdt}")
    v = Values(orc, *case[0], *case[1:], xdt)
    want = v.forward()
    err = _rms(v.call(ctx, torch.float32) - want) / _rms(want)
    assert "moefew" in ctx.last_kernel
    assert err <= FEW, f"{err:.2e}"


def _f16(v):
    """One f16 plane per 32 elements, the remainder plane lost."""
    b = v.reshape(-1, 32)
    s = 2.0 ** (14 - np.floor(np.log2(np.abs(b).max(1, keepdims=True))))
    return ((b * s).astype(np.float16).astype(np.float64) / s).reshape(v.shape)


def _without(i):
    def f(v):
        v = v.copy()
        v[i] = 0.0
        return v

    return f


@pytest.mark.parametrize("case", [c for c in FEW_CASES if c[0][0] * c[0][4] <= 64] + [((4, 256, 64, 65, 64), "q8_0", "q4_0")],
                         ids=_few_id)
def test_the_bound_sees_what_is_lost(orc, case):
    """On the CPU: forwards that lose the remainder plane of the rows or of the
    activations, the last element of either, or the last slot, are far outside
    the few-token bound."""
    v = Values(orc, *case[0], *case[1:], "f32")
    want = v.forward()
    far = 4 * FEW * _rms(want)
    assert _rms(v.forward(x=_f16) - want) > far
    assert _rms(v.forward(a=_f16) - want) > far
    assert _rms(v.forward(x=_without(-1)) - want) > far
    assert _rms(v.forward(a=_without(-1)) - want) > far
    if case[0][4] > 1:
        assert _rms(v.forward(slots=case[0][4] - 1) - want) > far
