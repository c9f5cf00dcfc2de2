"""The whole expert layer (rlxq_moe_layer) against float64, element by element.

Bounds.  A dot product of K elements with packed weights: the kernels split f32
activations into two halves (each element off by at most 2^-16 of itself) or
take bf16 ones as they are, and add code products to f32 sums, 32 additions in
a block whose partial sums stay below 20 times the block's sum |x| times its
largest |w| (codes carry an offset of up to 1152, or 8 to 10 times the largest
code, and a minimum may cancel half of d * code), then K / 32 blocks:
  d(x . w) <= (2^-16 + (32 * 20 + K / 32) * 2^-24) * sum_blocks (sum |x|) (max |w|).
silu has a slope of at most 1.1, and exp and the division keep 2^-20:
  da <= 1.1 |u| dg + |silu(g)| du + 1.1 dg du + 2^-20 |a|   (+ 2^-8 |a| where
a is rounded to bf16, half a step).  Softmax weights: the logits are off by
2^-24 of themselves (one rounding of an f64 sum), exp and the sums by (E + 8)
2^-23.  The weighted sum adds its own top_k roundings, a bf16 y 2^-8 |y|."""
import numpy as np
import pytest

from conftest import announce

pytestmark = pytest.mark.gpu

GGUF = {"q8_0": 1, "q4_0": 2, "q4_1": 3, "q4_k": 7, "q6_k": 8, "q5_k": 10, "q3_k": 11, "q2_k": 12, "q8_k": 13}
MX = 9


def _t(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _as(x32, xdt):
    import torch

    t = torch.from_numpy(np.ascontiguousarray(x32))
    if xdt == "f32":
        return t.cuda(), x32
    t = t.to(torch.bfloat16)
    return t.cuda(), t.float().numpy()


def _bank(orc, name, rng, rows, k, scale=0.05):
    """(packed, scales or None, values f64 [rows, k]) around `scale` in size."""
    if name == "mxfp4":
        codes = rng.integers(0, 256, (rows, k // 2), dtype=np.uint8)
        eb = rng.integers(119, 123, (rows, k // 32), dtype=np.uint8)
        return codes, eb, orc.mxfp4_dequantize(codes, eb, rows, k)
    w = (rng.standard_normal((rows, k)) * scale).astype(np.float32)
    if name in ("q8_0", "q4_0", "q4_1"):
        packed = orc.quantize(GGUF[name], w)
    else:
        packed = orc.synth(GGUF[name], rng, rows, k)
    return packed, None, orc.dequantize(GGUF[name], packed, k).astype(np.float64).reshape(rows, k)


class Layer:
    """A layer's inputs, on the device and as float64."""

    def __init__(self, orc, rng, rows, hidden, inter, experts, top_k, gu="q4_1", down="q4_1", xdt="f32", rdt="f32"):
        self.shape = (rows, hidden, inter, experts, top_k)
        self.names, self.xdt = (gu, down), xdt
        self.x, xv = _as(rng.standard_normal((rows, hidden)).astype(np.float32), xdt)
        self.r, rv = _as((rng.standard_normal((experts, hidden)) * 2 / hidden ** 0.5).astype(np.float32), rdt)
        self.xv, self.rv = xv.astype(np.float64), rv.astype(np.float64)
        g, gs, gv = _bank(orc, gu, rng, experts * 2 * inter, hidden)
        d, ds, dv = _bank(orc, down, rng, experts * hidden, inter)
        # (K-quant banks of the generator are larger than a trained layer's: activations to match)
        self.gv, self.dv = gv.reshape(experts, 2 * inter, hidden), dv.reshape(experts, hidden, inter)
        f = 1.0 / max(1.0, float(np.std(self.gv)) * hidden ** 0.5 / 2)
        if f < 1.0:
            x32 = (self.xv * 2.0 ** np.floor(np.log2(f))).astype(np.float32)
            self.x, xv = _as(x32, xdt)
            self.xv = xv.astype(np.float64)
        self.g, self.d = _t(g), _t(d)
        self.gs, self.ds = (None if s is None else _t(s) for s in (gs, ds))

    def call(self, ctx, **kw):
        from rlxq import MLX_MXFP4

        rows, hidden, inter, experts, top_k = self.shape
        sch = [MLX_MXFP4 if n == "mxfp4" else GGUF[n] for n in self.names]
        kw.setdefault("router", self.r)
        return ctx.moe_layer(kw.pop("x", self.x), kw.pop("router"), self.g, self.d, sch[0], sch[1], top_k, inter, experts,
                             gate_up_scales=self.gs, down_scales=self.ds, **kw)

    def route(self, renorm=True, logits=None):
        """(ids, probs) in float64, and the smallest gap at a row's border."""
        rows, _, _, experts, top_k = self.shape
        l = self.xv @ self.rv.T if logits is None else logits.astype(np.float64)
        order = np.argsort(-l, axis=1, kind="stable")
        s = np.take_along_axis(l, order, 1)
        gap = np.min(s[:, top_k - 1] - s[:, top_k]) if top_k < experts else 1.0
        p = np.exp(l - l.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        ids = order[:, :top_k]
        p = np.take_along_axis(p, ids, 1)
        return ids, p / p.sum(1, keepdims=True) if renorm else p, gap, np.max(np.abs(l))

    def exact(self, ids, p, big, act_eps=0.0, y_eps=0.0):
        """(y, bound) in float64, for the routing given."""
        rows, hidden, inter, experts, top_k = self.shape
        blk = lambda v: v.reshape(*v.shape[:-1], -1, 32)   # noqa: E731
        eps = lambda k: 2.0 ** -16 + (640 + k / 32) * 2.0 ** -24   # noqa: E731
        dp = 2 * 2.0 ** -24 * max(big, 1.0) + (experts + 8) * 2.0 ** -23
        y, tol = np.zeros((rows, hidden)), np.zeros((rows, hidden))
        gmax, dmax = np.abs(blk(self.gv)).max(-1), np.abs(blk(self.dv)).max(-1)
        for r in range(rows):
            xb = np.abs(blk(self.xv[r])).sum(-1)
            for j in range(top_k):
                e = ids[r, j]
                gu = self.gv[e] @ self.xv[r]
                de = eps(hidden) * (gmax[e] @ xb)
                g, u, dg, du = gu[:inter], gu[inter:], de[:inter], de[inter:]
                silu = g / (1 + np.exp(-g))
                a = silu * u
                da = 1.1 * np.abs(u) * dg + np.abs(silu) * du + 1.1 * dg * du + (2.0 ** -20 + act_eps) * np.abs(a)
                v = self.dv[e] @ a
                dv = np.abs(self.dv[e]) @ da + eps(inter) * (dmax[e] @ np.abs(blk(np.abs(a) + da)).sum(-1))
                y[r] += p[r, j] * v
                tol[r] += p[r, j] * dv + (dp + 2 * top_k * 2.0 ** -24) * p[r, j] * (np.abs(v) + dv)
        return y, tol * (1 + y_eps) + y_eps * np.abs(y)

    def check(self, got, ids, p, big, y_eps=0.0, act_eps=None):
        act_eps = (2.0 ** -8 if self.xdt == "bf16" else 0.0) if act_eps is None else act_eps
        want, tol = self.exact(ids, p, big, act_eps, y_eps)
        err = np.abs(got.double().cpu().numpy() - want)
        assert np.all(err <= tol), f"{np.max(err / tol):.2f} of the bound at worst, largest error {err.max():.3e}"


PAIRS = [(n, n) for n in GGUF] + [("mxfp4", "mxfp4"), ("q4_k", "q6_k"), ("q4_1", "mxfp4"), ("mxfp4", "q8_0")]


@pytest.mark.parametrize("xdt", ["bf16", "f32"])
@pytest.mark.parametrize("pair", PAIRS, ids=lambda p: "-".join(p))
def test_every_format(ctx, orc, pair, xdt):
    import torch

    for rows in (1, 5):
        announce(f"moe_layer {pair} x={xdt} rows={rows}")
        L = Layer(orc, np.random.default_rng(rows), rows, 512, 256, 12, 4, *pair, xdt=xdt)
        ids, p, gap, big = L.route()
        assert gap > 1e-5
        i = torch.empty((rows, 4), dtype=torch.int32, device="cuda")
        q = torch.empty((rows, 4), device="cuda")
        y = L.call(ctx, ids=i, probs=q)
        torch.cuda.synchronize()
        np.testing.assert_array_equal(i.cpu().numpy(), ids)
        np.testing.assert_allclose(q.cpu().numpy(), p, rtol=1e-5)
        L.check(y, ids, p, big)


# (rows, hidden, inter, experts, top_k): odd widths, one expert, all experts,
# more than 64 and 256 experts, many rows (the grouped kernels), wide rows
SHAPES = [(1, 32, 32, 1, 1), (3, 96, 160, 5, 5), (2, 544, 96, 70, 8), (4, 64, 64, 300, 10), (16, 1024, 352, 16, 8),
          (7, 2048, 768, 24, 8), (31, 256, 512, 8, 2), (9, 4096, 64, 6, 3), (2, 288, 4416, 4, 2), (70, 256, 128, 9, 3),
          (200, 512, 256, 4, 2)]


@pytest.mark.parametrize("xdt,ydt", [("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("name", ["mxfp4", "q4_1"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_shapes(ctx, orc, shape, name, xdt, ydt):
    import torch

    announce(f"moe_layer {shape} {name} x={xdt} y={ydt}")
    L = Layer(orc, np.random.default_rng(sum(shape)), *shape, name, name, xdt=xdt, rdt=xdt)
    ids, p, gap, big = L.route()
    assert gap > 1e-6
    y = L.call(ctx, y_dtype=torch.bfloat16 if ydt == "bf16" else torch.float32)
    torch.cuda.synchronize()
    L.check(y, ids, p, big, y_eps=2.0 ** -8 if ydt == "bf16" else 0.0)


@pytest.mark.parametrize("shape", [(3, 8192, 256, 4, 2), (2, 256, 12288, 3, 2), (1, 17408, 32, 2, 1)], ids=str)
def test_long_rows(ctx, orc, shape):
    import torch

    for xdt in ("bf16", "f32"):
        announce(f"moe_layer long rows {shape} x={xdt}")
        L = Layer(orc, np.random.default_rng(1), *shape, "mxfp4", "mxfp4", xdt=xdt)
        ids, p, gap, big = L.route()
        assert gap > 1e-6
        y = L.call(ctx)
        torch.cuda.synchronize()
        L.check(y, ids, p, big)


@pytest.mark.parametrize("rows", [2, 40])
def test_no_renorm_and_callers_logits(ctx, orc, rows):
    """The caller's logits in the place of the router, with and without
    renormalisation, and an expert masked by -inf."""
    import torch

    announce(f"moe_layer logits rows={rows}")
    rng = np.random.default_rng(3)
    L = Layer(orc, rng, rows, 256, 128, 10, 3, "q4_1", "q4_1")
    logits = rng.standard_normal((rows, 10)).astype(np.float32)
    logits[:, 4] = -np.inf
    for renorm in (True, False):
        ids, p, gap, _ = L.route(renorm, logits)
        assert gap > 1e-6 and not np.any(ids == 4)
        y = L.call(ctx, router=None, logits=_t(logits), renorm=renorm)
        torch.cuda.synchronize()
        L.check(y, ids, p, float(np.abs(logits[np.isfinite(logits)]).max()))


@pytest.mark.parametrize("rows", [3, 50])
def test_ties_go_to_the_lower_expert(ctx, orc, rows):
    import torch

    announce(f"moe_layer ties rows={rows}")
    L = Layer(orc, np.random.default_rng(4), rows, 256, 64, 130, 6)
    logits = np.zeros((rows, 130), np.float32)
    logits[0, [129, 7, 100]] = 1.0
    logits[1, ::2] = -0.0
    logits[2, 5:] = -3.0
    want = np.tile(np.arange(6), (rows, 1))
    want[0] = [7, 100, 129, 0, 1, 2]
    want[1] = [0, 1, 2, 3, 4, 5]   # (-0.0 and 0.0 are equal)
    i = torch.empty((rows, 6), dtype=torch.int32, device="cuda")
    L.call(ctx, router=None, logits=_t(logits), ids=i)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(i.cpu().numpy(), want)


@pytest.mark.parametrize("rows", [4, 60])
@pytest.mark.parametrize("via", ["logits", "router"])
def test_rows_without_a_softmax_are_nan(ctx, orc, rows, via):
    """NaN, +inf or nothing but -inf in a row's logits, or an activation that is
    not finite: that row's y is NaN, the others are as without it."""
    import torch

    announce(f"moe_layer NaN rows={rows} {via}")
    rng = np.random.default_rng(5)
    L = Layer(orc, rng, rows, 256, 96, 9, 2, "mxfp4", "mxfp4")
    if via == "logits":
        logits = rng.standard_normal((rows, 9)).astype(np.float32)
        clean = logits.copy()
        logits[0, 3], logits[2, 8], logits[3] = np.nan, np.inf, -np.inf
        y = L.call(ctx, router=None, logits=_t(logits))
        ids, p, gap, big = L.route(True, clean)
    else:
        x = L.x.clone()
        x[0, 3], x[2, 255], x[3, 0] = float("nan"), float("inf"), float("-inf")
        y = L.call(ctx, x=x)
        ids, p, gap, big = L.route()
    torch.cuda.synchronize()
    got = y.cpu().numpy()
    assert gap > 1e-6 and np.all(np.isnan(got[[0, 2, 3]]))
    want, tol = L.exact(ids, p, big)
    ok = [i for i in range(rows) if i not in (0, 2, 3)]
    assert np.all(np.abs(got[ok] - want[ok]) <= tol[ok])


def test_all_rows_on_one_expert(ctx, orc):
    """Every row takes the same experts (a crowded one, and others unused)."""
    import torch

    for rows in (8, 32, 90):
        announce(f"moe_layer one expert rows={rows}")
        rng = np.random.default_rng(6)
        L = Layer(orc, rng, rows, 512, 256, 16, 2, "q4_k", "q6_k")
        logits = rng.standard_normal((rows, 16)).astype(np.float32)
        logits[:, 11] += 20
        logits[:, 2] += 10
        ids, p, gap, big = L.route(True, logits)
        y = L.call(ctx, router=None, logits=_t(logits))
        torch.cuda.synchronize()
        L.check(y, ids, p, big)


@pytest.mark.parametrize("rows", [1, 16, 80])
def test_streams_and_graphs(ctx, orc, rows):
    """A side stream, then a captured call replayed on new inputs between eager
    calls on the same stream: the eager call's bits each time."""
    import torch

    announce(f"moe_layer streams and graphs rows={rows}")
    rng = np.random.default_rng(7)
    L = Layer(orc, rng, rows, 1024, 256, 32, 8, "mxfp4", "mxfp4", xdt="bf16")
    xs = [_as(rng.standard_normal((rows, 1024)).astype(np.float32), "bf16")[0] for _ in range(3)]
    eager = [L.call(ctx, x=x).cpu().numpy() for x in xs]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    x, y = xs[0].clone(), torch.empty((rows, 1024), device="cuda")
    with torch.cuda.stream(st):
        L.call(ctx, x=x, y=y)   # sizes the stream's scratch
    st.synchronize()
    np.testing.assert_array_equal(y.cpu().numpy(), eager[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        L.call(ctx, x=x, y=y)
    for i in (0, 1, 2, 1):
        x.copy_(xs[i])
        y.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(y.cpu().numpy(), eager[i])
        with torch.cuda.stream(st):
            z = L.call(ctx, x=xs[2])
        st.synchronize()
        np.testing.assert_array_equal(z.cpu().numpy(), eager[2])
    ctx.release_stream(stream=st.cuda_stream)

# many slots, many experts, few and many rows an expert, LDS-filling rows
FEW = [(1, 128, 192, 1024, 64, "q4_0", "q8_0"), (4, 256, 64, 65, 64, "q8_0", "q4_0"), (2, 512, 256, 700, 33, "q6_k", "q3_k"),
       (32, 96, 64, 96, 8, "mxfp4", "q4_1"), (32, 256, 256, 20, 4, "q5_k", "q2_k"), (21, 512, 288, 7, 2, "q4_k", "q4_1"),
       (17, 256, 512, 64, 15, "q2_k", "q5_k"), (24, 1056, 32, 12, 3, "q4_1", "mxfp4"), (13, 64, 2112, 5, 2, "q8_0", "q8_0")]


@pytest.mark.parametrize("xdt", ["bf16", "f32"])
@pytest.mark.parametrize("case", FEW, ids=lambda c: "x".join(map(str, c)))
def test_few_tokens(ctx, orc, case, xdt):
    """Both sides of the few-token kernels' own rules: one entry a pass and
    four, column tiles that do not divide the row, idle lanes, 64 slots."""
    import torch

    announce(f"moe_layer few tokens {case} x={xdt}")
    L = Layer(orc, np.random.default_rng(sum(case[:5])), *case[:5], *case[5:], xdt=xdt)
    ids, p, gap, big = L.route()
    assert gap > 1e-7
    y = L.call(ctx)
    torch.cuda.synchronize()
    L.check(y, ids, p, big)


def test_bank_beyond_32_bit_offsets(ctx):
    """An expert behind the first 4 GiB of the bank gives the bits it gives as a
    bank of its own (one row a pass, and several)."""
    import rlxq
    import torch

    H, I, E = 16384, 8192, 36
    for rows in (1, 5):
        announce(f"moe_layer large bank rows={rows}")
        gen = torch.Generator(device="cuda")
        gen.manual_seed(rows)
        g = torch.zeros(E * 2 * I * (H // 2), dtype=torch.uint8, device="cuda")
        d = torch.zeros(E * H * (I // 2), dtype=torch.uint8, device="cuda")
        gs = torch.full((E * 2 * I, H // 32), 110, dtype=torch.uint8, device="cuda")
        ds = torch.full((E * H, I // 32), 110, dtype=torch.uint8, device="cuda")
        assert g.numel() > 2 ** 32
        ge, de = g.view(E, -1)[-1], d.view(E, -1)[-1]
        for t in (ge, de):
            t.copy_(torch.randint(0, 256, t.shape, device="cuda", dtype=torch.uint8, generator=gen))
        x = torch.randn((rows, H), device="cuda", generator=gen)
        logits = torch.zeros((rows, E), device="cuda")
        logits[:, E - 1] = 50.0
        a = ctx.moe_layer(x, None, g, d, rlxq.MLX_MXFP4, rlxq.MLX_MXFP4, 1, I, E, logits=logits, gate_up_scales=gs,
                          down_scales=ds)
        b = ctx.moe_layer(x, None, ge, de, rlxq.MLX_MXFP4, rlxq.MLX_MXFP4, 1, I, 1, logits=logits[:, :1].contiguous(),
                          gate_up_scales=gs[-2 * I:], down_scales=ds[-H:])
        torch.cuda.synchronize()
        assert torch.isfinite(b).all() and b.abs().max() > 0
        assert torch.equal(a, b)
        del g, d, gs, ds


def test_more_rows_than_a_grid_dimension(ctx, orc):
    import torch

    announce("moe_layer 600000 rows")
    L = Layer(orc, np.random.default_rng(9), 40, 32, 32, 4, 1)
    x = L.x.repeat(15000, 1)
    i = torch.empty((600000, 1), dtype=torch.int32, device="cuda")
    L.shape = (600000,) + L.shape[1:]
    y = L.call(ctx, x=x, ids=i)
    torch.cuda.synchronize()
    L.shape = (40,) + L.shape[1:]
    ids, p, gap, big = L.route()
    assert gap > 1e-6
    np.testing.assert_array_equal(i.view(15000, 40).cpu().numpy(), np.broadcast_to(ids[:, 0], (15000, 40)))
    for at in (0, 262144 // 40, 7000, 14999):
        L.check(y.view(15000, 40, 32)[at], ids, p, big)


@pytest.mark.parametrize("rows", [4, 25, 60])
@pytest.mark.parametrize("xdt", ["bf16", "f32"])
def test_activations_not_finite_on_given_logits(ctx, orc, rows, xdt):
    """Finite logits of the caller's: a row of x with an infinity or a NaN leaves
    its y not finite, and the other rows are as without it.  (The infinity sits
    in the last block of a row whose blocks do not fill the lanes.)"""
    import torch

    announce(f"moe_layer x not finite rows={rows} x={xdt}")
    rng = np.random.default_rng(10)
    L = Layer(orc, rng, rows, 288, 96, 9, 2, "q4_1", "mxfp4", xdt=xdt)
    logits = rng.standard_normal((rows, 9)).astype(np.float32)
    x = L.x.clone()
    x[0, 287], x[2, 5], x[3, 100] = float("inf"), float("nan"), float("-inf")
    y = L.call(ctx, x=x, router=None, logits=_t(logits))
    torch.cuda.synchronize()
    got = y.cpu().numpy()
    ids, p, gap, big = L.route(True, logits)
    want, tol = L.exact(ids, p, big, act_eps=2.0 ** -8 if xdt == "bf16" else 0.0)
    assert gap > 1e-6 and not np.any(np.isfinite(got[[0, 2, 3]]))
    ok = [i for i in range(rows) if i not in (0, 2, 3)]
    assert np.all(np.abs(got[ok] - want[ok]) <= tol[ok])


def test_two_streams_at_once(ctx, orc):
    """Calls of one context under way on two streams, each with its scratch."""
    import torch

    announce("moe_layer and mxfp4_gemm on two streams")
    rng = np.random.default_rng(11)
    L = Layer(orc, rng, 12, 1024, 256, 32, 8, "mxfp4", "mxfp4", xdt="bf16")
    xs = [_as(rng.standard_normal((12, 1024)).astype(np.float32), "bf16")[0] for _ in range(2)]
    w, ws = ctx.quantize_mxfp4(_t(rng.standard_normal((512, 1024)).astype(np.float32)))
    want = [(L.call(ctx, x=x).clone(), ctx.mxfp4_gemm(x, w, ws, 512).clone()) for x in xs]
    torch.cuda.synchronize()
    st = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(20):
        for s, x, out in zip(st, xs, got):
            with torch.cuda.stream(s):
                out.append((L.call(ctx, x=x), ctx.mxfp4_gemm(x, w, ws, 512)))
    torch.cuda.synchronize()
    for out, (a, b) in zip(got, want):
        assert all(torch.equal(y, a) and torch.equal(z, b) for y, z in out)
    for s in st:
        ctx.release_stream(stream=s.cuda_stream)


@pytest.mark.parametrize("xdt", ["bf16", "f32"])
@pytest.mark.parametrize("pair", [("mxfp4", "q4_1"), ("q6_k", "q8_0"), ("q4_k", "q4_k")], ids=lambda p: "-".join(p))
def test_grouped_products_at_few_tokens(ctx, orc, pair, xdt, monkeypatch):
    """The composition of the grouped products, which serves what the few-token
    kernels do not take, within the same bounds on calls that they do."""
    import torch

    for rows in (1, 6, 30):
        announce(f"moe_layer grouped {pair} x={xdt} rows={rows}")
        L = Layer(orc, np.random.default_rng(20 + rows), rows, 512, 256, 12, 3, *pair, xdt=xdt)
        ids, p, gap, big = L.route()
        assert gap > 1e-6
        few = L.call(ctx)
        monkeypatch.setenv("RLXQ_MOE_LAYER", "grouped")
        grouped = L.call(ctx)
        monkeypatch.delenv("RLXQ_MOE_LAYER")
        torch.cuda.synchronize()
        L.check(few, ids, p, big)
        L.check(grouped, ids, p, big)


def test_two_graphs_on_one_scratch(ctx, orc):
    """Two graphs captured on one stream share its scratch: replayed in turns,
    with eager calls between, each gives the eager bits."""
    import torch

    announce("moe_layer and mxfp4_gemm graphs on one scratch")
    rng = np.random.default_rng(12)
    L = Layer(orc, rng, 9, 512, 256, 16, 4, "q4_1", "mxfp4", xdt="f32")
    v = _t(rng.standard_normal((70, 512)).astype(np.float32))
    w, ws = ctx.quantize_mxfp4(_t(rng.standard_normal((384, 512)).astype(np.float32)))
    a, b = L.call(ctx).clone(), ctx.mxfp4_gemm(v, w, ws, 384).clone()
    ya, yb = torch.empty_like(a), torch.empty_like(b)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):   # sizes the stream's scratch
        L.call(ctx, y=ya)
        ctx.mxfp4_gemm(v, w, ws, 384, y=yb)
    st.synchronize()
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga, stream=st):
        L.call(ctx, y=ya)
    with torch.cuda.graph(gb, stream=st):
        ctx.mxfp4_gemm(v, w, ws, 384, y=yb)
    for _ in range(4):
        ya.zero_()
        yb.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            ga.replay()
            gb.replay()
            z = L.call(ctx)
            ga.replay()
        st.synchronize()
        assert torch.equal(ya, a) and torch.equal(yb, b) and torch.equal(z, a)
    del ga, gb
    ctx.release_stream(stream=st.cuda_stream)


def test_quantised_experts_together(ctx, orc):
    """The set as it is used: float experts packed by quantize_mxfp4, a dense
    MXFP4 product on 4-bit activations in front, and the expert layer on its
    output."""
    import rlxq
    import torch

    announce("quantize_mxfp4 -> mxfp4_gemm -> moe_layer")
    rng = np.random.default_rng(8)
    H, I, E, K = 256, 128, 6, 2
    w = [(rng.standard_normal(s) * 0.06).astype(np.float32) for s in ((H, H), (E * 2 * I, H), (E * H, I))]
    (pc, ps), (gc, gs), (dc, ds) = (ctx.quantize_mxfp4(_t(v)) for v in w)
    x0 = _t(rng.standard_normal((5, H)).astype(np.float32))
    x = ctx.mxfp4_gemm(x0, pc, ps, H)
    router = _t((rng.standard_normal((E, H)) / 8).astype(np.float32))
    i = torch.empty((5, K), dtype=torch.int32, device="cuda")
    y = ctx.moe_layer(x, router, gc, dc, rlxq.MLX_MXFP4, rlxq.MLX_MXFP4, K, I, E, gate_up_scales=gs, down_scales=ds, ids=i)
    torch.cuda.synchronize()
    L = Layer.__new__(Layer)
    L.shape, L.xdt = (5, H, I, E, K), "f32"
    L.xv, L.rv = x.double().cpu().numpy(), router.double().cpu().numpy()
    L.gv = orc.mxfp4_dequantize(*orc.mxfp4_quantize(w[1]), E * 2 * I, H).reshape(E, 2 * I, H)
    L.dv = orc.mxfp4_dequantize(*orc.mxfp4_quantize(w[2]), E * H, I).reshape(E, H, I)
    xq = orc.mxfp4_dequantize(*orc.mxfp4_quantize(x0.cpu().numpy()), 5, H)
    pw = orc.mxfp4_dequantize(*orc.mxfp4_quantize(w[0]), H, H)
    assert np.all(np.abs(L.xv - xq @ pw.T) <= H * 2.0 ** -23 * (np.abs(xq) @ np.abs(pw).T))
    ids, p, gap, big = L.route()
    assert gap > 1e-6
    np.testing.assert_array_equal(i.cpu().numpy(), ids)
    L.check(y, ids, p, big)


def test_no_rows(ctx):
    import rlxq
    import torch

    announce("moe_layer rows=0")
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8, device="cuda")   # noqa: E731
    y = ctx.moe_layer(torch.zeros((0, 64), device="cuda"), torch.zeros((4, 64), device="cuda"), u8(4 * 64 * 40),
                      u8(4 * 64 * 20), rlxq.GGUF_Q4_1, rlxq.GGUF_Q4_1, 2, 32, 4)
    assert y.shape == (0, 64)


def test_status_codes(ctx):
    import ctypes as C

    import rlxq
    import torch

    announce("moe_layer status codes")
    f = lambda *s: torch.zeros(s, device="cuda")   # noqa: E731
    x, r, lg, y = f(2, 256), f(4, 256), f(2, 4), f(2, 256)
    g = torch.zeros(4 * 512 * 160, dtype=torch.uint8, device="cuda")
    d = torch.zeros(4 * 256 * 160, dtype=torch.uint8, device="cuda")
    p = lambda t, off=0: C.c_void_p(t.data_ptr() + off)   # noqa: E731
    base = dict(x=p(x), xd=0, r=p(r), rd=0, lg=None, gs=3, g=p(g), gsc=None, ds=3, d=p(d), dsc=None, rows=2, h=256, i=256,
                e=4, k=2, rn=1, ids=None, pr=None, y=p(y), yd=0)

    def call(**kw):
        return rlxq.lib().rlxq_moe_layer(ctx.h, *({**base, **kw}[n] for n in base), None)

    assert call() == rlxq.OK and call(rows=0) == rlxq.OK
    assert call(r=None) == rlxq.E_NULL and call(lg=p(lg)) == rlxq.E_NULL and call(r=None, lg=p(lg)) == rlxq.OK
    assert call(x=None) == rlxq.E_NULL and call(g=None) == rlxq.E_NULL and call(y=None) == rlxq.E_NULL
    assert call(gs=4) == rlxq.E_SCHEME and call(ds=6) == rlxq.E_SCHEME and call(gs=99) == rlxq.E_SCHEME
    assert call(gs=9) == rlxq.E_NULL   # MXFP4 without scales
    assert call(rows=-1) == rlxq.E_SHAPE and call(h=0) == rlxq.E_SHAPE and call(i=-32) == rlxq.E_SHAPE
    assert call(e=0) == rlxq.E_SHAPE and call(e=1025) == rlxq.E_SHAPE and call(k=0) == rlxq.E_SHAPE
    assert call(k=5) == rlxq.E_SHAPE and call(e=100, k=65) == rlxq.E_SHAPE
    assert call(h=48) == rlxq.E_SHAPE and call(ds=7, i=96) == rlxq.E_SHAPE and call(gs=1, h=96) == rlxq.E_ALIGN
    assert call(xd=2) == rlxq.E_DTYPE and call(yd=2) == rlxq.E_DTYPE and call(rd=2) == rlxq.E_DTYPE
    assert call(x=p(x, 4)) == rlxq.E_ALIGN and call(r=p(r, 8)) == rlxq.E_ALIGN and call(g=p(g, 2)) == rlxq.E_ALIGN
    torch.cuda.synchronize()
