"""MXFP4 quantiser and the MXFP4 x MXFP4 matmul (rlxq_quantize_mxfp4,
rlxq_mxfp4_gemm): codes and scales bit for bit against the encoder of
oracle.py, products against float64 sums of the decoded operands.

Tolerance of the products: the products of two E2M1 values and two powers of
two are exact, so only the f32 sums round, at most K of them, each by at most
2^-23 of a partial sum (2^-24 for a rounded addition, twice that where the
MFMA's inner adder truncates), and a partial sum is at most S = sum |x_q w_q|:
|error| <= K * 2^-23 * S.  A bf16 output adds 2^-8 |y|."""
import numpy as np
import pytest

from conftest import announce

pytestmark = pytest.mark.gpu


def _t(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _bf16(x32):
    """x rounded to bf16: (the tensor, its values as f32)."""
    import torch

    t = torch.from_numpy(x32).to(torch.bfloat16)
    return t.cuda(), t.float().numpy()


def _as(x32, xdt):
    return _bf16(x32) if xdt == "bf16" else (_t(x32), x32)


def _edge_rows(rng, k):
    """Rows whose blocks hold what the encoder can go wrong at."""
    rows = [rng.standard_normal(k).astype(np.float32) * np.float32(2.0 ** e) for e in (-126, -100, -3, 0, 9, 100, 125)]
    rows.append(np.zeros(k, np.float32))
    rows.append(np.full(k, -0.0, np.float32))
    mid = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], np.float32)   # ties, the largest value
    for sc in (1.0, 2.0 ** -40, 2.0 ** 60):
        rows.append((np.resize(np.concatenate([mid, -mid]), k) * np.float32(sc)).astype(np.float32))
        near = np.nextafter(np.resize(mid, k), np.float32(np.inf), dtype=np.float32)
        near[::32] = 6.0
        rows.append((near * np.float32(sc)).astype(np.float32))
    rows.append(np.resize(np.float32(2.0) ** np.arange(-149, 11, dtype=np.float32), k).astype(np.float32))   # subnormals
    rows.append(np.resize(np.ldexp(np.array([1, -3, 5, 0, 7], np.float32), -149), k).astype(np.float32))
    r = np.zeros(k, np.float32)   # a single element in each block: 1.5 * 2^q and its neighbours
    r[::32] = np.resize(np.array([1.5, np.nextafter(np.float32(1.5), np.float32(2)),
                                  np.nextafter(np.float32(1.5), np.float32(1)), 1.0, 2.0, 3.4e38], np.float32), k // 32)
    rows.append(r)
    return np.stack(rows)


@pytest.mark.parametrize("xdt", ["bf16", "f32"])
@pytest.mark.parametrize("shape", [(1, 32), (3, 96), (17, 4096), (5, 2080), (257, 160)], ids=str)
def test_quantize_matches_the_encoder(ctx, orc, shape, xdt):
    import torch

    announce(f"quantize_mxfp4 {shape} {xdt}")
    m, k = shape
    rng = np.random.default_rng(m + k)
    x, xv = _as((rng.standard_normal((m, k)) * np.exp(rng.standard_normal((m, k)))).astype(np.float32), xdt)
    codes, scales = ctx.quantize_mxfp4(x)
    torch.cuda.synchronize()
    wc, wb = orc.mxfp4_quantize(xv)
    np.testing.assert_array_equal(scales.cpu().numpy(), wb)
    np.testing.assert_array_equal(codes.cpu().numpy(), wc)


@pytest.mark.parametrize("xdt", ["bf16", "f32"])
def test_quantize_edges(ctx, orc, xdt):
    import torch

    announce(f"quantize_mxfp4 edges {xdt}")
    x, xv = _as(_edge_rows(np.random.default_rng(5), 320), xdt)
    codes, scales = ctx.quantize_mxfp4(x)
    torch.cuda.synchronize()
    wc, wb = orc.mxfp4_quantize(xv)
    np.testing.assert_array_equal(scales.cpu().numpy(), wb)
    np.testing.assert_array_equal(codes.cpu().numpy(), wc)


@pytest.mark.parametrize("xdt", ["bf16", "f32"])
def test_quantize_not_finite(ctx, orc, xdt):
    """Blocks with infinities or NaN: scale byte 127, +-6 for what is not
    finite, the rest as under scale 1; their neighbours as without them."""
    import torch

    announce(f"quantize_mxfp4 not finite {xdt}")
    rng = np.random.default_rng(6)
    x32 = (rng.standard_normal((4, 128)) * 2).astype(np.float32)
    x32[0, 3], x32[1, 40], x32[2, 127], x32[3, 64], x32[3, 65] = np.inf, -np.inf, np.nan, np.inf, -np.nan
    x, xv = _as(x32, xdt)
    codes, scales = ctx.quantize_mxfp4(x)
    torch.cuda.synchronize()
    wc, wb = orc.mxfp4_quantize(xv)
    np.testing.assert_array_equal(scales.cpu().numpy(), wb)
    np.testing.assert_array_equal(codes.cpu().numpy(), wc)


@pytest.mark.parametrize("xdt", ["bf16", "f32"])
def test_quantize_and_dequantize_large(ctx, orc, xdt):
    """The kernels of large matrices (several groups of elements per thread, the
    last workgroup part filled): sampled rows, the last ones among them."""
    import rlxq
    import torch

    m, k = 8201, 4128
    announce(f"quantize_mxfp4, dequantize {m}x{k} {xdt}")
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    x = torch.randn((m, k), device="cuda", generator=gen).to(torch.bfloat16 if xdt == "bf16" else torch.float32)
    codes, scales = ctx.quantize_mxfp4(x)
    v = ctx.dequantize(codes, rlxq.MLX_MXFP4, m, k, scales=scales)
    torch.cuda.synchronize()
    rows = np.unique(np.concatenate([np.arange(4), np.arange(m - 4, m), np.random.default_rng(2).integers(0, m, 60)]))
    at = torch.from_numpy(rows).cuda()
    wc, wb = orc.mxfp4_quantize(x[at].float().cpu().numpy())
    np.testing.assert_array_equal(scales[at].cpu().numpy(), wb)
    np.testing.assert_array_equal(codes[at].cpu().numpy(), wc)
    want = orc.mxfp4_dequantize(wc, wb, len(rows), k).astype(np.float32)
    np.testing.assert_array_equal(v[at].cpu().numpy(), want)


def test_quantize_then_dequantize_and_matmul(ctx, orc):
    """Together: rows packed on the device, decoded, and used as the weights of
    the dense op."""
    import rlxq
    import torch

    announce("quantize_mxfp4 -> dequantize, dequant_matmul")
    rng = np.random.default_rng(7)
    w32 = (rng.standard_normal((96, 256)) * 0.02).astype(np.float32)
    codes, scales = ctx.quantize_mxfp4(_t(w32))
    v = ctx.dequantize(codes, rlxq.MLX_MXFP4, 96, 256, scales=scales)
    x, xv = _bf16(rng.standard_normal((2, 256)).astype(np.float32))
    y = ctx.dequant_matmul(x, codes, rlxq.MLX_MXFP4, 96, scales=scales)
    torch.cuda.synchronize()
    want = orc.mxfp4_dequantize(*orc.mxfp4_quantize(w32), 96, 256)
    np.testing.assert_array_equal(v.cpu().numpy(), want.astype(np.float32))
    np.testing.assert_allclose(y.cpu().numpy(), xv.astype(np.float64) @ want.T, rtol=0, atol=1e-4)


def _want(orc, xv, codes, eb, n):
    """(y, S) in float64: the product of the decoded operands and of their
    magnitudes."""
    m, k = xv.shape
    xq = orc.mxfp4_dequantize(*orc.mxfp4_quantize(xv), m, k)
    wq = orc.mxfp4_dequantize(codes, eb, n, k)
    return xq @ wq.T, np.abs(xq) @ np.abs(wq).T


def _check(y, want, s, k, bf16):
    tol = k * 2.0 ** -23 * s + (2.0 ** -8 * np.abs(want) if bf16 else 0.0)
    # A true value past f32's largest, (2 - 2^-23) 2^127, has no finite f32: its
    # output is the infinity of its sign.  Where only S passes it, a partial sum
    # may, and no bound holds.
    top = float(np.finfo(np.float32).max)
    big = s > top
    past = np.abs(want) > top * (1 + 2.0 ** -24) + tol
    assert np.array_equal(y[past], np.sign(want[past]) * np.inf)
    err = np.where(big, 0.0, np.abs(np.where(big, 0.0, y) - np.where(big, 0.0, want)))
    assert np.all(err <= tol), f"worst {np.max(err - tol):.3e} over the bound, max err {np.max(err):.3e}"


def _weights(rng, n, k, lo=110, hi=130):
    return rng.integers(0, 256, (n, k // 2), dtype=np.uint8), rng.integers(lo, hi, (n, k // 32), dtype=np.uint8)


# (K in part of a span of 512 or 256 and of a stage of 128, more and fewer spans
# than waves, 16 and 32 weight rows a workgroup, activations quantised inside
# and ahead, one tile and many, edges in every direction)
SHAPES = [(1, 32, 1), (2, 1056, 6200), (3, 8704, 40), (12, 2176, 6176), (20, 160, 6190), (31, 9216, 130), (9, 4096, 520), (1, 4096, 512), (2, 96, 33), (5, 480, 17), (16, 512, 64), (17, 544, 100), (33, 1056, 250),
          (64, 2048, 384), (130, 800, 301), (200, 4096, 96), (257, 320, 513), (300, 1536, 640), (512, 288, 1025)]


@pytest.mark.parametrize("xdt,ydt", [("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_gemm(ctx, orc, shape, xdt, ydt):
    import torch

    m, k, n = shape
    announce(f"mxfp4_gemm {shape} x={xdt} y={ydt}")
    rng = np.random.default_rng(m * 7 + k + n)
    codes, eb = _weights(rng, n, k)
    x, xv = _as((rng.standard_normal((m, k)) * np.exp(rng.standard_normal(k))).astype(np.float32), xdt)
    y = ctx.mxfp4_gemm(x, _t(codes), _t(eb), n, y_dtype=torch.bfloat16 if ydt == "bf16" else torch.float32)
    torch.cuda.synchronize()
    assert ctx.last_kernel.startswith("rlxq_mx_")
    want, s = _want(orc, xv, codes, eb, n)
    _check(y.double().cpu().numpy(), want, s, k, ydt == "bf16")


@pytest.mark.parametrize("cfg", ["m256n256", "m256n256,3", "m128n128", "m128n128,2", "m128n64", "m128n64,4", "m64n64",
                                 "m64n64,2"])
@pytest.mark.parametrize("shape", [(1, 32, 1), (33, 96, 70), (70, 2336, 264), (130, 800, 301), (256, 256, 256),
                                   (300, 1536, 640), (512, 1152, 520)], ids=lambda s: "x".join(map(str, s)))
def test_gemm_every_tiling(ctx, orc, monkeypatch, shape, cfg):
    """Every tiling with and without K splits (an odd number of spans, of stages
    within the last one, more splits than spans), and weight blocks of scale 0."""
    import torch

    m, k, n = shape
    announce(f"mxfp4_gemm {cfg} {shape}")
    monkeypatch.setenv("RLXQ_MX_CFG", cfg)
    rng = np.random.default_rng(m + 3 * k + n)
    codes, eb = _weights(rng, n, k)
    for zeros, ydt in ((False, torch.bfloat16), (True, torch.float32)):
        if zeros:
            eb[rng.random(eb.shape) < 0.1] = 0
            eb[n // 2, 0] = 255
        x, xv = _as((rng.standard_normal((m, k)) * np.exp(rng.standard_normal(k))).astype(np.float32), "bf16")
        y = ctx.mxfp4_gemm(x, _t(codes), _t(eb), n, y_dtype=ydt)
        torch.cuda.synchronize()
        assert ctx.last_kernel == "rlxq_mx_gemm_" + cfg.split(",")[0]
        want, s = _want(orc, xv, codes, eb, n)
        _check(y.double().cpu().numpy(), want, s, k, ydt == torch.bfloat16)


def test_gemm_unknown_tiling(ctx, monkeypatch):
    import rlxq
    import torch

    monkeypatch.setenv("RLXQ_MX_CFG", "m7n7")
    w, s = torch.zeros((8, 32), dtype=torch.uint8, device="cuda"), torch.zeros((8, 2), dtype=torch.uint8, device="cuda")
    with pytest.raises(rlxq.RlxqError) as e:
        ctx.mxfp4_gemm(torch.zeros((2, 64), device="cuda"), w, s, 8)
    assert e.value.status == rlxq.E_NOKERNEL


def test_gemm_unaligned_output_and_scales(ctx, orc):
    """y and the scales at addresses that allow no wide access."""
    import torch

    for m, k, n in ((3, 352, 40), (200, 352, 264)):
        announce(f"mxfp4_gemm unaligned {m}x{k}x{n}")
        rng = np.random.default_rng(11)
        codes, eb = _weights(rng, n, k)
        buf = torch.zeros(n * k // 32 + 3, dtype=torch.uint8, device="cuda")
        s = buf[3:].view(n, k // 32)
        s.copy_(_t(eb))
        x, xv = _as(rng.standard_normal((m, k)).astype(np.float32), "f32")
        out = torch.full((m * n + 3,), 7.0, device="cuda")
        y = out[1:1 + m * n].view(m, n)
        ctx.mxfp4_gemm(x, _t(codes), s, n, y=y)
        torch.cuda.synchronize()
        want, sm = _want(orc, xv, codes, eb, n)
        _check(y.double().cpu().numpy(), want, sm, k, False)
        assert out[0] == 7.0 and torch.all(out[1 + m * n:] == 7.0)


@pytest.mark.parametrize("m", [1, 3, 40, 300])
def test_gemm_scale_bytes_0_and_255(ctx, orc, m):
    """Weight blocks of scale byte 0 are zeros, of 255 have scale 2^127 (as in
    rlxq_dequantize): the scaled MFMA reads those bytes otherwise."""
    import torch

    announce(f"mxfp4_gemm scale bytes 0, 255 m={m}")
    k, n = 1088, 300
    rng = np.random.default_rng(8 + m)
    codes, eb = _weights(rng, n, k)
    eb[rng.random(eb.shape) < 0.2] = 0
    # activations of 2^100 under zero weights: 2^-127 in place of 0 would show
    x32 = rng.standard_normal((m, k)).astype(np.float32)
    eb[:, 3] = 0
    x32[:, 96:128] *= np.float32(2.0 ** 120)
    # scale byte 255 against activations of 2^-126
    eb[:, 5] = 255
    x32[:, 160:192] *= np.float32(2.0 ** -126)
    x, xv = _as(x32, "f32")
    y = ctx.mxfp4_gemm(x, _t(codes), _t(eb), n)
    torch.cuda.synchronize()
    want, s = _want(orc, xv, codes, eb, n)
    _check(y.double().cpu().numpy(), want, s, k, False)


@pytest.mark.parametrize("m", [2, 50, 290])
@pytest.mark.parametrize("xdt", ["bf16", "f32"])
def test_gemm_rows_not_finite(ctx, orc, m, xdt):
    """A row with an infinity or a NaN is NaN in every column; the others are as
    without it.  Zero rows are zeros."""
    import torch

    announce(f"mxfp4_gemm rows not finite m={m} {xdt}")
    k, n = 608, 77
    rng = np.random.default_rng(9 + m)
    codes, eb = _weights(rng, n, k)
    x32 = rng.standard_normal((m, k)).astype(np.float32)
    clean = x32.copy()
    x32[0, 600] = np.inf
    if m > 2:
        x32[m - 1, 5] = np.nan
        x32[m // 2] = 0
        clean[m // 2] = 0
    x, _ = _as(x32, xdt)
    y = ctx.mxfp4_gemm(x, _t(codes), _t(eb), n)
    torch.cuda.synchronize()
    got = y.double().cpu().numpy()
    _, xv = _as(clean, xdt)
    want, s = _want(orc, xv, codes, eb, n)
    bad = [0] + ([m - 1] if m > 2 else [])
    assert np.all(np.isnan(got[bad]))
    ok = [i for i in range(m) if i not in bad]
    _check(got[ok], want[ok], s[ok], k, False)


def test_gemm_no_rows(ctx):
    import torch

    announce("mxfp4_gemm, quantize_mxfp4 m=0")
    w, s = torch.zeros((8, 32), dtype=torch.uint8, device="cuda"), torch.zeros((8, 2), dtype=torch.uint8, device="cuda")
    assert ctx.mxfp4_gemm(torch.zeros((0, 64), device="cuda"), w, s, 8).shape == (0, 8)
    c, b = ctx.quantize_mxfp4(torch.zeros((0, 64), device="cuda"))
    assert c.shape == (0, 32) and b.shape == (0, 2)


@pytest.mark.parametrize("m", [1, 20, 300])
def test_gemm_on_another_stream_and_in_a_graph(ctx, orc, m):
    """A side stream, and a captured call replayed with new inputs between eager
    calls on the same stream: every result as the eager one's bits."""
    import torch

    announce(f"mxfp4_gemm streams and graphs m={m}")
    k, n = 2048, 520
    rng = np.random.default_rng(10 + m)
    codes, eb = _weights(rng, n, k)
    w, s = _t(codes), _t(eb)
    xs = [_t(rng.standard_normal((m, k)).astype(np.float32)) for _ in range(3)]
    eager = [ctx.mxfp4_gemm(x, w, s, n).cpu().numpy() for x in xs]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    x, y = xs[0].clone(), torch.empty((m, n), device="cuda")
    with torch.cuda.stream(st):
        ctx.mxfp4_gemm(x, w, s, n, y=y)   # sizes the stream's scratch
    st.synchronize()
    np.testing.assert_array_equal(y.cpu().numpy(), eager[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        ctx.mxfp4_gemm(x, w, s, n, y=y)
    for i in (0, 1, 2, 1):
        x.copy_(xs[i])
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(y.cpu().numpy(), eager[i])
        with torch.cuda.stream(st):
            z = ctx.mxfp4_gemm(xs[2], w, s, n)
        st.synchronize()
        np.testing.assert_array_equal(z.cpu().numpy(), eager[2])
    ctx.release_stream(stream=st.cuda_stream)


def test_beyond_32_bit_offsets(ctx):
    """Rows behind the first 4 GiB: of the quantiser's input, of the codes, of
    the product's weights and of its output."""
    import rlxq
    import torch

    announce("mxfp4 beyond 4 GiB")
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    K, N = 4096, 2113536

    def values(t):
        c, sc = ctx.quantize_mxfp4(t)
        return ctx.dequantize(c, rlxq.MLX_MXFP4, *t.shape, scales=sc).view(t.shape).double()

    tail = torch.randn((48, K), device="cuda", generator=gen)
    x = torch.zeros((N, K), device="cuda")   # 35 GB
    x[-48:] = tail
    codes, scales = ctx.quantize_mxfp4(x)
    c0, s0 = ctx.quantize_mxfp4(tail)
    assert codes.numel() > 2 ** 32
    assert torch.equal(codes[-48:], c0) and torch.equal(scales[-48:], s0)
    back = ctx.dequantize(codes, rlxq.MLX_MXFP4, N, K, scales=scales, out=x)
    assert torch.equal(back.view(N, K)[-48:].double(), values(tail))
    del x, back
    # f32 sums of K exact products, in the order of the kernel: K 2^-24 of their size
    for m in (1, 20, 40):
        v = torch.randn((m, K), device="cuda", generator=gen)
        y = ctx.mxfp4_gemm(v, codes, scales, N)
        torch.cuda.synchronize()
        assert not y[:, :-48].any()
        vv, wv = values(v).cpu(), values(tail).cpu()
        assert ((y[:, -48:].cpu().double() - vv @ wv.T).abs() <= K * 2.0 ** -24 * (vv.abs() @ wv.abs().T)).all()
    del codes, scales, y
    v = torch.randn((33000, 64), device="cuda", generator=gen)   # an output of 33000 x 33024, 4.4 GB
    t = torch.randn((33024, 64), device="cuda", generator=gen)
    w, ws = ctx.quantize_mxfp4(t)
    y = ctx.mxfp4_gemm(v, w, ws, 33024)
    torch.cuda.synchronize()
    vv, wv = values(v[-40:].contiguous()).cpu(), values(t).cpu()
    assert ((y[-40:].cpu().double() - vv @ wv.T).abs() <= 64 * 2.0 ** -24 * (vv.abs() @ wv.abs().T)).all()


def test_status_codes(ctx):
    import ctypes as C

    import rlxq
    import torch

    announce("mxfp4 status codes")
    L = rlxq.lib()
    x = torch.zeros((4, 256), device="cuda")
    w, s = torch.zeros((8, 128), dtype=torch.uint8, device="cuda"), torch.zeros((8, 8), dtype=torch.uint8, device="cuda")
    y = torch.zeros((4, 8), device="cuda")
    p = lambda t, off=0: C.c_void_p(t.data_ptr() + off)   # noqa: E731

    def gemm(x_=None, xd=rlxq.F32, w_=None, s_=None, m=4, k=256, n=8, y_=None, yd=rlxq.F32):
        return L.rlxq_mxfp4_gemm(ctx.h, x_ or p(x), xd, w_ or p(w), s_ or p(s), m, k, n, y_ or p(y), yd, None)

    assert gemm() == rlxq.OK
    assert gemm(m=-1) == rlxq.E_SHAPE and gemm(n=0) == rlxq.E_SHAPE and gemm(k=0) == rlxq.E_SHAPE
    assert gemm(k=(1 << 24) + 32) == rlxq.E_SHAPE
    assert gemm(k=48) == rlxq.E_ALIGN
    assert gemm(x_=p(x, 4)) == rlxq.E_ALIGN and gemm(w_=p(w, 8)) == rlxq.E_ALIGN
    assert gemm(xd=rlxq.U8) == rlxq.E_DTYPE and gemm(yd=7) == rlxq.E_DTYPE
    assert L.rlxq_mxfp4_gemm(ctx.h, None, 0, p(w), p(s), 4, 256, 8, p(y), 0, None) == rlxq.E_NULL
    assert L.rlxq_mxfp4_gemm(ctx.h, p(x), 0, p(w), None, 4, 256, 8, p(y), 0, None) == rlxq.E_NULL
    c, b = torch.zeros((4, 128), dtype=torch.uint8, device="cuda"), torch.zeros((4, 8), dtype=torch.uint8, device="cuda")

    def quant(x_=None, xd=rlxq.F32, m=4, k=256, c_=None, b_=None):
        return L.rlxq_quantize_mxfp4(ctx.h, x_ or p(x), xd, m, k, c_ or p(c), b_ or p(b), None)

    assert quant() == rlxq.OK and quant(m=0) == rlxq.OK
    assert quant(m=-1) == rlxq.E_SHAPE and quant(k=0) == rlxq.E_SHAPE and quant(k=31) == rlxq.E_ALIGN
    assert quant(x_=p(x, 8)) == rlxq.E_ALIGN and quant(c_=p(c, 4)) == rlxq.E_ALIGN and quant(xd=2) == rlxq.E_DTYPE
    assert L.rlxq_quantize_mxfp4(ctx.h, p(x), 0, 4, 256, None, p(b), None) == rlxq.E_NULL
    torch.cuda.synchronize()
