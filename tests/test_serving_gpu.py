"""The operators around a served batch's packed products (rlxq.Serving) against
plain implementations in 64 bits.

Tolerances: with c the longest chain of f32 additions and S the sum of the
absolute values of what is added, an f32 sum is off by at most c 2^-24 S; a
rounding to bf16 by 2^-8 of the value (half a step, from above).  Where the
inputs are small integers every sum is exact and the outputs have to be equal.
A sampled token has to be equal: its kernel's sums are f64 or fixed point."""
import numpy as np
import pytest

from conftest import announce

pytestmark = pytest.mark.gpu

U32, UB = 2.0 ** -24, 2.0 ** -8


@pytest.fixture(scope="module")
def srv(ctx):
    import rlxq

    return rlxq.Serving(ctx)


def _dt(name):
    import torch

    return {"f32": torch.float32, "bf16": torch.bfloat16}[name]


def _gen(seed):
    import torch

    g = torch.Generator()
    g.manual_seed(seed)
    return g


# ---- low-rank adapters -----------------------------------------------------
def _lora_case(seed, m, k, n, rank, e, x, ab, y, segs=None, ints=False, ranks=False, scales=True, base=True):
    import torch

    g = _gen(seed)
    s = 1 if segs is None else len(segs)

    def values(lo, hi, *shape, size=1.0):
        if ints:
            return torch.randint(lo, hi + 1, shape, generator=g).float()
        return size * torch.randn(shape, generator=g)

    d = {"x": values(-2, 2, m, k).to(_dt(x)), "a": values(-1, 1, e, s * rank, k, size=k ** -0.5).to(_dt(ab)),
         "b": values(-1, 1, e, n, rank, size=0.3).to(_dt(ab)),
         "ids": torch.randint(-1, e + 1, (m,), generator=g).int(),   # (-1 and e: no adapter)
         "base": values(-99, 99, m, n).to(_dt(y)) if base else None,
         "ranks": torch.randint(0, rank + 1, (e,), generator=g).int() if ranks else None, "scales": None}
    if scales:
        d["scales"] = torch.tensor([0.5, 1.0, 2.0, -1.0])[torch.arange(e) % 4] if ints else torch.rand(e, generator=g) + 0.5
    return d


def _lora_f64(d, segs):
    """y and the sums of absolute values (base's included; v's terms; without base)."""
    import torch

    m, n, r = d["x"].shape[0], d["b"].shape[1], d["b"].shape[2]
    e = d["b"].shape[0]
    y = d["base"].double() if d["base"] is not None else torch.zeros((m, n), dtype=torch.float64)
    y, mag, dv = y.clone(), y.abs().clone(), torch.zeros_like(y)
    ends = np.cumsum([0] + (segs or [n])).tolist()
    for i in range(m):
        q = int(d["ids"][i])
        if not 0 <= q < e:
            continue
        s = float(d["scales"][q]) if d["scales"] is not None else 1.0
        rk = int(d["ranks"][q]) if d["ranks"] is not None else r
        x = d["x"][i].double()
        for j in range(len(ends) - 1):
            a = d["a"][q, j * r:j * r + rk].double()
            b = d["b"][q, ends[j]:ends[j + 1], :rk].double()
            v = a @ x
            y[i, ends[j]:ends[j + 1]] += s * (b @ v)
            mag[i, ends[j]:ends[j + 1]] += abs(s) * (b.abs() @ (a.abs() @ x.abs()))
            dv[i, ends[j]:ends[j + 1]] += abs(s) * (b.abs() @ v.abs())
    return y, mag, dv


def _cuda(d):
    return {k: v.cuda() if v is not None else None for k, v in d.items()}


def _run_lora(srv, d, segs, y=None, y_dtype=None, **kw):
    c = _cuda(d)
    return srv.lora_matmul(c["x"], c["ids"], c["a"], c["b"], ranks=c["ranks"], scales=c["scales"], segments=segs,
                           base=c["base"], y=y, y_dtype=y_dtype, **kw)


TYPES = [("bf16", "bf16", "bf16"), ("bf16", "bf16", "f32"), ("f32", "bf16", "f32"), ("f32", "f32", "f32"),
         ("bf16", "f32", "bf16"), ("f32", "f32", "bf16"), ("f32", "bf16", "bf16"), ("bf16", "f32", "f32")]
# (m, k, n, rank, adapters, segments)
LORA = [(1, 64, 40, 8, 1, None), (1, 4096, 6144, 16, 8, [4096, 1024, 1024]), (2, 72, 33, 16, 3, [16, 17]),
        (7, 256, 1, 24, 2, None), (15, 8, 130, 8, 4, [1, 129]), (16, 1032, 257, 40, 2, None),
        (17, 512, 96, 64, 1, [96]), (33, 520, 1023, 32, 5, [0, 1000, 23]), (64, 1024, 520, 64, 48, [260, 260]),
        (65, 136, 72, 128, 3, None), (130, 264, 300, 256, 2, [100, 100, 50, 50]), (257, 64, 200, 72, 70, None),
        (600, 520, 515, 16, 4, [515]), (1111, 128, 264, 64, 6, [132, 132])]


@pytest.mark.parametrize("types", TYPES, ids="_".join)
@pytest.mark.parametrize("case", LORA, ids=lambda c: "x".join(map(str, c[:5])))
def test_lora_integers_exact(srv, case, types):
    """Integers whose sums stay below 2^24 (below 2^16 in v, which takes part in
    two bf16 terms where y is bf16): equal up to y's own rounding."""
    import torch

    m, k, n, rank, e, segs = case
    announce(f"lora ints {case} {types}")
    d = _lora_case(m + k, m, k, n, rank, e, *types, segs=segs, ints=True, ranks=m % 2 == 1)
    y = _run_lora(srv, d, segs)
    torch.cuda.synchronize()
    want, mag, _ = _lora_f64(d, segs)
    assert float(mag.max()) < 2 ** 24
    assert torch.equal(y.cpu(), want.to(_dt(types[2])))


@pytest.mark.parametrize("types", TYPES, ids="_".join)
@pytest.mark.parametrize("case", LORA, ids=lambda c: "x".join(map(str, c[:5])))
def test_lora_values(srv, case, types):
    """Values: chains of at most k / 8 + rank + 40 additions (a lane's eight
    elements at a time, then lanes, waves and slices); bf16 y: v in two bf16 terms,
    2^-16 of it, and y's rounding."""
    import torch

    m, k, n, rank, e, segs = case
    announce(f"lora values {case} {types}")
    d = _lora_case(3 * m + k, m, k, n, rank, e, *types, segs=segs, ranks=m % 2 == 0, scales=m % 3 != 0, base=m % 5 != 0)
    y = _run_lora(srv, d, segs, y_dtype=_dt(types[2]))
    torch.cuda.synchronize()
    want, mag, dv = _lora_f64(d, segs)
    tol = (k / 8 + rank + 40) * U32 * mag + U32 * want.abs() + 1e-30
    if types[2] == "bf16":
        tol = tol + 2.0 ** -16 * dv + UB * (want.abs() + tol)
    assert y.dtype == _dt(types[2])
    worst = float(((y.cpu().double() - want).abs() / tol).max())
    assert worst <= 1, worst


@pytest.mark.parametrize("m", [1, 40, 300, 700])
@pytest.mark.parametrize("ydt", ["f32", "bf16"])
def test_lora_rows_without_adapter_and_in_place(srv, m, ydt):
    """Rows without an adapter are base's bits, NaN payloads too; base may be y;
    what adapters hold past their rank, and other adapters, may be NaN."""
    import torch

    announce(f"lora none m={m} {ydt}")
    k, n, rank, e = 264, 200, 32, 6
    d = _lora_case(m, m, k, n, rank, e, "bf16", "bf16", ydt, ranks=True)
    d["ids"] = (torch.arange(m) % 5 - 1).int()            # adapter 4, 5: nobody's
    d["ids"][torch.arange(m) % 5 == 4] = 2 ** 31 - 1
    d["ranks"][1] = 0                                     # an adapter of rank 0
    d["a"].view(e, rank, k)[4:] = float("nan")
    d["b"][4:] = float("inf")
    for q in range(4):
        d["a"].view(e, rank, k)[q, int(d["ranks"][q]):] = float("nan")
        d["b"][q, :, int(d["ranks"][q]):] = float("inf")
    it = torch.int32 if ydt == "f32" else torch.int16
    d["base"][0] = torch.randint(-2 ** 15, 2 ** 15, (n,), generator=_gen(9)).to(it).view(_dt(ydt)) if ydt == "bf16" else \
        torch.randint(-2 ** 31, 2 ** 31, (n,), generator=_gen(9)).to(it).view(_dt(ydt))
    clean = {**d, "base": d["base"].clone()}
    c = _cuda(d)
    y = srv.lora_matmul(c["x"], c["ids"], c["a"], c["b"], ranks=c["ranks"], scales=c["scales"], base=c["base"], y=c["base"])
    torch.cuda.synchronize()
    assert y.data_ptr() == c["base"].data_ptr()
    got, ids = y.cpu(), d["ids"]
    plain = (ids < 0) | (ids >= e)
    assert torch.equal(got.view(it)[plain], clean["base"].view(it)[plain])
    want, mag, dv = _lora_f64(clean, None)
    rest = ~plain
    tol = (k / 8 + rank + 40) * U32 * mag + U32 * want.abs() + 1e-30
    if ydt == "bf16":
        tol = tol + 2.0 ** -16 * dv + UB * (want.abs() + tol)
    if bool(rest.any()):
        assert bool(((got.double() - want).abs() <= tol)[rest].all())
    zero = ids == 1   # rank 0: base's values
    assert torch.equal(got[zero], clean["base"][zero])


@pytest.mark.parametrize("m", [3, 20, 400])
def test_lora_rows_stay_apart(srv, m):
    """A row or adapter that is not finite leaves its own rows not finite, the
    others alone; nothing behind the last row is written."""
    import torch

    announce(f"lora rows apart m={m}")
    k, n, rank, e = 136, 200, 16, 3
    d = _lora_case(5, m, k, n, rank, e, "f32", "bf16", "f32")
    d["ids"] = (torch.arange(m) % 2).int()
    c = _cuda(d)
    out = torch.full((m + 3, n), 7.0, device="cuda")
    clean = srv.lora_matmul(c["x"], c["ids"], c["a"], c["b"], scales=c["scales"], base=c["base"])
    x = c["x"].clone()
    x[1, 5] = float("nan")
    x[2, 7] = float("inf")
    y = srv.lora_matmul(x, c["ids"], c["a"], c["b"], scales=c["scales"], base=c["base"], y=out[:m])
    torch.cuda.synchronize()
    assert not bool(torch.isfinite(y[1:3]).any())
    keep = torch.ones(m, dtype=torch.bool)
    keep[1:3] = False
    assert torch.equal(y.cpu()[keep], clean.cpu()[keep])
    assert bool((out[m:] == 7).all())


def test_lora_unaligned_outputs(srv):
    """base and y at element offsets, an odd width."""
    import torch

    announce("lora unaligned")
    for ydt in ("f32", "bf16"):
        for m, n in ((3, 65), (300, 129), (20, 64)):
            d = _lora_case(m + n, m, 128, n, 16, 2, "bf16", "bf16", ydt, ints=True)
            c = _cuda(d)
            buf, bb = torch.zeros(m * n + 4, device="cuda", dtype=_dt(ydt)), torch.zeros(m * n + 4, device="cuda", dtype=_dt(ydt))
            bb[3:3 + m * n] = c["base"].view(-1)
            y = srv.lora_matmul(c["x"], c["ids"], c["a"], c["b"], scales=c["scales"], base=bb[3:3 + m * n].view(m, n),
                                y=buf[1:1 + m * n].view(m, n))
            torch.cuda.synchronize()
            assert torch.equal(y.cpu(), _lora_f64(d, None)[0].to(_dt(ydt)))
            assert float(buf[0]) == 0 and not bool(buf[1 + m * n:].any())


def test_lora_offsets_past_32_bits(srv):
    """Adapters and outputs whose element offsets pass 2^32 bytes and 2^31 elements."""
    import torch

    announce("lora offsets past 32 bits")
    e, k, rank, n = 70, 65536, 256, 131072   # a: 70 x 256 x 65536 bf16, b: 70 x 131072 x 256 bf16
    a = torch.zeros((e, rank, k), device="cuda", dtype=torch.bfloat16)
    b = torch.zeros((e, n, rank), device="cuda", dtype=torch.bfloat16)
    m = 5
    x = torch.ones((m, k), device="cuda", dtype=torch.bfloat16)
    for q, v in ((0, 1.0), (e - 1, 2.0)):
        a[q, rank - 1, k - 1] = v
        b[q, n - 1, rank - 1] = 3.0
    ids = torch.tensor([0, e - 1, 1, -1, e - 1], device="cuda", dtype=torch.int32)
    y = srv.lora_matmul(x, ids, a, b)
    torch.cuda.synchronize()
    assert y[:, n - 1].tolist() == [3.0, 6.0, 0.0, 0.0, 6.0] and not bool(y[:, :n - 1].any())
    del a, b
    m, n, k, rank, e = 20000, 120000, 8, 8, 2   # m x n past 2^31
    base = torch.zeros((m, n), device="cuda", dtype=torch.bfloat16)
    x = torch.ones((m, k), device="cuda", dtype=torch.bfloat16)
    a = torch.ones((e, rank, k), device="cuda", dtype=torch.bfloat16)
    b = torch.zeros((e, n, rank), device="cuda", dtype=torch.bfloat16)
    b[1, n - 1] = 1.0
    ids = torch.zeros(m, device="cuda", dtype=torch.int32)
    ids[m - 1] = 1
    srv.lora_matmul(x, ids, a, b, base=base, y=base)
    torch.cuda.synchronize()
    assert float(base[m - 1, n - 1]) == 64.0 and not bool(base[:m - 1].any()) and not bool(base[m - 1, :n - 1].any())


@pytest.mark.parametrize("m,e", [(300, 16384), (40, 16384), (257, 1), (700, 699)])
def test_lora_many_adapters(srv, m, e):
    """The most adapters a call takes, rows of nearly as many; and one for all."""
    import torch

    announce(f"lora many adapters m={m} e={e}")
    d = _lora_case(m + e, m, 16, 24, 8, e, "bf16", "bf16", "f32", ints=True, ranks=True)
    d["ids"][: m // 2] = e - 1
    y = _run_lora(srv, d, None)
    torch.cuda.synchronize()
    assert torch.equal(y.cpu(), _lora_f64(d, None)[0].float())


def test_lora_values_of_every_size(srv):
    """f32 x and A take part in bf16 terms: tiny, large and mixed magnitudes, signed zeros."""
    import torch

    announce("lora f32 magnitudes")
    for m in (5, 300):
        for x, ab in (("f32", "f32"), ("f32", "bf16"), ("bf16", "f32")):
            d = _lora_case(m, m, 256, 40, 16, 2, x, ab, "f32")
            g = _gen(m + 1)
            size = torch.exp2(torch.randint(-60, 61, (m, 1), generator=g).float())
            d["x"] = (d["x"].float() * size).to(_dt(x))
            d["x"][:, ::7] = -0.0
            d["a"] = (d["a"].float() * torch.exp2(torch.randint(-20, 21, (2, 16, 1), generator=g).float())).to(_dt(ab))
            d["base"].zero_()
            y = _run_lora(srv, d, None)
            torch.cuda.synchronize()
            want, mag, _ = _lora_f64(d, None)
            tol = (256 / 8 + 16 + 40) * U32 * mag + U32 * want.abs() + 1e-30
            assert bool(((y.cpu().double() - want).abs() <= tol).all())


# ---- residual norm ---------------------------------------------------------
def _norm_case(seed, rows, h, bdt, rdt, gdt, wdt, gate_rows, post, pre, block=True, resid=True):
    import torch

    g = _gen(seed)
    r = lambda *s: torch.randn(s, generator=g)   # noqa: E731
    return {"block": (3 * r(rows, h)).to(_dt(bdt)) if block else None, "resid": r(rows, h).to(_dt(rdt)) if resid else None,
            "gate": torch.sigmoid(r(gate_rows, h)).to(_dt(gdt)) if gate_rows else None,
            "post": (1 + 0.3 * r(h)).to(_dt(wdt)) if post else None, "pre": (1 + 0.3 * r(h)).to(_dt(wdt)) if pre else None}


def _norm_f64(d, alpha, eps, off):
    """h, y and the bounds of their f32 errors."""
    import torch

    first = d["block"] if d["block"] is not None else d["resid"]
    rows, h = first.shape
    c = h / 64 + 24   # a thread's run, lanes and waves; and the other roundings
    res = d["resid"].double() if d["resid"] is not None else torch.zeros((rows, h), dtype=torch.float64)
    t = torch.zeros_like(res)
    if d["block"] is not None:
        t = d["block"].double()
        if d["post"] is not None:
            t = t / (t.square().mean(1, keepdim=True) + eps).sqrt() * (off + d["post"].double())
        if d["gate"] is not None:
            t = t * d["gate"].double().repeat_interleave(rows // d["gate"].shape[0], 0)
    hh = res + alpha * t
    tol_h = U32 * (hh.abs() + c * abs(alpha) * t.abs()) + 1e-30
    if d["pre"] is None:
        return hh, tol_h, None, None
    inv = 1 / (hh.square().mean(1, keepdim=True) + eps).sqrt()
    w = off + d["pre"].double()
    y = hh * inv * w
    # (the sum of squares: each square off by twice h's error, then the chain)
    rel = (hh.abs() * tol_h).mean(1, keepdim=True) * inv * inv + c * U32
    return hh, tol_h, y, inv * w.abs() * tol_h + (rel + 8 * U32) * y.abs() + 1e-30


def _rounded(tol, want, dt):
    return tol + (UB if dt == "bf16" else U32) * (want.abs() + tol)


NORM = [(1, 8, 0), (1, 4096, 1), (3, 100, 3), (5, 1, 1), (7, 4097, 7), (12, 5120, 4), (64, 2048, 0), (9, 8192, 1),
        (6, 16384, 2), (2, 40000, 2), (300, 512, 100), (1000, 64, 10), (4, 24, 0), (2, 12288, 1)]


@pytest.mark.parametrize("types", [("f32", "f32", "f32", "f32", "f32"), ("bf16", "bf16", "bf16", "bf16", "bf16"),
                                   ("bf16", "f32", "f32", "f32", "bf16"), ("f32", "bf16", "bf16", "f32", "f32"),
                                   ("bf16", "f32", "bf16", "bf16", "f32")], ids="_".join)
@pytest.mark.parametrize("case", NORM, ids=lambda c: "x".join(map(str, c)))
def test_residual_norm_values(srv, case, types):
    """types: block, resid (and sum), gate, weights, y."""
    import torch

    rows, h, gate_rows = case
    for post, pre, block, resid, off, alpha in ((True, True, True, True, 0.0, 0.7), (False, True, True, True, 1.0, 1.0),
                                                (True, False, True, True, 1.0, -0.5), (False, True, False, True, 0.0, 1.0),
                                                (True, True, True, False, 0.0, 1.0)):
        announce(f"residual_norm {case} {types} post={post} pre={pre} block={block} resid={resid}")
        d = _norm_case(rows + h, rows, h, *types[:4], gate_rows if block else 0, post and block, pre, block, resid)
        c = _cuda(d)
        s, y = srv.residual_norm(c["block"], c["resid"], pre_weight=c["pre"], post_weight=c["post"], gate=c["gate"],
                                 scale=alpha, eps=1e-5, weight_offset=off, y_dtype=_dt(types[4]))
        torch.cuda.synchronize()
        hh, tol_h, want, tol_y = _norm_f64(d, alpha, 1e-5, off)
        sdt = types[1] if resid else "f32"
        assert s.dtype == _dt(sdt)
        assert bool(((s.cpu().double() - hh).abs() <= _rounded(tol_h, hh, sdt)).all())
        if pre:
            assert y.dtype == _dt(types[4])
            assert bool(((y.cpu().double() - want).abs() <= _rounded(tol_y, want, types[4])).all())
        else:
            assert y is None


@pytest.mark.parametrize("h", [64, 4096, 5000, 20000])
def test_residual_norm_in_place_and_special_rows(srv, h):
    """sum over resid, y over block; a row of zeros (eps alone), a row that is not
    finite leaves the others alone, one without any y."""
    import torch

    announce(f"residual_norm in place h={h}")
    d = _norm_case(h, 6, h, "f32", "f32", "f32", "f32", 2, True, True)
    d["block"][2], d["resid"][2] = 0, 0
    c = _cuda(d)
    s0, y0 = srv.residual_norm(c["block"], c["resid"], pre_weight=c["pre"], post_weight=c["post"], gate=c["gate"])
    assert not bool(y0[2].any()) and not bool(s0[2].any())
    bad = c["block"].clone()
    bad[4, h // 2] = float("nan")
    s1, y1 = srv.residual_norm(bad, c["resid"], pre_weight=c["pre"], post_weight=c["post"], gate=c["gate"])
    keep = [0, 1, 2, 3, 5]
    assert torch.equal(s1[keep], s0[keep]) and torch.equal(y1[keep], y0[keep]) and bool(torch.isnan(y1[4]).all())
    rb, bb = c["resid"].clone(), c["block"].clone()
    s2, y2 = srv.residual_norm(bb, rb, pre_weight=c["pre"], post_weight=c["post"], gate=c["gate"], sum=rb, y=bb)
    torch.cuda.synchronize()
    assert s2.data_ptr() == rb.data_ptr() and y2.data_ptr() == bb.data_ptr()
    assert torch.equal(s2, s0) and torch.equal(y2, y0)


def test_residual_norm_unaligned(srv):
    import torch

    announce("residual_norm unaligned")
    d = _norm_case(1, 5, 256, "bf16", "f32", "bf16", "f32", 1, True, True)
    c = _cuda(d)
    want = srv.residual_norm(c["block"], c["resid"], pre_weight=c["pre"], post_weight=c["post"], gate=c["gate"])

    def shifted(t):
        buf = torch.zeros(t.numel() + 1, device="cuda", dtype=t.dtype)
        buf[1:] = t.reshape(-1)
        return buf[1:].view(t.shape)

    got = srv.residual_norm(*(shifted(c[k]) for k in ("block", "resid")), pre_weight=shifted(c["pre"]),
                            post_weight=shifted(c["post"]), gate=shifted(c["gate"]))
    torch.cuda.synchronize()
    hh, tol_h, y, tol_y = _norm_f64(d, 1.0, 1e-6, 0.0)
    for o in (want, got):
        assert bool(((o[0].cpu().double() - hh).abs() <= _rounded(tol_h, hh, "f32")).all())
        assert bool(((o[1].cpu().double() - y).abs() <= _rounded(tol_y, y, "f32")).all())


def test_residual_norm_offsets_past_32_bits(srv):
    import torch

    announce("residual_norm offsets past 32 bits")
    rows, h = 140000, 16384   # 2.3e9 elements
    x = torch.zeros((rows, h), device="cuda", dtype=torch.bfloat16)
    x[rows - 1] = 2.0
    w = torch.ones(h, device="cuda")
    s, y = srv.residual_norm(None, x, pre_weight=w, sum=x, y_dtype=torch.bfloat16, eps=0.25)
    torch.cuda.synchronize()
    assert bool((y[rows - 1] == torch.tensor(2.0 / 4.25 ** 0.5).bfloat16()).all()) and not bool(y[:rows - 1].any())


# ---- sampling --------------------------------------------------------------
def _sample_row(l, t, k, p, q, u):
    """(token, probability) of one row of logits (numpy f32), in 64 bits."""
    if not (l < np.inf).all() or np.isnan(l).any() or (l == -np.inf).all() or np.isnan(t) or np.isnan(u):
        return -1, np.nan
    l = l.astype(np.float64) + 0.0
    order = np.argsort(-l, kind="stable")
    order = order[l[order] > -np.inf]
    if not t > 0:
        return int(order[0]), 1.0
    w = np.exp((l[order] - l[order[0]]) / float(t))
    n = min(int(k), len(order)) if 0 < k < len(l) else len(order)
    mass = np.cumsum(w[:n])
    if p < 1:
        n = min(n, 1 + int(np.searchsorted(mass, float(p) * mass[-1])))
    if q > 0:
        n = max(1, min(n, int((w >= min(float(q), 1.0)).sum())))
    kept = np.zeros(len(l))
    kept[order[:n]] = w[:n]
    mass = np.cumsum(kept)
    tok = min(int(np.searchsorted(mass, max(float(u), 0.0) * mass[-1], side="right")), int(kept.nonzero()[0].max()))
    return tok, kept[tok] / mass[-1]


def _check_sample(srv, logits, t, k, p, q, u, **kw):
    import torch

    def f(v, dt):
        return None if v is None else torch.tensor(np.asarray(v), dtype=dt).cuda()

    rows = logits.shape[0]
    tok, pr = srv.sample(logits.cuda(), f(u, torch.float32), temperature=f(t, torch.float32), top_k=f(k, torch.int32),
                         top_p=f(p, torch.float32), min_p=f(q, torch.float32), **kw)
    torch.cuda.synchronize()
    l = logits.float().numpy()
    f32 = lambda v, d: np.full(rows, d, np.float32) if v is None else np.asarray(v, np.float32)   # noqa: E731
    t, p, q, u = f32(t, 1), f32(p, 1), f32(q, 0), f32(u, 0)
    k = np.zeros(rows, np.int64) if k is None else np.asarray(k)
    want = [_sample_row(l[i], t[i], k[i], p[i], q[i], u[i]) for i in range(rows)]
    got = list(zip(tok.cpu().tolist(), pr.cpu().double().tolist()))
    for i, ((gt, gp), (wt, wp)) in enumerate(zip(got, want)):
        assert gt == wt, (i, gt, wt, t[i], k[i], p[i], q[i], u[i])
        # (f32 rounding, and sums in f64 or fixed point: far below it)
        assert (np.isnan(gp) and np.isnan(wp)) or abs(gp - wp) <= 2 * U32 * wp, (i, gp, wp)
    return tok, pr


def _settings(rng, rows, vocab):
    pick = rng.integers(0, 8, rows)
    t = np.where(pick == 0, 0.0, rng.uniform(0.2, 2.0, rows))
    k = np.where(pick & 1, rng.integers(1, max(2, min(vocab, 300)), rows), 0)
    p = np.where(pick & 2, rng.uniform(0.05, 0.999, rows), 1.0)
    q = np.where(pick & 4, 10.0 ** rng.uniform(-4, -0.5, rows), 0.0)
    return t, k, p, q, rng.random(rows)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1), (3, 2), (9, 7), (40, 64), (33, 257), (24, 1023), (16, 4096), (24, 5001),
                                   (9, 32000), (5, 50257), (64, 9999), (3, 151936), (300, 300)],
                         ids=lambda s: "x".join(map(str, s)))
def test_sample_mixed(srv, shape, dt):
    import torch

    rows, vocab = shape
    announce(f"sample {shape} {dt}")
    rng = np.random.default_rng(rows + vocab)
    logits = torch.from_numpy((2.5 * rng.standard_normal((rows, vocab)) + 6 * (rng.random((rows, vocab)) < 20 / vocab))
                              .astype(np.float32)).to(_dt(dt))
    _check_sample(srv, logits, *_settings(rng, rows, vocab))


def test_sample_defaults(srv):
    """No settings at all: temperature 1, the whole distribution; probs may be NULL."""
    import rlxq
    import torch

    announce("sample defaults")
    rng = np.random.default_rng(3)
    logits = torch.from_numpy(rng.standard_normal((12, 3001)).astype(np.float32))
    u = rng.random(12)
    tok, _ = _check_sample(srv, logits, None, None, None, None, u)
    out = torch.full((14,), 99, dtype=torch.int32, device="cuda")
    lc, uc = logits.cuda(), torch.tensor(u, dtype=torch.float32).cuda()
    rc = rlxq.lib().rlxq_sample(srv.ctx.h, lc.data_ptr(), 0, 12, 3001, None, None, None, None, uc.data_ptr(),
                                out.data_ptr(), None, None)
    torch.cuda.synchronize()
    assert rc == 0 and torch.equal(out[:12], tok) and out[12:].tolist() == [99, 99]


def test_sample_borders(srv):
    """Settings at and past their ends, tokens at both ends of u."""
    import torch

    announce("sample borders")
    rng = np.random.default_rng(4)
    v = 3000
    rows = [(0.0, 0, 1.0, 0.0, 0.3), (-1.0, 5, 0.5, 0.1, 0.3), (np.nan, 0, 1.0, 0.0, 0.3), (np.inf, 0, 1.0, 0.0, 0.7),
            (1e-30, 0, 1.0, 0.0, 0.7), (1e-3, 3, 0.9, 0.0, 0.9), (1e4, 0, 0.9, 0.0, 0.123), (1e4, 777, 0.7, 0.0, 0.99),
            (1e4, 0, 1.0, 0.999, 0.4), (30.0, 2900, 0.97, 1e-3, 0.77), (1.0, 1, 1.0, 0.0, 0.999), (1.0, v, 1.0, 0.0, 0.5),
            (1.0, v + 5, 0.5, 0.0, 0.5), (1.0, v - 1, 1.0, 0.0, 0.9), (1.0, -3, 1.0, 0.0, 0.1), (1.0, 2 ** 31 - 1, 1.0, 0.0, 0.1),
            (1.0, 0, 0.0, 0.0, 0.5), (1.0, 0, -1.0, 0.0, 0.5), (1.0, 0, 1e-9, 0.0, 0.5), (1.0, 0, np.nan, 0.0, 0.5),
            (1.0, 0, 2.0, 0.0, 0.5), (1.0, 0, 1.0, 1.0, 0.5), (1.0, 0, 1.0, 7.0, 0.5), (1.0, 0, 1.0, np.nan, 0.5),
            (1.0, 0, 1.0, -2.0, 0.5), (1.0, 0, 1.0, 0.0, 0.0), (1.0, 0, 1.0, 0.0, np.float32(1 - 2.0 ** -24)),
            (1.0, 0, 1.0, 0.0, 1.0), (1.0, 0, 1.0, 0.0, 5.0), (1.0, 0, 1.0, 0.0, -0.5), (1.0, 0, 1.0, 0.0, np.nan),
            (1.0, 40, 0.9, 0.0, 0.0), (1.0, 40, 0.9, 0.0, 1.0), (0.7, 0, 0.99999994, 0.0, 0.6), (5.0, 2999, 0.9999, 1e-5, 0.31)]
    cols = list(zip(*rows))
    for dt in ("f32", "bf16"):
        logits = torch.from_numpy((3 * rng.standard_normal((len(rows), v))).astype(np.float32)).to(_dt(dt))
        _check_sample(srv, logits, *cols)


@pytest.mark.parametrize("v", [5, 1000, 5000, 40000])
def test_sample_ties_and_masks(srv, v):
    """Equal logits (all, few levels, +0 and -0), masked tokens, rows masked but
    for some, one or none, NaN and +inf."""
    import torch

    announce(f"sample ties v={v}")
    rng = np.random.default_rng(v)
    n = 17
    levels = rng.integers(0, 4, (n, v)).astype(np.float32)
    zeros = np.where(rng.random((n, v)) < 0.5, 0.0, -0.0).astype(np.float32)
    masked = np.where(rng.random((n, v)) < 0.9, -np.inf, rng.standard_normal((n, v))).astype(np.float32)
    masked[:, v // 2] = 1.5
    few = np.full((n, v), -np.inf, np.float32)
    few[:, 3] = -7.0
    few[::2, 1] = -7.0
    far = np.full((n, v), -60.0, np.float32)   # a likely token over a floor of others
    far[:, 2] = 0.0
    bad = rng.standard_normal((n, v)).astype(np.float32)
    bad[0::4, v - 1], bad[1::4, 0], bad[2::4] = np.nan, np.inf, -np.inf
    bad[3, 1] = -np.nan
    big = (rng.integers(-5, 5, (n, v)) * 1e30).astype(np.float32)
    huge = (rng.integers(-2, 2, (n, v)) * 3.4e38 / 2).astype(np.float32)
    for logits in (levels, zeros, masked, few, far, bad, big, huge):
        t, k, p, q, u = _settings(rng, n, v)
        p[3], t[3], k[3], q[3] = 0.3, 1.0, 0, 0.0
        k[4], t[4], p[4], q[4] = max(1, v // 3), 1.0, 0.5, 0.0
        t[5], k[5], p[5], q[5] = 1.0, 0, 1.0, 0.0
        _check_sample(srv, torch.from_numpy(logits), t, k, p, q, u)
    # uniform rows: sums are whole numbers, borders exact
    const = torch.full((8, v), 0.25)
    _check_sample(srv, const, [1.0] * 8, [0, 4, 0, 0, v // 2, 0, 3, 0], [1, 1, 0.5, 0.25, 0.5, 1, 1, 0.75], [0, 0, 0, 0, 0, 1, 0.5, 0],
                  [0.5, 0.75, 0.5, 0.0, 0.25, 0.125, 0.0, 0.625])


def test_sample_unaligned_and_rows_behind(srv):
    import torch

    announce("sample unaligned")
    rng = np.random.default_rng(8)
    for dt in ("f32", "bf16"):
        for v in (4099, 8192, 20001):
            base = torch.from_numpy(rng.standard_normal(5 * v + 3).astype(np.float32)).to(_dt(dt)).cuda()
            l = base[3:].view(5, v)
            t, k, p, q, u = _settings(rng, 5, v)
            f = lambda a, d: torch.tensor(a, dtype=d).cuda()   # noqa: E731
            tok, pr = torch.full((7,), 99, dtype=torch.int32, device="cuda"), torch.full((7,), 99.0, device="cuda")
            srv.sample(l, f(u, torch.float32), temperature=f(t, torch.float32), top_k=f(k, torch.int32),
                       top_p=f(p, torch.float32), min_p=f(q, torch.float32), tokens=tok[:5], probs=pr[:5])
            torch.cuda.synchronize()
            t, p, q, u = (np.asarray(x, np.float32) for x in (t, p, q, u))
            want = [_sample_row(l[i].float().cpu().numpy(), t[i], k[i], p[i], q[i], u[i])[0] for i in range(5)]
            assert tok.tolist() == want + [99, 99] and pr[5:].tolist() == [99.0, 99.0]


def test_sample_hot_rows_with_masked_tokens(srv):
    """Temperatures past every difference of the logits: the tokens that are not
    masked alike, the masked ones none."""
    import torch

    announce("sample hot rows")
    rng = np.random.default_rng(21)
    for v in (300, 9000):
        l = np.where(rng.random((8, v)) < 0.5, -np.inf, 5 * rng.standard_normal((8, v))).astype(np.float32)
        _check_sample(srv, torch.from_numpy(l), [np.inf, 1e37, 3e38, 1e36, np.inf, 1e30, np.inf, 1e38],
                      [0, 0, 7, 0, v - 1, 0, 0, 100], [1, 0.5, 1, 1, 0.25, 0.75, 1, 0.5], [0, 0, 0, 0.5, 0, 0, 1, 0],
                      rng.random(8))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_sample_largest_vocabulary(srv, dt):
    """2^20 tokens, rows that start inside 16 bytes; flat ones among them."""
    import torch

    announce(f"sample 2^20 {dt}")
    v, rng = 1 << 20, np.random.default_rng(31)
    buf = torch.zeros(5 * v + 1, dtype=_dt(dt), device="cuda")
    l = torch.from_numpy(rng.standard_normal((5, v)).astype(np.float32)).to(_dt(dt))
    buf[1:] = l.view(-1).cuda()
    t, k, p, q, u = [1.0, 0.7, 8.0, 1.0, 1.3], [0, 700000, 0, 300, 0], [1.0, 0.9, 0.8, 1.0, 0.97], [0, 0, 0, 0, 1e-3], rng.random(5)
    f = lambda a, d: torch.tensor(a, dtype=d).cuda()   # noqa: E731
    tok, _ = srv.sample(buf[1:].view(5, v), f(u, torch.float32), temperature=f(t, torch.float32), top_k=f(k, torch.int32),
                        top_p=f(p, torch.float32), min_p=f(q, torch.float32))
    torch.cuda.synchronize()
    t, p, q, u = (np.asarray(x, np.float32) for x in (t, p, q, u))
    assert tok.tolist() == [_sample_row(l[i].float().numpy(), t[i], k[i], p[i], q[i], u[i])[0] for i in range(5)]


def test_sample_rows_past_a_batch(srv):
    """More rows than one pair of launches takes."""
    import torch

    announce("sample rows past a batch")
    rng = np.random.default_rng(41)
    rows, v = 26000, 9   # (a row of one chunk takes 5.3 KB of the 128 MB)
    logits = torch.from_numpy(rng.standard_normal((rows, v)).astype(np.float32))
    _check_sample(srv, logits, *_settings(rng, rows, v))


def test_sample_repeats_itself(srv):
    """The same call, again and on another stream: the same tokens and probabilities."""
    import torch

    announce("sample repeats")
    rng = np.random.default_rng(11)
    rows, v = 48, 30000
    logits = torch.from_numpy((2 * rng.standard_normal((rows, v))).astype(np.float32)).cuda()
    t, k, p, q, u = (torch.tensor(a, dtype=d).cuda() for a, d in zip(
        _settings(rng, rows, v), (torch.float32, torch.int32, torch.float32, torch.float32, torch.float32)))
    first = srv.sample(logits, u, temperature=t, top_k=k, top_p=p, min_p=q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            again = srv.sample(logits, u, temperature=t, top_k=k, top_p=p, min_p=q)
        here = srv.sample(logits, u, temperature=t, top_k=k, top_p=p, min_p=q)
        torch.cuda.synchronize()
        for o in (again, here):
            assert torch.equal(o[0], first[0]) and torch.equal(o[1], first[1])


# ---- together --------------------------------------------------------------
def _step(srv, orc, seed, rows):
    """A decode step's tail: block output and residual, norm, packed projection with
    adapters, packed head, tokens.  Returns run(stream) and the f64 tokens' check."""
    import torch

    rng = np.random.default_rng(seed)
    h, n, vocab, rank, e = 256, 512, 3000, 16, 4
    f = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda()   # noqa: E731
    w = torch.from_numpy(orc.synth_q4_1(rng, n, h)).cuda()
    head = torch.from_numpy(orc.synth_q4_1(rng, vocab, n)).cuda()
    d = {"block": f(rows, h), "resid": f(rows, h), "pre": f(h), "post": f(h), "a": f(e, 2 * rank, h) / 16,
         "b": f(e, n, rank) / 8, "ids": torch.from_numpy(rng.integers(-1, e, rows).astype(np.int32)).cuda(),
         "u": torch.from_numpy(rng.random(rows).astype(np.float32)).cuda(),
         "t": torch.from_numpy(rng.uniform(0, 2, rows).astype(np.float32)).cuda(),
         "k": torch.from_numpy(rng.integers(0, 60, rows).astype(np.int32)).cuda(),
         "p": torch.from_numpy(rng.uniform(0.3, 1.2, rows).astype(np.float32)).cuda()}
    out = {"sum": torch.empty_like(d["resid"]), "y": torch.empty((rows, h), device="cuda"),
           "z": torch.empty((rows, n), device="cuda"), "l": torch.empty((rows, vocab), device="cuda"),
           "tok": torch.empty(rows, dtype=torch.int32, device="cuda"), "pr": torch.empty(rows, device="cuda")}
    ctx = srv.ctx

    def run():
        srv.residual_norm(d["block"], d["resid"], pre_weight=d["pre"], post_weight=d["post"], sum=out["sum"], y=out["y"])
        ctx.dequant_matmul(out["y"], w, 3, n, y=out["z"])
        srv.lora_matmul(out["y"], d["ids"], d["a"], d["b"], segments=[300, 212], base=out["z"], y=out["z"])
        ctx.dequant_matmul(out["z"], head, 3, vocab, y=out["l"])
        srv.sample(out["l"], d["u"], temperature=d["t"], top_k=d["k"], top_p=d["p"], tokens=out["tok"], probs=out["pr"])

    return d, out, run, (w, head, h, n, vocab, rank)


@pytest.mark.parametrize("rows", [1, 5, 40, 300])
def test_step_of_a_served_batch(srv, orc, rows):
    """Each operator on the output of the one before: the chain against 64 bits
    (the packed products' own bar, 1e-3 of the largest), the tokens on the logits
    that the step computed."""
    import torch

    announce(f"step rows={rows}")
    d, out, run, (w, head, h, n, vocab, rank) = _step(srv, orc, rows, rows)
    run()
    torch.cuda.synchronize()
    c = {k: v.cpu() for k, v in d.items()}
    hh, _, y, _ = _norm_f64({"block": c["block"], "resid": c["resid"], "gate": None, "post": c["post"], "pre": c["pre"]}, 1.0,
                            1e-6, 0.0)
    z = torch.from_numpy(orc.matmul_f64(orc.Q4_1, y.float().numpy(), w.cpu().numpy(), n)).double()
    z = _lora_f64({"x": y, "a": c["a"], "b": c["b"], "ids": c["ids"], "base": z, "ranks": None, "scales": None}, [300, 212])[0]
    assert float((out["z"].cpu().double() - z).abs().max() / z.abs().max()) <= 1e-3
    l = torch.from_numpy(orc.matmul_f64(orc.Q4_1, z.float().numpy(), head.cpu().numpy(), vocab)).double()
    assert float((out["l"].cpu().double() - l).abs().max() / l.abs().max()) <= 2e-3
    got = out["l"].cpu().numpy()
    want = [_sample_row(got[i], *(c[k][i].numpy() for k in ("t", "k", "p")), np.float32(0), c["u"][i].numpy())[0]
            for i in range(rows)]
    assert out["tok"].tolist() == want


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_step_in_a_graph(srv, orc, rows):
    """Captured and replayed with other inputs, eager work on the same scratch in
    between, against eager runs bit for bit."""
    import torch

    announce(f"step graph rows={rows}")
    d, out, run, _ = _step(srv, orc, 7 * rows, rows)
    d2, out2, run2, _ = _step(srv, orc, 7 * rows + 1, rows + 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run2(), run()   # (the stream's scratch at its largest)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        run()
    for i in range(4):
        for k, s in (("block", 1.0 + i), ("a", 0.5 + i)):
            d[k].mul_(s)
        d["ids"].copy_(d["ids"].roll(1))
        run()
        torch.cuda.synchronize()
        want = {k: v.clone() for k, v in out.items()}
        for v in out.values():
            v.fill_(7)
        with torch.cuda.stream(side):
            run2()
            g.replay()
            run2()
        torch.cuda.synchronize()
        for k in out:
            assert torch.equal(out[k], want[k]), (i, k)


def test_two_streams_at_once(srv, orc):
    """Steps on two streams, each with its own scratch."""
    import torch

    announce("two streams")
    steps = [_step(srv, orc, s, r) for s, r in ((21, 30), (22, 90))]
    want = []
    for _, out, run, _ in steps:
        run()
        torch.cuda.synchronize()
        want.append({k: v.clone() for k, v in out.items()})
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(5):
        for _, out, _, _ in steps:
            for v in out.values():
                v.fill_(3)
        torch.cuda.synchronize()
        for st, (_, _, run, _) in zip(streams, steps):
            with torch.cuda.stream(st):
                run()
        torch.cuda.synchronize()
        for (_, out, _, _), w in zip(steps, want):
            assert all(torch.equal(out[k], w[k]) for k in out)


@pytest.mark.parametrize("types", TYPES[:4], ids="_".join)
@pytest.mark.parametrize("m", [30, 129, 256])
def test_lora_few_rows_of_few_adapters_many_columns(srv, m, types):
    """More than 3 2^20 outputs of at most 256 rows by few adapters, and fewer
    outputs: integers, as in test_lora_integers_exact."""
    import torch

    announce(f"lora m={m} n=24600 {types}")
    d = _lora_case(m, m, 136, 24600, 24, 3, *types, segs=[24000, 600], ints=True, ranks=True)
    y = _run_lora(srv, d, [24000, 600])
    torch.cuda.synchronize()
    want, mag, _ = _lora_f64(d, [24000, 600])
    assert float(mag.max()) < 2 ** 24
    assert torch.equal(y.cpu(), want.to(_dt(types[2])))
