"""The kernels that large calls of rlxq.Serving run on: several pieces of a row a
thread (norm), several chunks a workgroup (sampling), ranks past 128, slices of K
and wide column blocks with the list of tiles (adapters)."""
import numpy as np
import pytest

from conftest import announce
from test_serving_gpu import TYPES, _check_sample, _cuda, _dt, _lora_case, _norm_case, _norm_f64, _rounded, _settings

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24


@pytest.fixture(scope="module")
def srv(ctx):
    import rlxq

    return rlxq.Serving(ctx)


def _last_kernel(srv):
    import rlxq

    return rlxq.lib().rlxq_last_kernel(srv.ctx.h).decode()


# ---- residual norm: more than two rows a CU, 65 to 1024 pieces of eight ------
@pytest.mark.parametrize("types", [("f32", "f32", "f32", "f32", "f32"), ("bf16", "bf16", "bf16", "bf16", "bf16"),
                                   ("bf16", "f32", "f32", "f32", "bf16"), ("f32", "bf16", "bf16", "f32", "f32")], ids="_".join)
@pytest.mark.parametrize("case", [(513, 520, 0), (600, 4096, 3), (1030, 1000, 5), (520, 8192, 520), (2000, 1032, 1)],
                         ids=lambda c: "x".join(map(str, c)))
def test_norm_of_many_rows(srv, case, types):
    """types: block, resid (and sum), gate, weights, y."""
    import torch

    rows, h, gate_rows = case
    for post, block, resid in ((True, True, True), (False, True, True), (False, False, True), (True, True, False)):
        announce(f"norm of many rows {case} {types} post={post} block={block} resid={resid}")
        d = _norm_case(rows + h, rows, h, *types[:4], gate_rows if block else 0, post, True, block, resid)
        c = _cuda(d)
        s, y = srv.residual_norm(c["block"], c["resid"], pre_weight=c["pre"], post_weight=c["post"], gate=c["gate"], scale=0.7,
                                 eps=1e-5, y_dtype=_dt(types[4]))
        torch.cuda.synchronize()
        assert _last_kernel(srv).endswith("_c2")
        hh, tol_h, want, tol_y = _norm_f64(d, 0.7, 1e-5, 0.0)
        assert bool(((s.cpu().double() - hh).abs() <= _rounded(tol_h, hh, types[1] if resid else "f32")).all())
        assert bool(((y.cpu().double() - want).abs() <= _rounded(tol_y, want, types[4])).all())


# ---- sampling: two and three chunks a workgroup ------------------------------
@pytest.mark.parametrize("shape", [(640, 17001, "f32"), (960, 20001, "bf16"), (1700, 9001, "f32"), (700, 16390, "bf16")],
                         ids=lambda s: "x".join(map(str, s)))
def test_sample_of_many_rows(srv, shape):
    """Rows whose number of chunks is and is not a multiple of a workgroup's, that
    start anywhere in 16 bytes; with borders and without."""
    import torch

    rows, vocab, dt = shape
    announce(f"sample of many rows {shape}")
    rng = np.random.default_rng(rows)
    l = 2.5 * rng.standard_normal((rows, vocab)) + 6 * (rng.random((rows, vocab)) < 20 / vocab)
    l[::7] = np.where(rng.random(l[::7].shape) < 0.9, -np.inf, l[::7])
    l[3::50, 1] = np.nan
    l[4::50] = -np.inf
    logits = torch.from_numpy(l.astype(np.float32)).to(_dt(dt))
    t, k, p, q, u = _settings(rng, rows, vocab)
    _check_sample(srv, logits, t, k, p, q, u)
    _check_sample(srv, logits, np.where(t > 0, t, 1.0), None, None, None, u)


# ---- adapters with the list of tiles -----------------------------------------
def _lora_by_adapter(d, segs):
    """y and the sums of absolute values in f64, an adapter's rows at a time."""
    import torch

    e, n, r = d["b"].shape
    y = d["base"].double().clone()
    mag = y.abs()
    ends = np.cumsum([0] + (segs or [n])).tolist()
    for q in range(e):
        at = (d["ids"] == q).nonzero()[:, 0]
        s, rk = float(d["scales"][q]), int(d["ranks"][q]) if d["ranks"] is not None else r
        x = d["x"][at].double()
        for j in range(len(ends) - 1):
            a, b = d["a"][q, j * r:j * r + rk].double(), d["b"][q, ends[j]:ends[j + 1], :rk].double()
            y[at, ends[j]:ends[j + 1]] += s * ((x @ a.t()) @ b.t())
            mag[at, ends[j]:ends[j + 1]] += abs(s) * ((x.abs() @ a.abs().t()) @ b.abs().t())
    return y, mag


# (m, k, n, rank, adapters, segments)
LISTS = [(300, 264, 200, 256, 3, [100, 100]), (777, 136, 264, 136, 5, None), (513, 72, 129, 200, 2, None),     # ranks past 128
         (300, 4096, 72, 16, 3, None), (400, 2056, 130, 40, 4, [65, 65]), (260, 1544, 96, 128, 2, None),        # 8, 4, 3 slices of K
         (1100, 64, 16400, 32, 4, [9000, 7400]), (1100, 72, 16401, 24, 4, None),                                # 512 columns
         (4096, 64, 8200, 64, 6, [5000, 3200]), (2100, 64, 16384, 128, 3, None), (2100, 40, 16640, 136, 3, [8200, 200, 8240])]  # 1024


@pytest.mark.parametrize("types", TYPES, ids="_".join)
@pytest.mark.parametrize("case", LISTS, ids=lambda c: "x".join(map(str, c[:5])))
def test_lora_list_integers_exact(srv, case, types):
    """Every sum is a whole number below 2^24: equal up to y's own rounding."""
    import torch

    m, k, n, rank, e, segs = case
    announce(f"lora list ints {case} {types}")
    d = _lora_case(m + k, m, k, n, rank, e, *types, segs=segs, ints=True, ranks=k % 16 == 8)
    c = _cuda(d)
    y = srv.lora_matmul(c["x"], c["ids"], c["a"], c["b"], ranks=c["ranks"], scales=c["scales"], segments=segs, base=c["base"])
    torch.cuda.synchronize()
    assert "_many_" in _last_kernel(srv) and (rank <= 128 or _last_kernel(srv).endswith("_s8"))
    want, mag = _lora_by_adapter(d, segs)
    assert float(mag.max()) < 2 ** 24
    assert torch.equal(y.cpu(), want.to(_dt(types[2])))


@pytest.mark.parametrize("types", TYPES, ids="_".join)
@pytest.mark.parametrize("case", LISTS[:6], ids=lambda c: "x".join(map(str, c[:5])))
def test_lora_list_values(srv, case, types):
    """Chains of at most T k / 4 + 3 rank + 24 additions (a quarter of K a wave, T bf16
    products an f32 one, then waves, slices, and v's three terms by rank)."""
    import torch

    m, k, n, rank, e, segs = case
    announce(f"lora list values {case} {types}")
    d = _lora_case(3 * m + k, m, k, n, rank, e, *types, segs=segs, ranks=True)
    c = _cuda(d)
    y = srv.lora_matmul(c["x"], c["ids"], c["a"], c["b"], ranks=c["ranks"], scales=c["scales"], segments=segs, base=c["base"])
    torch.cuda.synchronize()
    want, mag = _lora_by_adapter(d, segs)
    terms = 1 if types[0] == types[1] == "bf16" else (8 if types[0] == types[1] else 3)
    tol = (terms * k / 4 + 3 * rank + 24) * U32 * mag + U32 * want.abs() + 1e-30
    if types[2] == "bf16":
        tol = tol + 2.0 ** -8 * (want.abs() + tol)
    assert bool(((y.cpu().double() - want).abs() <= tol).all())
