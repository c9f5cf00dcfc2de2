"""Sampling where a border or a token lies among weights far below the row's
largest: rows of a few equal likely tokens over a floor of equal others, whose
kept set follows from one division.

With h likely tokens of weight 1 and a floor of weight w, top-p keeps the likely
ones and the first r of the floor (by index), r the least whole number with h + r w
>= p M, M the mass of what top-k leaves.  u = 1 takes the last kept token, so the
token names the border itself.  A sum of f64 roundings moves (p M - h) / w by at
most some 8 2^-53 M / w, so cases whose fraction lies within that (and 0.01) of a whole number
are not taken."""
import numpy as np
import pytest

from conftest import announce

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def srv(ctx):
    import rlxq

    return rlxq.Serving(ctx)


def _row(v, heads, floor):
    l = np.full(v, floor, np.float32)
    l[heads] = 0.0
    return l


def _weight(floor, t=1.0):
    return np.exp(np.longdouble(np.float32(floor)) / np.longdouble(np.float32(t)))


def border(v, heads, floor, p, k=0, t=1.0):
    """(the last kept token, the kept mass, the weight of a floor token)."""
    h, w = len(heads), _weight(floor, t)
    mass = h + ((k if 0 < k < v else v) - h) * w
    x = (np.longdouble(np.float32(p)) * mass - h) / w
    away = abs(x - np.rint(x))
    assert x > 1 and away > 0.01 and away > 8 * 2.0 ** -53 * mass / w, (float(x), float(away))
    r = int(np.ceil(x))
    at = np.delete(np.arange(v), heads)[r - 1]   # the last one of the floor's
    return max(int(at), max(heads)), h + r * w, w


def _sample(srv, l, u, dt="f32", **kw):
    import torch

    rows = l.shape[0]
    types = {"top_k": torch.int32}
    l = torch.from_numpy(l).to({"f32": torch.float32, "bf16": torch.bfloat16}[dt]).cuda()
    f = lambda x, d: torch.tensor(np.asarray(x), dtype=d).cuda().expand(rows).contiguous()   # noqa: E731
    tok, pr = srv.sample(l, f(u, torch.float32), **{n: f(x, types.get(n, torch.float32)) for n, x in kw.items()})
    torch.cuda.synchronize()
    return tok.cpu().tolist(), pr.cpu().double().tolist()


# (vocabulary, floor, top-p, top-k, temperature): more floor tokens than are listed
FLOORS = [(151936, -23.0, 0.99999, 0, 1.0), (151936, -24.5, 1 - 2.0 ** -23, 0, 1.0),
          (60001, -12.0, 0.999999, 0, 0.5), (151936, -23.0, 0.99999, 140001, 1.0),
          (151936, -27.25, 1 - 2.0 ** -24, 150000, 1.0), (20003, -11.5, 0.999999, 0, 0.5)]


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("case", FLOORS, ids=lambda c: "_".join(map(str, c)))
def test_border_in_a_floor_past_the_list(srv, case, dt):
    v, floor, p, k, t = case
    announce(f"sample floor {case} {dt}")
    heads = [2]
    want, mass, w = border(v, heads, floor, p, k, t)
    tok, pr = _sample(srv, _row(v, heads, floor)[None], 1.0, dt, top_p=p, top_k=k, temperature=t)
    assert tok == [want]
    assert abs(pr[0] - float(w / mass)) <= 2.0 ** -23 * float(w / mass)


# (vocabulary, likely tokens, floor, top-p, top-k, temperature): the floor's share of a
# chunk that holds a likely token counts; the last three rows are listed as a whole
CHUNKS = [(1 << 20, [2], -30.0, 1 - 2.0 ** -24, 0, 1.0), (60000, [2], -26.0, 1 - 2.0 ** -23, 0, 1.0),
          (163840, [4096 * i + 7 for i in range(8)], -25.875, 1 - 2.0 ** -24, 0, 1.0),
          (163840, [4096 * i + 7 for i in range(20)], -24.875, 1 - 2.0 ** -24, 0, 1.0),
          (151936, [4096 * i + 4000 for i in range(12)], -25.25, 1 - 2.0 ** -24, 150001, 1.0),
          (60001, [4096 * i + 100 for i in range(3)], -12.9375, 1 - 2.0 ** -24, 0, 0.5),
          (8001, [2], -25.25, 1 - 2.0 ** -24, 0, 1.0), (8001, [2, 900], -24.75, 1 - 2.0 ** -24, 0, 1.0),
          (8001, [2, 900], -24.75, 1 - 2.0 ** -24, 7900, 1.0)]


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("case", CHUNKS, ids=lambda c: f"{c[0]}_{len(c[1])}_{c[2]}_{c[3]}_{c[4]}")
def test_border_in_a_floor_of_chunks_with_likely_tokens(srv, case, dt):
    v, heads, floor, p, k, t = case
    announce(f"sample chunks {case} {dt}")
    want, mass, w = border(v, heads, floor, p, k, t)
    assert want > max(heads)
    tok, pr = _sample(srv, _row(v, heads, floor)[None], 1.0, dt, top_p=p, top_k=k, temperature=t)
    assert tok == [want]
    assert abs(pr[0] - float(w / mass)) <= 2.0 ** -23 * float(w / mass)


# (vocabulary, floor, u): a likely token at 0 over a floor, no border at all
TOKENS = [(1 << 20, -30.0, 1 - 2.0 ** -24), (60000, -26.0, 1 - 2.0 ** -23), (60000, -25.5, 1 - 2.0 ** -22),
          (4000, -24.625, 1 - 2.0 ** -24), (151936, -23.0, 1 - 2.0 ** -18)]


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("case", TOKENS, ids=lambda c: "_".join(map(str, c)))
def test_token_in_a_floor(srv, case, dt):
    """u M lies in the floor: index i, the first with 1 + i w > u M."""
    v, floor, u = case
    announce(f"sample token {case} {dt}")
    w = _weight(floor)
    mass = 1 + (v - 1) * w
    x = (np.longdouble(np.float32(u)) * mass - 1) / w
    away = abs(x - np.rint(x))
    assert 1 < x < v - 1 and away > 0.01 and away > 8 * 2.0 ** -53 * mass / w
    tok, pr = _sample(srv, _row(v, [0], floor)[None], u, dt)
    assert tok == [int(np.floor(x)) + 1]
    assert abs(pr[0] - float(w / mass)) <= 2.0 ** -23 * float(w / mass)


def _floor_token(v, floor, k, u):
    """The token of u, from one likely token at 0 over the first k - 1 of a floor."""
    w = _weight(floor)
    mass = 1 + (k - 1) * w
    x = (np.longdouble(np.float32(u)) * mass - 1) / w
    away = abs(x - np.rint(x))
    assert 1 < x < k - 1 and away > 0.01 and away > 8 * 2.0 ** -53 * mass / w
    return int(np.floor(x)) + 1, float(w / mass)


# (vocabulary, floor, top-k, u): what top-k keeps of a floor, the last row listed
KEPT = [(163840, -27.0, 150001, 1 - 2.0 ** -24), (60000, -26.25, 59001, 1 - 2.0 ** -24), (163840, -25.625, 120000, 1 - 2.0 ** -23),
        (8001, -25.25, 7000, 1 - 2.0 ** -24)]


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("case", KEPT, ids=lambda c: "_".join(map(str, c)))
def test_token_among_a_floor_that_is_kept(srv, case, dt):
    v, floor, k, u = case
    announce(f"sample kept {case} {dt}")
    want, share = _floor_token(v, floor, k, u)
    tok, pr = _sample(srv, _row(v, [0], floor)[None], u, dt, top_k=k)
    assert tok == [want] and abs(pr[0] - share) <= 2.0 ** -23 * share


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("v", [3000, 9001, 40000, 151936])
def test_least_u_takes_the_first_that_is_kept(srv, v, dt):
    """However little it weighs: sums of what lies ahead of the likely token are not
    lost.  Rows differ in the floor; top-k leaves one of it out, min-p nothing."""
    announce(f"sample least u v={v} {dt}")
    floors = [-20.0, -40.0, -60.0, -88.0, -300.0]
    likely, l = v - 100, np.stack([_row(v, [v - 100], f) for f in floors])
    p = 1 - 2.0 ** -24
    for kw, kept in (({}, floors), ({"top_k": v - 1}, floors), ({"top_k": v - 1, "top_p": p}, [f for f in floors if v * _weight(f) > 1 - p]),
                     ({"min_p": 1e-38}, [f for f in floors if _weight(f) >= 1e-38])):
        for u in (0.0, -1.0, 1.5e-45):
            tok, _ = _sample(srv, l, u, dt, **kw)
            assert tok == [0 if f in kept and _weight(f) > u else likely for f in floors], (kw, u)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("v", [300, 5000, 50257, 151936])
def test_u_from_1_up_takes_the_last_that_is_kept(srv, v, dt):
    """However little it weighs beside what the sums round to."""
    announce(f"sample last v={v} {dt}")
    import torch

    rng = np.random.default_rng(v)
    l = (3 * rng.standard_normal((12, v))).astype(np.float32)
    top = l.max(1, keepdims=True)
    l[:, v - 3:] = top - 38   # 2^-54 of the largest
    l[:, 1:2] = top - 45      # (what top-k of v - 1 leaves out)
    rounded = torch.from_numpy(l).to({"f32": torch.float32, "bf16": torch.bfloat16}[dt]).float().numpy()
    best = [int(max(np.argsort(-r, kind="stable")[:200])) for r in rounded]
    for kw, want in (({}, [v - 1] * 12), ({"top_k": v - 1}, [v - 1] * 12), ({"min_p": 1e-18}, [v - 1] * 12), ({"top_k": 200}, best)):
        for u in (1.0, 5.0, np.inf):
            assert _sample(srv, l, u, dt, **kw)[0] == want, (kw, u)


@pytest.mark.parametrize("v", [300, 3000, 40000])
def test_least_u_and_the_smallest_weights(srv, v):
    """A weight counts as long as f64 has it, denormals among them: e^-745 is one,
    e^-750 is 0."""
    announce(f"sample smallest weights v={v}")
    floors = [-690.0, -701.0, -720.0, -744.0, -750.0, -2000.0]
    l = np.stack([_row(v, [v - 100], f) for f in floors])
    for dt in ("f32", "bf16"):
        for kw in ({}, {"top_k": v - 1}, {"temperature": 0.5}):
            t, x = kw.get("temperature", 1.0), l if dt == "f32" else np.round(l / 4) * 4   # (bf16: multiples of 4)
            first = [0 if np.exp(np.float64(f) / t) > 0 else v - 100 for f in x[:, 0]]
            assert _sample(srv, x, 0.0, dt, **kw)[0] == first, kw
            assert _sample(srv, x, 1.0, dt, **kw)[0] == [v - 1 - ("top_k" in kw) if f == 0 else v - 100 for f in first], kw


# (vocabulary, likely tokens, floor, top-p, temperature, the likely tokens' logit)
FAR = [(163840, [4096 * i + 7 for i in range(8)], -25.875, 1 - 2.0 ** -24, 1.0, 1e6), (60001, [4096 * i + 100 for i in range(3)], -26.0, 1 - 2.0 ** -24, 1.0, -8e6),
       (60001, [4096 * i + 100 for i in range(3)], -12.875, 1 - 2.0 ** -24, 0.5, 2.0 ** 20),
       (163840, [4096 * i + 7 for i in range(20)], -24.75, 1 - 2.0 ** -24, 1.0, 3e5), (8001, [2, 900], -24.75, 1 - 2.0 ** -24, 1.0, -1e6)]


@pytest.mark.parametrize("case", FAR, ids=lambda c: f"{c[0]}_{len(c[1])}_{c[2]}_{c[5]}")
def test_border_in_a_floor_of_rows_far_from_0(srv, case):
    v, heads, floor, p, t, at = case
    announce(f"sample far {case}")
    want, _, _ = border(v, heads, floor, p, 0, t)
    l = _row(v, heads, floor) + np.float32(at)
    assert l[0] - np.float32(at) == floor
    assert _sample(srv, l[None], 1.0, top_p=p, temperature=t)[0] == [want]


# (vocabulary, the likely token, the token that u falls into, top-k): both in one chunk, most also in one thread's eight
AHEAD = [(12288, 6000, 5000, 0), (12288, 5003, 5000, 12287), (60001, 39990, 39987, 0), (60001, 39990, 37001, 60000),
         (300, 250, 120, 299), (300, 122, 120, 250), (4000, 498, 497, 500)]


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("case", AHEAD, ids=lambda c: "_".join(map(str, c)))
def test_u_ahead_of_a_likely_token(srv, case, dt):
    """What lies ahead of a likely token by index is summed by itself: u M in a floor of
    2^-58 to 2^-130 of it, index i the first with (i + 1) w > u M."""
    v, likely, token, k = case
    announce(f"sample ahead {case} {dt}")
    for floor in (-40.0, -58.0, -80.0):
        w = _weight(floor)
        mass = 1 + ((k if k else v) - 1) * w
        u = np.float32((token + 0.5) * w / mass)
        x = np.longdouble(u) * mass / w
        assert abs(x - np.rint(x)) > 0.3 and int(x) == token
        tok, pr = _sample(srv, _row(v, [likely], floor)[None], u, dt, top_k=k)
        assert tok == [token], floor
        assert abs(pr[0] - float(w / mass)) <= 2.0 ** -23 * float(w / mass) + 1e-45
