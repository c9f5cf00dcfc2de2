"""Performance cases of the operators around the packed products of a served
batch, in plain torch and through the library's calls.

Three operators: `lora` (low-rank adapters of many requests, each row its own,
added to a shared projection's output), `norm` (a block's output normalised,
gated, added to the residual stream, and the sum normalised for the next block)
and `sample` (a token per row under temperature, top-k, top-p and min-p, from
given random numbers).

Sizes: the Qwen3-8B linear shapes (hidden 4096, q|k|v 6144, gate|up 24576, down
12288 -> 4096), hidden 5120, and generic ranks, batches and vocabularies.
"""
from __future__ import annotations

import sys
from pathlib import Path

import numpy as np
import torch

own = False   # True: the library's calls; False: elementary torch operations

_ROOT = Path(__file__).resolve().parent.parent
_DT = {"f32": torch.float32, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "bf16": 2}

_ops = None


def _serving():
    """The library's serving operators (imported at the first call)."""
    global _ops
    if _ops is None:
        if str(_ROOT / "rlx-models_amd") not in sys.path:
            sys.path.insert(0, str(_ROOT / "rlx-models_amd"))
        import rlxq

        _ops = rlxq.Serving(rlxq.Context(0))
    return _ops


# ---- the cases -------------------------------------------------------------
def _case(name, **c):
    return {"name": name, **c} if name else c


def _lora(name, m, k, n, rank, adapters, x, ab, y, segs=1, ragged=False):
    """segs: 1, 2 (halves) or 3 (two thirds and two sixths, as q|k|v); ragged:
    the adapters' ranks differ."""
    return _case(name, op="lora", m=m, k=k, n=n, rank=rank, adapters=adapters, x=x, ab=ab, y=y, segs=segs, ragged=ragged)


def _norm(name, m, h, x, y, post=True, gate="none", resid="f32"):
    """gate: none, channel (one for all rows), group (one for each of 4 or fewer
    groups of rows) or row."""
    return _case(name, op="norm", m=m, h=h, x=x, y=y, post=post, gate=gate, resid=resid)


def _sample(name, m, vocab, x, mode):
    """mode: chat (top-k and top-p), top_p, free (temperature and min-p) or mixed
    (every request its own, greedy ones among them)."""
    return _case(name, op="sample", m=m, vocab=vocab, x=x, mode=mode)


def listed():
    return [
        # single-stream decode, q|k|v: launch latency and little else
        _lora("lora_m1_4096_6144_r16_bf16", 1, 4096, 6144, 16, 8, "bf16", "bf16", "bf16", segs=3),
        # 64 decoding streams over 48 adapters, gate|up: the adapters' bytes
        _lora("lora_m64_4096_24576_r64_bf16", 64, 4096, 24576, 64, 48, "bf16", "bf16", "bf16", segs=2),
        # a few streams with drafted tokens, f32 throughout, the down projection
        _lora("lora_m33_12288_4096_r32_f32", 33, 12288, 4096, 32, 5, "f32", "f32", "f32"),
        # short prompts of several requests, ranks that differ
        _lora("lora_m777_4096_4096_r128_f32", 777, 4096, 4096, 128, 6, "f32", "bf16", "f32", ragged=True),
        # long prompts of eight requests, gate|up: the largest
        _lora("lora_m4096_4096_24576_r64_bf16", 4096, 4096, 24576, 64, 8, "bf16", "bf16", "bf16", segs=2),
        # one decoding stream
        _norm("norm_1x4096_f32", 1, 4096, "f32", "f32", post=False),
        # a short prompt of an odd length, gated by request
        _norm("norm_197x5120_bf16", 197, 5120, "bf16", "bf16", gate="group"),
        # long prompts, gated by channel
        _norm("norm_16384x4096_bf16", 16384, 4096, "bf16", "bf16", gate="channel", resid="bf16"),
        # one chat
        _sample("sample_1x151936_chat", 1, 151936, "f32", "chat"),
        # a few requests, an odd vocabulary, bf16 logits
        _sample("sample_7x50257_mixed", 7, 50257, "bf16", "mixed"),
        # a served batch, every request its own settings
        _sample("sample_64x151936_mixed", 64, 151936, "f32", "mixed"),
        # rollouts: many rows, the whole distribution
        _sample("sample_256x128000_free", 256, 128000, "bf16", "free"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """A case of the listed ones' ranges: 1 to 4096 rows (16384 of the norm's),
    widths that are no multiple of any tile, ranks 8 to 128 of 1 to 64 adapters,
    vocabularies of 1000 to 160000."""
    op = rng.choice(["lora", "lora", "norm", "sample", "sample"])
    x = rng.choice(["f32", "bf16"])
    if op == "norm":
        h = 8 * _log_int(rng, 16, 1100)
        return _norm(None, _log_int(rng, 1, min(16384, 6 * 10 ** 7 // h)), h, x, rng.choice(["f32", "bf16"]),
                     post=rng.random() < 0.6, gate=rng.choice(["none", "channel", "group", "row"]),
                     resid=rng.choice(["f32", "bf16"]))
    if op == "sample":
        vocab = _log_int(rng, 1000, 160000)
        return _sample(None, _log_int(rng, 1, min(256, 2 * 10 ** 7 // vocab)), vocab, x,
                       rng.choice(["chat", "top_p", "free", "mixed"]))
    rank = 8 * _log_int(rng, 1, 16)
    m, k, n = _log_int(rng, 1, 3000), 8 * _log_int(rng, 16, 1536), _log_int(rng, 100, 20000)
    n = min(n, 4 * 10 ** 7 // m)
    segs = rng.randint(1, 3)
    most = min(64, 2048 // rank, 10 ** 8 // (rank * (n + segs * k)))
    return _lora(None, m, k, n, rank, _log_int(rng, 1, max(1, most)), x, rng.choice(["f32", "bf16"]),
                 rng.choice(["f32", "bf16"]), segs=segs, ragged=rng.random() < 0.5)


def _widths(case):
    n = case["n"]
    if case["segs"] == 3:
        return [n - 2 * (n // 6), n // 6, n // 6]
    return [n - n // 2, n // 2] if case["segs"] == 2 else [n]


# ---- inputs ----------------------------------------------------------------
def _rows(m, k, dtype, gen, size=1.0):
    """Activations: order one, some channels much larger."""
    channel = torch.exp(0.5 * torch.randn(k, device="cuda", generator=gen))
    return (size * torch.randn((m, k), device="cuda", generator=gen) * channel).to(dtype)


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    m = case["m"]

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    def uniform(*shape):
        return torch.rand(shape, device="cuda", generator=gen)

    if case["op"] == "lora":
        k, n, r, e, s, dt = case["k"], case["n"], case["rank"], case["adapters"], case["segs"], _DT[case["ab"]]
        d = {"x": _rows(m, k, _DT[case["x"]], gen), "base": _rows(m, n, _DT[case["y"]], gen)}
        d["a"] = (normal(e, s * r, k) / k ** 0.5).to(dt)
        d["b"] = (normal(e, n, r) * 0.2 / r ** 0.5).to(dt)
        d["scales"] = 0.5 + 2 * uniform(e)
        d["ranks"] = torch.full((e,), r, device="cuda", dtype=torch.int32)
        if case["ragged"]:
            d["ranks"] = (r * (1 + torch.randint(0, 4, (e,), device="cuda", generator=gen)) // 4).int()
        ids = torch.arange(m, device="cuda") % e
        if m > 256:   # prompts: a run of rows for each request
            ids = torch.sort(ids).values
        else:         # decoding streams in any order
            ids = torch.randperm(e, device="cuda", generator=gen)[ids][torch.randperm(m, device="cuda", generator=gen)]
        # (one stream in sixteen without an adapter)
        d["ids"] = torch.where(torch.arange(m, device="cuda") % 16 == 15, -1, ids).int()
        return d
    if case["op"] == "norm":
        h = case["h"]
        d = {"block": _rows(m, h, _DT[case["x"]], gen, 0.3), "resid": _rows(m, h, _DT[case["resid"]], gen, 3.0),
             "pre": 1 + 0.2 * normal(h), "post": 1 + 0.2 * normal(h) if case["post"] else None, "gate": None}
        if case["gate"] != "none":
            groups = next(g for g in (4, 3, 2, 1) if m % g == 0)
            d["gate"] = torch.sigmoid(normal({"channel": 1, "group": groups, "row": m}[case["gate"]], h)).to(_DT[case["x"]])
        return d
    v, mode = case["vocab"], case["mode"]
    # a few likely tokens over a broad rest, as a head's logits are
    d = {"logits": (2.5 * normal(m, v) + 6 * (uniform(m, v) < 20 / v)).to(_DT[case["x"]]), "u": uniform(m)}
    d["temperature"] = 0.5 + uniform(m) if mode != "chat" else torch.full((m,), 0.8, device="cuda")
    d["top_k"] = torch.full((m,), 50 if mode == "chat" else 0, device="cuda", dtype=torch.int32)
    d["top_p"] = torch.full((m,), 0.95 if mode in ("chat", "top_p") else 1.0, device="cuda")
    d["min_p"] = torch.zeros(m, device="cuda")
    if mode == "free":
        d["min_p"] = torch.where(uniform(m) < 0.25, 0.01, 0.0)
    if mode == "mixed":
        kind = torch.arange(m, device="cuda") % 6   # greedy, top-k, top-p, both, min-p, all three
        d["temperature"] = torch.where(kind == 0, 0.0, d["temperature"])
        k = torch.randint(1, 200, (m,), device="cuda", generator=gen)
        d["top_k"] = torch.where((kind == 1) | (kind == 3) | (kind == 5), k, 0).int()
        d["top_p"] = torch.where((kind == 2) | (kind == 3) | (kind == 5), 0.5 + 0.5 * uniform(m), 1.0)
        d["min_p"] = torch.where(kind >= 4, 0.1 * uniform(m), 0.0)
    return d


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    m = case["m"]
    if case["op"] == "lora":
        s["y"] = torch.empty_like(s["base"])
    elif case["op"] == "norm":
        s["sum"] = torch.empty_like(s["resid"])
        s["y"] = torch.empty((m, case["h"]), device="cuda", dtype=_DT[case["y"]])
    else:
        s["tokens"] = torch.empty(m, device="cuda", dtype=torch.int32)
        s["probs"] = torch.empty(m, device="cuda")
    return s


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    ops, c = _serving(), s["case"]
    if c["op"] == "lora":
        return ops.lora_matmul(s["x"], s["ids"], s["a"], s["b"], ranks=s["ranks"], scales=s["scales"],
                               segments=_widths(c), base=s["base"], y=s["y"])
    if c["op"] == "norm":
        return ops.residual_norm(s["block"], s["resid"], pre_weight=s["pre"], post_weight=s["post"], gate=s["gate"],
                                 scale=0.7, eps=1e-6, sum=s["sum"], y=s["y"])
    return ops.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                      min_p=s["min_p"], tokens=s["tokens"], probs=s["probs"])


# ---- the plain forms -------------------------------------------------------
def _run_plain(s):
    return {"lora": _plain_lora, "norm": _plain_norm, "sample": _plain_sample}[s["case"]["op"]](s)


def _plain_lora(s):
    c, x = s["case"], s["x"].float()
    e, g, r, k, m = c["adapters"], c["segs"], c["rank"], c["k"], c["m"]
    used = torch.arange(r, device=x.device) < s["ranks"][:, None]
    a = torch.where(used[:, None, :, None], s["a"].float().view(e, g, r, k), 0.0)
    b = torch.where(used[:, None, :], s["b"].float(), 0.0)
    on = (s["ids"] >= 0) & (s["ids"] < e)
    ids = torch.where(on, s["ids"], 0).long()
    factor = torch.where(on, s["scales"][ids], 0.0)
    if m <= 64:   # a few rows: their adapters gathered
        v = torch.bmm(a[ids].view(m, g * r, k), x[:, :, None]).view(m, g, r) * factor[:, None, None]
        d = [torch.bmm(w, v[:, j, :, None])[:, :, 0] for j, w in enumerate(torch.split(b[ids], _widths(c), dim=1))]
    else:         # many: the adapters side by side, a row's others at zero
        v = (x @ a.view(e * g * r, k).t()).view(m, e, g, r)
        v = v * torch.nn.functional.one_hot(ids, e)[:, :, None, None] * factor[:, None, None, None]
        d = [v[:, :, j].reshape(m, e * r) @ w.permute(0, 2, 1).reshape(e * r, -1)
             for j, w in enumerate(torch.split(b, _widths(c), dim=1))]
    return (s["base"].float() + torch.cat(d, 1)).to(_DT[c["y"]])


def _plain_norm(s):
    def unit(t):
        return t * torch.rsqrt((t * t).mean(1, keepdim=True) + 1e-6)

    t = s["block"].float()
    if s["post"] is not None:
        t = unit(t) * s["post"]
    if s["gate"] is not None:
        t = t * s["gate"].float().repeat_interleave(t.shape[0] // s["gate"].shape[0], 0)
    h = s["resid"].float() + 0.7 * t
    return h.to(s["resid"].dtype), (unit(h) * s["pre"]).to(_DT[s["case"]["y"]])


def _plain_sample(s):
    # sums and borders in 64 bits: a token's border lies next to the random number
    x, top_k, u = s["logits"].float(), s["top_k"], s["u"].double()[:, None]
    t, p, q = (s[n].double()[:, None] for n in ("temperature", "top_p", "min_p"))
    v, order = torch.sort(x, dim=1, descending=True, stable=True)
    v = v.double()
    rank = torch.arange(v.shape[1], device=x.device)
    w = torch.exp((v - v[:, :1]) / torch.where(t > 0, t, 1.0))
    w = torch.where(rank < torch.where(top_k > 0, top_k, v.shape[1])[:, None], w, 0.0)
    mass = torch.cumsum(w, 1)
    before = torch.cat([torch.zeros_like(t), mass[:, :-1]], 1)
    keep = ((p >= 1) | (before < p * mass[:, -1:])) & (w >= q) & (t > 0)
    w = torch.where(keep | (rank == 0), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)
    mass = torch.cumsum(w, 1)
    last = (w > 0).long().mul(rank).amax(1)
    tokens = torch.minimum((mass <= u * mass[:, -1:]).sum(1), last)
    probs = w.gather(1, tokens[:, None]) / mass[:, -1:]
    bad = ~(v[:, 0] < torch.inf) | (v[:, 0] == -torch.inf)
    return torch.where(bad, -1, tokens).int(), torch.where(bad, torch.nan, probs[:, 0]).float()


# ---- what a pass cannot do without -----------------------------------------
def work(case):
    m = case["m"]
    if case["op"] == "lora":
        k, n, r, g = case["k"], case["n"], case["rank"] * (0.625 if case["ragged"] else 1.0), case["segs"]
        return {"bytes": int(min(m, case["adapters"]) * r * (g * k + n) * _SIZE[case["ab"]] + m * k * _SIZE[case["x"]] +
                             2 * m * n * _SIZE[case["y"]]),
                "flops": int(2 * m * r * (g * k + n))}
    if case["op"] == "norm":
        return {"bytes": m * case["h"] * (_SIZE[case["x"]] * (2 if case["gate"] == "row" else 1) +
                                          2 * _SIZE[case["resid"]] + _SIZE[case["y"]]), "flops": 10 * m * case["h"]}
    return {"bytes": m * (case["vocab"] * _SIZE[case["x"]] + 28), "flops": 4 * m * case["vocab"]}


# ---- float64 ---------------------------------------------------------------
def exact(case, seed):
    d = _inputs(case, seed)
    if case["op"] == "lora":
        y, r = d["base"].double(), case["rank"]
        ends = np.cumsum([0] + _widths(case)).tolist()
        for e in range(case["adapters"]):
            at = (d["ids"] == e).nonzero()[:, 0]
            q = int(d["ranks"][e])
            for j in range(case["segs"]):
                v = d["x"][at].double() @ d["a"][e, j * r:j * r + q].double().t()
                y[at, ends[j]:ends[j + 1]] += d["scales"][e].double() * (v @ d["b"][e, ends[j]:ends[j + 1], :q].double().t())
        return y
    if case["op"] == "norm":
        t, h = d["block"].double(), case["h"]
        if case["post"]:
            t = d["post"].double() * t / (t.square().sum(1, keepdim=True) / h + 1e-6).sqrt()
        if d["gate"] is not None:
            g = d["gate"].double()
            t = (t.view(g.shape[0], -1, h) * g[:, None]).view(-1, h)
        t = d["resid"].double() + 0.7 * t
        return t, d["pre"].double() * t / (t.square().sum(1, keepdim=True) / h + 1e-6).sqrt()
    x = d["logits"].float().cpu().numpy().astype(np.longdouble)
    t, k, p, q, u = (d[n].cpu().numpy().astype(np.float64) for n in ("temperature", "top_k", "top_p", "min_p", "u"))
    tokens, probs = np.zeros(case["m"], np.int32), np.zeros(case["m"])
    for i, l in enumerate(x):
        order = np.argsort(-l, kind="stable")
        if t[i] <= 0:
            tokens[i], probs[i] = order[0], 1.0
            continue
        w = np.exp((l[order] - l[order[0]]) / t[i])
        n = int(k[i]) if 0 < k[i] < len(l) else len(l)
        mass = np.cumsum(w[:n])
        if p[i] < 1:
            n = min(n, 1 + int(np.searchsorted(mass, p[i] * mass[-1])))
        n = max(1, min(n, int((w >= q[i]).sum())))
        kept = np.zeros_like(l)
        kept[order[:n]] = w[:n]
        mass = np.cumsum(kept)
        tokens[i] = min(int(np.searchsorted(mass, u[i] * mass[-1], side="right")), int(kept.nonzero()[0].max()))
        probs[i] = kept[tokens[i]] / mass[-1]
    return torch.from_numpy(tokens), torch.from_numpy(probs)
