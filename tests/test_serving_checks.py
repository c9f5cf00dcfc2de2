"""CPU tests of rlxq.Serving: what its methods and the C entry points refuse
before anything is queued, and the stream that they pass."""
import ctypes as C
import types

import pytest
import torch

import rlxq

X, IDS = torch.zeros((3, 64)), torch.zeros(3, dtype=torch.int32)
A, B, B2 = torch.zeros((2, 8, 64)), torch.zeros((2, 10, 8)), torch.zeros((2, 16, 64))
L, U = torch.zeros((3, 50)), torch.zeros(3)
BF = torch.bfloat16

CALLS = {
    "lora_matmul": lambda s, **k: s.lora_matmul(X, IDS, A, B, **k),
    "residual_norm": lambda s, **k: s.residual_norm(X, X.clone(), pre_weight=torch.ones(64), **k),
    "sample": lambda s, **k: s.sample(L, U, **k),
}


def test_sizes_that_fit():
    rlxq.check_lora_matmul(X, IDS, A, B, ranks=torch.zeros(2, dtype=torch.int32), scales=torch.ones(2),
                           base=torch.zeros((3, 10)), y=torch.zeros((3, 10)))
    rlxq.check_lora_matmul(X, IDS, B2, B, segments=[4, 6])
    rlxq.check_residual_norm(X, X, pre_weight=torch.ones(64), gate=torch.ones((3, 64)), sum=X, y=X)
    rlxq.check_sample(L, U, temperature=U, top_k=IDS, top_p=U, min_p=U, tokens=IDS, probs=U)


@pytest.mark.parametrize("kw", [
    dict(x=X.double()), dict(x=X[0]), dict(x=torch.zeros((64, 3)).t()), dict(ids=IDS.long()), dict(ids=IDS[:2]),
    dict(ids=IDS[:, None]), dict(a=A[:, :7]), dict(a=A[:, :, :32].contiguous()), dict(a=A[:1]), dict(a=A.to(BF)), dict(b=B.to(BF)),
    dict(b=B[:1]), dict(segments=[4, 6]), dict(a=B2), dict(a=B2, segments=[4, 5]), dict(a=B2, segments=[-1, 11]),
    dict(segments=[]), dict(ranks=torch.zeros(2)), dict(ranks=torch.zeros(3, dtype=torch.int32)),
    dict(scales=torch.zeros(3)), dict(scales=torch.zeros(2, dtype=BF)), dict(base=torch.zeros((3, 9))),
    dict(base=torch.zeros((3, 10)), y=torch.zeros((3, 10), dtype=BF)), dict(y=torch.zeros((10, 3)).t()),
    dict(y=torch.zeros((3, 10), dtype=torch.float16)), dict(x=None), dict(ids=None)])
def test_lora_refuses(kw):
    args = {"x": X, "ids": IDS, "a": A, "b": B, **kw}
    with pytest.raises(ValueError):
        rlxq.check_lora_matmul(args.pop("x"), args.pop("ids"), args.pop("a"), args.pop("b"), **args)


@pytest.mark.parametrize("kw", [
    dict(block=None, resid=None), dict(block=None, gate=torch.ones((1, 64))), dict(block=None, post_weight=torch.ones(64)),
    dict(y=X), dict(resid=X[:2]), dict(block=X.double()), dict(pre_weight=torch.ones(63)), dict(post_weight=torch.ones((1, 64))),
    dict(pre_weight=torch.ones(64), post_weight=torch.ones(64, dtype=BF)), dict(sum=torch.zeros((3, 64), dtype=BF)),
    dict(gate=torch.ones((2, 64))), dict(gate=torch.ones((6, 64))), dict(gate=torch.ones((0, 64))), dict(gate=torch.ones((1, 63))),
    dict(gate=torch.ones(64)), dict(sum=torch.zeros((64, 3)).t())])
def test_residual_norm_refuses(kw):
    args = {"block": X, "resid": X, **kw}
    with pytest.raises(ValueError):
        rlxq.check_residual_norm(args.pop("block"), args.pop("resid"), **args)


@pytest.mark.parametrize("kw", [
    dict(logits=L.double()), dict(logits=L[0]), dict(logits=torch.zeros((50, 3)).t()), dict(u=None), dict(u=U.double()), dict(u=U[:2]),
    dict(temperature=torch.zeros(4)), dict(top_k=U), dict(top_p=U.double()), dict(min_p=U[None]), dict(tokens=IDS.long()),
    dict(probs=torch.zeros(2))])
def test_sample_refuses(kw):
    args = {"logits": L, "u": U, **kw}
    with pytest.raises(ValueError):
        rlxq.check_sample(args.pop("logits"), args.pop("u"), **args)


def _serving(device):
    c = rlxq.Context.__new__(rlxq.Context)
    c.h, c.device = None, device
    return rlxq.Serving(c)


@pytest.mark.parametrize("name", CALLS)
def test_tensors_off_the_contexts_device(name):
    with pytest.raises(ValueError, match="context is on cuda:0"):
        CALLS[name](_serving(0))


@pytest.mark.parametrize("name", CALLS)
def test_stream_of_the_contexts_device(name, monkeypatch):
    got = {}

    class Lib:
        def __getattr__(self, fn):
            def call(*args):
                got[fn] = args
                return 0

            return call

    monkeypatch.setattr(rlxq, "lib", Lib)
    monkeypatch.setattr(rlxq, "_on_device", lambda device, **t: None)
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d: types.SimpleNamespace(cuda_stream=1000 + d))
    for kw, want in (({}, 1003), ({"stream": 77}, 77)):
        got.clear()
        CALLS[name](_serving(3), **kw)
        assert got["rlxq_" + name][-1] == want


def test_every_method_with_a_stream_is_here():
    import inspect

    have = {n for n, f in inspect.getmembers(rlxq.Serving, inspect.isfunction) if "stream" in inspect.signature(f).parameters}
    assert have == set(CALLS)


def test_null_context():
    lib = rlxq.lib()
    assert lib.rlxq_lora_matmul(None, None, 0, None, None, None, 0, None, None, None, 1, 1, 8, 8, 8, 1, None, None, 0,
                                None) == rlxq.E_NULL
    assert lib.rlxq_residual_norm(None, None, 0, None, 0, None, 0, 1, None, None, 0, 0.0, 1.0, 1e-6, 1, 8, None, None, 0,
                                  None) == rlxq.E_NULL
    assert lib.rlxq_sample(None, None, 0, 1, 8, None, None, None, None, None, None, None, None) == rlxq.E_NULL


# ---- the C entry points' refusals: need a context, launch nothing -------------
P = 1 << 20   # an aligned address that no refused call reads


def _lora(ctx, x=P, x_dtype=0, ids=P, a=P, b=P, ab=0, ranks=None, scales=None, ends=None, segs=1, m=4, k=64, n=32, rank=8, e=2,
          base=None, y=P, y_dtype=0):
    e_ = (C.c_int64 * len(ends))(*ends) if ends is not None else None
    return rlxq.lib().rlxq_lora_matmul(ctx.h, x, x_dtype, ids, a, b, ab, ranks, scales, e_, segs, m, k, n, rank, e, base, y,
                                       y_dtype, None)


def _norm(ctx, block=P, bd=0, resid=P, rd=0, gate=None, gd=0, gr=1, post=None, pre=P, wd=0, off=0.0, scale=1.0, eps=1e-6, rows=4,
          h=64, sum=P, y=P, yd=0):
    return rlxq.lib().rlxq_residual_norm(ctx.h, block, bd, resid, rd, gate, gd, gr, post, pre, wd, off, scale, eps, rows, h, sum,
                                         y, yd, None)


def _sample(ctx, l=P, ld=0, rows=4, v=50, t=None, k=None, p=None, q=None, u=P, tok=P, pr=None):
    return rlxq.lib().rlxq_sample(ctx.h, l, ld, rows, v, t, k, p, q, u, tok, pr, None)


REFUSED = [
    (_lora, dict(m=-1), "E_SHAPE"), (_lora, dict(n=-1), "E_SHAPE"), (_lora, dict(k=0), "E_SHAPE"), (_lora, dict(m=2 ** 24 + 1), "E_SHAPE"),
    (_lora, dict(m=2 ** 62), "E_SHAPE"), (_lora, dict(n=2 ** 62), "E_SHAPE"), (_lora, dict(k=2 ** 62), "E_SHAPE"),
    (_lora, dict(m=2 ** 24, n=2 ** 24), "E_SHAPE"),
    (_lora, dict(rank=0), "E_SHAPE"), (_lora, dict(rank=12), "E_SHAPE"), (_lora, dict(rank=264), "E_SHAPE"), (_lora, dict(e=0), "E_SHAPE"),
    (_lora, dict(e=2 ** 14 + 1), "E_SHAPE"), (_lora, dict(k=60), "E_ALIGN"), (_lora, dict(x_dtype=2), "E_DTYPE"),
    (_lora, dict(ab=2), "E_DTYPE"), (_lora, dict(y_dtype=7), "E_DTYPE"), (_lora, dict(segs=2), "E_NULL"), (_lora, dict(segs=0), "E_NULL"),
    (_lora, dict(ends=[32], segs=0), "E_SHAPE"), (_lora, dict(ends=[8, 16, 20, 24, 32], segs=5), "E_SHAPE"),
    (_lora, dict(ends=[31], segs=1), "E_SHAPE"), (_lora, dict(ends=[33], segs=1), "E_SHAPE"), (_lora, dict(ends=[-1, 32], segs=2), "E_SHAPE"),
    (_lora, dict(ends=[20, 10, 32], segs=3), "E_SHAPE"), (_lora, dict(x=None), "E_NULL"), (_lora, dict(ids=None), "E_NULL"),
    (_lora, dict(a=None), "E_NULL"), (_lora, dict(b=None), "E_NULL"), (_lora, dict(y=None), "E_NULL"), (_lora, dict(x=P + 8), "E_ALIGN"),
    (_lora, dict(a=P + 4), "E_ALIGN"), (_lora, dict(b=P + 2), "E_ALIGN"), (_lora, dict(y=P + 2), "E_ALIGN"),
    (_lora, dict(base=P + 1, y_dtype=1), "E_ALIGN"), (_lora, dict(ids=P + 2), "E_ALIGN"),
    (_norm, dict(rows=-1), "E_SHAPE"), (_norm, dict(h=0), "E_SHAPE"), (_norm, dict(h=2 ** 24 + 1), "E_SHAPE"), (_norm, dict(rows=2 ** 62), "E_SHAPE"),
    (_norm, dict(bd=2), "E_DTYPE"), (_norm, dict(rd=3), "E_DTYPE"), (_norm, dict(wd=2), "E_DTYPE"), (_norm, dict(yd=2), "E_DTYPE"),
    (_norm, dict(gate=P, gd=2), "E_DTYPE"), (_norm, dict(gate=P, gr=3), "E_SHAPE"), (_norm, dict(gate=P, gr=0), "E_SHAPE"),
    (_norm, dict(gate=P, gr=8), "E_SHAPE"), (_norm, dict(eps=-1.0), "E_SHAPE"), (_norm, dict(eps=float("nan")), "E_SHAPE"),
    (_norm, dict(block=None, resid=None), "E_NULL"), (_norm, dict(block=None, gate=P), "E_NULL"), (_norm, dict(block=None, post=P), "E_NULL"),
    (_norm, dict(sum=None, y=None, pre=None), "E_NULL"), (_norm, dict(y=None), "E_NULL"), (_norm, dict(pre=None), "E_NULL"),
    (_norm, dict(block=P + 2), "E_ALIGN"), (_norm, dict(sum=P + 1, rd=1), "E_ALIGN"),
    (_sample, dict(rows=-1), "E_SHAPE"), (_sample, dict(v=0), "E_SHAPE"), (_sample, dict(v=2 ** 20 + 1), "E_SHAPE"),
    (_sample, dict(rows=2 ** 40), "E_SHAPE"), (_sample, dict(ld=2), "E_DTYPE"), (_sample, dict(l=None), "E_NULL"), (_sample, dict(u=None), "E_NULL"),
    (_sample, dict(tok=None), "E_NULL"), (_sample, dict(l=P + 2), "E_ALIGN"), (_sample, dict(l=P + 1, ld=1), "E_ALIGN"),
    (_sample, dict(tok=P + 2), "E_ALIGN"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(len(REFUSED)), ids=lambda i: REFUSED[i][0].__name__[1:] + "-" + "-".join(
    f"{k}={v}" for k, v in REFUSED[i][1].items()))
def test_entry_point_refuses(ctx, i):
    call, kw, status = REFUSED[i]
    assert call(ctx, **kw) == getattr(rlxq, status)
    assert rlxq.lib().rlxq_last_error(ctx.h)


@pytest.mark.gpu
def test_empty_calls(ctx):
    """No rows (or columns): fine, with NULL pointers too."""
    for kw in (dict(m=0), dict(n=0), dict(m=0, x=None, ids=None, a=None, b=None, y=None)):
        assert _lora(ctx, **kw) == rlxq.OK
    assert _norm(ctx, rows=0) == rlxq.OK and _norm(ctx, rows=0, block=None, resid=None, sum=None, y=None) == rlxq.OK
    assert _sample(ctx, rows=0) == rlxq.OK and _sample(ctx, rows=0, l=None, u=None, tok=None) == rlxq.OK
