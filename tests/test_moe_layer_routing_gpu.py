"""Routing of the expert layer past the few-token kernels: the router product's
two kernels (a wave per expert and four rows, or per four experts and eight rows)
in every type, with experts and rows that do not divide, and the top-k kernels
for up to 64, 128, 256 and 1024 experts.  ids and weights against float64; y, of
sampled rows, within the bounds of test_moe_layer_gpu.py."""
import numpy as np
import pytest

from conftest import announce
from test_moe_layer_gpu import Layer


def _kernels(rows, experts):
    """What layer_logits and layer_pick choose (moe_host.cpp)."""
    big = ((experts + 3) // 4) * ((rows + 7) // 8) >= 1024
    return "e4r8" if big else "e1r4", 1 if experts <= 64 else 2 if experts <= 128 else 4 if experts <= 256 else 16


# (rows, hidden, inter, experts, top_k), kernels
CASES = [((40, 256, 64, 128, 8), ("e1r4", 2)), ((261, 256, 64, 128, 8), ("e4r8", 2)), ((257, 544, 32, 127, 5), ("e4r8", 2)),
         ((262, 96, 32, 129, 6), ("e4r8", 4)), ((37, 288, 32, 129, 4), ("e1r4", 4)), ((40, 64, 32, 300, 10), ("e1r4", 16)),
         ((109, 64, 32, 299, 10), ("e4r8", 16)), ((35, 96, 32, 1023, 64), ("e4r8", 16)), ((515, 160, 32, 63, 3), ("e4r8", 1)),
         ((66, 2048, 32, 64, 8), ("e1r4", 1))]


def test_the_cases_reach_every_kernel():
    assert all(_kernels(s[0], s[3]) == k for s, k in CASES)
    assert {k for _, k in CASES} >= {(b, n) for b in ("e1r4", "e4r8") for n in (1, 2, 4, 16)}


@pytest.mark.gpu
@pytest.mark.parametrize("xdt,rdt", [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[0])) + "-" + c[1][0])
def test_routing(ctx, orc, case, xdt, rdt):
    import torch

    shape = rows, hidden, inter, experts, top_k = case[0]
    announce(f"moe_layer routing {shape} x={xdt} router={rdt}")
    L = Layer(orc, np.random.default_rng(sum(shape)), *shape, "q4_1", "q4_1", xdt=xdt, rdt=rdt)
    i = torch.empty((rows, top_k), dtype=torch.int32, device="cuda")
    q = torch.empty((rows, top_k), device="cuda")
    y = L.call(ctx, ids=i, probs=q)
    torch.cuda.synchronize()
    got = i.cpu().numpy()
    ids, p, _, big = L.route()
    # equal but for logits that agree to their rounding (2^-24 of the largest,
    # twice): those may change places
    l = L.xv @ L.rv.T
    diff = np.abs(np.take_along_axis(l, got.astype(np.int64), 1) - np.take_along_axis(l, ids, 1))
    assert np.all((got == ids) | (diff <= 2 * 2.0 ** -24 * big))
    assert all(len(set(r)) == top_k for r in got.tolist()) and np.mean(got == ids) > 0.999
    # l - max: two rounded logits and the difference's own rounding; expf, the sums
    # over E and over the slots and two divisions (E + 16 times 2^-23)
    np.testing.assert_allclose(q.cpu().numpy(), p, rtol=4 * 2.0 ** -24 * big + (experts + 16) * 2.0 ** -23)
    at = np.unique(np.r_[0, 1, rows - 2, rows - 1, np.random.default_rng(0).integers(0, rows, 4)])
    L.shape = (len(at),) + shape[1:]
    L.xv = L.xv[at]
    L.check(y[torch.from_numpy(at).cuda()], got[at], p[at], big)
