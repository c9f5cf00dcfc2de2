"""Low-rank adapters: v takes part in the second product with all of its bits, and
up to the largest float, whatever y's type."""
import numpy as np
import pytest

from conftest import announce

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def srv(ctx):
    import rlxq

    return rlxq.Serving(ctx)


def _dt(name):
    import torch

    return {"f32": torch.float32, "bf16": torch.bfloat16}[name]


@pytest.mark.parametrize("ydt", ["bf16", "f32"])
@pytest.mark.parametrize("xdt", ["bf16", "f32"])
@pytest.mark.parametrize("m", [1, 20, 300])
@pytest.mark.parametrize("rank", [8, 40, 72, 256])
def test_base_that_nearly_cancels(srv, rank, m, xdt, ydt):
    """Integers: v has 20 bits, at most eight of a column's b are 1 or -1, so that
    every sum stays below 2^24 and is exact; base is the bf16 next to minus the
    adapter's part: y is what is left, up to its own rounding."""
    import torch

    announce(f"lora cancel rank={rank} m={m} x={xdt} y={ydt}")
    g = torch.Generator()
    g.manual_seed(rank + m)
    k, n, e = 64, 136, 3
    x = torch.randint(100, 129, (m, k), generator=g).double()
    a = torch.randint(100, 129, (e, rank, k), generator=g).double()
    b = torch.zeros(e, n, rank, dtype=torch.float64)
    at = torch.randint(0, rank, (e, n, 8), generator=g)
    b.scatter_(2, at, (2 * torch.randint(0, 2, (e, n, 8), generator=g) - 1).double())
    ids = torch.randint(0, e, (m,), generator=g)
    v = torch.einsum("erk,mk->mer", a, x)[torch.arange(m), ids]
    part = (b[ids] * v[:, None]).sum(2)
    assert float(v.max()) > 2 ** 18 and float((b[ids].abs() * v[:, None].abs()).sum(2).max()) < 2 ** 23
    base = -part.float().bfloat16().float()
    want = (base.double() + part).float().to(_dt(ydt))
    c = lambda t, dt: t.to(dt).cuda()   # noqa: E731
    y = srv.lora_matmul(c(x, _dt(xdt)), c(ids, torch.int32), c(a, torch.bfloat16), c(b, torch.bfloat16), base=c(base, _dt(ydt)))
    torch.cuda.synchronize()
    assert torch.equal(y.cpu(), want)


@pytest.mark.parametrize("ydt", ["bf16", "f32"])
@pytest.mark.parametrize("m", [3, 300])
def test_largest_v(srv, m, ydt):
    """v at the largest float, above the largest bf16: finite, and so is y."""
    import torch

    announce(f"lora largest v m={m} y={ydt}")
    big = float(np.finfo(np.float32).max)
    x = torch.zeros(m, 16)
    x[:, 3] = big * torch.where(torch.arange(m) % 2 == 0, 1.0, -1.0)
    a, b = torch.zeros(2, 8, 16), torch.zeros(2, 40, 8)
    a[:, 5, 3] = 1.0
    b[:, :, 5] = 2.0 ** -torch.arange(1, 41).float()
    want = (x[:, 3:4].double() * b[0, :, 5].double()).float().to(_dt(ydt))
    y = srv.lora_matmul(x.cuda(), (torch.arange(m) % 2).int().cuda(), a.bfloat16().cuda(), b.bfloat16().cuda(), y_dtype=_dt(ydt))
    torch.cuda.synchronize()
    assert torch.equal(y.cpu(), want)
