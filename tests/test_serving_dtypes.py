"""CPU tests of rlxq.Serving: an output type that contradicts a given tensor's is
refused, one that agrees is not."""
import pytest
import torch

import rlxq

F, BF = torch.float32, torch.bfloat16
X, IDS, A, B = torch.zeros((3, 64)), torch.zeros(3, dtype=torch.int32), torch.zeros((2, 8, 64)), torch.zeros((2, 10, 8))
W = torch.ones(64)


@pytest.fixture
def srv(monkeypatch):
    """A context on no device: the tensors' device is not looked at, no call is made."""
    class Lib:
        def __getattr__(self, fn):
            return lambda *args: 0

    monkeypatch.setattr(rlxq, "lib", Lib)
    monkeypatch.setattr(rlxq, "_on_device", lambda device, **t: None)
    monkeypatch.setattr(rlxq, "_stream", lambda stream, device: 0)
    c = rlxq.Context.__new__(rlxq.Context)
    c.h, c.device = None, -1   # (where CPU tensors are)
    return rlxq.Serving(c)


@pytest.mark.parametrize("dt,other", [(F, BF), (BF, F)])
def test_lora_y_dtype(srv, dt, other):
    t = torch.zeros((3, 10), dtype=dt)
    for kw in ({"base": t}, {"y": t}, {"base": t, "y": t}):
        with pytest.raises(ValueError, match="y_dtype"):
            srv.lora_matmul(X, IDS, A, B, y_dtype=other, **kw)
        assert srv.lora_matmul(X, IDS, A, B, y_dtype=dt, **kw).dtype is dt
        assert srv.lora_matmul(X, IDS, A, B, **kw).dtype is dt
    assert srv.lora_matmul(X, IDS, A, B, y_dtype=dt).dtype is dt
    assert srv.lora_matmul(X, IDS, A, B).dtype is F
    with pytest.raises(ValueError, match="y_dtype"):
        srv.lora_matmul(X, IDS, A, B, y_dtype=torch.float16)


@pytest.mark.parametrize("dt,other", [(F, BF), (BF, F)])
def test_residual_norm_y_dtype(srv, dt, other):
    y = torch.zeros((3, 64), dtype=dt)
    with pytest.raises(ValueError, match="y_dtype"):
        srv.residual_norm(X, X, pre_weight=W, y=y, y_dtype=other)
    assert srv.residual_norm(X, X, pre_weight=W, y=y, y_dtype=dt)[1] is y
    assert srv.residual_norm(X, X, pre_weight=W, y_dtype=dt)[1].dtype is dt
    assert srv.residual_norm(X.to(dt), X.to(dt), pre_weight=W)[1].dtype is dt
    assert srv.residual_norm(X, X, post_weight=W, y_dtype=dt)[1] is None   # (no y is asked for)
