"""The forms that a branch output may take in front of the norm that leaves rows in 8 bits: all of them are checked before the launch."""

import pytest
import torch


@pytest.fixture
def launches(monkeypatch):
    """The kernels' calls recorded instead of made, tensors of the CPU let through otherwise checked."""
    from pyre_b200.kernels import ops
    seen = []

    def check(t, name, dtype=None, dim=None):
        if dtype is not None and t.dtype != dtype:
            raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
        if dim is not None and t.dim() != dim:
            raise ValueError(f"{name} must have {dim} dimensions")

    monkeypatch.setattr(ops, "_check", check)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops.lib, "call", lambda name, *args: seen.append((name, args)))
    return seen


def test_a_deferred_product_of_another_type_is_refused(launches, monkeypatch):
    """Its bfloat16 rows would be read as float32, twice as far as they go."""
    from pyre_b200.kernels import ops
    T, H = 3, 64
    x, w = torch.zeros((T, H)), torch.ones(H)
    y = torch.zeros((T, H), dtype=torch.bfloat16)
    deferred = ops.DeferredProduct(torch.zeros((T, 32), dtype=torch.bfloat16), torch.zeros((H, 32), dtype=torch.bfloat16), torch.bfloat16)
    monkeypatch.setattr(ops, "gemm_tc", lambda *a, **kw: y)
    ops.add_rmsnorm_rows8(x, deferred, w, 1e-6)
    name, args = launches.pop()
    assert name == "pyre_norm_rows8" and args[1] == y.data_ptr() and args[2] is None
    with pytest.raises(ValueError, match="delta must be torch.float32"):
        ops.add_rmsnorm_rows8(x, deferred, w, 1e-6, dtype=torch.float32)
    assert not launches


def test_partial_sums_and_plain_branches(launches):
    from pyre_b200.kernels import ops
    T, H = 3, 64
    x, w = torch.zeros((T, H)), torch.ones(H)
    parts = ops.PartialSums(torch.zeros((2, T, H)), torch.bfloat16)
    for dtype in (torch.bfloat16, torch.float32):
        ops.add_rmsnorm_rows8(x, parts, w, 1e-6, dtype=dtype)
        args = launches.pop()[1]
        assert args[1] is None and args[2] == parts.parts.data_ptr() and args[3] == 2 and args[4] == T * H
        ops.add_rmsnorm_rows8(x, None, w, 1e-6, dtype=dtype)
        assert launches.pop()[1][1:4] == (None, None, 0)
    with pytest.raises(ValueError, match="delta must be"):
        ops.add_rmsnorm_rows8(x, torch.zeros((T, H), dtype=torch.bfloat16), w, 1e-6, dtype=torch.float32)
    with pytest.raises(ValueError, match="delta shape"):
        ops.add_rmsnorm_rows8(x, ops.PartialSums(torch.zeros((2, T, H + 1)), torch.bfloat16), w, 1e-6)
