"""What the operators' Python side refuses before anything reaches a device."""
import types

import pytest

import jieyu_amd

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("cap", [0, 0.0, -1.0, 1e-50, -1e-50, float("nan")])
def test_caps_that_float32_does_not_hold(cap):
    """one that rounds to 0 would count as none"""
    from jieyu_amd import batch
    pool = types.SimpleNamespace(_b=batch._bind(), device=torch.device("cpu"))
    with pytest.raises(jieyu_amd.JyError, match="cap"):
        batch.PagePool._rules(pool, 1, 1, cap, None, None)
    assert batch.PagePool._rules(pool, 1, 1, 1e-30, None, None).cap > 0
