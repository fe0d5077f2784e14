"""Temperatures whose square leaves fp32: the distance has it as a factor, and would be 0, infinite or NaN."""
import pytest
import torch

from dizo_amd import _lib as L
from dizo_amd import token_loss as T
from dizo_amd._lib import DzError

P = 4096  # a pointer that is not NULL; nothing reads through it


def _call(temperature, batch):
    lib = L.load()
    rc = lib.dz_topk_distill(P, L.DZ_DTYPE_F16, batch, 3, 10, 30, 10, P, P, 4, temperature, 1, P, None, 0, 0, None, 0, 0, None)
    return rc, lib.dz_last_error().decode()


@pytest.mark.parametrize("temperature", [3e-39, 1e-25, 2.0**-64, 2.0**64, 1e20, 3e38])
def test_a_temperature_whose_square_leaves_fp32_is_refused(temperature, monkeypatch):
    rc, msg = _call(temperature, 2)
    assert rc < 0 and "temperature" in msg and "square" in msg
    monkeypatch.setattr(T, "_check_logits", lambda what, logits: 0)
    x, val, at = torch.zeros(3, 8), torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int64)
    with pytest.raises(DzError, match="temperature"):
        T.topk_distill(x, val, at, temperature=temperature)
    with pytest.raises(DzError, match="temperature"):
        T.topk_distill_grad(x, val, at, torch.ones(3), temperature=temperature)


@pytest.mark.parametrize("temperature", [2.0**-63, 0.01, 1.0, 100.0, 1.8e19])
def test_a_temperature_whose_square_is_of_fp32_is_not(temperature):
    assert _call(temperature, 0)[0] == 0  # no rows: the checks alone
