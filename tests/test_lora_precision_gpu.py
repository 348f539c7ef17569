"""What the adapters' inner values x A^T keep of their bits, and rows in different company (capi.lora)."""
import math

import pytest
import torch

from oracle import serving_ref as ref
from tests.test_lora_gpu import HALF16, make, run_lora

pytestmark = pytest.mark.gpu


def cancelled(gpu, d):
    """The rows with the base that leaves least of the result: what shows are the sums' errors, not the rounding
    to fp16 of a result of their size.  Checked against the oracle's bound."""
    for t in d["t"]:
        full, _ = ref.lora(t["x"], t["a"], t["b"], torch.zeros_like(t["base"]), d["ids"], d["scale"])
        t["base"] = -full.half()
    for t, y in zip(d["t"], run_lora(gpu, d)):
        want, err = ref.lora(t["x"], t["a"], t["b"], t["base"], d["ids"], d["scale"])
        assert (want.abs() <= full.abs().max() * HALF16).all()
        bad = (y.cpu().double() - want).abs() > err + HALF16 * (want.abs() + err) + 2.0 ** -25
        assert not bad.any(), (int(bad.sum()), float(((y.cpu().double() - want).abs() / err).max()))


@pytest.mark.parametrize("last", [8, 12, 14])
@pytest.mark.parametrize("m,R,K", [(20, 16, 256), (150, 32, 512)])
def test_ranks_of_different_sizes(gpu, m, R, K, last):
    """A's rows from 1 down to 2^-last and B's columns inversely: every rank counts for as much in the result,
    however small its inner value is beside the row's largest."""
    d = make(m, 2, R, [(64, K)], seed=last + R, none=0.0)
    f = torch.exp2(-torch.linspace(0, last, R).round())
    t = d["t"][0]
    t["a"], t["b"] = (t["a"].float() * f[:, None]).half(), (t["b"].float() / f).half()
    assert t["b"].abs().max() < 60000
    cancelled(gpu, d)
