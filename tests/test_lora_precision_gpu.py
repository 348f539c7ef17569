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


def test_an_infinite_rank_leaves_the_others_finite(gpu):
    """One rank of an adapter overflows (an infinity in A) beside inner values beyond fp16's range: the result is
    that infinity, not the NaN of two."""
    m, R, K, N = 5, 8, 64, 16
    a = torch.ones(1, R, K).half()
    a[0, 0, 0] = float("inf")
    x = torch.full((m, K), 8192.0).half()    # inner values of 2^19 where finite
    x[3] = 2.0
    b = torch.full((1, N, R), -2.0 ** -10).half()
    b[0, ::2, 0] = 2.0 ** -10                # (odd columns: of the same sign as the others)
    d = {"ids": torch.zeros(m, dtype=torch.int32), "scale": None,
         "t": [{"x": x, "a": a, "b": b, "base": torch.zeros(m, N).half()}]}
    y = run_lora(gpu, d)[0].float().cpu()
    assert (y[:, ::2] == float("inf")).all() and (y[:, 1::2] == -float("inf")).all()


@pytest.mark.parametrize("K", [200, 2048, 8192])
def test_a_row_in_different_company(gpu, K):
    """A row alone, among other adapters' rows, and among 20, 40 and 200 of its own adapter's: operands straight
    into registers or through LDS, K in few and many parts.  Each is within the sums' bound of the exact value and
    rounded once, so any two are within twice the bound and a whole step of fp16 of each other."""
    N, R, G = 264, 24, 4
    d = make(240, G, R, [(N, K)], seed=K, none=0.0)
    t = d["t"][0]
    d["ids"][:] = 1
    want, err = ref.lora(t["x"][:1], t["a"], t["b"], t["base"][:1], d["ids"][:1], d["scale"])
    got = []
    for own, others in ((1, 0), (1, 39), (20, 0), (40, 0), (40, 200), (200, 0), (200, 40)):
        ids = torch.ones(own + others, dtype=torch.int32)
        ids[own:] = torch.tensor([-1, 0, 2, 3], dtype=torch.int32).repeat(others // 4 + 1)[:others]
        e = {"ids": ids, "scale": d["scale"], "t": [{**t, "x": t["x"][:own + others], "base": t["base"][:own + others]}]}
        got.append(run_lora(gpu, e)[0][:1].cpu().double())
        assert ((got[-1] - want).abs() <= err + HALF16 * (want.abs() + err) + 2.0 ** -25).all()
    for y in got[1:]:
        assert ((y - got[0]).abs() <= 2 * err + 2 * HALF16 * (want.abs() + err) + 2.0 ** -24).all()
