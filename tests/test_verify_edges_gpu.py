"""Verification of drafted tokens (capi.verify_drafts) at the ends of its numbers: logits at the ends of
fp32's range, weights that underflow, very many drafts."""
import pytest
import torch

from tests.test_verify_gpu import check, make

pytestmark = pytest.mark.gpu

F = torch.finfo(torch.float32).max
INF = float("inf")


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("V", [4, 1000, 4096, 8192, 140000])
@pytest.mark.parametrize("filt", [{}, {"top_k": 1}, {"top_k": 3, "top_p": 0.9}, {"top_k": 700}, {"top_p": 0.6},
                                  {"temperature": 1000.0}], ids=["all", "k1", "k3p90", "k700", "p60", "hot"])
def test_infinities_beside_the_ends_of_the_range(gpu, V, probs, filt):
    """-inf counts as the lowest finite value and +inf as the largest, so they are tied with entries that hold
    those: in one part of the row, and in parts of their own."""
    d = make(8, 3, V, seed=61 + V, half=False, probs=probs)
    l = d["logits"]
    l[0, :], l[0, :, 1::2] = -F, -INF
    l[1, :], l[1, :, : V // 2] = -F, -INF
    l[2, :], l[2, :, V - 1] = -INF, -F
    l[3, :, 0], l[3, :, 1] = INF, F
    l[4, :, 0], l[4, :, V - 1] = F, INF
    l[5, :, V // 2:] = F
    l[5, :, 0] = INF
    l[6, :], l[6, :, ::2], l[6, :, 3] = -INF, -F, 1.0
    l[7, :, 1], l[7, :, 2:] = F, -INF
    d["n_draft"][:] = 3
    check(gpu, d, **filt)
