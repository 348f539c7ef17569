"""Verification of drafted tokens (capi.verify_drafts) at the ends of its numbers: logits at the ends of
fp32's range, weights that underflow, very many drafts."""
import pytest
import torch

from tests.test_verify_gpu import check, make
from vkwr_amd import capi

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


def test_uniform_of_zero_on_weights_that_underflow(gpu):
    """Without a filter a segment's sum is kept relative to its group's largest logit: in units of the row's it
    may be a denormal where every single weight is 0 (here 2^-1039 beside 2^-1010 in its group, 1 in the next).
    A uniform of 0 has to fall on an entry that has a weight, in vocabulary order."""
    V = 4096
    for drafted in (0, 1):
        l = torch.full((2, drafted + 1, V), -INF)
        l[:, :, 3:200] = -720.0
        l[:, :, 256:260] = -700.0
        l[:, :, 2048:2050] = 0.0
        tokens = torch.full((2, drafted + 1), -5, dtype=torch.int32, device=gpu)
        accepted = torch.empty(2, dtype=torch.int32, device=gpu)
        u = torch.zeros(2, drafted + 1)
        u[:, 0] = 0.0 if drafted == 0 else 0.9  # the draft, half of the row's mass, is rejected
        capi.verify_drafts(l.to(gpu), torch.full((2, drafted), 2048, dtype=torch.int32, device=gpu), u.to(gpu), tokens,
                           accepted)
        assert tokens[:, 0].tolist() == [256, 256] and accepted.tolist() == [0, 0]


@pytest.mark.parametrize("filt", [{}, {"top_p": 0.95}, {"top_k": 2, "top_p": 0.95}], ids=["all", "p95", "k2p95"])
@pytest.mark.parametrize("reject", [3, 63, 64, 65, 100000, 262143])
def test_hundreds_of_thousands_of_drafts(gpu, filt, reject):
    """The work has to grow with the drafts, not with their square: what each row tests of those before it is
    bounded.  (One sequence; entry 1 of 8 holds all but e^-20 of each row, and is drafted up to `reject`.)"""
    K, V = 262143, 8
    l = torch.full((1, K + 1, V), -20.0)
    l[:, :, 1] = 0.0
    drafts = torch.ones(1, K, dtype=torch.int32)
    if reject < K:
        drafts[0, reject] = 2
    u = torch.full((1, K + 1), 0.5)
    args = [t.to(gpu) for t in (l.half(), drafts, u)]
    tokens = torch.full((1, K + 1), -5, dtype=torch.int32, device=gpu)
    accepted = torch.empty(1, dtype=torch.int32, device=gpu)
    ws = torch.empty(capi.verify_workspace_bytes(1, K, V), dtype=torch.uint8, device=gpu)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    capi.verify_drafts(*args, tokens, accepted, workspace=ws, **filt)
    end.record()
    torch.cuda.synchronize()
    assert accepted.item() == reject
    assert (tokens[0, :reject + 1] == 1).all() and (tokens[0, reject + 1:] == -1).all()
    assert start.elapsed_time(end) < 2000.0  # milliseconds
