"""Beam selection where the other tests do not go: many groups of many beams, offsets past 32 bits, what a workspace
held before, and scores so far from zero that tokens' scores are equal in 64 bits.
"""
import pytest
import torch

from oracle import beam_ref
from tests.test_beam_gpu import check, inputs, run
from vkwr_amd import capi

pytestmark = pytest.mark.gpu
INF = float("inf")


def oracle(l, s, n, e, end, alpha):
    """(the logits stay on the GPU: sorting millions of them on the host would take minutes)"""
    return beam_ref.select(l.cuda(), s, n, e, end, alpha)


# keys of a row: W times the groups of 8192 entries; above 256 they are ranked by walking the groups' lists
@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("B,W,V", [(2, 32, 65537), (1, 32, 73728), (2, 17, 131073), (3, 3, 2 ** 20), (1, 5, 400000),
                                   (1, 20, 2 ** 20), (1, 32, 2 ** 20)])
def test_many_keys_a_row(B, W, V, half):
    a = inputs(B, W, V, half, seed=B + W + V, ended=0.1)
    check(run(*a, end=3, alpha=0.7), oracle(*a, 3, 0.7))


@pytest.mark.parametrize("half", [True, False])
def test_many_keys_in_few_groups(half):
    """All of a beam's best in one group, in the last one, and spread evenly; beams with next to nothing allowed."""
    W, V = 32, 90000
    l, s, n, e = inputs(1, W, V, half, seed=3)
    s[:] = torch.linspace(-1.0, -1.5, W)
    l[0, 0, 5000:5100] += 30.0
    l[0, 1, V - 50:] += 30.0
    l[0, 2, ::2500] += 30.0
    l[0, 3] = -INF
    l[0, 3, [7, 80000]] = 1.0
    l[0, 4] = -INF
    l[0, 5, :82000] = -INF
    check(run(l, s, n, e), oracle(l, s, n, e, -1, 0.0))


@pytest.mark.parametrize("W", [2, 17, 32])
def test_ties_among_many_keys(W):
    V = 2 ** 17 + 5
    l = torch.zeros(3, W, V)
    l[1, :, ::3] = 1.0
    l[1, :, 0] = -0.0
    l[2] = torch.randint(0, 3, (W, V), generator=torch.Generator().manual_seed(3)).float()
    s, n, e = torch.full((3, W), -1.5), torch.full((3, W), 3, dtype=torch.int32), torch.zeros(3, W, dtype=torch.int32)
    for t in (l, l.half()):
        check(run(t, s, n, e), oracle(t, s, n, e, -1, 0.0))


def test_offsets_past_32_bits():
    """The last of 2080 rows of 2^20 fp16 logits; the requests before it are one row over and over."""
    B, W, V = 65, 32, 2 ** 20
    g = torch.Generator(device="cuda").manual_seed(1)
    l = torch.empty(B, W, V, dtype=torch.float16, device="cuda")
    l[:] = torch.randn(V, generator=g, device="cuda").half()
    l[-1] = (3.0 * torch.randn(W, V, generator=g, device="cuda")).half()
    s = -torch.rand(B, W, generator=torch.Generator().manual_seed(2)).sort(1).values
    n, e = torch.ones(B, W, dtype=torch.int32), torch.zeros(B, W, dtype=torch.int32)
    got = run(l, s, n, e)
    one = run(l[-1:], s[-1:], n[-1:], e[-1:])
    for a, b in zip(got, one):
        assert torch.equal(a[-1:], b)
    check(one, oracle(l[-1:], s[-1:], n[-1:], e[-1:], -1, 0.0))


@pytest.mark.parametrize("byte", [0, 0x7f, 0xff])
def test_what_the_workspace_held_does_not_matter(byte):
    """Rows that offer nothing or only themselves are not written there: NaN, infinities and large keys stay in."""
    B, W, V = 6, 5, 20000
    l, s, n, e = inputs(B, W, V, True, seed=4, ended=0.4)
    s[1, 1:] = -INF
    s[2] = -INF
    e[3] = 1
    l[4, 2] = -INF
    ws = torch.full((capi.beam_workspace_bytes(B, W, V),), byte, dtype=torch.uint8, device="cuda")
    check(run(l, s, n, e, end=1, alpha=0.6, ws=ws), beam_ref.select(l, s, n, e, 1, 0.6))


@pytest.mark.parametrize("half", [True, False])
def test_equal_scores_of_different_logits(half):
    """At a score of -2^100 every token's score is that number: within a beam the larger logit still goes first, and
    equal logits by the lowest token; among beams of equal scores the lower one goes first."""
    B, W, V = 1, 3, 20000
    l = inputs(B, W, V, half, seed=5)[0]
    l[0, 0, 400] = l[0, 0, 9] = 20.0
    s = torch.full((B, W), -2.0 ** 100)
    n, e = torch.ones(B, W, dtype=torch.int32), torch.zeros(B, W, dtype=torch.int32)
    got = run(l, s, n, e)
    rest = l[0, 0].clone()
    rest[[400, 9]] = -INF
    assert got[0].tolist() == [[9, 400, int(rest.argmax())]] and got[1].tolist() == [[0, 0, 0]]
    assert (got[2].cpu() == -2.0 ** 100).all()
