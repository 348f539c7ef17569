"""Beam selection and the reordering of states against plain implementations in 64 bits and on lists.

Whole numbers have to be equal.  Scores are rounded to fp32 once (2^-24) behind log-sums whose terms are
fp32: an exponential is within 2^-22 + |d| 2^-23 of its value (terms with |d| > 16 weigh less than 2^-23),
a lane's sum of at most 32 terms within 31 2^-24: below 2^-17 in all.
"""
import math

import pytest
import torch

from oracle import beam_ref
from vkwr_amd import capi

pytestmark = pytest.mark.gpu
INF = math.inf


def run(logits, scores, lengths, ended, end=-1, alpha=0.0, ws=None):
    B, W, _ = logits.shape
    i32 = lambda: torch.full((B, W), -9, dtype=torch.int32, device="cuda")  # noqa: E731
    out = [i32(), i32(), torch.full((B, W), 9.0, device="cuda"), i32(), i32()]
    capi.beam_select(logits.cuda(), scores.cuda(), lengths.cuda(), ended.cuda(), *out, end=end, length_penalty=alpha,
                     workspace=ws)
    return out


def check(got, want):
    names = ("tokens", "parents", "scores", "lengths", "ended")
    for name, g, w in zip(names, got, want):
        if name == "scores":
            g = g.cpu().double()
            assert torch.equal(g == -INF, w == -INF)
            fin = w > -INF
            assert ((g - w).abs()[fin] <= 2.0 ** -17 + w.abs()[fin] * 2.0 ** -24).all(), (g, w)
        else:
            assert torch.equal(g.cpu(), w), (name, g.cpu(), w)


def inputs(B, W, V, half, seed, ended=0.0, banned=0.0):
    g = torch.Generator().manual_seed(seed)
    l = 2.0 * torch.randn(B, W, V, generator=g)
    l.scatter_add_(2, torch.randint(0, V, (B, W, 5), generator=g), 5.0 + 2.0 * torch.randn(B, W, 5, generator=g))
    if banned:
        l[torch.rand(B, W, V, generator=g) < banned] = -INF
    s = -torch.sort(6.0 * torch.rand(B, W, generator=g), dim=1).values
    e = (torch.rand(B, W, generator=g) < ended).to(torch.int32)
    n = torch.randint(1, 40, (B, W), generator=g, dtype=torch.int32)
    return (l.half() if half else l), s, n, e


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("B,W,V", [(1, 1, 1), (1, 4, 3), (2, 5, 7), (1, 1, 1000), (3, 2, 8192), (2, 3, 8193), (1, 4, 65536),
                                   (4, 8, 5003), (2, 16, 16384), (1, 32, 40000), (5, 13, 1001), (1, 7, 131072), (17, 6, 2048)])
def test_select(B, W, V, half):
    a = inputs(B, W, V, half, seed=B + W + V)
    check(run(*a, end=min(2, V - 1)), beam_ref.select(*a, min(2, V - 1), 0.0))


@pytest.mark.parametrize("alpha", [0.0, 0.6, 1.0, 2.5])
@pytest.mark.parametrize("ended,banned", [(0.3, 0.0), (0.9, 0.5), (1.0, 0.0), (0.2, 0.999)])
def test_finished_banned_and_length(alpha, ended, banned):
    a = inputs(6, 5, 3001, True, seed=int(10 * alpha), ended=ended, banned=banned)
    check(run(*a, end=7, alpha=alpha), beam_ref.select(*a, 7, alpha))


def test_first_step_counts_one_beam():
    l, s, n, e = inputs(3, 6, 2000, True, seed=1)
    l = l[:, :1].repeat(1, 6, 1)
    s = torch.full((3, 6), -INF)
    s[:, 0] = 0.0
    n.zero_()
    got = run(l, s, n, e)
    check(got, beam_ref.select(l, s, n, e, -1, 0.0))
    assert (got[1] == 0).all()


def test_nothing_left():
    """Rows whose mask leaves nothing, requests with fewer candidates than beams or none at all."""
    l, s, n, e = inputs(5, 4, 600, False, seed=2)
    l[0] = -INF                      # nothing
    l[1, :, 2:] = -INF               # two tokens a beam
    l[1, 1:] = -INF                  # in one beam: two candidates for four rows
    l[2, 2] = float("nan")           # a beam of NaN
    s[3, :] = -INF                   # dead beams
    s[4, 1] = float("nan")
    got = run(l, s, n, e)
    check(got, beam_ref.select(l, s, n, e, -1, 0.0))
    assert (got[0][0] == -1).all() and (got[4][0] == 1).all() and (got[0][3] == -1).all()
    assert (got[1][1].cpu() == torch.tensor([0, 0, -1, -1])).all()


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("W", [1, 4, 9, 32])
def test_ties(W, half):
    """Equal logits, many or all: the lowest index of the lowest beam."""
    V = 20000
    l = torch.zeros(4, W, V)
    l[1, :, ::3] = 1.0
    l[2] = torch.randint(0, 3, (W, V), generator=torch.Generator().manual_seed(3)).float()
    l[3, :, 15000:] = 2.0
    l[3, :, 5] = -0.0
    l[:, :, 100] = -INF
    l = l.half() if half else l
    s, n, e = torch.full((4, W), -1.5), torch.full((4, W), 3, dtype=torch.int32), torch.zeros(4, W, dtype=torch.int32)
    got = run(l, s, n, e)
    check(got, beam_ref.select(l, s, n, e, -1, 0.0))


def test_lowest_value_and_infinities():
    """A mask of the type's lowest value leaves the tokens choosable; +inf takes all of the probability."""
    for dtype in (torch.float16, torch.float32):
        low = torch.finfo(dtype).min
        l, s, n, e = inputs(3, 3, 1000, dtype == torch.float16, seed=4)
        l[0] = low
        l[1, :, 1:] = low
        l[2, 1, 77] = INF
        l[2, 1, 500] = INF
        got = run(l, s, n, e)
        want = beam_ref.select(l, s, n, e, -1, 0.0)
        for i in (0, 1, 3, 4):
            assert torch.equal(got[i].cpu(), want[i])
        near = (got[2].cpu().double() - want[2]).abs() <= 2.0 ** -17 + want[2].abs() * 2.0 ** -24
        assert (near | (got[2].cpu().double() == want[2])).all()


def test_request_alone_and_among_others():
    l, s, n, e = inputs(9, 4, 30000, True, seed=5, ended=0.2)
    whole = run(l, s, n, e, end=0, alpha=0.7)
    for b in (0, 4, 8):
        one = run(l[b:b + 1], s[b:b + 1], n[b:b + 1], e[b:b + 1], end=0, alpha=0.7)
        for w, o in zip(whole, one):
            assert torch.equal(w[b:b + 1], o)


def test_select_unaligned_logits():
    l, s, n, e = inputs(2, 3, 1024, True, seed=6)
    flat = torch.zeros(l.numel() + 1, dtype=torch.float16, device="cuda")
    flat[1:] = l.reshape(-1).cuda()
    check(run(flat[1:].view(2, 3, 1024), s, n, e), beam_ref.select(l, s, n, e, -1, 0.0))


# ---------------------------------------------------------------- states

def pools_of(layers, n_slots, C, seed, dev="cuda"):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [torch.randn(layers, n_slots, C // 64, 64, 64, generator=g, device=dev),
            torch.randn(layers, n_slots, C, generator=g, device=dev).half(),
            torch.randint(0, 99, (1, n_slots, 4), generator=g, device=dev, dtype=torch.int32)]


@pytest.mark.parametrize("B,W,layers,C", [(1, 1, 2, 64), (1, 4, 3, 128), (3, 5, 2, 256), (2, 32, 1, 64), (40, 8, 2, 64),
                                          (300, 3, 1, 64), (7, 31, 1, 128), (1024, 4, 1, 64)])
def test_reorder(B, W, layers, C):
    g = torch.Generator().manual_seed(B * W)
    n_slots = B * W + 5
    for trial in range(3):
        slots = torch.randperm(n_slots, generator=g)[:B * W].view(B, W).to(torch.int32)
        parents = torch.randint(-1 if trial else 0, W, (B, W), generator=g, dtype=torch.int32)
        if trial == 1:
            parents[0] = 0
        if trial == 2:
            parents[-1] = torch.arange(W - 1, -1, -1, dtype=torch.int32)
        skip = (torch.rand(B, W, generator=g) < 0.3 * trial).to(torch.int32)
        pools = pools_of(layers, n_slots, C, seed=trial)
        want, want_pools = beam_ref.reorder(slots, parents, skip, n_slots, pools)
        out = torch.full((B, W), -7, dtype=torch.int32, device="cuda")
        capi.beam_reorder(slots.cuda(), parents.cuda(), out, pools, skip=skip.cuda() if trial else None)
        assert torch.equal(out.cpu(), want)
        for p, w in zip(pools, want_pools):
            assert torch.equal(p, w)
        assert sorted(out.cpu().reshape(-1).tolist()) == sorted(slots.reshape(-1).tolist())


def test_reorder_bad_slots_and_parents():
    """Slots outside the pool and parents outside the beams copy nothing."""
    pools = pools_of(2, 6, 64, seed=1)
    slots = torch.tensor([[0, 99, 2], [3, 4, -5]], dtype=torch.int32)
    parents = torch.tensor([[1, 1, 0], [0, 0, 77]], dtype=torch.int32)
    want, want_pools = beam_ref.reorder(slots, parents, torch.zeros_like(slots), 6, pools)
    out = torch.empty(2, 3, dtype=torch.int32, device="cuda")
    capi.beam_reorder(slots.cuda(), parents.cuda(), out, pools)
    assert torch.equal(out.cpu(), want)
    for p, w in zip(pools, want_pools):
        assert torch.equal(p, w)


def test_reorder_without_pools():
    slots = torch.tensor([[4, 1, 0]], dtype=torch.int32, device="cuda")
    parents = torch.tensor([[2, 2, 2]], dtype=torch.int32, device="cuda")
    out = torch.empty_like(slots)
    capi.beam_reorder(slots, parents, out, [])
    assert out.tolist() == [[0, 4, 1]]


def test_reorder_refuses_pools_of_different_slots():
    slots = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    a, b = torch.zeros(2, 3, 4, device="cuda"), torch.zeros(2, 4, 4, device="cuda")
    with pytest.raises(ValueError, match="pool 1"):
        capi.beam_reorder(slots, slots, slots.clone(), [a, b])
    with pytest.raises(TypeError):
        capi.beam_reorder(slots, slots, slots.clone(), [a.transpose(0, 2)])


def test_step_captured():
    """Selection and reordering in one graph, replayed with eager work between: every replay as the eager calls."""
    B, W, V, n_slots = 3, 4, 9000, 14
    l, s, n, e = (t.cuda() for t in inputs(B, W, V, True, seed=8))
    slots = torch.randperm(n_slots, generator=torch.Generator().manual_seed(1))[:B * W].view(B, W).to(torch.int32).cuda()
    pools = pools_of(2, n_slots, 64, seed=3)
    i32 = lambda: torch.empty(B, W, dtype=torch.int32, device="cuda")  # noqa: E731
    out = [i32(), i32(), torch.empty(B, W, device="cuda"), i32(), i32()]
    new = i32()
    ws = torch.empty(capi.beam_workspace_bytes(B, W, V), dtype=torch.uint8, device="cuda")

    def step():
        capi.beam_select(l, s, n, e, *out, end=1, length_penalty=0.5, workspace=ws)
        capi.beam_reorder(slots, out[1], new, pools, skip=out[4])

    keep = [p.clone() for p in pools]
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for seed in (1, 2, 3):
        for p, k in zip(pools, keep):
            p.copy_(k)
        l.copy_(inputs(B, W, V, True, seed=seed)[0])
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*out, new, *pools)]
        for p, k in zip(pools, keep):
            p.copy_(k)
        step()
        for a, b in zip(got, (*out, new, *pools)):
            assert torch.equal(a, b)
        check(got[:5], beam_ref.select(l.cpu(), s.cpu(), n.cpu(), e.cpu(), 1, 0.5))
