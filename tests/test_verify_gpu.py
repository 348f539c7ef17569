"""Verification of drafted tokens (capi.verify_drafts) against the 64-bit oracle: whole numbers, so
every one has to be equal."""
import math

import numpy as np
import pytest
import torch

from oracle import serving_ref as ref
from vkwr_amd import capi


def make(B, K, V, seed, half=True, probs=True, sharp=3.0, near=0.7):
    g = torch.Generator().manual_seed(seed)
    logits = 1.5 * torch.randn(B, K + 1, V, generator=g)
    top = torch.randint(0, V, (B, K + 1, min(8, V)), generator=g)
    logits.scatter_add_(2, top, sharp * torch.randn(top.shape, generator=g))
    logits = logits.half() if half else logits
    q = torch.softmax(logits[:, :K].float() + near * torch.randn(B, K, V, generator=g), dim=-1)
    drafts = (torch.multinomial(q.reshape(B * K, V), 1, generator=g).view(B, K) if K else torch.zeros(B, 0)).to(torch.int32)
    return {"logits": logits, "drafts": drafts, "u": torch.rand(B, K + 1, generator=g),
            "n_draft": torch.randint(0, K + 1, (B,), generator=g, dtype=torch.int32), "q": q if probs else None}


def check(gpu, d, **filt):
    B, T, V = d["logits"].shape
    c = lambda t: None if t is None else t.to(gpu)  # noqa: E731
    tokens = torch.full((B, T), 77, dtype=torch.int32, device=gpu)
    accepted = torch.full((B,), 77, dtype=torch.int32, device=gpu)
    capi.verify_drafts(c(d["logits"]), c(d["drafts"]), c(d["u"]), tokens, accepted, n_draft=c(d["n_draft"]),
                       draft_probs=c(d["q"]), **filt)
    wt, wa = ref.verify(d["logits"].numpy(), d["drafts"].numpy(), d["u"].numpy(),
                        None if d["n_draft"] is None else d["n_draft"].numpy(),
                        None if d["q"] is None else d["q"].numpy(), **filt)
    np.testing.assert_array_equal(accepted.cpu().numpy(), wa)
    np.testing.assert_array_equal(tokens.cpu().numpy(), wt)
    return wt, wa


@pytest.mark.gpu
@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("B,K,V", [(1, 1, 4), (3, 4, 1000), (7, 3, 4096), (5, 8, 4100), (4, 2, 20004), (3, 4, 65536)])
@pytest.mark.parametrize("filt", [{}, {"top_k": 40, "top_p": 0.9, "temperature": 0.8}, {"top_p": 0.95}, {"top_k": 5}],
                         ids=["all", "k40p90", "p95", "k5"])
def test_against_64_bits(gpu, B, K, V, half, probs, filt):
    wt, wa = check(gpu, make(B, K, V, seed=B + K + V, half=half, probs=probs), **filt)
    assert (wa >= 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("filt", [{}, {"top_k": 100, "top_p": 0.8}], ids=["all", "filtered"])
@pytest.mark.parametrize("V", [65540, 200000, 1048576])
def test_large_vocabularies(gpu, V, filt):
    check(gpu, make(2, 2, V, seed=V, half=False), **filt)


@pytest.mark.gpu
@pytest.mark.parametrize("filt", [{"temperature": 0.001}, {"temperature": 1000.0}, {"temperature": 1000.0, "top_p": 0.5},
                                  {"temperature": 20.0, "top_k": 3000}, {"top_k": 1}, {"top_p": 0.0}, {"top_p": 1e-6},
                                  {"top_k": 20004}, {"top_k": 20003}, {"top_p": 0.999999}, {"top_k": -5, "top_p": 2.0}])
def test_extreme_filters(gpu, filt):
    check(gpu, make(6, 3, 20004, seed=17), **filt)


@pytest.mark.gpu
@pytest.mark.parametrize("filt", [{}, {"top_k": 50}, {"top_k": 3000, "top_p": 0.7}], ids=["all", "k50", "k3000p70"])
def test_ties(gpu, filt):
    """Logits of few distinct values: thousands of entries tied at the threshold share its budget."""
    d = make(4, 3, 20000, seed=5)
    d["logits"] = (d["logits"] * 0.5).round().half()
    check(gpu, d, **filt)
    d["logits"] = torch.zeros_like(d["logits"])  # every entry tied
    check(gpu, d, **filt)


@pytest.mark.gpu
@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("filt", [{}, {"top_k": 40, "top_p": 0.9}, {"top_k": 3000}, {"temperature": 50.0, "top_p": 0.6}])
def test_masked_and_non_finite_logits(gpu, half, filt):
    """Vocabulary entries masked with -inf or the type's lowest value, NaN (as 0) and +inf."""
    V = 8192
    d = make(6, 3, V, seed=23, half=half)
    l = d["logits"]
    low = torch.finfo(l.dtype).min
    l[0, :, 5:] = -float("inf")
    l[1, :, : V - 7] = low
    l[2, :, ::2] = float("nan")
    l[3, 0] = -float("inf")       # nothing left: the entries are tied
    l[3, 1, 100] = float("inf")
    l[3, 2, 200:203] = float("inf")
    l[4] = low
    d["n_draft"][:] = 3
    check(gpu, d, **filt)


@pytest.mark.gpu
@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("V,k", [(65536, 40), (65536, 64), (20004, 200), (4096, 64), (2000, 64), (131072, 20), (8192, 300)])
def test_largest_entries_side_by_side(gpu, V, k, probs):
    """The top_k entries in one stretch of the vocabulary, in a few stretches, and spread: what a part
    of the row holds of them is anything from none to all."""
    d = make(6, 3, V, seed=29 + V, probs=probs)
    l = d["logits"].float()
    l[0], l[1] = l[0].sort(dim=-1, descending=True)[0], l[1].sort(dim=-1)[0]
    l[2, :, 100:100 + 2 * k] += 9.0
    l[3, :, -k:] += 9.0
    l[4] = torch.floor(l[4])  # and ties
    d["logits"] = l.half()
    d["n_draft"][:] = 3
    for filt in ({"top_k": k}, {"top_k": k, "top_p": 0.9}, {"top_k": k, "top_p": 0.999, "temperature": 4.0}):
        check(gpu, d, **filt)


@pytest.mark.gpu
@pytest.mark.parametrize("left", [1, 3, 50])
def test_few_entries_left_by_a_mask(gpu, left):
    """Fewer entries than top_k (and than a list would hold) are not masked."""
    d = make(4, 2, 65536, seed=37)
    keep = torch.randperm(65536, generator=torch.Generator().manual_seed(left))[:left]
    mask = torch.full((65536,), -float("inf"))
    mask[keep] = 0.0
    d["logits"] = (d["logits"].float() + mask).half()
    for filt in ({}, {"top_k": 40}, {"top_k": 40, "top_p": 0.9}, {"top_p": 0.9}):
        check(gpu, d, **filt)


@pytest.mark.gpu
def test_uniforms_at_their_ends(gpu):
    for u in (0.0, 1.0 - 2.0 ** -24):
        for probs in (True, False):
            d = make(5, 4, 1000, seed=31, probs=probs)
            d["u"] = torch.full_like(d["u"], u)
            check(gpu, d, top_k=100)


@pytest.mark.gpu
def test_drafter_equal_to_target_accepts_all(gpu):
    d = make(9, 5, 1000, seed=41, half=False)
    d["q"] = torch.softmax(d["logits"][:, :5], dim=-1)
    d["u"] = d["u"] * 0.999
    d["n_draft"] = None
    _, wa = check(gpu, d)
    assert (wa == 5).all()


@pytest.mark.gpu
def test_unnormalised_drafter_falls_back_to_the_target(gpu):
    d = make(4, 2, 512, seed=43)
    d["q"] = torch.full_like(d["q"], 2.0)  # p - q < 0 everywhere
    d["u"][:, :2] = 0.9
    d["n_draft"] = None
    _, wa = check(gpu, d)
    assert (wa == 0).all()


@pytest.mark.gpu
def test_lengths_and_bad_entries(gpu):
    d = make(6, 3, 1000, seed=47, probs=False)
    d["n_draft"] = torch.tensor([0, 3, -1, 4, 1, 2], dtype=torch.int32)
    d["drafts"][1, 0], d["drafts"][4, 0], d["drafts"][5, 1] = -7, 1000, 2 ** 31 - 1
    wt, wa = check(gpu, d)
    assert wa[2] == wa[3] == -1 and (wt[2:4] == -1).all()
    d["q"] = make(6, 3, 1000, seed=47)["q"]
    check(gpu, d)
    check(gpu, make(5, 0, 1000, seed=48, probs=False))  # no drafts: plain sampling


@pytest.mark.gpu
def test_law_of_the_new_token(gpu):
    """Over many uniforms the emitted first token follows p, whatever the drafter proposes: counts
    within 6 standard deviations."""
    n, V = 20000, 8
    g = torch.Generator().manual_seed(3)
    logits = torch.randn(1, 2, V, generator=g).expand(n, 2, V).contiguous()
    q = torch.softmax(torch.randn(1, 1, V, generator=g), -1).expand(n, 1, V).contiguous()
    drafts = torch.multinomial(q[:, 0], 1, generator=g).to(torch.int32)
    tokens = torch.empty(n, 2, dtype=torch.int32, device=gpu)
    accepted = torch.empty(n, dtype=torch.int32, device=gpu)
    capi.verify_drafts(logits.to(gpu), drafts.to(gpu), torch.rand(n, 2, generator=g).to(gpu), tokens, accepted,
                       draft_probs=q.to(gpu))
    first = tokens[:, 0].cpu().numpy()
    p = ref.probabilities(logits[0, 0].numpy())
    counts = np.bincount(first, minlength=V)
    assert (np.abs(counts - n * p) <= 6 * np.sqrt(n * p * (1 - p)) + 1).all()


@pytest.mark.gpu
def test_batch_independence_graph_and_stream(gpu):
    d = make(8, 4, 8192, seed=53)
    c = lambda t: t.to(gpu)  # noqa: E731
    ins = [c(d[k]) for k in ("logits", "drafts", "u")]
    nd, q = c(d["n_draft"]), c(d["q"])
    tokens = torch.empty(8, 5, dtype=torch.int32, device=gpu)
    accepted = torch.empty(8, dtype=torch.int32, device=gpu)
    ws = torch.empty(capi.verify_workspace_bytes(8, 4, 8192), dtype=torch.uint8, device=gpu)
    capi.verify_drafts(*ins, tokens, accepted, n_draft=nd, draft_probs=q, top_k=50, top_p=0.9, workspace=ws)
    want_t, want_a = tokens.clone(), accepted.clone()
    for b in range(8):
        t1, a1 = tokens.new_empty(1, 5), accepted.new_empty(1)
        capi.verify_drafts(*[x[b:b + 1] for x in ins], t1, a1, n_draft=nd[b:b + 1], draft_probs=q[b:b + 1], top_k=50,
                           top_p=0.9)
        assert torch.equal(t1[0], want_t[b]) and a1[0] == want_a[b]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        capi.verify_drafts(*ins, tokens, accepted, n_draft=nd, draft_probs=q, top_k=50, top_p=0.9, workspace=ws)
    for _ in range(3):
        tokens.fill_(5)
        accepted.fill_(5)
        ws.fill_(255)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(tokens, want_t) and torch.equal(accepted, want_a)


@pytest.mark.gpu
def test_masses_that_all_round_down(gpu):
    """2^20 - 2 equal weights, each rounded down by a third of 2^-43: the kept mass is 4e-8 short, and the
    first draft's acceptance, whose border lies in between, may fall either way, but what follows it has to
    fit: the second draft's row is then judged, or not looked at.  (The weights are exp(l / temperature); N
    x = 1 + 4e-8 puts 1/2 between 1 / (mass as rounded) and 1 / mass.)"""
    V = 1 << 20
    x = (1.0 + 4e-8) / (V - 2)
    assert 0.2 < x * 2.0 ** 43 % 1.0 < 0.45
    l = torch.full((1, 3, V), -13.875)
    l[..., 0], l[..., V - 1] = 0.0, -30.0
    drafts = torch.zeros(1, 2, dtype=torch.int32)
    u = torch.tensor([[0.5, 0.9, 0.0]])
    tokens, accepted = torch.empty(1, 3, dtype=torch.int32, device=gpu), torch.empty(1, dtype=torch.int32, device=gpu)
    ws = torch.full((capi.verify_workspace_bytes(1, 2, V),), 255, dtype=torch.uint8, device=gpu)
    capi.verify_drafts(l.to(gpu), drafts.to(gpu), u.to(gpu), tokens, accepted, temperature=-13.875 / math.log(x),
                       top_p=1.0 - 1e-9, workspace=ws)
    assert (accepted.item(), tokens[0].tolist()) in ((1, [0, 1, -1]), (0, [1, -1, -1]))


@pytest.mark.gpu
@pytest.mark.parametrize("K", [63, 64, 130])
@pytest.mark.parametrize("filt", [{}, {"top_k": 40, "top_p": 0.9}, {"top_p": 0.95}, {"top_k": 300}],
                         ids=["all", "k40p90", "p95", "k300"])
def test_many_drafts(gpu, K, filt):
    """More rows per sequence than a wave has lanes; the first rejection anywhere among them."""
    d = make(6, K, 1000, seed=K, probs=False)
    d["drafts"] = d["logits"][:, :K].float().argmax(-1).to(torch.int32)
    d["u"][:, :K] *= 1e-9
    for b, at in enumerate((0, 62, 63, 64, K - 1)):
        if at < K:
            d["u"][b, at] = 1.0 - 2.0 ** -24
    d["n_draft"] = torch.tensor([K, K, K, K, K, min(K, 64)], dtype=torch.int32)
    wt, wa = check(gpu, d, **filt)
    assert wa[5] == min(K, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("filt", [{}, {"top_k": 40, "top_p": 0.9}, {"top_p": 0.95}], ids=["all", "k40p90", "p95"])
def test_offsets_past_32_bits(gpu, filt, probs):
    """The last sequences of more than 2^31 logits, as in a call of their own."""
    B, K, V, last = 8400, 3, 65536, 3
    d = make(last, K, V, seed=71)
    logits = torch.zeros(B, K + 1, V, dtype=torch.float16, device=gpu)
    logits[-last:] = d["logits"].to(gpu)
    drafts, u = torch.zeros(B, K, dtype=torch.int32, device=gpu), torch.zeros(B, K + 1, device=gpu)
    drafts[-last:], u[-last:] = d["drafts"].to(gpu), d["u"].to(gpu)
    n = torch.zeros(B, dtype=torch.int32, device=gpu)
    n[-last:] = d["n_draft"].to(gpu)
    q = None
    if probs:
        q = torch.zeros(B, K, V, device=gpu)
        q[-last:] = d["q"].to(gpu)
    outs = []
    for s in (slice(0, B), slice(B - last, B)):
        tokens = torch.empty(s.stop - s.start, K + 1, dtype=torch.int32, device=gpu)
        accepted = torch.empty(s.stop - s.start, dtype=torch.int32, device=gpu)
        capi.verify_drafts(logits[s], drafts[s], u[s], tokens, accepted, n_draft=n[s],
                           draft_probs=None if q is None else q[s], **filt)
        outs.append((tokens[-last:], accepted[-last:]))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


@pytest.mark.gpu
@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("V", [65536, 20004, 1220, 131076])
@pytest.mark.parametrize("filt", [{"top_p": 0.95}, {"top_p": 0.6, "temperature": 0.7}, {"top_k": 5000, "top_p": 0.9}],
                         ids=["p95", "p60", "k5000p90"])
def test_nucleus_of_peaked_and_flat_rows(gpu, V, half, probs, filt):
    """Rows whose kept entries are a few, hundreds, and most of the row, next to each other in a sequence;
    replayed over scratch that holds anything."""
    d = make(9, 4, V, seed=V + 1, half=False, probs=probs)
    f = torch.tensor([0.3, 1.0, 3.0, 8.0, 20.0])
    l = d["logits"] * f[torch.randint(0, 5, (9, 5, 1), generator=torch.Generator().manual_seed(V))]
    d["logits"] = l.half() if half else l
    d["n_draft"][:] = 4
    if not probs:
        d["drafts"] = l[:, :4].argmax(-1).to(torch.int32)
    wt, wa = check(gpu, d, **filt)
    c = lambda t: None if t is None else t.to(gpu)  # noqa: E731
    ins, q = [c(d[k]) for k in ("logits", "drafts", "u")], c(d["q"])
    tokens = torch.empty(9, 5, dtype=torch.int32, device=gpu)
    accepted = torch.empty(9, dtype=torch.int32, device=gpu)
    ws = torch.zeros(capi.verify_workspace_bytes(9, 4, V), dtype=torch.uint8, device=gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        capi.verify_drafts(*ins, tokens, accepted, draft_probs=q, workspace=ws, **filt)
    for fill in (255, 1, 0):
        ws.fill_(fill)
        tokens.fill_(5)
        g.replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(tokens.cpu().numpy(), wt)
        np.testing.assert_array_equal(accepted.cpu().numpy(), wa)
