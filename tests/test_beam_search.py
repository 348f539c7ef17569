"""The beam search's own logic on the CPU: an engine whose logits are a fixed function of a sequence's tokens,
and the 64-bit oracle in place of the kernels."""
import types

import pytest
import torch

from oracle import beam_ref
from vkwr.model_executor import BeamSearch
from vkwr_amd import capi

V, END = 12, 3


def logits_of(tokens):
    g = torch.Generator().manual_seed(hash(tuple(tokens)) % 2 ** 31)
    return 2.0 * torch.randn(V, generator=g).half().float()


class Engine:
    """A sequence's tokens are its state: their number, then the tokens."""

    def __init__(self, max_rows=64, max_seqs=64):
        self.max_rows, self.max_seqs, self.calls = max_rows, max_seqs, []
        self.cfg = types.SimpleNamespace(vocab=V)
        self.model = types.SimpleNamespace(head=torch.empty(0))
        self.adapters = None

    def step(self, state, decode=None, prefill=(), adapter_ids=None):
        out, rows = [], 0
        groups = ([(decode[0][:, None], decode[1])] if decode else []) + list(prefill)
        for tokens, slots in groups:
            rows += tokens.numel()
            assert len(set(slots.tolist())) == slots.numel()
            for t, slot in zip(tokens.tolist(), slots.tolist()):
                s = state.wkv[0, slot]
                n = int(s[0])
                s[1 + n:1 + n + len(t)] = torch.tensor(t).float()
                s[0] = n + len(t)
                out.append(logits_of(s[1:1 + n + len(t)].int().tolist()))
        assert rows <= self.max_rows and len(out) <= self.max_seqs
        self.calls.append((rows, None if adapter_ids is None else adapter_ids.tolist()))
        return torch.stack(out).half()


def make_state(n_slots):
    g = torch.Generator().manual_seed(0)
    return types.SimpleNamespace(n_slots=n_slots, wkv=torch.randn(1, n_slots, 300, generator=g),
                                 att_shift=torch.randn(2, n_slots, 4, generator=g), ffn_shift=torch.zeros(2, n_slots, 4))


@pytest.fixture(autouse=True)
def oracle(monkeypatch):
    def select(logits, scores, lengths, ended, tokens, parents, scores2, lengths2, ended2, end=-1, length_penalty=0.0,
               workspace=None):
        for dst, src in zip((tokens, parents, scores2, lengths2, ended2),
                            beam_ref.select(logits, scores, lengths, ended, end, length_penalty)):
            dst.copy_(src)

    def reorder(slots, parents, slots2, pools, skip=None):
        new, after = beam_ref.reorder(slots, parents, skip, pools[0].shape[1], pools)
        slots2.copy_(new)
        for p, a in zip(pools, after):
            p.copy_(a)

    monkeypatch.setattr(capi, "beam_select", select)
    monkeypatch.setattr(capi, "beam_reorder", reorder)


PROMPTS = [[1, 2, 3, 1, 2], [7], [4] * 11, [9, 8, 9, 8, 9, 0, 0, 5], [0, 0]]


@pytest.mark.parametrize("width,end,alpha", [(1, -1, 0.0), (3, -1, 0.0), (4, END, 0.0), (4, END, 0.8), (5, END, 2.0), (8, END, 0.6)])
@pytest.mark.parametrize("steps", [1, 2, 11])
def test_equals_search_over_sequences(width, end, alpha, steps):
    search = BeamSearch(Engine(), make_state(45), width, max_requests=2, max_new_tokens=11, end=end, length_penalty=alpha,
                        slots=range(44, 44 - 2 * width, -1), chunk=4, max_prefill_chunks=2)
    for trial in range(2):  # the second call on slots that the first has used
        got = search.generate(PROMPTS, steps)
        for p, hyps in zip(PROMPTS, got):
            want = beam_ref.search(logits_of, p, width, steps, end, alpha)
            assert len(hyps) == len(want)
            for h, (tokens, score, over) in zip(hyps, want):
                assert h.tokens == tokens and h.finished == over
                assert abs(h.score - score) < 1e-4 * max(1.0, abs(score))  # kept in fp32
                assert h.normalised == pytest.approx(h.score / max(len(tokens), 1) ** alpha)


def test_width_one_is_greedy():
    search = BeamSearch(Engine(), make_state(3), 1, max_requests=3, max_new_tokens=9)
    for p, hyps in zip(PROMPTS, search.generate(PROMPTS, 9)):
        out = []
        for _ in range(9):
            out.append(int(logits_of(p + out).argmax()))
        assert [h.tokens for h in hyps] == [out]


def test_few_candidates(monkeypatch):
    """A vocabulary that leaves fewer candidates than beams."""
    def only_two(tokens):
        l = torch.full((V,), float("-inf"))
        l[END] = 0.0
        l[5] = -0.5
        return l

    monkeypatch.setitem(globals(), "logits_of", only_two)
    for hyps in BeamSearch(Engine(), make_state(16), 8, max_requests=2, max_new_tokens=30, end=END).generate(PROMPTS[:2], 2):
        assert sorted(h.tokens for h in hyps) == [[END], [5, END], [5, 5]]


def test_stops_when_all_beams_are_finished(monkeypatch):
    def at_once(tokens):
        l = torch.full((V,), -8.0)
        l[END] = 8.0
        return l

    monkeypatch.setitem(globals(), "logits_of", at_once)
    e = Engine()
    hyps = BeamSearch(e, make_state(4), 2, max_requests=2, max_new_tokens=200, end=END).generate(PROMPTS[:2], 200)
    assert len(e.calls) < 40 and all(h.finished for hs in hyps for h in hs)
    assert hyps[0][0].tokens == [END]


def test_prefill_in_chunks_and_adapters():
    e = Engine(max_rows=8, max_seqs=8)
    e.adapters = object()
    search = BeamSearch(e, make_state(8), 4, max_requests=2, max_new_tokens=3, chunk=5, max_prefill_chunks=3)
    got = search.generate(PROMPTS[2:4], 3, adapters=[5, -1])
    for p, hyps in zip(PROMPTS[2:4], got):
        assert [h.tokens for h in hyps] == [s for s, _, _ in beam_ref.search(logits_of, p, 4, 3)]
    assert [c[0] for c in e.calls[-2:]] == [8, 8] and e.calls[-1][1] == [5] * 4 + [-1] * 4
    assert all(c[0] <= 8 for c in e.calls)


def test_refusals():
    e, s = Engine(max_rows=16, max_seqs=16), make_state(16)
    for kw in ({"width": 0}, {"width": 33}, {"width": 4, "max_requests": 5}, {"width": 2, "max_requests": 0},
               {"width": 2, "slots": [1]}, {"width": 2, "slots": [1, 1]}, {"width": 2, "slots": [1, 16]}, {"width": 2, "end": V},
               {"width": 2, "end": -2}, {"width": 2, "chunk": 0}, {"width": 2, "max_new_tokens": 0},
               {"width": 2, "max_prefill_chunks": 0}):
        with pytest.raises(ValueError):
            BeamSearch(e, s, **kw)
    b = BeamSearch(e, s, 2, max_new_tokens=4)
    for args in (([[]], 2), ([[1]], 0), ([[1]], 5), ([[1]], 2, [0]), ([[1, V]], 2), ([[0], [-1]], 2)):
        with pytest.raises(ValueError):
            b.generate(*args)
    assert b.generate([], 3) == []
