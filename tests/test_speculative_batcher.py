"""The batchers' own logic on the CPU: an engine whose logits are a fixed function of a sequence's last tokens,
and the 64-bit oracle in place of the verification kernel."""
import types

import pytest
import torch

from oracle import serving_ref
from vkwr.model_executor import ContinuousBatcher, Request, SpeculativeBatcher
from vkwr_amd import capi

V = 16


def logits_of(tokens):
    """Small whole numbers, so that the largest are tied more often than not."""
    g = torch.Generator().manual_seed(hash(tuple(tokens[-2:])) % 2 ** 31)
    return torch.randint(0, 4, (V,), generator=g).float()


class Engine:
    """A sequence's tokens are its state: their number, then the tokens."""

    def __init__(self, draft_seqs=4, max_draft=3, max_rows=64):
        self.draft_seqs, self.max_draft, self.max_rows, self.max_seqs = draft_seqs, max_draft, max_rows, max_rows
        self.cfg = types.SimpleNamespace(vocab=V)
        self.model = types.SimpleNamespace(head=torch.empty(0))
        self.kept = None

    def _tokens(self, state, slot):
        s = state.wkv[0, slot]
        return s[1:1 + int(s[0])].int().tolist()

    def _append(self, state, slot, tokens):
        s = state.wkv[0, slot]
        n = int(s[0])
        s[1 + n:1 + n + len(tokens)] = torch.tensor(tokens).float()
        s[0] = n + len(tokens)

    def step(self, state, decode=None, prefill=(), adapter_ids=None, flush=True):
        out = []
        groups = ([(decode[0][:, None], decode[1])] if decode else []) + list(prefill)
        for tokens, slots in groups:
            for t, slot in zip(tokens.tolist(), slots.tolist()):
                self._append(state, slot, t)
                out.append(logits_of(self._tokens(state, slot)))
        return torch.stack(out)

    def draft_step(self, state, tokens, slots, adapter_ids=None):
        assert self.kept is None
        self.kept = (state, tokens.tolist(), slots)
        return torch.stack([torch.stack([logits_of(self._tokens(state, slot) + t[:i + 1]) for i in range(len(t))])
                            for t, slot in zip(tokens.tolist(), slots)])

    def accept(self, accepted):
        (state, tokens, slots), self.kept = self.kept, None
        for t, slot, n in zip(tokens, slots, accepted.tolist()):
            self._append(state, slot, t[:n + 1])

    def drop(self, slots, state=None):
        pass


def make_state(n_slots=4):
    return types.SimpleNamespace(n_slots=n_slots, wkv=torch.zeros(1, n_slots, 200), att_shift=torch.zeros(1, n_slots, 1),
                                 ffn_shift=torch.zeros(1, n_slots, 1))


@pytest.fixture
def oracle(monkeypatch):
    def verify_drafts(logits, drafts, uniforms, tokens, accepted, n_draft=None, draft_probs=None, workspace=None, **filt):
        wt, wa = serving_ref.verify(logits.numpy(), drafts.numpy(), uniforms.numpy(),
                                    None if n_draft is None else n_draft.numpy(), draft_probs, **filt)
        tokens.copy_(torch.from_numpy(wt))
        accepted.copy_(torch.from_numpy(wa))

    monkeypatch.setattr(capi, "verify_drafts", verify_drafts)


def run(batcher, prompts):
    reqs = [batcher.submit(p, 5 + 4 * i) for i, p in enumerate(prompts)]
    batcher.run()
    return [r.output for r in reqs]


PROMPTS = [[1, 2, 3, 1, 2], [7], [4, 4, 4, 4], [9, 8, 9, 8, 9], [0, 0], [15, 3, 2]]


@pytest.mark.parametrize("filt", [{}, {"top_k": 1, "top_p": 0.5}, {"top_k": 7, "top_p": 0.0}])
def test_greedy_tokens_are_the_first_of_the_largest(oracle, filt):
    """Whatever the seed, the drafts and the other sequences of a step, and the tokens of plain decoding; the
    drafts here are often right, tied with the right one, or behind a short draft."""
    want = run(ContinuousBatcher(Engine(), make_state(), max_decode=4, chunk=3), PROMPTS)
    tied = 0
    for p, o in zip(PROMPTS, want):
        for i, t in enumerate(o):
            l = logits_of((p + o[:i]))
            assert t == int((l == l.max()).nonzero()[0])
            tied += int((l == l.max()).sum()) > 1
    assert tied > 10

    def largest(tokens, n):  # the last of the largest
        out = []
        for _ in range(n if len(tokens) % 3 else 1):
            l = logits_of(tokens + out)
            out.append(int((l == l.max()).nonzero()[-1 if len(out) else 0]))
        return out[:n]

    def zeros(tokens, n):
        return [0] * (n - len(tokens) % 2)

    for seed in (0, 1):
        for draft in ({}, {"draft": largest}, {"draft": zeros}):
            b = SpeculativeBatcher(Engine(), make_state(), max_decode=4, chunk=3, seed=seed, **draft, **filt)
            assert run(b, PROMPTS) == want
    for n in (1, 3):
        assert run(SpeculativeBatcher(Engine(n), make_state(2), chunk=3, draft=largest, **filt), PROMPTS) == want


def test_accepted_drafts_save_steps(oracle):
    def exact(tokens, n):
        out = []
        for _ in range(n):
            l = logits_of(tokens + out)
            out.append(int(l.argmax()))
        return out

    b = SpeculativeBatcher(Engine(), make_state(), draft=exact, chunk=8)
    run(b, PROMPTS[:1] * 4)
    assert b.accepted == b.drafted > 0


def test_request_fields_keep_their_places():
    """Fields that came later stand behind those that callers may give by position."""
    r = Request([1, 2, 3], 4, 5, 6, 2, [9])
    assert (r.rid, r.slot, r.pos, r.output, r.adapter) == (5, 6, 2, [9], -1) and r.prefilling


def test_a_sample_function_is_refused():
    """(It would not be called: the verification draws the tokens.)"""
    with pytest.raises(TypeError):
        SpeculativeBatcher(Engine(), make_state(), chunk=8, sample=lambda logits: logits.argmax(-1))
    SpeculativeBatcher(Engine(), make_state(), chunk=8, sample=None)


class Counted(int):
    """A token that counts its comparisons."""
    count = 0

    def __eq__(self, other):
        Counted.count += 1
        return int(self) == int(other)

    __hash__ = int.__hash__


def test_looked_up_drafts_are_prompt_lookups(oracle):
    """What the batcher looks up is what prompt_lookup finds in the whole sequence, at every step."""
    from vkwr.model_executor.scheduler import prompt_lookup
    seen = []

    def spy(tokens, n):
        seen.append((tuple(tokens), n))
        return prompt_lookup(tokens, n)

    outs = [run(SpeculativeBatcher(Engine(), make_state(), chunk=3, **kw), PROMPTS) for kw in ({}, {"draft": spy})]
    assert outs[0] == outs[1]
    calls = []
    b = SpeculativeBatcher(Engine(), make_state(), chunk=3)
    draft = b._draft
    b._draft = lambda r, n: calls.append((tuple(r.prompt + r.output), n, draft(r, n))) or calls[-1][2]
    assert run(b, PROMPTS) == outs[0] and not b.lookups
    assert [c[:2] for c in calls] == seen
    assert all(d == prompt_lookup(list(t), n) for t, n, d in calls) and any(d for _, _, d in calls)


def test_lookups_of_growing_sequences():
    from vkwr.model_executor.scheduler import _Lookup, prompt_lookup
    g = torch.Generator().manual_seed(3)
    for trial in range(40):
        r = Request(torch.randint(0, 4, (1 + trial % 5,), generator=g).tolist(), 100)
        look = _Lookup(r.prompt)
        for _ in range(30):
            n = int(torch.randint(0, 5, (1,), generator=g))
            assert look(r, n) == prompt_lookup(r.prompt + r.output, n)
            r.output += torch.randint(0, 4, (1 + n,), generator=g).tolist()


def test_looking_up_drafts_does_not_walk_the_sequence(oracle):
    """A prompt of different tokens: a step compares no more than a few of them."""
    import vkwr.model_executor.scheduler as scheduler

    class Long(Engine):
        def step(self, state, decode=None, prefill=(), adapter_ids=None, flush=True):
            return torch.stack([logits_of(t) for tokens, _ in prefill for t in tokens.tolist()])

        def draft_step(self, state, tokens, slots, adapter_ids=None):
            return torch.stack([torch.stack([logits_of(t[:i + 1]) for i in range(len(t))]) for t in tokens.tolist()])

        def accept(self, accepted):
            pass

    b = scheduler.SpeculativeBatcher(Long(max_rows=4000), make_state(), chunk=3000)
    b.submit([Counted(i) for i in range(3000)], 12)
    b.step()
    Counted.count = 0
    for _ in range(5):
        b.step()
    assert Counted.count < 1000


@pytest.mark.parametrize("filt", [{}, {"top_k": 5}])
def test_the_default_type_does_not_matter(monkeypatch, filt):
    """The uniforms are fp32, as the verification takes them, whatever torch makes by default."""
    seen = []

    def verify_drafts(logits, drafts, uniforms, tokens, accepted, **kw):
        seen.append(uniforms.dtype)
        tokens.fill_(3)
        accepted.zero_()

    monkeypatch.setattr(capi, "verify_drafts", verify_drafts)
    torch.set_default_dtype(torch.float64)
    try:
        run(SpeculativeBatcher(Engine(), make_state(), chunk=8, **filt), PROMPTS[:2])
    finally:
        torch.set_default_dtype(torch.float32)
    assert set(seen) == {torch.float32}
