"""Calls that the beam search refuses, on the CPU: what it refuses is left as it was."""
import types

import pytest
import torch

from tests.test_beam_search import PROMPTS, Engine, make_state, oracle  # noqa: F401  (the fixture replaces the kernels)
from vkwr.model_executor import BeamSearch


class Drafts(Engine):
    """An engine that keeps drafts of `state` between two of its calls, as DraftEngine does."""

    def __init__(self, state):
        super().__init__()
        self.open = (state, [0])

    def drop(self, slots, state=None):
        if self.open is not None and self.open[0].wkv is state.wkv:
            raise RuntimeError("drop: the last step's drafts are not accepted yet")

    def step(self, *args, **kw):
        if self.open is not None:
            raise RuntimeError("step: the last step's drafts are not accepted yet")
        return super().step(*args, **kw)


@pytest.mark.parametrize("same", [True, False])
def test_between_a_draft_step_and_its_accept(same):
    """Refused before any state is reset, whichever state the drafts are of."""
    state = make_state(6)
    engine = Drafts(state if same else make_state(6))
    search = BeamSearch(engine, state, 2, max_requests=2, max_new_tokens=3)
    before = [t.clone() for t in (state.wkv, state.att_shift, state.ffn_shift)]
    with pytest.raises(RuntimeError, match="accepted"):
        search.generate(PROMPTS[:2], 3)
    for a, b in zip(before, (state.wkv, state.att_shift, state.ffn_shift)):
        assert torch.equal(a, b)
    engine.open = None
    want = BeamSearch(Engine(), make_state(6), 2, max_requests=2, max_new_tokens=3).generate(PROMPTS[:2], 3)
    assert search.generate(PROMPTS[:2], 3) == want


@pytest.mark.parametrize("adapters", [[2, 0], [0, 2], [5, -1]])
def test_adapters_outside_the_pool(adapters):
    """Refused (their rows' logits are NaN: such a prompt would have no hypothesis); any negative number means none."""
    engine = Engine()
    engine.adapters = types.SimpleNamespace(pool=types.SimpleNamespace(n_adapters=2))
    search = BeamSearch(engine, make_state(6), 2, max_requests=2, max_new_tokens=3)
    with pytest.raises(ValueError, match="adapter"):
        search.generate(PROMPTS[:2], 3, adapters=adapters)
    assert engine.calls == []
    assert [len(h) for h in search.generate(PROMPTS[:2], 3, adapters=[1, -7])] == [2, 2]


def test_more_beams_than_a_call_reorders(monkeypatch):
    """129 requests of 32 beams: run in parts of at most 4096 beams, which is what the reordering takes."""
    from vkwr_amd import capi
    seen = []
    inner = capi.beam_reorder

    def reorder(slots, *args, **kw):
        seen.append(slots.numel())
        assert slots.numel() <= 4096
        inner(slots, *args, **kw)

    monkeypatch.setattr(capi, "beam_reorder", reorder)
    engine = Engine(max_rows=5000, max_seqs=5000)
    search = BeamSearch(engine, make_state(129 * 32), 32, max_requests=129, max_new_tokens=1, max_prefill_chunks=129)
    prompts = [[i % 12, i // 12] for i in range(129)]
    got = search.generate(prompts, 1)
    assert seen == [4096, 32] and len(got) == 129
    for i in (0, 127, 128):
        alone = BeamSearch(Engine(), make_state(32), 32, max_new_tokens=1).generate([prompts[i]], 1)
        assert got[i] == alone[0]
