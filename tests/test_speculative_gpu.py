"""Speculative decoding on the tiny RWKV-7 shape: tied logits, and kept tokens of sequences that are gone."""
import pytest
import torch

from tests.test_drafts_adapters_gpu import _i32, _tiny

pytestmark = pytest.mark.gpu


def test_greedy_takes_the_lowest_of_tied_logits(gpu):
    """Vocabulary entries 2 i and 2 i + 1 share their head's row, so every logit is tied with its neighbour's:
    even tokens only, whatever the seed, and though the drafts are odd ones too."""
    from vkwr.model_executor import DraftEngine, SpeculativeBatcher
    cfg, model, state = _tiny(gpu, 4)
    model.head[1::2] = model.head[::2]
    outs = []

    def either(tokens, n):
        return [(known[len(tokens) + i] + i % 2) if len(tokens) + i < len(known) else 0 for i in range(n)]

    known = []
    for seed, kw in ((0, {}), (1, {}), (2, {"draft": either}), (3, {"draft": either, "top_p": 0.0, "top_k": 5})):
        sched = SpeculativeBatcher(DraftEngine(model, 3, 3, max_rows=32), state, max_prefill_chunks=2, chunk=8, seed=seed, **kw)
        reqs = [sched.submit([6, 8, 6, 8, 6], 16) for _ in range(3)]
        sched.run()
        outs.append([r.output for r in reqs])
        known = reqs[0].prompt + reqs[0].output
        assert all(t % 2 == 0 for r in reqs for t in r.output)
    assert outs[0] == outs[1]
    assert sched.drafted > sched.accepted > 0


def test_sequences_that_end_leave_another_states_kept_tokens(gpu):
    """One engine for two states: a request that ends on the one in slot 2 has nothing to do with the tokens kept
    of slot 2 of the other."""
    from vkwr.model_executor import DraftEngine, RWKV7State, SpeculativeBatcher
    from vkwr_amd import capi
    cfg, model, state = _tiny(gpu, 4)
    eng = DraftEngine(model, 2, 2, max_rows=24)
    eng.draft_step(state, _i32([[5, 6, 7], [8, 9, 10]], gpu), [2, 0])
    eng.accept(_i32([2, 1], gpu))
    before = state.wkv.clone()
    other = SpeculativeBatcher(eng, RWKV7State(cfg, 4, gpu, std=0.0, layout=capi.WKV_STATE_STD), max_prefill_chunks=4, chunk=4)
    reqs = [other.submit([1 + i, 2, 3], 1) for i in range(4)]
    assert len(other.run()) == 4 and all(len(r.output) == 1 for r in reqs)
    assert set(eng.rows_of) == {0, 2}
    eng.flush(state)
    changed = (state.wkv != before).flatten(2).any(-1).any(0)
    assert changed.tolist() == [True, False, True, False]


@pytest.mark.parametrize("plain", [False, True])
def test_a_new_sequence_takes_no_kept_tokens_of_the_slots_last_user(gpu, plain):
    """A batcher that is left in the middle of its requests, then another one on the same engine and state."""
    from vkwr.model_executor import ContinuousBatcher, DraftEngine, SpeculativeBatcher
    cfg, model, state = _tiny(gpu, 3)

    def serve(eng):
        if plain:
            sched = ContinuousBatcher(eng, state, max_decode=3, max_prefill_chunks=3, chunk=8)
        else:
            sched = SpeculativeBatcher(eng, state, max_prefill_chunks=3, chunk=8)
        reqs = [sched.submit([2 + i, 4, 2 + i, 4], 8) for i in range(3)]
        sched.run()
        return [r.output for r in reqs], state.wkv.clone()

    want = serve(DraftEngine(model, 3, 2, max_rows=32))
    eng = DraftEngine(model, 3, 2, max_rows=32)
    left = SpeculativeBatcher(eng, state, max_prefill_chunks=3, chunk=8)
    for _ in range(3):
        left.submit([9, 7, 5, 9, 7], 40)
    for _ in range(3):
        left.step()
    assert set(eng.rows_of) == {0, 1, 2}
    got = serve(eng)
    assert got[0] == want[0] and torch.equal(got[1], want[1])


def test_drop_waits_for_accept(gpu):
    """Between a draft step and its accept nothing is kept yet: a drop there would be undone by the accept."""
    from vkwr.model_executor import DraftEngine, RWKV7State
    from vkwr_amd import capi
    cfg, model, state = _tiny(gpu, 4)
    other = RWKV7State(cfg, 4, gpu, layout=capi.WKV_STATE_STD)
    eng = DraftEngine(model, 2, 2)
    eng.draft_step(state, _i32([[5, 6], [8, 9]], gpu), [2, 0])
    for args in (([2],), ([2], state)):
        with pytest.raises(RuntimeError):
            eng.drop(*args)
    eng.drop([2], other)
    eng.accept(_i32([1, 1], gpu))
    eng.drop([2], other)
    assert set(eng.rows_of) == {0, 2}
    eng.drop([2], state)
    assert set(eng.rows_of) == {0}
