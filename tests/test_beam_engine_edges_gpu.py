"""Beam search on a draft engine, on another stream, and over 8-bit weights that are replaced under a captured step.

The searches compared take the same steps in the same batches, so their results are equal bit for bit.  Logits behind kept
tokens are compared at the engine tests' tolerance (5e-2).
"""
import pytest
import torch

from tests.test_int8_beam_engine_gpu import TOL, _clone, _i32, _prompts, _tiny

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("capture", [False, True])
def test_on_a_draft_engine(gpu, capture):
    """Kept tokens of the search's own slots are forgotten, those of other slots stay that sequence's; between a draft
    step and its accept a search is refused and changes nothing."""
    from vkwr.model_executor import BeamSearch, DraftEngine, MixedEngine
    cfg, model, state = _tiny(gpu, 14)
    prompts = _prompts(cfg)
    kw = dict(max_requests=3, max_new_tokens=9, end=5, length_penalty=0.5, chunk=8, slots=range(1, 13))
    want = BeamSearch(MixedEngine(model, 40, max_seqs=16), _clone(state), 4, **kw).generate(prompts, 9)
    drafts = torch.randint(0, cfg.vocab, (2, 3), generator=torch.Generator().manual_seed(7)).to(torch.int32).to(gpu)
    more = torch.tensor([[3, 4]], dtype=torch.int32, device=gpu)

    def continued(search_between):
        eng, st = DraftEngine(model, 8, 4), _clone(state)
        search = BeamSearch(eng, st, 4, capture=capture, **kw) if search_between else None
        eng.draft_step(st, drafts, [13, 2])
        if search:
            before = _clone(st)
            with pytest.raises(RuntimeError, match="accepted"):
                search.generate(prompts, 9)
            for a, b in ((before.wkv, st.wkv), (before.att_shift, st.att_shift), (before.ffn_shift, st.ffn_shift)):
                assert torch.equal(a, b)
        eng.accept(torch.tensor([1, 2], dtype=torch.int32, device=gpu))
        if search:
            for _ in range(2):
                assert search.generate(prompts, 9) == want
        return eng.draft_step(st, more, [13]).float().cpu()

    assert (continued(True) - continued(False)).abs().max().item() <= TOL


def test_on_another_stream(gpu):
    from vkwr.model_executor import BeamSearch, MixedEngine
    cfg, model, state = _tiny(gpu, 12)
    prompts = _prompts(cfg)
    eng = MixedEngine(model, 40, max_seqs=12)
    kw = dict(max_requests=3, max_new_tokens=12, end=9, chunk=8)
    want = BeamSearch(eng, state, 4, **kw).generate(prompts, 12)
    search = BeamSearch(eng, state, 4, capture=True, **kw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            assert search.generate(prompts, 12) == want
    torch.cuda.current_stream().wait_stream(s)
    assert search.generate(prompts, 12) == want


def test_weights_replaced_under_a_captured_step(gpu):
    from vkwr.model_executor import BeamSearch, Int8Weights, MixedEngine
    cfg, model, state = _tiny(gpu, 12)
    prompts = _prompts(cfg)
    w = Int8Weights(model)
    eng = MixedEngine(model, 40, max_seqs=12, int8=w)
    kw = dict(max_requests=3, max_new_tokens=12, chunk=8)
    eager, captured = BeamSearch(eng, state, 4, **kw), BeamSearch(eng, state, 4, capture=True, **kw)
    first = eager.generate(prompts, 12)
    assert captured.generate(prompts, 12) == first
    g = torch.Generator().manual_seed(3)
    for l, L in enumerate(model.layers):
        for n in ("Wr", "value"):
            N, K = L[n].shape
            w.load(l, n, torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8).to(gpu),
                   torch.full((N,), 0.0005, device=gpu))
    second = eager.generate(prompts, 12)
    assert second != first and captured.generate(prompts, 12) == second
