"""8-bit weights in the mixed and draft steps, and beam search on top of them, on the tiny RWKV-7 shape.

The 8-bit engine's logits are compared with the float32 model (oracle/model_ref) whose large projections round
their rows and weights to 8 bits by the same formula, at the end-to-end tolerance of the engine tests (5e-2).
Hypotheses are scored again by running their tokens one at a time through the same engine: logits of a row
may differ by the tolerance between batches, a log-probability by twice that.
"""
import copy
import types

import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = 5e-2
ALL = ("Wr", "Wk", "Wv", "Wo", "key", "value")


def _tiny(gpu, n_slots, seed=0):
    from vkwr.model_executor import RWKV7Config, RWKV7Model, RWKV7State
    from vkwr_amd import capi
    cfg = RWKV7Config.preset("tiny")
    return cfg, RWKV7Model(cfg, gpu, seed=seed), RWKV7State(cfg, n_slots, gpu, std=0.1, seed=seed + 1,
                                                            layout=capi.WKV_STATE_STD)


def _clone(state):
    s = copy.copy(state)
    s.wkv, s.att_shift, s.ffn_shift = state.wkv.clone(), state.att_shift.clone(), state.ffn_shift.clone()
    return s


def _i32(x, gpu):
    return torch.tensor(x, dtype=torch.int32, device=gpu)


def _rounded(x):
    top = x.double().abs().amax(-1, keepdim=True)
    q = torch.round(127.0 * x.double() / torch.where(top > 0, top, 1.0))
    return (q * top / 127.0).float()


class _Reference:
    """model_ref with rows and weights of the named projections rounded to 8 bits; adapters: layer, name ->
    (A, B, scale) added to the product of the unrounded rows."""

    def __init__(self, model, names, monkeypatch, adapters=None):
        from oracle import model_ref
        self.ref = model_ref
        marked = {}
        layers = []
        for l, L in enumerate(model.layers):
            d = {k: v.float().cpu() for k, v in L.items()}
            for n in names:
                d[n] = _rounded(d[n])
                marked[id(d[n])] = (l, n)
            layers.append(d)
        self.model = types.SimpleNamespace(cfg=model.cfg, layers=layers, emb=model.emb.cpu(), ln_out_w=model.ln_out_w.cpu(),
                                           ln_out_b=model.ln_out_b.cpu(), head=model.head.cpu())
        adapters = adapters or {}

        def linear(x, W, rd):
            at = marked.get(id(W))
            y = (_rounded(x) if at else x) @ W.t()
            if at in adapters:
                A, B, scale = adapters[at]
                y = y + scale * ((x @ A.float().cpu().t()) @ B.float().cpu().t())
            return y

        def channel_mix(W, o, res, prev, rd):
            res, xx = model_ref.add_layer_norm(o, res, W["ln2_w"], W["ln2_b"], rd)
            act = torch.relu(linear(model_ref.lerp(xx, prev, W["x_k_ffn"], rd), W["key"], rd)) ** 2
            return res, linear(act, W["value"], rd), xx

        monkeypatch.setattr(model_ref, "linear", linear)
        monkeypatch.setattr(model_ref, "channel_mix", channel_mix)

    def run(self, state, tokens, slot):
        st = [state.wkv.cpu().clone(), state.att_shift.cpu().float(), state.ffn_shift.cpu().float()]
        for t in tokens:
            out = self.ref.decode_step(self.model, *st, t.reshape(1), torch.tensor([slot]), round_fp16=False)
        return out[0]


@pytest.mark.parametrize("names", [ALL, ("key", "value"), ("Wv",)])
def test_mixed_step_matches_rounded_model(gpu, monkeypatch, names):
    from vkwr.model_executor import Int8Weights, MixedEngine
    cfg, model, state = _tiny(gpu, 12)
    g = torch.Generator().manual_seed(5)
    tok = torch.randint(0, cfg.vocab, (5,), generator=g).to(torch.int32)
    pre = torch.randint(0, cfg.vocab, (2, 40), generator=g).to(torch.int32)
    slots = [7, 0, 3, 11, 5, 2, 9]
    eng = MixedEngine(model, 100, int8=Int8Weights(model, names))
    got = eng.step(_clone(state), decode=(tok.to(gpu), _i32(slots[:5], gpu)), prefill=[(pre.to(gpu), _i32(slots[5:], gpu))])
    got = got.float().cpu()
    ref = _Reference(model, names, monkeypatch)
    for q, slot in enumerate(slots):
        want = ref.run(state, [tok[q]] if q < 5 else pre[q - 5], slot)
        assert (got[q] - want).abs().max().item() <= TOL, q


def test_int8_with_adapters(gpu, monkeypatch):
    from vkwr.model_executor import AdapterPool, Int8Weights, MixedEngine
    cfg, model, state = _tiny(gpu, 6)
    pool = AdapterPool(model, 2, 8)
    g = torch.Generator(device=gpu).manual_seed(3)
    given = [{n: ((torch.randn(8, L[n].shape[1], generator=g, device=gpu) / L[n].shape[1] ** 0.5).half(),
                  (0.1 * torch.randn(L[n].shape[0], 8, generator=g, device=gpu)).half()) for n in ALL} for L in model.layers]
    pool.load(1, given, scale=0.75)
    eng = MixedEngine(model, 16, adapters=pool, int8=Int8Weights(model))
    tok, slots = torch.tensor([3, 900, 17], dtype=torch.int32), [4, 0, 2]
    got = eng.step(_clone(state), decode=(tok.to(gpu), _i32(slots, gpu)), adapter_ids=_i32([1, -1, 1], gpu)).float().cpu()
    for ids, rows in (({(l, n): (*given[l][n], 0.75) for l in range(cfg.n_layer) for n in ALL}, (0, 2)), ({}, (1,))):
        with monkeypatch.context() as m:
            ref = _Reference(model, ALL, m, ids)
            for q in rows:
                assert (got[q] - ref.run(state, [tok[q]], slots[q])).abs().max().item() <= TOL


def test_loaded_8_bit_weights(gpu, monkeypatch):
    """Weights given in 8 bits replace the rounded ones, in place."""
    from vkwr.model_executor import Int8Weights, MixedEngine
    cfg, model, state = _tiny(gpu, 4)
    w = Int8Weights(model, ("value",))
    eng = MixedEngine(model, 8, int8=w)
    g = torch.Generator().manual_seed(9)
    for l, L in enumerate(model.layers):
        N, K = L["value"].shape
        q = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8)
        q[:, 0] = 127  # so that rounding the values again gives them back
        scale = 0.0002 * (1 + torch.rand(N, generator=g))
        w.load(l, "value", q.to(gpu), scale.to(gpu))
        L["value"] = (q.double() * scale.double()[:, None]).float().to(gpu)
    with pytest.raises(ValueError):
        w.load(0, "value", torch.zeros(3, 4, dtype=torch.int8, device=gpu), torch.zeros(3, device=gpu))
    tok = torch.tensor([5, 77], dtype=torch.int32)
    got = eng.step(_clone(state), decode=(tok.to(gpu), _i32([1, 3], gpu))).float().cpu()
    ref = _Reference(model, ("value",), monkeypatch)
    for q, slot in enumerate((1, 3)):
        assert (got[q] - ref.run(state, [tok[q]], slot)).abs().max().item() <= TOL


def test_draft_steps_on_8_bit_weights(gpu):
    """A draft step's logits are those of single steps of the 8-bit mixed engine."""
    from vkwr.model_executor import DraftEngine, Int8Weights, MixedEngine
    cfg, model, state = _tiny(gpu, 6)
    w = Int8Weights(model)
    one, drafts = MixedEngine(model, 8, int8=w), DraftEngine(model, 2, 2, int8=w)
    tok = torch.randint(0, cfg.vocab, (2, 3), generator=torch.Generator().manual_seed(1)).to(torch.int32).to(gpu)
    a, b = _clone(state), _clone(state)
    got = drafts.draft_step(a, tok, [4, 1]).float()
    for t in range(3):
        want = one.step(b, decode=(tok[:, t].contiguous(), _i32([4, 1], gpu))).float()
        assert (got[:, t] - want).abs().max().item() <= TOL


def test_refusals(gpu):
    from vkwr.model_executor import Int8Weights, MixedEngine
    cfg, model, _ = _tiny(gpu, 2)
    for names in ((), ("head",), ("key", "key")):
        with pytest.raises(ValueError):
            Int8Weights(model, names)
    weights = Int8Weights(model)
    whole, weights.layers = weights.layers, weights.layers[:-1]
    with pytest.raises(ValueError, match="layers"):
        MixedEngine(model, 4, int8=weights)
    weights.layers = whole
    weights.layers[1]["key"], weights.layers[1]["value"] = weights.layers[1]["value"], weights.layers[1]["key"]
    with pytest.raises(ValueError, match="sizes"):
        MixedEngine(model, 4, int8=weights)


def _prompts(cfg, seed=2):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, cfg.vocab, (n,), generator=g).tolist() for n in (5, 1, 23)]


@pytest.mark.parametrize("width,end,alpha", [(1, -1, 0.0), (4, -1, 0.0), (3, 11, 0.7)])
def test_hypotheses_scored_again(gpu, width, end, alpha):
    """Scores, order, and the states that the last beams leave in their slots."""
    from vkwr.model_executor import BeamSearch, Int8Weights, MixedEngine
    cfg, model, state = _tiny(gpu, 20)
    eng = MixedEngine(model, 40, max_seqs=16, int8=Int8Weights(model))
    before = _clone(state)
    search = BeamSearch(eng, state, width, max_requests=3, max_new_tokens=7, end=end, length_penalty=alpha, chunk=8,
                        slots=range(2, 2 + 3 * width))
    prompts = _prompts(cfg)
    got = search.generate(prompts, 7)
    slots = search._views(search.now, 3)[3].tolist()
    untouched = [i for i in range(20) if not 2 <= i < 2 + 3 * width]
    assert torch.equal(state.wkv[:, untouched], before.wkv[:, untouched])
    for b, (p, hyps) in enumerate(zip(prompts, got)):
        assert len(hyps) == width and len({tuple(h.tokens) for h in hyps}) == width
        assert [h.normalised for h in hyps] == sorted((h.normalised for h in hyps), reverse=True)
        for w, h in enumerate(hyps):
            s = _clone(before)
            for pool in (s.wkv, s.att_shift, s.ffn_shift):
                pool[:, 0].zero_()
            logits = eng.step(s, prefill=[(_i32([p], gpu), _i32([0], gpu))])[0].double()
            score = 0.0
            for i, t in enumerate(h.tokens):
                score += float(torch.log_softmax(logits, 0)[t])
                if i + 1 < len(h.tokens):
                    logits = eng.step(s, decode=(_i32([t], gpu), _i32([0], gpu)))[0].double()
            assert abs(score - h.score) <= 2 * TOL * len(h.tokens)
            if not h.finished:
                at = slots[b][w]
                assert (state.wkv[:, at] - s.wkv[:, 0]).abs().max().item() <= 1e-2
                assert (state.att_shift[:, at].float() - s.att_shift[:, 0].float()).abs().max().item() <= 1e-1


def test_width_one_is_greedy(gpu):
    from vkwr.model_executor import BeamSearch, ContinuousBatcher, MixedEngine
    cfg, model, state = _tiny(gpu, 4)
    prompts = _prompts(cfg)
    eng = MixedEngine(model, 32, max_seqs=8)
    best = BeamSearch(eng, state, 1, max_new_tokens=6).generate(prompts, 6)
    for p, hyps in zip(prompts, best):
        b = ContinuousBatcher(eng, state, max_decode=1, max_prefill_chunks=1, chunk=31)
        r = b.submit(p, 6)
        b.run()
        assert hyps[0].tokens == r.output


@pytest.mark.parametrize("int8", [False, True])
def test_captured_search_equals_eager(gpu, int8):
    """Steps replayed from a graph, over several calls with eager work between, give the eager results bit for
    bit; a call of fewer requests has a graph of its own."""
    from vkwr.model_executor import BeamSearch, Int8Weights, MixedEngine
    cfg, model, state = _tiny(gpu, 12)
    eng = MixedEngine(model, 40, max_seqs=12, int8=Int8Weights(model) if int8 else None)
    kw = dict(max_requests=3, max_new_tokens=24, end=9, length_penalty=0.6, chunk=8)
    eager, captured = BeamSearch(eng, state, 4, **kw), BeamSearch(eng, state, 4, capture=True, **kw)
    for seed in (2, 3):
        for prompts in (_prompts(cfg, seed), _prompts(cfg, seed + 10)[:2]):
            a, b = eager.generate(prompts, 24), captured.generate(prompts, 24)
            assert a == b
    assert set(captured.graphs) == {(3, False), (2, False)}


def test_beam_search_with_adapters(gpu):
    from vkwr.model_executor import AdapterPool, BeamSearch, MixedEngine
    cfg, model, state = _tiny(gpu, 9)
    pool = AdapterPool(model, 1, 8)
    g = torch.Generator(device=gpu).manual_seed(3)
    pool.load(0, [{n: ((torch.randn(8, L[n].shape[1], generator=g, device=gpu) / L[n].shape[1] ** 0.5).half(),
                       (0.1 * torch.randn(L[n].shape[0], 8, generator=g, device=gpu)).half()) for n in ALL}
                  for L in model.layers])
    eng = MixedEngine(model, 40, max_seqs=16, adapters=pool)
    p = _prompts(cfg)[0]
    plain, mixed = (BeamSearch(eng, state, 3, max_requests=2, max_new_tokens=6, capture=c) for c in (False, True))
    without = plain.generate([p], 6)[0]
    both = mixed.generate([p, p], 6, adapters=[0, -1])
    assert both == plain.generate([p, p], 6, adapters=[0, -1])
    assert [h.tokens for h in both[0]] != [h.tokens for h in without]
    with pytest.raises(ValueError):
        plain.generate([p], 6, adapters=[0, 0])
