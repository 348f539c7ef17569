"""Adapters per request in the mixed step, draft steps and the speculative batcher, on the tiny RWKV-7
shape.

The adapters' logits are compared with the float32 model (oracle/model_ref) whose weights have the adapter
merged in, at the end-to-end tolerance of the engine tests (5e-2); draft steps with the same tokens run one
at a time through MixedEngine, at the tolerances those tests use for states and shift rows; generated
tokens with a teacher-forced replay: each must be within that tolerance of the replay's largest logit.
"""
import copy
import types

import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = 5e-2


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


def _pool(model, gpu, n=3, ranks=(8, 16, 5), names=("Wr", "Wk", "Wv", "Wo", "key", "value"), seed=3):
    from vkwr.model_executor import AdapterPool
    g = torch.Generator(device=gpu).manual_seed(seed)
    pool = AdapterPool(model, n, max(ranks), names)
    given = []
    for i in range(n):
        layers = []
        for L in model.layers:
            d = {}
            for k, name in enumerate(names):
                if (i + k) % 4 == 3:
                    continue  # not every adapter has every projection
                N, K = L[name].shape
                d[name] = ((torch.randn(ranks[i], K, generator=g, device=gpu) / K ** 0.5).half(),
                           (0.1 * torch.randn(N, ranks[i], generator=g, device=gpu)).half())
            layers.append(d)
        pool.load(i, layers, scale=0.5 + i)
        given.append(layers)
    return pool, given


def _merged(model, layers, scale):
    out = []
    for L, A in zip(model.layers, layers):
        d = {k: v.float() for k, v in L.items()}
        for n, (a, b) in A.items():
            d[n] = d[n] + scale * (b.float() @ a.float())
        out.append(d)
    return types.SimpleNamespace(cfg=model.cfg, layers=out, emb=model.emb, ln_out_w=model.ln_out_w,
                                 ln_out_b=model.ln_out_b, head=model.head)


def _shift_close(a, b):
    _, e = torch.frexp(b.float().abs())
    ulp = torch.ldexp(torch.ones_like(b, dtype=torch.float32), e - 11)
    return ((a.float() - b.float()).abs() / torch.clamp(ulp, min=2e-3)).max().item() <= 4


@pytest.mark.parametrize("names", [("Wr", "Wk", "Wv", "Wo", "key", "value"), ("Wr", "Wv", "Wo", "value")])
def test_mixed_step_with_adapters_matches_merged_weights(gpu, names):
    """Rows without an adapter keep their bits where the key is not adapted; where it is, their FFN keys
    too are rounded to fp16 before the square, which follows the adapters' launch."""
    from oracle import model_ref
    from vkwr.model_executor import MixedEngine
    cfg, model, state = _tiny(gpu, 12)
    pool, given = _pool(model, gpu, names=names)
    g = torch.Generator().manual_seed(5)
    tok = torch.randint(0, cfg.vocab, (5,), generator=g).to(torch.int32)
    pre = torch.randint(0, cfg.vocab, (2, 6), generator=g).to(torch.int32)
    ids, slots = [1, -1, 0, 2, 1, 2, -1], [7, 0, 3, 11, 5, 2, 9]
    eng = MixedEngine(model, 64, adapters=pool)
    s2 = _clone(state)
    got = eng.step(s2, decode=(tok.to(gpu), _i32(slots[:5], gpu)), prefill=[(pre.to(gpu), _i32(slots[5:], gpu))],
                   adapter_ids=_i32(ids, gpu)).float().cpu()
    plain = MixedEngine(model, 64).step(_clone(state), decode=(tok.to(gpu), _i32(slots[:5], gpu)),
                                        prefill=[(pre.to(gpu), _i32(slots[5:], gpu))]).float().cpu()
    for q, (i, slot) in enumerate(zip(ids, slots)):
        m = _merged(model, given[i], 0.5 + i) if i >= 0 else model
        st = [state.wkv.cpu().clone(), state.att_shift.cpu().float(), state.ffn_shift.cpu().float()]
        for t in ([tok[q]] if q < 5 else pre[q - 5]):
            want = model_ref.decode_step(m, *st, t.reshape(1), torch.tensor([slot]), round_fp16=False)
        assert (got[q] - want[0]).abs().max().item() <= TOL
        if i >= 0:
            assert (got[q] - plain[q]).abs().max().item() > 0.1  # the adapter matters
        elif "key" not in names:
            assert torch.equal(got[q], plain[q])


def test_step_without_ids_keeps_its_results(gpu):
    from vkwr.model_executor import MixedEngine
    cfg, model, state = _tiny(gpu, 6)
    pool, _ = _pool(model, gpu)
    dec = (_i32([3, 900, 17], gpu), _i32([4, 0, 2], gpu))
    a, b = _clone(state), _clone(state)
    assert torch.equal(MixedEngine(model, 8).step(a, decode=dec), MixedEngine(model, 8, adapters=pool).step(b, decode=dec))
    assert torch.equal(a.wkv, b.wkv)
    with pytest.raises(ValueError):
        MixedEngine(model, 8).step(a, decode=dec, adapter_ids=_i32([0, 0, 0], gpu))


@pytest.mark.parametrize("with_adapters", [False, True])
def test_draft_steps_equal_single_steps(gpu, with_adapters):
    """Four draft steps with changing batches, lengths, orders and acceptances (none, some, all) against
    the kept tokens run one at a time; then flush, after which the whole state is that of those steps."""
    from vkwr.model_executor import DraftEngine, MixedEngine
    cfg, model, state = _tiny(gpu, 10)
    pool = _pool(model, gpu)[0] if with_adapters else None
    eng = DraftEngine(model, 4, 4, adapters=pool)
    ref = MixedEngine(model, 8, adapters=pool)
    s1, s2 = _clone(state), _clone(state)
    g = torch.Generator().manual_seed(11)
    ada = [0, -1, 2, 1, 1, 0, -1, 2, 0, 1]
    for slots, T, acc in (([7, 1, 4], 5, [4, 0, 2]), ([4, 7, 1, 2], 3, [2, 1, 0, 1]), ([2, 9], 5, [3, -1]),
                          ([1, 4, 9, 2], 1, [0, 0, 0, 0])):
        tokens = torch.randint(0, cfg.vocab, (len(slots), T), generator=g).to(torch.int32).to(gpu)
        ids = _i32([ada[i] for i in slots], gpu) if pool else None
        got = eng.draft_step(s1, tokens, slots, adapter_ids=ids).float().clone()
        eng.accept(_i32(acc, gpu))
        for b, slot in enumerate(slots):
            one = _clone(s2)
            for t in range(T):
                lg = ref.step(one, decode=(tokens[b, t:t + 1].contiguous(), _i32([slot], gpu)),
                              adapter_ids=None if ids is None else ids[b:b + 1]).float()
                assert (got[b, t] - lg[0]).abs().max().item() <= TOL, (slots, b, t)
                if t == acc[b]:
                    s2.wkv[:, slot] = one.wkv[:, slot]
                    s2.att_shift[:, slot], s2.ffn_shift[:, slot] = one.att_shift[:, slot], one.ffn_shift[:, slot]
        assert _shift_close(s1.att_shift, s2.att_shift) and _shift_close(s1.ffn_shift, s2.ffn_shift)
    eng.flush(s1)
    assert (s1.wkv - s2.wkv).abs().max().item() <= 2e-2
    assert torch.equal(s1.wkv[:, [0, 3, 5, 6, 8]], state.wkv[:, [0, 3, 5, 6, 8]])


def test_draft_engine_refuses_and_drops(gpu):
    from vkwr.model_executor import DraftEngine, RWKV7State
    cfg, model, state = _tiny(gpu, 6)
    eng = DraftEngine(model, 2, 2)
    tok = torch.zeros(2, 2, dtype=torch.int32, device=gpu)
    with pytest.raises(RuntimeError):
        eng.accept(_i32([0, 0], gpu))
    for slots in ([0], [0, 0], [0, 6], [-1, 2]):
        with pytest.raises(ValueError):
            eng.draft_step(state, tok, slots)
    with pytest.raises(ValueError):
        eng.draft_step(state, torch.zeros(2, 4, dtype=torch.int32, device=gpu), [0, 1])
    with pytest.raises(ValueError):
        eng.draft_step(RWKV7State(cfg, 6, gpu), tok, [0, 1])
    before = state.wkv.clone()
    eng.draft_step(state, tok, [3, 5])
    with pytest.raises(RuntimeError):
        eng.draft_step(state, tok, [3, 5])
    with pytest.raises(RuntimeError):
        eng.flush(state)
    eng.accept(_i32([1, 1], gpu))
    assert torch.equal(state.wkv, before)
    eng.drop([3])
    eng.flush(state)
    assert torch.equal(state.wkv[:, 3], before[:, 3]) and not torch.equal(state.wkv[:, 5], before[:, 5])
    eng.flush(state)  # nothing left


def _replay(model, req, gpu, pool=None):
    """Every generated token is within TOL of the replay's largest logit."""
    from vkwr.model_executor import MixedEngine, RWKV7State
    from vkwr_amd import capi
    state = RWKV7State(model.cfg, 1, gpu, std=0.0, layout=capi.WKV_STATE_STD)
    eng = MixedEngine(model, 4, adapters=pool)
    ids = _i32([req.adapter], gpu) if pool is not None and req.adapter >= 0 else None
    fed = req.prompt + req.output[:-1]
    for i, t in enumerate(fed):
        lg = eng.step(state, decode=(_i32([t], gpu), _i32([0], gpu)), adapter_ids=ids)[0].float()
        if i >= len(req.prompt) - 1:
            out = req.output[i - len(req.prompt) + 1]
            assert lg[out] >= lg.max() - TOL, (i, out)


@pytest.mark.parametrize("with_adapters", [False, True])
def test_speculative_batcher_generates_the_greedy_tokens(gpu, with_adapters):
    """More requests than slots and than draft rows; drafts looked up, exact, and wrong ones."""
    from vkwr.model_executor import DraftEngine, SpeculativeBatcher
    cfg, model, state = _tiny(gpu, 5)
    pool = _pool(model, gpu)[0] if with_adapters else None
    g = torch.Generator().manual_seed(21)
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=g).tolist() for n in (1, 9, 17, 5, 12, 3, 30)]
    prompts = [p + p[:4] for p in prompts]

    def wrong(tokens, n):
        return [(tokens[-1] + 1 + i) % cfg.vocab for i in range(n)]

    outs = []
    for draft in (None, wrong):
        eng = DraftEngine(model, 3, 3, adapters=pool, max_rows=32)
        kw = {} if draft is None else {"draft": draft}
        sched = SpeculativeBatcher(eng, state, max_prefill_chunks=2, chunk=8, **kw)
        reqs = [sched.submit(p, 3 + 2 * i, adapter=(i % 4 - 1) if pool else -1) for i, p in enumerate(prompts)]
        done = sched.run()
        assert len(done) == len(reqs) and all(len(r.output) == r.max_new_tokens for r in reqs)
        assert sched.slots.available == state.n_slots and not eng.rows_of
        for r in reqs:
            _replay(model, r, gpu, pool)
        outs.append([r.output for r in reqs])
    # an exact drafter: most drafts are accepted and the steps get fewer
    known = {tuple(p): o for p, o in zip(prompts, outs[0])}

    def exact(tokens, n):
        for p, o in known.items():
            if tuple(tokens[:len(p)]) == p and tokens[len(p):] == o[:len(tokens) - len(p)]:
                return o[len(tokens) - len(p):][:n]
        return []

    eng = DraftEngine(model, 3, 3, adapters=pool, max_rows=32)
    sched = SpeculativeBatcher(eng, state, draft=exact, max_prefill_chunks=2, chunk=8)
    reqs = [sched.submit(p, 3 + 2 * i, adapter=(i % 4 - 1) if pool else -1) for i, p in enumerate(prompts)]
    sched.run()
    assert sched.accepted >= 0.8 * sched.drafted > 0
    for r in reqs:
        _replay(model, r, gpu, pool)


def test_sampled_speculation_with_filter(gpu):
    """top-k / top-p sampling: tokens of the kept set only, as many as asked for, and the same from the
    same seed."""
    from vkwr.model_executor import DraftEngine, SpeculativeBatcher
    cfg, model, state = _tiny(gpu, 4)
    runs = []
    for _ in range(2):
        eng = DraftEngine(model, 2, 4, max_rows=24)
        sched = SpeculativeBatcher(eng, state, temperature=0.9, top_k=20, top_p=0.9, seed=5, max_prefill_chunks=2,
                                   chunk=8)
        reqs = [sched.submit([5, 6, 7, 5, 6], 12) for _ in range(3)]
        sched.run()
        runs.append([r.output for r in reqs])
        assert all(len(o) == 12 and all(0 <= t < cfg.vocab for t in o) for o in runs[-1])
    assert runs[0] == runs[1]


def test_step_writes_the_kept_tokens_first(gpu):
    """A plain step after a draft step equals one after an explicit flush; another state's step leaves the
    kept tokens for theirs."""
    from vkwr.model_executor import DraftEngine
    cfg, model, state = _tiny(gpu, 6)
    g = torch.Generator().manual_seed(31)
    tok = torch.randint(0, cfg.vocab, (2, 3), generator=g).to(torch.int32).to(gpu)
    pre = torch.randint(0, cfg.vocab, (1, 4), generator=g).to(torch.int32).to(gpu)
    runs = []
    for explicit in (True, False):
        eng, s, other = DraftEngine(model, 2, 2, max_rows=16), _clone(state), _clone(state)
        eng.draft_step(s, tok, [3, 5])
        with pytest.raises(RuntimeError):
            eng.step(s, decode=(_i32([1], gpu), _i32([3], gpu)))
        eng.accept(_i32([2, 0], gpu))
        eng.step(other, decode=(_i32([1], gpu), _i32([3], gpu)))
        assert set(eng.rows_of) == {3, 5}
        if explicit:
            eng.flush(s, [5, 3, 5])
        out = eng.step(s, decode=(_i32([7], gpu), _i32([3], gpu)), prefill=[(pre, _i32([5], gpu))]).clone()
        assert not eng.rows_of
        runs.append((out, s.wkv, s.att_shift))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_padding_behind_short_drafts_is_free(gpu):
    from vkwr.model_executor import DraftEngine
    cfg, model, state = _tiny(gpu, 4)
    outs = []
    for pad in (0, -1, 2 ** 31 - 1):
        eng, s = DraftEngine(model, 2, 3), _clone(state)
        tok = _i32([[5, 6, pad, pad], [9, 10, 11, 12]], gpu)
        lg = eng.draft_step(s, tok, [2, 0]).clone()
        eng.accept(_i32([1, 2], gpu))
        eng.flush(s)
        outs.append((lg[0, :2], lg[1], s.wkv, s.att_shift))
    for o in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(o, outs[0]))


def test_engines_refuse_wrong_counts(gpu):
    from vkwr.model_executor import DraftEngine
    cfg, model, state = _tiny(gpu, 4)
    eng = DraftEngine(model, 2, 2, adapters=_pool(model, gpu)[0])
    dec = (_i32([3, 9], gpu), _i32([0, 2], gpu))
    tok = _i32([[1, 2], [3, 4]], gpu)
    before = state.wkv.clone()
    for ids in (_i32([1], gpu), _i32([1, 0, 2], gpu), torch.tensor([1, 0], device=gpu)):
        with pytest.raises(ValueError):
            eng.step(state, decode=dec, adapter_ids=ids)
        with pytest.raises(ValueError):
            eng.draft_step(state, tok, [0, 2], adapter_ids=ids)
    assert torch.equal(state.wkv, before)
    eng.draft_step(state, tok, [0, 2], adapter_ids=_i32([1, -1], gpu))
    for acc in (_i32([1], gpu), torch.tensor([1, 1], device=gpu), torch.tensor([1, 1], dtype=torch.int32)):
        with pytest.raises(ValueError):
            eng.accept(acc)
    eng.accept(_i32([1, 1], gpu))  # still open
    eng.flush(state)


def test_more_prompt_chunks_than_draft_rows(gpu):
    from vkwr.model_executor import DraftEngine, SpeculativeBatcher
    cfg, model, state = _tiny(gpu, 6)
    eng = DraftEngine(model, 1, 7, max_rows=64)
    sched = SpeculativeBatcher(eng, state, max_prefill_chunks=6, chunk=8)
    reqs = [sched.submit([3 + i, 4, 5, 3 + i, 4], 4) for i in range(6)]
    assert len(sched.run()) == 6
    for r in reqs:
        _replay(model, r, gpu)


def test_adapters_scratch_is_whole_from_the_start(gpu):
    """Steps of every size, in any order, run in the scratch that the engine was built with."""
    from vkwr.model_executor import MixedEngine
    cfg, model, state = _tiny(gpu, 8)
    eng = MixedEngine(model, 64, adapters=_pool(model, gpu)[0])
    at = eng.adapters.ws.data_ptr()
    for T in (1, 9, 2, 60):
        tok = torch.ones(1, T, dtype=torch.int32, device=gpu)
        eng.step(state, prefill=[(tok, _i32([1], gpu))], adapter_ids=_i32([2], gpu))
    assert eng.adapters.ws.data_ptr() == at


def test_captured_steps_follow_the_adapter_indices(gpu):
    """A captured mixed step with adapters, replayed with other indices, tokens and slots: the eager step's
    logits and states."""
    from vkwr.model_executor import MixedEngine
    cfg, model, state = _tiny(gpu, 8)
    pool, _ = _pool(model, gpu)
    eng, eager = MixedEngine(model, 32, adapters=pool), MixedEngine(model, 32, adapters=pool)
    tok, slots, ids = _i32([1, 2, 3], gpu), _i32([0, 1, 2], gpu), _i32([0, 1, -1, 2], gpu)
    pre, pslot = torch.ones(1, 5, dtype=torch.int32, device=gpu), _i32([3], gpu)
    s1 = _clone(state)

    def step(e, s):
        return e.step(s, decode=(tok, slots), prefill=[(pre, pslot)], adapter_ids=ids)

    step(eng, _clone(state))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(eng, s1)
    s2 = _clone(s1)
    for seed in (1, 2, 3):
        g = torch.Generator().manual_seed(seed)
        tok.copy_(torch.randint(0, cfg.vocab, (3,), generator=g))
        pre.copy_(torch.randint(0, cfg.vocab, (1, 5), generator=g))
        ids.copy_(torch.randint(-1, 3, (4,), generator=g))
        perm = torch.randperm(8, generator=g)
        slots.copy_(perm[:3])
        pslot.copy_(perm[3:4])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step(eager, s2))
        assert torch.equal(s1.wkv, s2.wkv) and torch.equal(s1.att_shift, s2.att_shift)


def test_no_drafts_at_all(gpu):
    """max_draft = 0: plain decoding through the draft step."""
    from vkwr.model_executor import DraftEngine, SpeculativeBatcher
    cfg, model, state = _tiny(gpu, 4)
    eng = DraftEngine(model, 2, 0, max_rows=24)
    sched = SpeculativeBatcher(eng, state, max_decode=1, max_prefill_chunks=1, chunk=8)
    reqs = [sched.submit([5, 6, 7, 5, 6], n) for n in (1, 2, 5)]
    assert len(sched.run()) == 3 and sched.drafted == 0
    for r in reqs:
        assert len(r.output) == r.max_new_tokens
        _replay(model, r, gpu)
