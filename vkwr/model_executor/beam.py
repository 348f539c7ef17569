"""Beam search over the slot pools.

`BeamSearch.generate` runs up to `max_requests` prompts with `width` beams each on a MixedEngine.  A prompt
is prefilled once, in the slot of its first beam; every further step runs all beams of all requests as
decode rows (finished ones too: a step's rows are fixed), then

  capi.beam_select   the best continuations of each request's beams, on the device
  capi.beam_reorder  their states follow: the first child of a beam stays in its slot, others get a copy

and nothing comes back to the host but, every few steps, whether all beams are finished.  Tokens and parents
of each step are kept on the device and walked back at the end.  With capture=True a step is recorded into
a HIP graph once per number of requests and replayed.
"""
from dataclasses import dataclass

import torch

from vkwr_amd import capi

CHECK_EVERY = 8  # steps between looks at whether all beams are finished


@dataclass
class Hypothesis:
    tokens: list         # generated tokens, `end` included where it was generated
    score: float         # sum of their log-probabilities
    normalised: float    # score / length^length_penalty, by which hypotheses are ordered
    finished: bool       # ends with `end`


class BeamSearch:
    """`slots`: max_requests * width distinct slot numbers that the search may use (default: the first ones);
    their states are reset by every call.  end: the token that finishes a beam (-1: none).  max_new_tokens:
    the most that a call may ask for."""

    def __init__(self, engine, state, width, max_requests=1, max_new_tokens=1024, end=-1, length_penalty=0.0, slots=None,
                 max_prefill_chunks=4, chunk=512, capture=False):
        n, vocab = max_requests * width, engine.cfg.vocab
        if not 1 <= width <= capi.MAX_BEAMS or max_requests < 1 or max_new_tokens < 1:
            raise ValueError(f"beam search: {max_requests} requests of {width} beams (1 to {capi.MAX_BEAMS}), "
                             f"{max_new_tokens} tokens")
        if n > engine.max_rows or n > engine.max_seqs or min(max_prefill_chunks, max_requests) > engine.max_seqs:
            raise ValueError(f"beam search: {n} beams, {max_prefill_chunks} chunks; the engine has {engine.max_rows} rows "
                             f"and logits for {engine.max_seqs}")
        if chunk < 1 or max_prefill_chunks < 1 or not -1 <= end < vocab:
            raise ValueError(f"beam search: chunks of {chunk}, {max_prefill_chunks} at a time, end token {end} of {vocab}")
        slots = list(range(n)) if slots is None else [int(s) for s in slots]
        if len(slots) != n or len(set(slots)) != n or not all(0 <= s < state.n_slots for s in slots):
            raise ValueError(f"beam search: needs {n} distinct slots below {state.n_slots}, got {slots}")
        self.engine, self.state, self.width, self.max_requests = engine, state, width, max_requests
        self.max_new_tokens, self.end, self.length_penalty = max_new_tokens, end, length_penalty
        self.slots, self.max_prefill_chunks, self.chunk = slots, max_prefill_chunks, min(chunk, engine.max_rows)
        self.capture, self.graphs = capture, {}
        dev = self.device = engine.model.head.device
        i32 = dict(dtype=torch.int32, device=dev)
        # scores (fp32 bits), lengths, ended, slots of the beams: before a step and after it
        self.now, self.new = torch.zeros(4 * n, **i32), torch.zeros(4 * n, **i32)
        self.parents, self.tokens, self.ids = torch.zeros(n, **i32), torch.zeros(n, **i32), torch.zeros(n, **i32)
        self.hist = torch.zeros(2, max_new_tokens, n, **i32)  # tokens, parents
        self.at = torch.zeros(1, dtype=torch.int64, device=dev)
        self.first = torch.zeros(n, vocab, dtype=torch.float16, device=dev)
        self.ws = torch.empty(capi.beam_workspace_bytes(max_requests, width, vocab), dtype=torch.uint8, device=dev)

    def _views(self, buf, B):
        n = B * self.width
        s, le, e, sl = (buf[i * n:(i + 1) * n].view(B, self.width) for i in range(4))
        return s.view(torch.float32), le, e, sl

    def _reset(self, B):
        used = self.slots[:B * self.width]
        st, at = self.state, torch.tensor(used).to(self.device)
        for pool in (st.wkv, st.att_shift, st.ffn_shift):
            pool.index_fill_(1, at, 0)
        drop = getattr(self.engine, "drop", None)  # a DraftEngine: what it keeps of the slots' last users
        if drop is not None:
            drop(used, st)
        scores, lengths, ended, slots = self._views(self.now, B)
        scores.fill_(float("-inf"))
        scores[:, 0].zero_()  # a request's beams are one behind its prompt
        lengths.zero_()
        ended.zero_()
        slots.copy_(torch.tensor(used, dtype=torch.int32).view(B, self.width))
        self.at.zero_()

    def _prefill(self, prompts, adapters):
        """The prompts, in the slots of the first beams; the logits behind them into rows of `first`."""
        W, left = self.width, [0] * len(prompts)
        while True:
            groups, rows = {}, 0
            for b, p in enumerate(prompts):
                t = min(self.chunk, len(p) - left[b], self.engine.max_rows - rows)
                if t <= 0:
                    continue
                groups.setdefault(t, []).append(b)
                rows += t
                if sum(len(g) for g in groups.values()) == self.max_prefill_chunks:
                    break
            if not groups:
                return
            i32 = lambda v: torch.tensor(v, dtype=torch.int32).to(self.device)  # noqa: E731
            order = [b for g in groups.values() for b in g]
            kw = {} if adapters is None else {"adapter_ids": i32([adapters[b] for b in order])}
            logits = self.engine.step(self.state, prefill=[
                (i32([prompts[b][left[b]:left[b] + t] for b in g]), i32([self.slots[b * W] for b in g]))
                for t, g in groups.items()], **kw)
            for i, b in enumerate(order):
                left[b] += next(t for t, g in groups.items() if b in g)
                if left[b] == len(prompts[b]):
                    self.first[b * W].copy_(logits[i])

    def _choose(self, logits, B):
        """One step behind the model's: the next beams, their states, and what the next step reads."""
        n = B * self.width
        scores, lengths, ended, slots = self._views(self.now, B)
        scores2, lengths2, ended2, slots2 = self._views(self.new, B)
        tokens, parents = self.tokens[:n].view(B, -1), self.parents[:n].view(B, -1)
        capi.beam_select(logits, scores, lengths, ended, tokens, parents, scores2, lengths2, ended2, end=self.end,
                         length_penalty=self.length_penalty, workspace=self.ws)
        st = self.state
        capi.beam_reorder(slots, parents, slots2, [st.wkv, st.att_shift, st.ffn_shift], skip=ended2)
        self.hist[0, :, :n].index_copy_(0, self.at, self.tokens[None, :n])
        self.hist[1, :, :n].index_copy_(0, self.at, self.parents[None, :n])
        self.at += 1
        self.tokens[:n].clamp_(min=0)  # (a beam that is not there is stepped with some token)
        self.now.copy_(self.new)

    def _step(self, B, adapters):
        n = B * self.width
        kw = {"adapter_ids": self.ids[:n]} if adapters else {}
        logits = self.engine.step(self.state, decode=(self.tokens[:n], self._views(self.now, B)[3].view(-1)), **kw)
        self._choose(logits.view(B, self.width, -1), B)

    def _run_step(self, B, adapters):
        if not self.capture:
            return self._step(B, adapters)
        graph = self.graphs.get((B, adapters))
        if graph is None:
            self.graphs[B, adapters] = False
            return self._step(B, adapters)  # (first as it is: libraries load and allocate on first use)
        if graph is False:
            torch.cuda.synchronize(self.device)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                self._step(B, adapters)
            self.graphs[B, adapters] = graph
        graph.replay()

    def generate(self, prompts, max_new_tokens, adapters=None):
        """prompts: lists of tokens; adapters (engines with adapters): an index per prompt, -1 for none.
        Returns a list of Hypothesis per prompt, the best first (at most `width`)."""
        prompts = [list(p) for p in prompts]
        vocab = self.engine.cfg.vocab
        if any(not 0 <= t < vocab for p in prompts for t in p):
            raise ValueError(f"beam search: a token outside the vocabulary of {vocab}")
        if not all(prompts) or not 1 <= max_new_tokens <= self.max_new_tokens:
            raise ValueError(f"beam search: an empty prompt, or {max_new_tokens} new tokens (1 to {self.max_new_tokens})")
        if adapters is not None and (len(adapters) != len(prompts) or getattr(self.engine, "adapters", None) is None):
            raise ValueError(f"beam search: {len(adapters)} adapters for {len(prompts)} prompts, or an engine without")
        pool = getattr(getattr(self.engine, "adapters", None), "pool", None)
        if adapters is not None and pool is not None and any(a >= pool.n_adapters for a in adapters):
            raise ValueError(f"beam search: adapters {list(adapters)} of {pool.n_adapters}")
        if getattr(self.engine, "open", None) is not None:  # a DraftEngine, whose step would refuse it when states are reset
            raise RuntimeError("beam search: the engine's last drafts are not accepted yet")
        out = []
        at_once = min(self.max_requests, capi.MAX_BEAM_ROWS // self.width)
        for i in range(0, len(prompts), at_once):
            part = slice(i, i + at_once)
            out += self._generate(prompts[part], max_new_tokens, None if adapters is None else list(adapters[part]))
        return out

    def _generate(self, prompts, steps, adapters):
        B, W = len(prompts), self.width
        n = B * W
        self._reset(B)
        self._prefill(prompts, adapters)
        if adapters is not None:
            self.ids[:n].copy_(torch.tensor(adapters, dtype=torch.int32).repeat_interleave(W))
        self._choose(self.first[:n].view(B, W, -1), B)
        done = 1
        ended = self._views(self.now, B)[2]
        while done < steps:
            if self.end >= 0 and done % CHECK_EVERY == 0 and bool((ended != 0).all()):
                break
            self._run_step(B, adapters is not None)
            done += 1
        scores, lengths, ended, _ = (t.tolist() for t in self._views(self.now, B))
        tokens, parents = self.hist[:, :done, :n].cpu().view(2, done, B, W).tolist()
        return [self._walk(scores[b], lengths[b], ended[b], [t[b] for t in tokens], [p[b] for p in parents]) for b in range(B)]

    def _walk(self, scores, lengths, ended, tokens, parents):
        """Every beam's tokens, from the last step's parents back."""
        out = []
        for w, score in enumerate(scores):
            if score == float("-inf"):
                continue
            at, seq = w, []
            for tok, par in zip(reversed(tokens), reversed(parents)):
                seq.append(tok[at])
                at = par[at]
            n = lengths[w]  # behind a finished beam's end there is only the end again
            seq = seq[::-1][:n]
            out.append(Hypothesis(seq, score, score / max(n, 1) ** self.length_penalty, bool(ended[w])))
        return out


__all__ = ["BeamSearch", "Hypothesis"]
