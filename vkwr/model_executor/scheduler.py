"""Continuous batching over a WKV slot pool (the reference has no serving code).

Requests arrive with a prompt and a generation budget.  The batcher admits them
into free slots of the recurrent-state pool (resetting the slot's WKV state and
both shift rows), then every step runs one MixedEngine forward over

  * up to `max_decode` sequences that are generating (one token each: the last
    token they produced), and
  * up to `max_prefill_chunks` prompt chunks of at most `chunk` tokens from
    sequences still consuming their prompt (chunks of equal length share one
    prefill group),

within `max_rows` rows in total.  A sequence's first generated token comes from
the logits of its last prompt chunk; each later one from its decode row.
Finished sequences release their slot immediately, so waiting requests are
admitted the next step (256 decode rows + 4 x 512 prefill
rows per step, 2048-slot pool).  The default sampler is greedy (argmax); pass
`sample` to use another, e.g. a ``GpuSampler`` (temperature / top-k / top-p on
the vkwr_sampling kernels).  A request may name an adapter of the engine's pool.

`SpeculativeBatcher` does the same on a `DraftEngine`: generating sequences run
their last token and up to `max_draft` drafts in one draft step, `verify_drafts`
accepts or rejects them, and a sequence advances by one token or more.
"""
from collections import deque
from dataclasses import dataclass, field

import torch

from vkwr_amd import capi


@dataclass
class Request:
    prompt: list
    max_new_tokens: int
    rid: int = -1
    slot: int = -1
    pos: int = 0                       # prompt tokens consumed
    output: list = field(default_factory=list)
    adapter: int = -1                  # of the engine's AdapterPool; -1: none

    @property
    def prefilling(self):
        return self.pos < len(self.prompt)

    @property
    def done(self):
        return len(self.output) >= self.max_new_tokens


class SlotAllocator:
    """Free list over the state pool's slots (FIFO reuse).  Freeing a slot that is out of
    range or not allocated raises RuntimeError, so the slot lists the batcher builds from
    allocated slots are distinct and in range: it checks them on the host and passes
    them to the kernels without a device-side check."""

    def __init__(self, n_slots):
        self.n_slots = n_slots
        self._free = deque(range(n_slots))
        self._used = set()

    def alloc(self):
        if not self._free:
            return None
        slot = self._free.popleft()
        self._used.add(slot)
        return slot

    def free(self, slot):
        if not (0 <= slot < self.n_slots) or slot not in self._used:
            raise RuntimeError(f"slot {slot} is not allocated (pool of {self.n_slots})")
        self._used.remove(slot)
        self._free.append(slot)

    @property
    def available(self):
        return len(self._free)


class ContinuousBatcher:
    def __init__(self, engine, state, max_decode=256, max_prefill_chunks=4, chunk=512, sample=None):
        assert chunk >= 1 and max_decode + chunk <= engine.max_rows
        # every decode row and every chunk's sequence gets a logits row
        assert max_decode + max_prefill_chunks <= engine.max_seqs, (max_decode, max_prefill_chunks, engine.max_seqs)
        self.engine, self.state = engine, state
        self.max_decode, self.max_prefill_chunks, self.chunk = max_decode, max_prefill_chunks, chunk
        self.max_rows = engine.max_rows
        self.slots = SlotAllocator(state.n_slots)
        self.waiting = deque()
        self.running = []
        self.sample = sample or (lambda logits: torch.argmax(logits.float(), dim=-1))
        self.device = engine.model.head.device
        self._next_id = 0
        self._rr = 0  # round-robin start among the decoding sequences
        self.steps = 0
        self.tokens_processed = 0

    def submit(self, prompt, max_new_tokens, adapter=-1):
        assert len(prompt) >= 1 and max_new_tokens >= 1
        adapters = getattr(self.engine, "adapters", None)
        n = 0 if adapters is None else adapters.pool.n_adapters
        if not -1 <= adapter < n:
            raise ValueError(f"adapter {adapter} of {n}")
        req = Request(list(prompt), max_new_tokens, rid=self._next_id, adapter=adapter)
        self._next_id += 1
        self.waiting.append(req)
        return req

    def _reset_slot(self, slot):
        st = self.state
        st.wkv[:, slot].zero_()
        st.att_shift[:, slot].zero_()
        st.ffn_shift[:, slot].zero_()
        drop = getattr(self.engine, "drop", None)  # a DraftEngine: what it keeps of the slot's last user
        if drop is not None:
            drop([slot], st)

    def _i32(self, values):
        return torch.tensor(values, dtype=torch.int32).to(self.device, non_blocking=True)

    def _check_slots(self, reqs):
        """Host-side slot-table check of one step (no device sync): every slot allocated,
        each used by one sequence only."""
        slots = [r.slot for r in reqs]
        if len(set(slots)) != len(slots) or any(s not in self.slots._used for s in slots):
            raise RuntimeError(f"invalid slot table for this step: {slots}")

    def _adapter_ids(self, reqs):
        """The step's argument for these requests' adapters, where one of them has any."""
        ids = [r.adapter for r in reqs]
        return {"adapter_ids": self._i32(ids)} if any(i >= 0 for i in ids) else {}

    def _admit(self):
        while self.waiting and self.slots.available:
            req = self.waiting.popleft()
            req.slot = self.slots.alloc()
            self._reset_slot(req.slot)
            self.running.append(req)

    def _decoding(self):
        """The generating sequences of this step."""
        decoding = [r for r in self.running if not r.prefilling]
        if len(decoding) > self.max_decode:
            # more generating sequences than decode rows: rotate, so none starves
            start = self._rr % len(decoding)
            self._rr = start + self.max_decode
            return (decoding[start:] + decoding[:start])[: self.max_decode]
        return decoding

    def _chunks(self, rows):
        """Prompt chunks of this step beside `rows` decode rows: chunk length -> requests."""
        groups = {}
        n_chunks = 0
        for r in self.running:
            if not r.prefilling or n_chunks == self.max_prefill_chunks:
                continue
            t = min(self.chunk, len(r.prompt) - r.pos, self.max_rows - rows)
            if t <= 0:
                break
            groups.setdefault(t, []).append(r)
            rows += t
            n_chunks += 1
        return groups

    def step(self):
        """Runs one forward step; returns the requests that finished in it."""
        self._admit()
        dec = self._decoding()
        groups = self._chunks(len(dec))
        rows = len(dec) + sum(t * len(reqs) for t, reqs in groups.items())
        if rows == 0:
            return []
        self._check_slots(dec + [r for reqs in groups.values() for r in reqs])
        decode = None
        if dec:
            decode = (self._i32([r.output[-1] for r in dec]), self._i32([r.slot for r in dec]))
        prefill, order = [], []
        for t, reqs in groups.items():
            toks = self._i32([r.prompt[r.pos:r.pos + t] for r in reqs])
            prefill.append((toks, self._i32([r.slot for r in reqs])))
            order.append((t, reqs))
        logits = self.engine.step(self.state, decode=decode, prefill=prefill,
                                  **self._adapter_ids(dec + [r for _, reqs in order for r in reqs]))
        nxt = self.sample(logits).tolist()
        for i, r in enumerate(dec):
            r.output.append(nxt[i])
        j = len(dec)
        for t, reqs in order:
            for r in reqs:
                r.pos += t
                if not r.prefilling:
                    r.output.append(nxt[j])
                j += 1
        self.steps += 1
        self.tokens_processed += rows
        finished = [r for r in self.running if r.done]
        for r in finished:
            self.slots.free(r.slot)
        self.running = [r for r in self.running if not r.done]
        return finished

    def run(self, max_steps=1 << 30):
        """Steps until every submitted request finished; returns them in completion order."""
        done = []
        while (self.waiting or self.running) and self.steps < max_steps:
            done += self.step()
        return done


def prompt_lookup(tokens, n, match=2):
    """Up to n drafts: what followed the latest earlier occurrence of the last `match` tokens."""
    if len(tokens) <= match:
        return []
    tail = tokens[-match:]
    for i in range(len(tokens) - match - 1, -1, -1):
        if tokens[i:i + match] == tail:
            return tokens[i + match:i + match + n]
    return []


class _Lookup:
    """prompt_lookup of one growing sequence by an index of its pairs of tokens: the steps of a call are the
    tokens that came since the last, not the sequence's (a list scanned anew took 0.66 ms of 8192 tokens, once a
    sequence and step)."""

    def __init__(self, prompt):
        self.tokens, self.places, self.seen = list(prompt), {}, 0

    def __call__(self, request, n):
        t = self.tokens
        t += request.output[len(t) - len(request.prompt):]
        for i in range(self.seen, len(t) - 2):  # all pairs but the last
            self.places[t[i], t[i + 1]] = i
        self.seen = max(len(t) - 2, 0)
        at = self.places.get(tuple(t[-2:]))
        return [] if at is None else t[at + 2:at + 2 + n]


class SpeculativeBatcher(ContinuousBatcher):
    """Continuous batching with drafted tokens on a DraftEngine.  `draft(tokens, n)` proposes up to n
    tokens behind a sequence's tokens (default: looked up in them); top_k = 1 generates greedily, the lowest
    index among equal logits, whatever the drafts and the seed.
    Prompt chunks run as in ContinuousBatcher, in a step of their own before the drafts'."""

    def __init__(self, engine, state, draft=prompt_lookup, temperature=1.0, top_k=1, top_p=1.0, seed=0, **kw):
        if kw.get("sample") is not None:
            raise TypeError("tokens are drawn by verify_drafts (temperature, top_k, top_p): no sample function")
        kw.setdefault("max_decode", engine.draft_seqs)
        if kw["max_decode"] > engine.draft_seqs:
            raise ValueError(f"{kw['max_decode']} generating sequences, the engine drafts {engine.draft_seqs}")
        super().__init__(engine, state, **kw)
        B, T = engine.draft_seqs, engine.max_draft + 1
        self.draft, self.filter = draft, dict(temperature=temperature, top_k=top_k, top_p=top_p)
        self.gen = torch.Generator(device=self.device).manual_seed(seed)
        V = engine.cfg.vocab
        # top_k = 1 (top_p = 0 stands for it): a row of its own per token
        self.greedy = top_k == 1 or top_p == 0
        P = self.max_prefill_chunks
        sizes = ((B * T, 0), (P, 0)) if self.greedy else ((B, T - 1), (P, 0))
        need = max(capi.verify_workspace_bytes(b, k, V) for b, k in sizes)
        self.ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        self.zeros = torch.zeros(max(B * T, P), 1, dtype=torch.float32, device=self.device)
        self.drafted = self.accepted = 0
        self.lookups = {}  # request id -> _Lookup

    def _draft(self, r, n):
        if self.draft is prompt_lookup:
            if r.rid not in self.lookups:
                self.lookups[r.rid] = _Lookup(r.prompt)
            return self.lookups[r.rid](r, n)
        return list(self.draft(r.prompt + r.output, n))[:self.engine.max_draft]

    def _verify(self, logits, drafts, n_draft):
        """logits [B, T, V], n_draft: the drafts' lengths (host); (tokens, accepted) on the device."""
        B, T, _ = logits.shape
        if self.greedy:
            return self._verify_greedy(logits, drafts, n_draft)
        tokens = torch.empty(B, T, dtype=torch.int32, device=self.device)
        accepted = torch.empty(B, dtype=torch.int32, device=self.device)
        u = torch.rand(B, T, generator=self.gen, dtype=torch.float32, device=self.device)
        capi.verify_drafts(logits, drafts, u, tokens, accepted, n_draft=self._i32(n_draft), workspace=self.ws,
                           **self.filter)
        return tokens, accepted

    def _verify_greedy(self, logits, drafts, n_draft):
        """As _verify, where only a row's first largest logit will do (fp16 logits are often tied, and the filter
        keeps all entries that are): every row's token is drawn with the uniform 0, which falls on the first kept
        entry, and compared with the draft.  Rows behind a short draft (a length of -1) are not looked at."""
        B, T, V = logits.shape
        best = torch.empty(B * T, 1, dtype=torch.int32, device=self.device)
        count = torch.empty(B * T, dtype=torch.int32, device=self.device)
        capi.verify_drafts(logits.view(B * T, 1, V), drafts.new_empty(B * T, 0), self.zeros[:B * T], best, count,
                           n_draft=self._i32([0 if t <= n else -1 for n in n_draft for t in range(T)]),
                           workspace=self.ws, **self.filter)
        best = best.view(B, T)
        # (behind a short draft: drafts of -1, which no row's token is)
        accepted = (best[:, :T - 1] == drafts).to(torch.int32).cumprod(1).sum(1, dtype=torch.int32)
        kept = torch.arange(T, device=self.device) <= accepted[:, None]
        return torch.where(kept, best, -1), accepted

    def _finish(self):
        finished = [r for r in self.running if r.done]
        for r in finished:
            self.engine.drop([r.slot], self.state)
            self.lookups.pop(r.rid, None)
            self.slots.free(r.slot)
        self.running = [r for r in self.running if not r.done]
        return finished

    def step(self):
        """Prompt chunks, then one draft step of the generating sequences; returns the requests that
        finished."""
        self._admit()
        groups = self._chunks(0)
        if groups:
            order = [(t, reqs) for t, reqs in groups.items()]
            flat = [r for _, reqs in order for r in reqs]
            self._check_slots(flat)
            prefill = [(self._i32([r.prompt[r.pos:r.pos + t] for r in reqs]), self._i32([r.slot for r in reqs]))
                       for t, reqs in order]
            # (a prompt's slot is fresh: no kept tokens)
            logits = self.engine.step(self.state, prefill=prefill, flush=False, **self._adapter_ids(flat))
            none = torch.empty(len(flat), 0, dtype=torch.int32, device=self.device)
            nxt = self._verify(logits[:, None, :], none, [0] * len(flat))[0][:, 0].tolist()
            for (t, r), token in zip([(t, r) for t, reqs in order for r in reqs], nxt):
                r.pos += t
                self.tokens_processed += t
                if not r.prefilling:
                    r.output.append(token)
            done = self._finish()
        else:
            done = []
        dec = self._decoding()
        if dec:
            self._check_slots(dec)
            K = self.engine.max_draft
            drafts = [self._draft(r, min(K, r.max_new_tokens - len(r.output) - 1)) for r in dec]
            T = 1 + max(len(d) for d in drafts)
            rows = self._i32([[r.output[-1]] + d + [-1] * (T - 1 - len(d)) for r, d in zip(dec, drafts)])
            logits = self.engine.draft_step(self.state, rows, [r.slot for r in dec], **self._adapter_ids(dec))
            tokens, accepted = self._verify(logits, rows[:, 1:].contiguous(), [len(d) for d in drafts])
            self.engine.accept(accepted)
            for r, d, new, n in zip(dec, drafts, tokens.tolist(), accepted.tolist()):
                r.output += new[:min(n + 1, r.max_new_tokens - len(r.output))]
                self.drafted += len(d)
                self.accepted += n
            self.tokens_processed += rows.numel()
        if groups or dec:
            self.steps += 1
        return done + self._finish()


__all__ = ["Request", "SlotAllocator", "ContinuousBatcher", "SpeculativeBatcher", "prompt_lookup"]
