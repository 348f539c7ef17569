"""Speculative decoding: a step over drafted tokens, whose state is written once it is known how many
of them stay.

`DraftEngine.draft_step` runs T tokens of each sequence (the last one generated, then T - 1 drafts) through
the model in one pass and returns the logits behind every one of them; `accept` then says how many drafts
each sequence keeps (capi.verify_drafts decides, from the logits).  A recurrent state cannot drop the
rejected tokens again, so the step leaves the states alone:

  WKV     the step's w, k', v, -kk, kk*a of every layer are kept, and the next draft step's WKV launches
          take the kept tokens from them before they run their own drafts (vkwr_wkv7_fp32_drafts_slots):
          one read and one write of each state per step, whatever T is.
  shift   the LayerNorm rows of every layer are kept, and `accept` copies the last kept token's into the
          shift pools.

Between steps the WKV pool is behind by the kept tokens of the sequences of the last draft step: `flush`
writes them (before the pool is read by anything else), `drop` forgets them (finished sequences, slots that
are reset).  Sequences that a draft step leaves out are flushed by it, all of them by `step`.

Per layer as MixedEngine's step, with the fused LayerNorm + shift launches replaced by LayerNorm (its rows
kept) and a token shift on gathered shift rows.
"""
import torch

from vkwr_amd import capi
from vkwr.model_executor.mixed import TMIX_MIX, MixedEngine

PENDING = ("w", "new_k", "v", "neg_kk", "kka")


class DraftEngine(MixedEngine):
    """Draft steps of up to `max_seqs` sequences of up to `max_draft` drafts; also a MixedEngine (prompts,
    plain decode steps) of max_seqs * (max_draft + 1) rows, or max_rows if that is more."""

    def __init__(self, model, max_seqs, max_draft, max_rows=0, adapters=None):
        self.draft_rows = max_seqs * (max_draft + 1)
        super().__init__(model, max(max_rows, self.draft_rows), max_seqs=self.draft_rows, adapters=adapters)
        cfg, dev, R, C = model.cfg, model.head.device, self.draft_rows, model.cfg.n_embd
        self.max_draft, self.draft_seqs = max_draft, max_seqs

        def buf(*shape):
            return torch.empty(*shape, dtype=torch.float16, device=dev)

        # the vectors of two steps (this one's and the one before's), per layer
        self.pend = [[{n: buf(R, C) for n in PENDING} for _ in model.layers] for _ in range(2)]
        self.ys = [buf(cfg.n_layer, R, C) for _ in range(2)]  # LN1 and LN2 rows of the step
        self.which = 0           # the set that holds the last step's vectors
        self.open = None         # the draft step that waits for accept: (state, slots, B, T, shift rows before)
        self.rows_of = {}        # slot -> its sequence in the last draft step, where tokens are to be written
        self.T, self.kept = 0, None
        self.pool_of = None
        if adapters is not None:  # layer 0's values go to the kept vectors
            self.adapted_first = [self._adapted_rkv(0, self.pend[i][0]["v"]) for i in range(2)]

    def step(self, state, decode=None, prefill=(), adapter_ids=None, flush=True):
        """MixedEngine's step, the kept tokens written first.  flush=False: not (for the caller whose
        slots here have none)."""
        if self.open is not None:
            raise RuntimeError("step: the last step's drafts are not accepted yet")
        if flush and self.pool_of is state.wkv:
            self.flush(state)
        return super().step(state, decode, prefill, adapter_ids)

    def draft_step(self, state, tokens, slots, adapter_ids=None):
        """tokens [B, T] int32 on the device (the last generated token, then the drafts; anything behind a
        short draft: a number outside the vocabulary runs as the nearest inside), slots: B distinct slot
        numbers (host).  Returns logits [B, T, V] (a view valid until the next step); `accept` has to follow."""
        B, T = tokens.shape
        slots = [int(i) for i in slots]
        if self.open is not None:
            raise RuntimeError("draft_step: the last step's drafts are not accepted yet")
        if not (0 < B <= self.draft_seqs and 1 <= T <= self.max_draft + 1) or len(slots) != B:
            raise ValueError(f"draft_step: {B} sequences of {T} tokens, {len(slots)} slots; at most "
                             f"{self.draft_seqs} of {self.max_draft + 1}")
        if len(set(slots)) != B or not all(0 <= i < state.n_slots for i in slots):
            raise ValueError(f"draft_step: slots must be distinct and below {state.n_slots}: {slots}")
        if state.layout != capi.WKV_STATE_STD:
            raise ValueError("draft_step: the row-major WKV pool is needed")
        if self.rows_of and self.pool_of is not state.wkv:
            raise RuntimeError("draft_step: kept tokens of another state are not written yet (flush)")
        adapters = self._begin_adapters([(B, T, 0, None, 0)], adapter_ids)
        self.flush(state, [i for i in self.rows_of if i not in set(slots)])
        cfg, m, s = self.cfg, self.model, self
        C, H, R, ws = cfg.n_embd, cfg.n_head, B * T, self.ws
        dev = tokens.device
        sl = torch.tensor(slots, dtype=torch.int32).to(dev, non_blocking=True)
        sl64 = sl.long()
        # kept tokens of the step before
        kept = rows = None
        if self.rows_of:
            r = torch.tensor([self.rows_of.get(i, -1) for i in slots], dtype=torch.int32).to(dev, non_blocking=True)
            kept = torch.where(r >= 0, self.kept[r.clamp(min=0).long()], 0).to(torch.int32)
            rows = r.clamp(min=0)
        before, now = self.pend[self.which], self.pend[self.which ^ 1]
        att = state.att_shift.index_select(1, sl64)  # [L, B, C]
        ffn = state.ffn_shift.index_select(1, sl64)
        att0, ffn0 = att.clone(), ffn.clone()
        s.tok[:R].copy_(tokens.reshape(-1).clamp(0, cfg.vocab - 1))
        torch.index_select(m.emb, 0, s.tok[:R], out=s.x0[:R])
        own = s.w, s.v_first, s.v_new
        x, res_in = s.x0[:R], None
        try:
            for l, L in enumerate(m.layers):
                first = l == 0
                N = now[l]
                s.w = N["w"]
                if first:
                    s.v_first = N["v"]
                else:
                    s.v_new = N["v"]
                res = x if first else s.res[1][:R]  # layer 0: the embedding is the residual stream
                y = self.ys[0][l, :R]
                capi.layer_norm(x, L["ln1_w"], L["ln1_b"], y, residual=res_in, x_out=None if first else res)
                capi.token_shift(B, T, C, y, att[l], [L[k] for k in TMIX_MIX], [t[:R] for t in s.mix])
                capi.gemm(self._proj(L, s.lw[l], R, first), ws)
                if adapters is not None:
                    adapters.add(self.adapted_first[self.which ^ 1] if first else self.adapted[l]["rkv"])
                capi.gemm(self._rank_out(L, s.lw[l], R, first), ws)
                v = N["v"][:R]
                capi.kk_a_gate(R, 1, C, H, s.k[:R], L["k_k"], L["a0"], s.a12[:R], L["k_a"], N["new_k"][:R],
                               N["neg_kk"][:R], N["kka"][:R])
                P = before[l]
                pending = None if kept is None else tuple(P[n][:self.B * self.T].view(self.B, self.T, C) for n in PENDING)
                capi.wkv_drafts_slots(B, T, C, H, state.wkv[l], sl, s.r[:R], N["w"][:R], N["new_k"][:R], v,
                                      N["neg_kk"][:R], N["kka"][:R], s.y[:R], kept=kept, pending=pending,
                                      pending_rows=rows)
                capi.groupnorm_bonus_gate(R, 1, C, H, s.y[:R], s.r[:R], N["new_k"][:R], v, L["r_k"], L["lnx_w"],
                                          L["lnx_b"], s.g[:R], s.o_in[:R])
                capi.gemm([capi.gemm_problem(s.o_in[:R], L["Wo"], s.o[:R])], ws)
                if adapters is not None:
                    adapters.add(self.adapted[l]["o"])
                res2 = s.res[0][:R]
                y = self.ys[1][l, :R]
                capi.layer_norm(s.o[:R], L["ln2_w"], L["ln2_b"], y, residual=res, x_out=res2)
                capi.token_shift(B, T, C, y, ffn[l], [L["x_k_ffn"]], [s.xk[:R]])
                self._ffn(l, L, R, adapters)
                x, res_in = s.ffn[:R], res2
        finally:
            s.w, s.v_first, s.v_new = own
        capi.add_last_layer_norm(R, 1, C, x, res_in, m.ln_out_w, m.ln_out_b, s.h[:R])
        capi.gemm(self._head_problem(R), ws)
        self.which ^= 1
        self.B, self.T, self.rows_of, self.pool_of = B, T, {}, None  # the step before is written now
        self.open = (state, slots, sl64, att0, ffn0)
        return s.logits[:R].view(B, T, -1)

    def accept(self, accepted):
        """accepted [B] int32 on the device: the drafts that each sequence of the last draft step keeps (its
        first token stays in any case; below 0, as verify_drafts reports a bad draft length: nothing)."""
        if self.open is None:
            raise RuntimeError("accept: no draft step is open")
        state, slots, sl, att0, ffn0 = self.open
        B, T = self.B, self.T
        if tuple(accepted.shape) != (B,) or accepted.dtype != torch.int32 or accepted.device != sl.device:
            raise ValueError(f"accept: expected int32 [{B}] on {sl.device}, got {accepted.dtype} "
                             f"{tuple(accepted.shape)} on {accepted.device}")
        self.open = None
        self.kept = (accepted + 1).clamp(min=0, max=T).to(torch.int32)
        last = (self.kept - 1).clamp(min=0).long()
        some = (self.kept > 0)[None, :, None]
        for pool, ys, old in ((state.att_shift, self.ys[0], att0), (state.ffn_shift, self.ys[1], ffn0)):
            at = torch.arange(B, device=last.device) * T + last
            pool.index_copy_(1, sl, torch.where(some, ys.index_select(1, at), old))
        self.rows_of = {slot: b for b, slot in enumerate(slots)}
        self.pool_of = state.wkv

    def flush(self, state, slots=None):
        """Writes the kept tokens of these slots (None: all) to the WKV pool."""
        if self.open is not None:
            raise RuntimeError("flush: the last step's drafts are not accepted yet")
        todo = [i for i in dict.fromkeys(self.rows_of if slots is None else slots) if i in self.rows_of]
        if not todo:
            return
        if self.pool_of is not state.wkv:
            raise RuntimeError("flush: the kept tokens are another state's")
        cfg, C, H, P = self.cfg, self.cfg.n_embd, self.cfg.n_head, self.T
        dev = self.kept.device
        rows = torch.tensor([self.rows_of[i] for i in todo], dtype=torch.int32).to(dev, non_blocking=True)
        sl = torch.tensor(todo, dtype=torch.int32).to(dev, non_blocking=True)
        kept = self.kept[rows.long()]
        for l in range(cfg.n_layer):
            N = self.pend[self.which][l]
            pending = tuple(N[n][:self.B * P].view(self.B, P, C) for n in PENDING)
            capi.wkv_drafts_slots(len(todo), 0, C, H, state.wkv[l], sl, *[None] * 7, kept=kept, pending=pending,
                                  pending_rows=rows)
        self.drop(todo)

    def drop(self, slots, state=None):
        """Forgets the kept tokens of these slots (sequences that end); given a state, only if they are its.
        Not between a draft step and its accept, which is what says that tokens are kept."""
        if self.open is not None and (state is None or self.open[0].wkv is state.wkv):
            raise RuntimeError("drop: the last step's drafts are not accepted yet")
        if state is not None and self.pool_of is not state.wkv:
            return
        for i in slots:
            self.rows_of.pop(i, None)


__all__ = ["DraftEngine"]
