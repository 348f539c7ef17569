"""CPU oracle (64 bits, plain lists) of beam search -- test infrastructure only: one selection, one
reordering of states, and a whole search over a function that gives a sequence's next log-probabilities."""
import math

import torch

INF = math.inf


def select(logits, scores, lengths, ended, end=-1, alpha=0.0):
    """The W best continuations of each request's W beams: tokens, parents, scores (float64), lengths, ended."""
    B, W, V = logits.shape
    out = [[], [], [], [], []]
    for b in range(B):
        cands = []
        for w in range(W):
            s, n = float(scores[b, w]), int(lengths[b, w])
            if not s > -INF:
                continue
            if ended[b, w]:
                cands.append((s * max(n, 1) ** -alpha, w, end, s, n, 1))
                continue
            l = logits[b, w].double()
            l = torch.where(l.isnan(), -INF, l)
            top = float(l.max())
            if top == -INF:
                continue
            d = torch.where(l == top, 0.0, l - top)
            lp = d - torch.log(torch.exp(d).sum())
            kth = float(torch.sort(lp, descending=True).values[min(W, V) - 1])
            keep = (lp > kth).nonzero()[:, 0].tolist() + (lp == kth).nonzero()[:W, 0].tolist()
            for v in keep:
                x = float(lp[v])
                if x > -INF:
                    cands.append(((s + x) * max(n + 1, 1) ** -alpha, w, v, s + x, n + 1, int(v == end)))
        cands = sorted(cands, key=lambda c: (-c[0], c[1], c[2]))[:W]
        rows = [(c[2], c[1], c[3], c[4], c[5]) for c in cands] + [(-1, -1, -INF, 0, 1)] * (W - len(cands))
        for o, r in zip(out, zip(*rows)):
            o.append(list(r))
    return [torch.tensor(o, dtype=torch.float64 if i == 2 else torch.int32) for i, o in enumerate(out)]


def reorder(slots, parents, skip, n_slots, pools):
    """(slots of the new beams, pools after the copies); skip may be None."""
    pools = [p.clone() for p in pools]
    new, moves = [], []
    W = slots.shape[1]
    skip = torch.zeros_like(slots) if skip is None else skip
    for s, p, k in zip(slots.tolist(), parents.tolist(), skip.tolist()):
        carry = [0 <= x < W and not y for x, y in zip(p, k)]
        first = {}
        for c in range(W):
            if carry[c]:
                first.setdefault(p[c], c)
        left = [s[b] for b in range(W) if b not in first]
        row = []
        for c in range(W):
            if carry[c] and first[p[c]] == c:
                row.append(s[p[c]])
            else:
                row.append(left.pop(0))
                if carry[c]:
                    moves.append((s[p[c]], row[-1]))
        new.append(row)
    for pool in pools:
        for a, b in moves:
            if 0 <= a < n_slots and 0 <= b < n_slots:
                pool[:, b] = pool[:, a]
    return torch.tensor(new, dtype=torch.int32), pools


def search(logits_of, prompt, width, steps, end=-1, alpha=0.0):
    """[(tokens, score, finished)], the best first; logits_of(tokens) gives a sequence's next logits."""
    beams = [([], 0.0, False)]
    for _ in range(steps):
        cands = []
        for w, (seq, score, over) in enumerate(beams):
            if over:
                cands.append((score * max(len(seq), 1) ** -alpha, w, end, seq, score, True))
                continue
            lp = torch.log_softmax(logits_of(list(prompt) + seq).double(), 0)
            for v in range(lp.numel()):
                x = score + float(lp[v])
                if x > -INF:
                    cands.append((x * (len(seq) + 1) ** -alpha, w, v, seq + [v], x, v == end))
        cands.sort(key=lambda c: (-c[0], c[1], c[2]))
        beams = [(c[3], c[4], c[5]) for c in cands[:width]]
    return beams
