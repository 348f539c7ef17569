"""Serving operators as measurable cases: projections with 8-bit weights, one step of beam search,
and the reordering of recurrent states behind it.

A case is a dict of plain values; `prepare` makes its inputs on the GPU from a seed, `run`
makes one pass over them, `work` states the bytes and operations that the pass cannot do
without and `exact` computes the same outputs in 64 bits.  `listed` holds the named cases,
`draw` gives further ones of the same ranges.  With `own` False, `run` computes the operators
from elementary torch operations; with `own` True it calls the package's entry points.

Kinds of work (field "kind"):

  linear   y = f(s_i t_j sum_k q_ik w_jk): every row x_i of fp16 activations is rounded to 8 bits
           with a scale of its own (s_i = max|x_i| / 127, halves to even) and multiplied with 8-bit
           weights that have a scale t_j per output channel, for the projections that "targets"
           lists (N x K each, an activation matrix of its own for each).  "square": f is the squared
           ReLU of the FFN key.  "x": "ln" activations as they leave a LayerNorm and token shift
           (some channels much larger than others), "relu2" as they leave a squared ReLU.
  beam     the W best continuations of each request's W beams by score + log p, normalised by
           length^alpha; a finished beam stays as the one candidate it is.  "first": the step behind
           the prompt, where only a request's first beam counts.  "banned": share of the vocabulary
           that a grammar or a word list rules out (-inf).
  reorder  the recurrent states (WKV and both token-shift rows, all layers) follow the beams that
           were chosen: the first child of a beam keeps its slot, further ones get a copy in the
           slots of beams without a child.

Sizes: widths 1024 to 4096 (states: 768 to 4096) with heads of 64 and any odd projection, 1 to 2304
rows; 1 to 64 requests of 1 to 16 beams; vocabularies of 1000 to 131072.
"""
import math

import torch

own = False

HEAD = 64
NEG = -math.inf


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # One user, one token: the time mix's three projections; launch latency counts.
        {"name": "linear 1 row r,k,v", "kind": "linear", "m": 1, "targets": "2048x2048,2048x2048,2048x2048", "square": False,
         "x": "ln"},
        # A decode batch (16 requests of 8 beams) through the FFN key.
        {"name": "linear 128 rows ffn key", "kind": "linear", "m": 128, "targets": "8192x2048", "square": True, "x": "ln"},
        # Prompt chunks and decode rows as they come, through the down projection.
        {"name": "linear 433 rows value", "kind": "linear", "m": 433, "targets": "2048x8192", "square": False, "x": "relu2"},
        # A projection whose sizes divide by nothing (a pruned or foreign layer), a ragged batch.
        {"name": "linear 77 rows odd", "kind": "linear", "m": 77, "targets": "1003x2501", "square": False, "x": "ln"},
        # A continuous-batching step of the wide model: 256 decode rows and 4 chunks of 512.
        {"name": "linear 2304 rows ffn key", "kind": "linear", "m": 2304, "targets": "16384x4096", "square": True, "x": "ln"},
        # One user, four beams.
        {"name": "beam 1x4", "kind": "beam", "B": 1, "W": 4, "V": 65536, "fp16": True, "alpha": 0.0, "ended": 0.0,
         "first": False, "banned": 0.0},
        # A decode batch, scores by length, some beams finished.
        {"name": "beam 16x8 by length", "kind": "beam", "B": 16, "W": 8, "V": 65536, "fp16": True, "alpha": 0.7, "ended": 0.2,
         "first": False, "banned": 0.0},
        # The largest batch, fp32 logits.
        {"name": "beam 64x8 fp32", "kind": "beam", "B": 64, "W": 8, "V": 65536, "fp16": False, "alpha": 0.0, "ended": 0.0,
         "first": False, "banned": 0.0},
        # A small odd vocabulary with a grammar's mask, many beams, behind the prompt.
        {"name": "beam 5x13 small vocab", "kind": "beam", "B": 5, "W": 13, "V": 5003, "fp16": True, "alpha": 0.0, "ended": 0.0,
         "first": True, "banned": 0.5},
        # One user, four beams of a small model: latency.
        {"name": "reorder 1x4 small", "kind": "reorder", "B": 1, "W": 4, "layers": 12, "H": 12, "skip": 0.0},
        # A few requests of the wide model.
        {"name": "reorder 3x5 wide", "kind": "reorder", "B": 3, "W": 5, "layers": 32, "H": 64, "skip": 0.0},
        # A decode batch of beams; finished beams take no state along.
        {"name": "reorder 16x8", "kind": "reorder", "B": 16, "W": 8, "layers": 24, "H": 32, "skip": 0.1},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choice(("linear", "beam", "reorder"))
    if kind == "linear":
        C = rng.choice((1024, 2048, 2560, 4096))
        shape = rng.choice(("rkv", "o", "key", "value", "odd"))
        targets = {"rkv": ",".join([f"{C}x{C}"] * 3), "o": f"{C}x{C}", "key": f"{4 * C}x{C}", "value": f"{C}x{4 * C}",
                   "odd": f"{_log_int(rng, 20, 20000)}x{_log_int(rng, 20, 12000)}"}[shape]
        return {"kind": "linear", "m": _log_int(rng, 1, 2304), "targets": targets, "square": shape == "key",
                "x": "relu2" if shape == "value" else "ln"}
    if kind == "beam":
        return {"kind": "beam", "B": _log_int(rng, 1, 64), "W": rng.choice((1, 2, 3, 4, 5, 8, 12, 16)),
                "V": rng.choice((65536, _log_int(rng, 1000, 131072))), "fp16": rng.random() < 0.7,
                "alpha": rng.choice((0.0, 0.6, 1.0)), "ended": rng.choice((0.0, 0.0, 0.3)), "first": rng.random() < 0.15,
                "banned": rng.choice((0.0, 0.0, 0.5, 0.99))}
    layers, H = rng.choice(((2, 4), (12, 12), (24, 32), (32, 40), (32, 64)))
    return {"kind": "reorder", "B": _log_int(rng, 1, 32), "W": rng.choice((2, 3, 4, 5, 8, 12)), "layers": layers, "H": H,
            "skip": rng.choice((0.0, 0.1, 0.5))}


def draw(rng):
    """One more case, no larger than the largest listed one of its kind."""
    most = {}
    for c in listed():
        most[c["kind"]] = max(most.get(c["kind"], 0), _size(c))
    while True:
        c = _draw(rng)
        if _size(c) <= most[c["kind"]]:
            return c


def _size(case):
    if case["kind"] == "linear":
        return work(case)["flops"]
    if case["kind"] == "beam":
        return case["B"] * case["W"] * case["V"] * (2 if case["fp16"] else 4)
    return case["B"] * case["W"] * case["layers"] * case["H"]


# ---------------------------------------------------------------- projections with 8-bit weights

def _targets(case):
    return [tuple(int(v) for v in t.split("x")) for t in case["targets"].split(",")]


def _prepare_linear(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    m = case["m"]
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    st = {"targets": [], "square": case["square"]}
    for N, K in _targets(case):
        x = torch.relu(rn(m, K)).square() if case["x"] == "relu2" else rn(m, K) * torch.exp(0.6 * rn(K))
        w = 0.02 * rn(N, K) * torch.exp(0.3 * rn(N, 1))
        top = w.abs().amax(1, keepdim=True)
        st["targets"].append({"x": x.half(), "w": torch.round(w * (127.0 / top)).to(torch.int8), "t": (top / 127.0)[:, 0],
                              "y": torch.empty(m, N, dtype=torch.float16, device="cuda")})
    if own:  # what an engine does once: the weights laid out, the launch described, the scratch
        from vkwr_amd import capi
        epi = capi.EPI_RELU_SQUARE if case["square"] else capi.EPI_NONE
        st["calls"] = [capi.linear_i8_problem(t["x"], capi.i8_weight(t.pop("w"), t["t"]), t["y"], epilogue=epi)
                       for t in st["targets"]]
        st["ws"] = torch.empty(capi.linear_i8_workspace_bytes(st["calls"]), dtype=torch.uint8, device="cuda")
    return st


def _run_linear(st):
    if own:
        from vkwr_amd import capi
        capi.linear_i8(st["calls"], st["ws"])
        return [t["y"] for t in st["targets"]]
    for t in st["targets"]:
        x = t["x"].float()
        top = x.abs().amax(1, keepdim=True)
        # in 64 bits: halves are exact there, and nothing else rounds to one
        q = torch.round(x.double() * 127.0 / torch.where(top > 0, top, 1.0).double()).float()
        y = (q @ t["w"].float().t()) * (top / 127.0) * t["t"]
        if st["square"]:
            y = torch.clamp(y, min=0.0).square()
        t["y"].copy_(y)
    return [t["y"] for t in st["targets"]]


def _exact_linear(case, seed):
    out = []
    st = _prepare_plain(case, seed)
    for t in st["targets"]:
        x = t["x"].double()
        y = torch.empty(x.shape[0], t["w"].shape[0], dtype=torch.float64, device="cuda")
        w = t["w"].double() * t["t"].double()[:, None]
        for r in range(0, x.shape[0], 512):
            rows = x[r:r + 512]
            step = rows.abs().max(dim=1).values[:, None]
            step[step == 0] = 1.0
            levels = (127.0 * rows / step).round()  # 127 x is exact, so a quotient that ends in .5 is too
            y[r:r + 512] = torch.mm(levels, w.t()) * (step / 127.0)
        out.append(torch.where(y > 0, y * y, torch.zeros_like(y)) if case["square"] else y)
    return out


def _prepare_plain(case, seed):
    """The inputs as the plain form has them."""
    global own
    was, own = own, False
    try:
        return _PREPARE[case["kind"]](case, seed)
    finally:
        own = was


def _work_linear(case):
    m = case["m"]
    b = f = 0
    for N, K in _targets(case):
        b += 2 * m * K + N * K + 4 * N + 2 * m * N
        f += 2 * m * N * K
    return {"bytes": b, "flops": f}


# ---------------------------------------------------------------- one step of beam search

def _prepare_beam(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, W, V = case["B"], case["W"], case["V"]
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    rand = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    # a language model's rows: a broad floor with a handful of likely tokens, which the beams of a
    # request share in part
    logits = 1.5 * rn(B, W, V)
    both = torch.randint(0, V, (B, 1, 6), generator=g, device="cuda").expand(B, W, 6)
    each = torch.randint(0, V, (B, W, 6), generator=g, device="cuda")
    logits.scatter_add_(2, torch.cat([both, each], 2), 6.0 + 3.0 * rn(B, W, 12))
    if case["banned"] > 0:
        logits.masked_fill_(rand(B, 1, V) < case["banned"], NEG)
    logits = logits.half() if case["fp16"] else logits
    scores = -torch.sort(20.0 * rand(B, 1) + 4.0 * rand(B, W), dim=1).values
    ended = (rand(B, W) < case["ended"]).to(torch.int32)
    lengths = torch.randint(1, 200, (B, 1), generator=g, device="cuda", dtype=torch.int32).repeat(1, W)
    lengths = torch.where(ended > 0, (lengths.float() * (0.5 + 0.5 * rand(B, W))).to(torch.int32).clamp_(min=1), lengths)
    if case["first"]:
        logits = logits[:, :1].repeat(1, W, 1)
        scores = torch.where(torch.arange(W, device="cuda") == 0, 0.0, NEG).expand(B, W).contiguous()
        ended, lengths = torch.zeros_like(ended), torch.zeros_like(lengths)
    st = {"logits": logits, "scores": scores, "ended": ended, "lengths": lengths, "end": 0, "alpha": case["alpha"]}
    if own:
        from vkwr_amd import capi
        i32 = lambda: torch.empty(B, W, dtype=torch.int32, device="cuda")  # noqa: E731
        st["out"] = [i32(), i32(), torch.empty(B, W, device="cuda"), i32(), i32()]
        st["ws"] = torch.empty(capi.beam_workspace_bytes(B, W, V), dtype=torch.uint8, device="cuda")
    return st


def _run_beam(st):
    """tokens, parents, scores, lengths, ended, each [B, W]"""
    if own:
        from vkwr_amd import capi
        capi.beam_select(st["logits"], st["scores"], st["lengths"], st["ended"], *st["out"], end=st["end"],
                         length_penalty=st["alpha"], workspace=st["ws"])
        return st["out"]
    # in 64 bits: candidates of different beams are compared across sums over the vocabulary
    l, end = st["logits"].double(), st["end"]
    B, W, V = l.shape
    ended = st["ended"] > 0
    top = l.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), 0.0, top)
    raw = st["scores"].double()[:, :, None] + (l - top - torch.log(torch.exp(l - top).sum(-1, keepdim=True)))
    raw = torch.where(torch.isnan(raw), NEG, raw)  # a row without a token
    stay = torch.where(torch.arange(V, device=l.device) == end, st["scores"].double()[:, :, None], NEG)
    raw = torch.where(ended[:, :, None], stay, raw)
    length = st["lengths"] + (~ended).to(torch.int32)
    rank = raw * torch.pow(length.clamp(min=1).double(), -st["alpha"])[:, :, None]
    best, at = torch.sort(rank.view(B, W * V), dim=1, descending=True, stable=True)
    best, at = best[:, :W], at[:, :W]
    none = best == NEG
    parents = torch.where(none, -1, at // V)
    tokens = torch.where(none, -1, at % V)
    p = parents.clamp(min=0)
    scores = torch.where(none, NEG, torch.gather(raw.view(B, W * V), 1, at))
    lengths = torch.where(none, 0, torch.gather(length, 1, p))
    done = none | torch.gather(ended, 1, p) | (tokens == end)
    return [tokens.to(torch.int32), parents.to(torch.int32), scores.float(), lengths.to(torch.int32), done.to(torch.int32)]


def _exact_beam(case, seed):
    st = _prepare_plain(case, seed)
    B, W, V = st["logits"].shape
    out = [[], [], [], [], []]
    for b in range(B):
        ended, lengths, old = st["ended"][b].tolist(), st["lengths"][b].tolist(), st["scores"][b].double().tolist()
        raw = torch.full((W, V), NEG, dtype=torch.float64, device="cuda")
        for w in range(W):
            if ended[w]:
                raw[w, st["end"]] = old[w]
            elif old[w] > NEG:
                raw[w] = old[w] + torch.log_softmax(st["logits"][b, w].double(), 0)
        grown = [n + (not e) for n, e in zip(lengths, ended)]
        rank = raw * torch.tensor([max(n, 1) ** -case["alpha"] for n in grown], dtype=torch.float64, device="cuda")[:, None]
        rows = [[], [], [], [], []]
        for _ in range(W):
            best = float(rank.max())
            if not best > NEG:
                row = (-1, -1, NEG, 0, 1)
            else:
                i = int((rank.view(-1) == best).nonzero()[0])
                p, v = divmod(i, V)
                row = (v, p, float(raw[p, v]), grown[p], int(bool(ended[p]) or v == st["end"]))
                rank[p, v] = NEG
            for dst, value in zip(rows, row):
                dst.append(value)
        for dst, row in zip(out, rows):
            dst.append(row)
    kinds = (torch.int32, torch.int32, torch.float64, torch.int32, torch.int32)
    return [torch.tensor(o, dtype=k, device="cuda") for o, k in zip(out, kinds)]


def _work_beam(case):
    B, W, V = case["B"], case["W"], case["V"]
    rows = B * (1 if case["first"] else W * (1.0 - case["ended"]))  # beams that are over have no logits to look at
    return {"bytes": int(rows * V * (2 if case["fp16"] else 4)) + 32 * B * W, "flops": int(4 * rows * V)}


# ---------------------------------------------------------------- states behind the beams

def _beam_parents(case, g, dev):
    """Parents as beam search leaves them: better beams have more children."""
    u = torch.rand(case["B"], case["W"], generator=g, device=dev)
    skip = (torch.rand(case["B"], case["W"], generator=g, device=dev) < case["skip"]).to(torch.int32)
    return (case["W"] * u * u).to(torch.int32).clamp_(0, case["W"] - 1), skip


def _prepare_reorder(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, W, L, H = case["B"], case["W"], case["layers"], case["H"]
    n_slots = B * W + 3
    parents, skip = _beam_parents(case, g, "cuda")
    half = lambda: torch.randn(L, n_slots, H * HEAD, generator=g, device="cuda").half()  # noqa: E731
    return {"pools": [0.3 * torch.randn(L, n_slots, H, HEAD, HEAD, generator=g, device="cuda"), half(), half()],
            "slots": torch.randperm(n_slots, generator=g, device="cuda")[:B * W].to(torch.int32).view(B, W),
            "parents": parents, "skip": skip, "out": torch.empty(B, W, dtype=torch.int32, device="cuda")}


def _run_reorder(st):
    """slots of the new beams, and the pools"""
    if own:
        from vkwr_amd import capi
        capi.beam_reorder(st["slots"], st["parents"], st["out"], st["pools"], skip=st["skip"])
        return [st["out"], *st["pools"]]
    slots, parents = st["slots"], st["parents"].long()
    B, W = slots.shape
    at = torch.arange(W, device=slots.device)
    carry = st["skip"] == 0
    child = (parents[:, None, :] == at[None, :, None]) & carry[:, None, :]  # [B, parent, child]
    before = torch.cumsum(child.int(), 2) - child.int()
    keeps = ((before == 0) & child).any(1)                      # the first carrying child of its parent
    free = ~child.any(2)                                        # beams whose slot is left over
    nth_free = torch.sort((~free).int(), dim=1, stable=True).indices
    nth = torch.cumsum((~keeps).int(), 1) - 1                   # of the children that take such a slot
    own_slot = torch.gather(slots, 1, parents)
    new = torch.where(keeps, own_slot, torch.gather(slots, 1, torch.gather(nth_free, 1, nth.clamp(min=0))))
    src = torch.where(carry, own_slot, new).view(-1).long()
    dst = new.view(-1).long()
    for pool in st["pools"]:
        pool.index_copy_(1, dst, pool.index_select(1, src))
    st["out"].copy_(new)
    return [st["out"], *st["pools"]]


def _exact_reorder(case, seed):
    st = _prepare_plain(case, seed)
    new, moves = [], []
    for slots, parents, skip in zip(st["slots"].tolist(), st["parents"].tolist(), st["skip"].tolist()):
        kept = {}
        for child, (p, s) in enumerate(zip(parents, skip)):
            if not s:
                kept.setdefault(p, child)
        left = [slots[p] for p in range(len(slots)) if p not in kept]
        row = []
        for child, (p, s) in enumerate(zip(parents, skip)):
            if not s and kept[p] == child:
                row.append(slots[p])
                continue
            row.append(left.pop(0))
            if not s:
                moves.append((slots[p], row[-1]))
        new.append(row)
    for pool in st["pools"]:
        for src, dst in moves:
            pool[:, dst] = pool[:, src]
    return [torch.tensor(new, dtype=torch.int32, device="cuda"), *[pool.double() for pool in st["pools"]]]


def _work_reorder(case):
    parents, skip = _beam_parents(case, torch.Generator().manual_seed(0), "cpu")
    copies = 0
    for p, s in zip(parents.tolist(), skip.tolist()):
        carried = [i for i, x in zip(p, s) if not x]
        copies += len(carried) - len(set(carried))
    C = case["H"] * HEAD
    return {"bytes": 2 * copies * case["layers"] * (4 * C * HEAD + 4 * C) + 16 * case["B"] * case["W"], "flops": 0}


# ---------------------------------------------------------------- by kind

_PREPARE = {"linear": _prepare_linear, "beam": _prepare_beam, "reorder": _prepare_reorder}
_RUN = {"linear": _run_linear, "beam": _run_beam, "reorder": _run_reorder}
_EXACT = {"linear": _exact_linear, "beam": _exact_beam, "reorder": _exact_reorder}
_WORK = {"linear": _work_linear, "beam": _work_beam, "reorder": _work_reorder}


def prepare(case, seed):
    st = _PREPARE[case["kind"]](case, seed)
    st["kind"] = case["kind"]
    return st


def run(state):
    return _RUN[state["kind"]](state)


def exact(case, seed):
    return _EXACT[case["kind"]](case, seed)


def work(case):
    return _WORK[case["kind"]](case)
