"""Serving operators as measurable cases: adapters of many requests, verification of drafted
tokens, and the WKV-7 recurrence over drafted tokens.

A case is a dict of plain values; `prepare` makes its inputs on the GPU from a seed, `run`
makes one pass over them, `work` states the bytes and operations that the pass cannot do
without and `exact` computes the same outputs in 64 bits.  `listed` holds the named cases,
`draw` gives further ones of the same ranges.  With `own` False, `run` computes the operators
from elementary torch operations; with `own` True it calls the package's entry points.

Kinds of work (field "kind"):

  lora    y = epilogue(base + scale (x A^T) B^T) with A, B and scale of each row's own adapter,
          for the projections of a layer that read rows of a step: `names` lists them
          (r, k, v, o: [C, C]; key: [4C, C] with the squared ReLU; value: [C, 4C]).  Decode
          batches have one row per request, prefill chunks runs of rows of one request; some
          requests have no adapter.  The plan (rows ordered by adapter) is made in the pass.
  verify  drafted tokens against the target's logits: probabilities under temperature / top-k /
          top-p, the accept test of each draft, and the token after the last accepted one,
          drawn from what the target has beyond the drafter (or from the target itself where
          all are accepted).  "probs" False: the drafter proposes single tokens (looked up in
          the prompt), True: it gives its distribution.
  wkv     the WKV-7 recurrence of a step with drafts: the state of each sequence takes the
          tokens that the step before kept, and the drafts run on from it without being
          written.  T = 0 only writes the kept tokens, P = 0 only runs drafts.

Sizes: widths 1024 to 4096 (recurrence: 768 to 4096) with heads of 64, ranks 8 to 64, 1 to 64 adapters, 1 to 2304 rows;
1 to 128 sequences with 1 to 8 drafts; vocabularies of 1000 to 131072.
"""
import math

import torch

own = False

HEAD = 64
FLT_MAX = torch.finfo(torch.float32).max


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # A few users, each with a fine-tuned variant, one token each: launch latency counts.
        {"name": "lora 5 rows 5 adapters", "kind": "lora", "decode": 5, "chunks": "", "C": 2048, "R": 16, "G": 8,
         "names": "r,k,v", "plain_share": 0.0},
        # A full decode batch over popular and rare adapters, a quarter of it on the base model.
        {"name": "lora 128 rows ffn key", "kind": "lora", "decode": 128, "chunks": "", "C": 2048, "R": 32, "G": 40,
         "names": "key", "plain_share": 0.25},
        # One layer of a continuous-batching step of the wide model: decode rows and prompt chunks.
        {"name": "lora mixed 256 + 4x512", "kind": "lora", "decode": 256, "chunks": "512,512,512,512", "C": 4096, "R": 64,
         "G": 32, "names": "r,k,v,o", "plain_share": 0.1},
        # Prompt chunks as they come, odd lengths, small rank, through the down projection.
        {"name": "lora chunks 333 + 90 value", "kind": "lora", "decode": 11, "chunks": "333,90", "C": 2048, "R": 8, "G": 16,
         "names": "value", "plain_share": 0.0},
        # One user, drafts looked up in the prompt, the model's own distribution.
        {"name": "verify 1 seq lookup", "kind": "verify", "B": 1, "K": 4, "V": 65536, "fp16": True, "probs": False,
         "temperature": 1.0, "top_k": -1, "top_p": 1.0},
        # A decode batch with drafts of a small model and the usual truncation.
        {"name": "verify 24 seqs truncated", "kind": "verify", "B": 24, "K": 5, "V": 65536, "fp16": True, "probs": True,
         "temperature": 0.8, "top_k": 40, "top_p": 0.9},
        # The largest batch, a drafter's distribution, fp32 logits, nucleus only.
        {"name": "verify 128 seqs nucleus", "kind": "verify", "B": 128, "K": 4, "V": 65536, "fp16": False, "probs": True,
         "temperature": 1.0, "top_k": -1, "top_p": 0.95},
        # A small odd vocabulary (a multiple of 4, as the samplers take), ragged draft lengths.
        {"name": "verify 37 seqs small vocab", "kind": "verify", "B": 37, "K": 7, "V": 20004, "fp16": True, "probs": False,
         "temperature": 1.3, "top_k": 200, "top_p": 1.0},
        # One user: 4 drafts behind the token, up to 5 kept of the step before.
        {"name": "wkv 1 seq 5 + 5", "kind": "wkv", "B": 1, "H": 32, "P": 5, "T": 5},
        # A moderate batch, short drafts.
        {"name": "wkv 24 seqs 3 + 3", "kind": "wkv", "B": 24, "H": 32, "P": 3, "T": 3},
        # A full batch of the wide model.
        {"name": "wkv 128 seqs 5 + 5", "kind": "wkv", "B": 128, "H": 64, "P": 5, "T": 5},
        # Kept tokens written before the sequences go on elsewhere (a plain decode step, a copy).
        {"name": "wkv 37 seqs write 7", "kind": "wkv", "B": 37, "H": 40, "P": 7, "T": 0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choice(("lora", "verify", "wkv"))
    if kind == "lora":
        decode = _log_int(rng, 1, 256)
        chunks = [str(_log_int(rng, 2, 512)) for _ in range(rng.choice((0, 0, 1, 2, 4)))]
        return {"kind": "lora", "decode": decode, "chunks": ",".join(chunks), "C": rng.choice((1024, 2048, 2560, 4096)),
                "R": rng.choice((8, 16, 24, 32, 64)), "G": _log_int(rng, 1, 64),
                "names": rng.choice(("r", "r,k,v", "r,k,v,o", "o", "key", "value")),
                "plain_share": rng.choice((0.0, 0.1, 0.3, 0.9))}
    if kind == "verify":
        return {"kind": "verify", "B": _log_int(rng, 1, 128), "K": rng.randint(1, 8),
                "V": rng.choice((65536, 4 * _log_int(rng, 250, 32768))), "fp16": rng.random() < 0.7,
                "probs": rng.random() < 0.5, "temperature": round(rng.uniform(0.3, 1.5), 3),
                "top_k": rng.choice((-1, 1, _log_int(rng, 2, 1000))),
                "top_p": rng.choice((1.0, round(rng.uniform(0.3, 0.99), 3)))}
    P, T = rng.randint(0, 9), rng.randint(0, 9)
    return {"kind": "wkv", "B": _log_int(rng, 1, 128), "H": rng.choice((12, 32, 40, 64)), "P": P, "T": T if P else max(T, 1)}


def draw(rng):
    """One more case, no larger than the largest listed one of its kind."""
    most = {}
    for c in listed():
        most[c["kind"]] = max(most.get(c["kind"], 0), work(c)["bytes"])
    while True:
        c = _draw(rng)
        if work(c)["bytes"] <= most[c["kind"]]:
            return c


# ---------------------------------------------------------------- adapters

def _targets(case):
    """(name, N, K, squared ReLU) of the adapted projections."""
    C = case["C"]
    size = {"key": (4 * C, C, True), "value": (C, 4 * C, False)}
    return [(n, *size.get(n, (C, C, False))) for n in case["names"].split(",")]


def _chunks(case):
    return [int(t) for t in case["chunks"].split(",") if t]


def _lora_rows(case):
    return case["decode"] + sum(_chunks(case))


def _lora_adapters(case, g):
    """Adapter of each row (-1: none): popular adapters come more often; a chunk is one request."""
    G, n = case["G"], case["decode"] + len(_chunks(case))
    u = torch.rand(n, generator=g)
    ids = (G * u * u).to(torch.int32).clamp_(0, G - 1)
    ids[torch.rand(n, generator=g) < case["plain_share"]] = -1
    return torch.repeat_interleave(ids, torch.tensor([1] * case["decode"] + _chunks(case)))


def _prepare_lora(case, seed):
    g = torch.Generator().manual_seed(seed)
    d = torch.Generator(device="cuda").manual_seed(seed + 1)
    m, R, G = _lora_rows(case), case["R"], case["G"]
    rn = lambda *s: torch.randn(*s, generator=d, device="cuda")  # noqa: E731
    st = {"ids": _lora_adapters(case, g).cuda(), "scale": (0.5 + torch.rand(G, generator=g)).cuda(), "targets": []}
    for _, N, K, sq in _targets(case):
        st["targets"].append({
            "x": rn(m, K).half(), "a": (rn(G, R, K) / math.sqrt(K)).half(), "b": (0.3 * rn(G, N, R) / math.sqrt(R)).half(),
            "base": rn(m, N).half(), "y": torch.empty(m, N, dtype=torch.float16, device="cuda"), "sq": sq})
    if own:  # what an engine allocates and describes once: the plan's buffer, the targets, the scratch
        from vkwr_amd import capi
        st["plan"] = capi.lora_plan_empty(m, G, "cuda")
        st["calls"] = [capi.lora_target(t["x"], t["a"], t["b"], t["y"], base=t["base"],
                                        epilogue=capi.EPI_RELU_SQUARE if t["sq"] else capi.EPI_NONE)
                       for t in st["targets"]]
        st["ws"] = torch.empty(capi.lora_workspace_bytes(m, G, st["calls"]), dtype=torch.uint8, device="cuda")
    return st


def _run_lora(st):
    if own:
        from vkwr_amd import capi
        capi.lora_plan(st["ids"], st["plan"])
        capi.lora(st["plan"], st["calls"], scale=st["scale"], workspace=st["ws"])
        return [t["y"] for t in st["targets"]]
    out = []
    G = st["scale"].shape[0]
    # every adapter's product for every row, the other adapters' columns masked out
    mine = (st["ids"][:, None] == torch.arange(G, device="cuda", dtype=torch.int32)).float() * st["scale"]
    for t in st["targets"]:
        R, K = t["a"].shape[1:]
        h = (t["x"].float() @ t["a"].float().reshape(G * R, K).t()).view(-1, G, R) * mine[:, :, None]
        y = t["base"].float() + h.view(-1, G * R) @ t["b"].float().transpose(1, 2).reshape(G * R, -1)
        if t["sq"]:
            y = torch.clamp(y, min=0.0).square()
        t["y"].copy_(y)
        out.append(t["y"])
    return out


def _exact_lora(case, seed):
    st = _prepare_lora(case, seed)
    out = []
    for t in st["targets"]:
        y = t["base"].double()
        for a in sorted(set(st["ids"].tolist()) - {-1}):
            rows = (st["ids"] == a).nonzero()[:, 0]
            h = t["x"][rows].double() @ t["a"][a].double().t()
            y[rows] += float(st["scale"][a]) * (h @ t["b"][a].double().t())
        out.append(torch.where(y > 0, y * y, torch.zeros_like(y)) if t["sq"] else y)
    return out


def _work_lora(case):
    m, R = _lora_rows(case), case["R"]
    ids = _lora_adapters(case, torch.Generator().manual_seed(0))
    used = len(set(ids.tolist()) - {-1})
    rows = int((ids >= 0).sum())
    b = f = 0
    for _, N, K, _ in _targets(case):
        b += 2 * (rows * K + 2 * m * N + used * R * (N + K))
        f += 2 * rows * R * (N + K)
    return {"bytes": b, "flops": f}


# ---------------------------------------------------------------- verification

def _prepare_verify(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, K, V = case["B"], case["K"], case["V"]
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    # a language model's rows: a broad floor with a handful of likely tokens
    logits = 1.5 * rn(B, K + 1, V)
    top = torch.randint(0, V, (B, K + 1, 12), generator=g, device="cuda")
    logits.scatter_add_(2, top, 6.0 + 3.0 * rn(B, K + 1, 12))
    logits = logits.half() if case["fp16"] else logits
    # the drafter: the same rows, disturbed
    q = torch.softmax((logits[:, :K].float() + 0.7 * rn(B, K, V)) / case["temperature"], dim=-1)
    drafts = torch.multinomial(q.reshape(B * K, V), 1, generator=g).view(B, K).to(torch.int32)
    n_draft = torch.randint(0, K + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    n_draft = torch.where(torch.rand(B, generator=g, device="cuda") < 0.7, K, n_draft).to(torch.int32)
    st = {"logits": logits, "drafts": drafts, "n_draft": n_draft, "q": q if case["probs"] else None,
          "u": torch.rand(B, K + 1, generator=g, device="cuda"),
          "temperature": case["temperature"], "top_k": case["top_k"], "top_p": case["top_p"]}
    if own:
        from vkwr_amd import capi
        st["tokens"] = torch.empty(B, K + 1, dtype=torch.int32, device="cuda")
        st["accepted"] = torch.empty(B, dtype=torch.int32, device="cuda")
        st["ws"] = torch.empty(capi.verify_workspace_bytes(B, K, V), dtype=torch.uint8, device="cuda")
    return st


def _run_verify(st):
    if own:
        from vkwr_amd import capi
        capi.verify_drafts(st["logits"], st["drafts"], st["u"], st["tokens"], st["accepted"], n_draft=st["n_draft"],
                           draft_probs=st["q"], temperature=st["temperature"], top_k=st["top_k"], top_p=st["top_p"],
                           workspace=st["ws"])
        return [st["tokens"], st["accepted"]]
    # in 64 bits throughout: accept tests and draws sit next to borders of sums over the vocabulary
    logits, drafts, q = st["logits"], st["drafts"].long(), st["q"]
    B, T, V = logits.shape
    K = T - 1
    dev = logits.device
    top_k = st["top_k"] if 0 < st["top_k"] <= V else V
    l = logits.double()
    x = torch.exp((l - l.amax(-1, keepdim=True)) / st["temperature"])
    if top_k < V or st["top_p"] < 1.0:
        ls, _ = torch.sort(l, dim=-1, descending=True)
        cum = torch.cumsum(torch.exp((ls - ls[..., :1]) / st["temperature"]), dim=-1)
        enough = torch.arange(1, V + 1, device=dev) >= top_k
        goal = st["top_p"] * cum[..., -1:]
        if st["top_p"] < 1.0:
            enough = enough | (cum >= goal)
        at = enough.expand(B, T, V).to(torch.int8).argmax(-1, keepdim=True)
        tau = torch.gather(ls, -1, at)
        eq = l == tau
        n_gt, n_eq = (l > tau).sum(-1, keepdim=True), eq.sum(-1, keepdim=True)
        comp = (top_k - n_gt).double() / n_eq
        if st["top_p"] < 1.0:
            m_gt = torch.where(l > tau, x, 0.0).sum(-1, keepdim=True)
            x_tau = torch.exp((tau - ls[..., :1]) / st["temperature"])
            comp = torch.minimum(comp, (goal - m_gt) / (x_tau * n_eq))
        x = torch.where(l > tau, x, torch.where(eq, x * comp.clamp(0.0, 1.0), 0.0))
        del ls, cum, eq
    p = x / x.sum(-1, keepdim=True)
    pd = torch.gather(p[:, :K], -1, drafts[..., None])[..., 0]
    qd = torch.ones_like(pd) if q is None else torch.gather(q, -1, drafts[..., None])[..., 0].double()
    pos = torch.arange(K, device=dev)
    ok = (st["u"][:, :K].double() * qd < pd) & (pos < st["n_draft"][:, None])
    accepted = torch.cumprod(ok.long(), dim=1).sum(1)
    rejected = accepted < st["n_draft"]
    row = torch.gather(p, 1, accepted[:, None, None].expand(B, 1, V))[:, 0]
    at = accepted.clamp(max=K - 1)
    if q is None:
        minus = torch.zeros_like(row).scatter_(1, torch.gather(drafts, 1, at[:, None]), 2.0)
    else:
        minus = torch.gather(q, 1, at[:, None, None].expand(B, 1, V))[:, 0].double()
    rest = torch.clamp(row - minus, min=0.0)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0.0, rest, row)
    w = torch.where(rejected[:, None], rest, row)
    cdf = torch.cumsum(w, dim=-1)
    new = (cdf > st["u"][:, K:].double() * cdf[:, -1:]).to(torch.int8).argmax(-1)
    pos = torch.arange(T, device=dev)
    tokens = torch.full((B, T), -1, dtype=torch.long, device=dev)
    tokens[:, :K] = torch.where(pos[:K] < accepted[:, None], drafts, -1)
    tokens.scatter_(1, accepted[:, None], new[:, None])
    return [tokens.to(torch.int32), accepted.to(torch.int32)]


def _exact_row(l, temperature, top_k, top_p):
    """p of one row of logits by the definition, over its distinct values."""
    V = l.numel()
    e = torch.exp((l - l.max()) / temperature)
    if not 0 < top_k <= V:
        top_k = V
    if top_k == V and top_p >= 1.0:
        return e / e.sum()
    vals, inv, cnt = torch.unique(l, return_inverse=True, return_counts=True)
    ev = torch.exp((vals - vals[-1]) / temperature) * cnt
    n_ge = torch.flip(torch.cumsum(torch.flip(cnt, (0,)), 0), (0,))
    m_ge = torch.flip(torch.cumsum(torch.flip(ev, (0,)), 0), (0,))
    goal = top_p * ev.sum()
    big = (n_ge >= top_k) | ((m_ge >= goal) if top_p < 1.0 else torch.zeros_like(n_ge, dtype=torch.bool))
    i = int(big.nonzero()[-1])
    share = float(top_k - (n_ge[i] - cnt[i])) / float(cnt[i])
    if top_p < 1.0:
        share = min(share, float((goal - (m_ge[i] - ev[i])) / ev[i]))
    part = (torch.arange(vals.numel(), device=l.device) > i).double()
    part[i] = min(max(share, 0.0), 1.0)
    e = e * part[inv]
    return e / e.sum()


def _exact_verify(case, seed):
    st = _prepare_verify(case, seed)
    logits, drafts, q, u = st["logits"], st["drafts"].tolist(), st["q"], st["u"].double().tolist()
    B, T, V = logits.shape
    tokens, accepted = [], []
    for b, n in enumerate(st["n_draft"].tolist()):
        out, i = [], 0
        while True:
            p = _exact_row(logits[b, i].double(), st["temperature"], st["top_k"], st["top_p"])
            if i == n:
                break
            d = drafts[b][i]
            if not u[b][i] * (1.0 if q is None else float(q[b, i, d])) < float(p[d]):
                beyond = p.clone()
                if q is None:
                    beyond[d] = 0.0
                else:
                    beyond = torch.clamp(beyond - q[b, i].double(), min=0.0)
                p = beyond if float(beyond.sum()) > 0.0 else p
                break
            out.append(d)
            i += 1
        c = torch.cumsum(p, 0)
        out.append(int(torch.searchsorted(c, (u[b][T - 1] * c[-1]).reshape(1), right=True)[0]))
        tokens.append(out + [-1] * (T - len(out)))
        accepted.append(i)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return [i32(tokens), i32(accepted)]


def _work_verify(case):
    B, T, V = case["B"], case["K"] + 1, case["V"]
    rows = B * (0.85 * case["K"] + 1)  # behind a short draft there are no rows to look at
    b = int(rows * V) * (2 if case["fp16"] else 4) + 4 * B * (4 * T + 2)
    if case["probs"]:
        b += B * V * 4  # the drafter's row at the rejected position
    return {"bytes": b, "flops": int(4 * rows * V)}


# ---------------------------------------------------------------- the recurrence over drafts

def _prepare_wkv(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, H, P, T = case["B"], case["H"], case["P"], case["T"]
    C, n_slots = H * HEAD, B + B // 2 + 2
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731

    def tokens(n):
        kk = torch.nn.functional.normalize(rn(B, n, H, HEAD), dim=-1).view(B, n, C)
        lr = torch.sigmoid(rn(B, n, C))
        return {"r": rn(B, n, C).half(), "w": (2.0 * rn(B, n, C) - 1.0).half(), "k": (0.5 * rn(B, n, C)).half(),
                "v": rn(B, n, C).half(), "a": (-kk).half(), "b": (kk * lr).half()}

    st = {"pool": 0.3 * rn(n_slots, H, HEAD, HEAD),
          "slots": torch.randperm(n_slots, generator=g, device="cuda")[:B].to(torch.int32),
          "kept": torch.randint(1, P + 1, (B,), generator=g, device="cuda", dtype=torch.int32) if P else None,
          "pending": tokens(P), "new": tokens(T), "B": B, "H": H, "P": P, "T": T, "C": C,
          "y": torch.empty(B, T, C, dtype=torch.float16, device="cuda")}
    return st


def _run_wkv(st):
    B, H, P, T, C = (st[k] for k in "BHPTC")
    pend, new, y = st["pending"], st["new"], st["y"]
    if own:
        from vkwr_amd import capi
        capi.wkv_drafts_slots(B, T, C, H, st["pool"], st["slots"], new["r"], new["w"], new["k"], new["v"], new["a"], new["b"],
                              y, kept=st["kept"],
                              pending=(pend["w"], pend["k"], pend["v"], pend["a"], pend["b"]) if P else None)
        return [y, st["pool"]] if T else [st["pool"]]
    slots = st["slots"].long()
    S = st["pool"][slots]

    def token(S, src, t):
        w, k, v, a, b = (src[n][:, t].float().view(B, H, HEAD) for n in ("w", "k", "v", "a", "b"))
        d = torch.exp(-math.exp(-0.5) * torch.sigmoid(w))
        sa = (S * a[:, :, None, :]).sum(-1)
        return S * d[:, :, None, :] + sa[..., None] * b[:, :, None, :] + v[..., None] * k[:, :, None, :]

    for t in range(P):
        S = torch.where((t < st["kept"])[:, None, None, None], token(S, pend, t), S)
    if P:
        st["pool"][slots] = S
    for t in range(T):
        S = token(S, new, t)
        y[:, t] = (S * new["r"][:, t].float().view(B, H, 1, HEAD)).sum(-1).view(B, C)
    return [y, st["pool"]] if T else [st["pool"]]


def _exact_wkv(case, seed):
    st = _prepare_wkv(case, seed)
    B, H, P, T, C = (st[k] for k in "BHPTC")
    pool = st["pool"].double()
    ys = []
    S = pool.index_select(0, st["slots"].long()).view(B * H, HEAD, HEAD)

    def vec(src, n, t):
        return src[n][:, t].double().reshape(B * H, HEAD)

    def step(S, src, t):
        d = torch.exp(-torch.sigmoid(vec(src, "w", t)) / math.sqrt(math.e))
        change = torch.bmm(torch.bmm(S, vec(src, "a", t)[:, :, None]), vec(src, "b", t)[:, None, :])
        return S * d[:, None, :] + change + torch.bmm(vec(src, "v", t)[:, :, None], vec(src, "k", t)[:, None, :])

    for t in range(P):
        live = (st["kept"] > t).repeat_interleave(H)
        S[live] = step(S, st["pending"], t)[live]
    if P:
        pool.index_copy_(0, st["slots"].long(), S.view(B, H, HEAD, HEAD))
    for t in range(T):
        S = step(S, st["new"], t)
        ys.append(torch.bmm(S, vec(st["new"], "r", t)[:, :, None]).view(B, C))
    return [torch.stack(ys, 1), pool] if T else [pool]


def _work_wkv(case):
    B, H, P, T = case["B"], case["H"], case["P"], case["T"]
    C, states = H * HEAD, 4 * B * H * HEAD * HEAD
    kept = (P + 1) / 2  # tokens kept of P, on average
    return {"bytes": int(states * (2 if P else 1) + 2 * B * C * (5 * kept * (P > 0) + 7 * T)),
            "flops": int(B * H * HEAD * HEAD * (7 * kept * (P > 0) + 9 * T))}


# ---------------------------------------------------------------- by kind

_PREPARE = {"lora": _prepare_lora, "verify": _prepare_verify, "wkv": _prepare_wkv}
_RUN = {"lora": _run_lora, "verify": _run_verify, "wkv": _run_wkv}
_EXACT = {"lora": _exact_lora, "verify": _exact_verify, "wkv": _exact_wkv}
_WORK = {"lora": _work_lora, "verify": _work_verify, "wkv": _work_wkv}


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
