"""WKV-7 over drafted tokens (capi.wkv_drafts_slots) against the 64-bit recurrence, and bit for bit
against the decode steps that it stands for."""
import pytest
import torch

from oracle import serving_ref as ref
from vkwr_amd import capi

HALF16 = 2.0 ** -11  # half a step of fp16, relative


def tokens(n_rows, n, H, gen, spread=1.0):
    C = H * 64
    rn = lambda: torch.randn(n_rows, n, C, generator=gen)  # noqa: E731
    kk = torch.nn.functional.normalize(torch.randn(n_rows, n, H, 64, generator=gen), dim=-1).view(n_rows, n, C)
    return {"r": rn().half(), "w": (2 * rn() - 1).half(), "k": (0.5 * spread * rn()).half(), "v": (spread * rn()).half(),
            "a": (-kk).half(), "b": (kk * torch.sigmoid(rn())).half()}


def make(B, P, T, H, seed, n_slots=None, n_pending=None, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    n_slots = n_slots or B + 3
    return {"pool": 0.3 * spread * torch.randn(n_slots, H, 64, 64, generator=g),
            "slots": torch.randperm(n_slots, generator=g)[:B].to(torch.int32),
            "kept": torch.randint(0, P + 1, (B,), generator=g, dtype=torch.int32) if P else None,
            "pending": tokens(n_pending or B, P, H, g, spread), "new": tokens(B, T, H, g, spread)}


def run(gpu, B, P, T, H, d, pending_rows=None, pool=None):
    C = H * 64
    pool = d["pool"].to(gpu) if pool is None else pool
    y = torch.full((B, T, C), 7.0, dtype=torch.float16, device=gpu)
    new = [d["new"][n].to(gpu) for n in "rwkvab"]
    pend = tuple(d["pending"][n].to(gpu) for n in "wkvab") if P else None
    capi.wkv_drafts_slots(B, T, C, H, pool, d["slots"].to(gpu), *new, y,
                          kept=d["kept"].to(gpu) if P else None, pending=pend,
                          pending_rows=None if pending_rows is None else pending_rows.to(gpu))
    return y, pool


@pytest.mark.gpu
@pytest.mark.parametrize("B,P,T,H", [(1, 0, 1, 1), (1, 5, 5, 2), (3, 4, 1, 3), (2, 16, 17, 1), (2, 1, 16, 2), (5, 3, 0, 2),
                                     (2, 37, 20, 1), (1, 0, 33, 1)])
def test_against_64_bits(gpu, B, P, T, H):
    d = make(B, P, T, H, seed=B + 10 * P + 100 * T)
    y, pool = run(gpu, B, P, T, H, d)
    ry, ey, rp, ep = ref.wkv_drafts(d["pool"], d["slots"], d["kept"], d["pending"], None, d["new"], H)
    assert ((pool.cpu().double() - rp).abs() <= ep).all()
    assert ((y.cpu().double() - ry).abs() <= ey + HALF16 * (ry.abs() + ey) + 2.0 ** -25).all()


@pytest.mark.gpu
@pytest.mark.parametrize("B,P,T,H", [(2, 4, 5, 2), (9, 3, 4, 32), (70, 5, 5, 16), (150, 2, 3, 8), (3, 20, 21, 40)])
def test_bits_of_single_steps(gpu, B, P, T, H):
    """kept tokens, then drafts: the bits of as many single decode steps, at batches on every split."""
    C = H * 64
    d = make(B, P, T, H, seed=3 * B + T)
    y, pool = run(gpu, B, P, T, H, d)
    want = d["pool"].to(gpu)
    dummy = torch.empty(1, C, dtype=torch.float16, device=gpu)
    for i in range(B):
        one = d["slots"][i:i + 1].to(gpu)
        seq = [("pending", t) for t in range(int(d["kept"][i]))] + [("new", t) for t in range(T)]
        for n, (src, t) in enumerate(seq):
            if src == "new" and t == 0:
                saved = want[int(d["slots"][i])].clone()
            out = y.new_empty(1, C) if src == "new" else dummy
            r = d["new"]["r"][i:i + 1, min(t, T - 1)]
            v = [d[src][c][i:i + 1, t].contiguous().to(gpu) for c in "wkvab"]
            capi.wkv_step_rows_slots(1, C, H, want, one, r.contiguous().to(gpu), *v, out)
            if src == "new":
                assert torch.equal(out[0], y[i, t]), (i, t)
        if T:
            want[int(d["slots"][i])] = saved
    assert torch.equal(want, pool)


@pytest.mark.gpu
def test_pending_rows_and_repeated_steps(gpu):
    """Three steps of a loop whose batch changes its order: the state of the tokens kept so far."""
    B, T, H = 6, 4, 2
    d = make(B, T, T, H, seed=5, n_slots=9)
    pool = d["pool"].to(gpu)
    run(gpu, B, 0, T, H, d, pool=pool)
    assert torch.equal(pool.cpu(), d["pool"])  # drafts alone leave the pool
    rows = torch.tensor([3, 0, 5, 1, 4, 2], dtype=torch.int32)
    e = make(B, T, T, H, seed=6, n_slots=9)
    e["pending"], e["slots"] = d["new"], d["slots"][rows.long()]
    y, pool = run(gpu, B, T, T, H, e, pending_rows=rows, pool=pool)
    ry, ey, rp, ep = ref.wkv_drafts(d["pool"], e["slots"], e["kept"], e["pending"], rows, e["new"], H)
    assert ((pool.cpu().double() - rp).abs() <= ep).all()
    assert ((y.cpu().double() - ry).abs() <= ey + HALF16 * (ry.abs() + ey) + 2.0 ** -25).all()


@pytest.mark.gpu
def test_bad_entries_give_nan_and_leave_the_pool(gpu):
    B, P, T, H = 6, 2, 3, 2
    d = make(B, P, T, H, seed=8)
    n = d["pool"].shape[0]
    d["slots"][0], d["slots"][1] = -1, n
    d["kept"][:] = 1
    d["kept"][2], d["kept"][3] = -1, P + 1
    rows = torch.tensor([0, 1, 2, 3, B, 5], dtype=torch.int32)
    y, pool = run(gpu, B, P, T, H, d, pending_rows=rows)
    assert torch.isnan(y[:5]).all() and not torch.isnan(y[5]).any()
    same = torch.ones(n, dtype=torch.bool)
    same[int(d["slots"][5])] = False
    assert torch.equal(pool.cpu()[same], d["pool"][same])
    assert not torch.equal(pool.cpu()[~same], d["pool"][~same])


@pytest.mark.gpu
def test_large_state_and_nan_stay_in_their_sequence(gpu):
    B, P, T, H = 3, 2, 2, 2
    d = make(B, P, T, H, seed=9)
    d["kept"][:] = P
    clean, _ = run(gpu, B, P, T, H, d)
    d["new"]["k"][1] = float("nan")
    d["pending"]["v"][1] = float("inf")
    y, pool = run(gpu, B, P, T, H, d)
    assert torch.equal(y[[0, 2]], clean[[0, 2]]) and not torch.isfinite(y[1]).all()


@pytest.mark.gpu
def test_graph_replays_and_another_stream(gpu):
    B, P, T, H = 4, 3, 4, 4
    C = H * 64
    d = make(B, P, T, H, seed=11)
    want_y, want_pool = run(gpu, B, P, T, H, d)
    want2_y, want2_pool = run(gpu, B, P, T, H, d, pool=want_pool.clone())
    pool, y = d["pool"].to(gpu), torch.empty(B, T, C, dtype=torch.float16, device=gpu)
    new = [d["new"][n].to(gpu) for n in "rwkvab"]
    pend = tuple(d["pending"][n].to(gpu) for n in "wkvab")
    slots, kept = d["slots"].to(gpu), d["kept"].to(gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        capi.wkv_drafts_slots(B, T, C, H, pool, slots, *new, y, kept=kept, pending=pend)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want_y) and torch.equal(pool, want_pool)
    y.fill_(1.0)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want2_y) and torch.equal(pool, want2_pool)
    with torch.cuda.stream(side):
        p2 = d["pool"].to(gpu)
        y2, p2 = run(gpu, B, P, T, H, d, pool=p2)
    side.synchronize()
    assert torch.equal(y2, want_y) and torch.equal(p2, want_pool)


@pytest.mark.gpu
def test_pool_past_32_bits(gpu):
    """Slots on either side of the pool's 2^31st entry."""
    B, P, T, H = 2, 2, 2, 64
    d = make(B, P, T, H, seed=5, n_slots=2)
    y, pool = run(gpu, B, P, T, H, d)
    big = torch.zeros(8400, H, 64, 64, device=gpu)
    at = [8191, 8399]
    big[at] = d["pool"].to(gpu)
    e = {**d, "slots": torch.tensor([at[i] for i in d["slots"].tolist()], dtype=torch.int32)}
    y2, _ = run(gpu, B, P, T, H, e, pool=big)
    assert torch.equal(y, y2) and torch.equal(big[at], pool) and not big[:8191].any() and not big[8192:8399].any()
