"""Adapters of many requests (capi.lora) against the 64-bit oracle."""
import math

import pytest
import torch

from oracle import serving_ref as ref
from vkwr_amd import capi

HALF16 = 2.0 ** -11


def make(m, G, R, sizes, seed, none=0.2, run=1, scale=True):
    """sizes: (N, K) per target; run: rows of one request in a row."""
    g = torch.Generator().manual_seed(seed)
    n = -(-m // run)
    ids = torch.randint(0, G, (n,), generator=g, dtype=torch.int32)
    ids[torch.rand(n, generator=g) < none] = -1
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return {"ids": ids.repeat_interleave(run)[:m].contiguous(), "scale": 0.5 + torch.rand(G, generator=g) if scale else None,
            "t": [{"x": rn(m, K).half(), "a": (rn(G, R, K) / math.sqrt(K)).half(), "b": (0.3 * rn(G, N, R)).half(),
                   "base": rn(m, N).half()} for N, K in sizes]}


def run_lora(gpu, d, epilogue=capi.EPI_NONE, inplace=False):
    m, G = d["ids"].numel(), d["t"][0]["a"].shape[0]
    plan = capi.lora_plan_empty(m, G, gpu)
    capi.lora_plan(d["ids"].to(gpu), plan)
    ts, ys = [], []
    for t in d["t"]:
        base = t["base"].to(gpu)
        y = base if inplace else torch.full_like(base, 9.0)
        ts.append(capi.lora_target(t["x"].to(gpu), t["a"].to(gpu), t["b"].to(gpu), y, base=None if inplace else base,
                                   epilogue=epilogue))
        ys.append(y)
    ws = torch.full((capi.lora_workspace_bytes(m, G, ts),), 255, dtype=torch.uint8, device=gpu)  # NaN where unwritten
    capi.lora(plan, ts, scale=None if d["scale"] is None else d["scale"].to(gpu), workspace=ws)
    return ys


def check(gpu, d, epilogue=capi.EPI_NONE, inplace=False):
    for y, t in zip(run_lora(gpu, d, epilogue, inplace), d["t"]):
        want, err = ref.lora(t["x"], t["a"], t["b"], t["base"], d["ids"], d["scale"], epilogue == capi.EPI_RELU_SQUARE)
        got = y.cpu().double()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        ok = (got - want).abs() <= err + HALF16 * (want.abs() + err) + 2.0 ** -25
        assert (ok | torch.isnan(want)).all(), float(((got - want).abs() - err).nan_to_num().max())


@pytest.mark.gpu
@pytest.mark.parametrize("m,G,R,N,K", [(1, 1, 8, 8, 8), (1, 3, 16, 256, 256), (5, 8, 16, 264, 40), (17, 4, 24, 72, 1000),
                                       (33, 40, 32, 520, 328), (64, 1, 64, 128, 64), (65, 1, 48, 64, 2048),
                                       (130, 2, 128, 304, 512), (200, 3, 72, 1000, 72), (7, 1000, 40, 96, 136)])
def test_against_64_bits(gpu, m, G, R, N, K):
    check(gpu, make(m, G, R, [(N, K)], seed=m + R))


@pytest.mark.gpu
@pytest.mark.parametrize("epilogue", [capi.EPI_NONE, capi.EPI_RELU_SQUARE])
@pytest.mark.parametrize("inplace", [False, True])
def test_targets_epilogues_and_runs(gpu, epilogue, inplace):
    """Several projections of different sizes at once; prompt chunks as runs of one adapter."""
    check(gpu, make(150, 5, 16, [(256, 128), (64, 320), (1024, 64)], seed=3, run=1), epilogue, inplace)
    check(gpu, make(300, 5, 16, [(256, 128), (64, 320)], seed=4, run=70), epilogue, inplace)
    check(gpu, make(40, 6, 8, [(64, 64)] * 8, seed=5, scale=False), epilogue, inplace)


@pytest.mark.gpu
@pytest.mark.parametrize("none", [0.0, 1.0])
def test_all_or_no_rows_with_adapters(gpu, none):
    for ep in (capi.EPI_NONE, capi.EPI_RELU_SQUARE):
        check(gpu, make(70, 4, 16, [(128, 128)], seed=6, none=none), ep)


@pytest.mark.gpu
def test_indices_out_of_range(gpu):
    d = make(20, 4, 16, [(128, 64)], seed=7)
    d["ids"][3], d["ids"][4], d["ids"][9], d["ids"][11] = 4, 2 ** 31 - 1, -2 ** 31, -5
    check(gpu, d)
    check(gpu, d, capi.EPI_RELU_SQUARE, True)


@pytest.mark.gpu
def test_whole_numbers_are_exact(gpu):
    """Small whole numbers: every sum is exact in fp32 and in fp16, whatever its order and split."""
    g = torch.Generator().manual_seed(1)
    m, G, R, N, K = 100, 7, 32, 192, 256
    ri = lambda lo, hi, *s: torch.randint(lo, hi + 1, s, generator=g).half()  # noqa: E731
    d = {"ids": torch.randint(-1, G, (m,), generator=g, dtype=torch.int32), "scale": None,
         "t": [{"x": ri(-1, 1, m, K) * (torch.rand(m, K, generator=g) < 0.1), "a": ri(-1, 1, G, R, K),
                "b": ri(-1, 1, G, N, R), "base": ri(-8, 8, m, N)}]}
    want, _ = ref.lora(*(d["t"][0][k] for k in ("x", "a", "b", "base")), d["ids"])
    assert want.abs().max() < 2048
    assert torch.equal(run_lora(gpu, d)[0].cpu().double(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [2.0 ** -13, 2.0 ** 9])
def test_inner_values_far_from_one(gpu, size):
    """x A^T beyond fp16's range at either end, brought back by B: the split holds 22 bits of it."""
    d = make(50, 3, 16, [(128, 256)], seed=8, none=0.0, scale=False)
    t = d["t"][0]
    t["x"], t["a"] = (t["x"].float() * size).half(), (t["a"].float() * size * 4).half()
    t["b"] = (t["b"].float() / max(size * size, 2.0 ** -14)).half()
    check(gpu, d)


@pytest.mark.gpu
def test_non_finite_values_stay_in_their_rows(gpu):
    d = make(40, 2, 16, [(128, 64)], seed=9, none=0.0)
    clean = run_lora(gpu, d)[0]
    d["t"][0]["x"][5, 3], d["t"][0]["x"][17, 0] = float("inf"), float("nan")
    y = run_lora(gpu, d)[0]
    rest = torch.ones(40, dtype=torch.bool)
    rest[[5, 17]] = False
    assert torch.equal(y[rest], clean[rest])
    assert not torch.isfinite(y[5]).any() and torch.isnan(y[17]).all()


@pytest.mark.gpu
def test_row_results_do_not_depend_on_the_batch(gpu):
    """A row alone, in a batch and in a run of 200: within one rounding of each other, and the same
    bits in the same batch shape under any order of the rows."""
    d = make(90, 3, 32, [(256, 512)], seed=10, none=0.1)
    y = run_lora(gpu, d)[0]
    perm = torch.randperm(90, generator=torch.Generator().manual_seed(2))
    e = {"ids": d["ids"][perm].contiguous(), "scale": d["scale"],
         "t": [{**d["t"][0], "x": d["t"][0]["x"][perm], "base": d["t"][0]["base"][perm]}]}
    assert torch.equal(run_lora(gpu, e)[0], y[perm.to(gpu)])


@pytest.mark.gpu
def test_graph_replays_with_other_adapters(gpu):
    """A captured plan + projections follow the adapter indices that the buffer holds at replay."""
    d = make(64, 6, 16, [(256, 128), (128, 256)], seed=12)
    ids = d["ids"].to(gpu)
    plan = capi.lora_plan_empty(64, 6, gpu)
    ys = [torch.empty_like(t["base"], device=gpu) for t in d["t"]]
    ts = [capi.lora_target(t["x"].to(gpu), t["a"].to(gpu), t["b"].to(gpu), y, base=t["base"].to(gpu))
          for t, y in zip(d["t"], ys)]
    ws = torch.empty(capi.lora_workspace_bytes(64, 6, ts), dtype=torch.uint8, device=gpu)
    scale = d["scale"].to(gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        capi.lora_plan(ids, plan)
        capi.lora(plan, ts, scale=scale, workspace=ws)
    for seed in (1, 2, 3):
        new = torch.randint(-1, 6, (64,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)
        ids.copy_(new)
        g.replay()
        torch.cuda.synchronize()
        d["ids"] = new
        for y, want in zip(ys, run_lora(gpu, d)):
            assert torch.equal(y, want)


@pytest.mark.gpu
def test_plan_of_many_rows(gpu):
    """Long runs, scattered rows and thousands of adapters in one plan."""
    g = torch.Generator().manual_seed(4)
    ids = torch.cat([torch.full((1500,), 17), torch.randint(-1, 5000, (700,), generator=g), torch.full((333,), 4999),
                     torch.full((129,), -1)]).to(torch.int32)
    m, G, R, N, K = ids.numel(), 5000, 8, 16, 16
    d = {"ids": ids, "scale": None, "t": [{"x": torch.randn(m, K, generator=g).half(),
                                           "a": torch.randn(G, R, K, generator=g).half(),
                                           "b": (0.2 * torch.randn(G, N, R, generator=g)).half(),
                                           "base": torch.randn(m, N, generator=g).half()}]}
    check(gpu, d)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [17, 65, 70, 97, 150])
def test_equal_rows_of_an_adapter_are_equal(gpu, n):
    """The plan puts an adapter's rows into its tiles, the last of which is shorter, in any order: equal rows
    have to get equal bits wherever they are."""
    d = make(n + 40, 3, 16, [(256, 4096), (72, 200)], seed=n)
    d["ids"][:] = 1
    d["ids"][n:] = torch.arange(40, dtype=torch.int32) % 2 * 2
    for t in d["t"]:
        t["x"][:n] = t["x"][0].clone()
    for t in d["t"]:
        t["base"][:] = 0
    for t, y in zip(d["t"], run_lora(gpu, d)):
        t["base"][:n] = -y[0].cpu()  # what is left are the fp32 sums' last bits
    first = None
    for _ in range(3):
        ys = [y.cpu() for y in run_lora(gpu, d)]
        for y in ys:
            assert torch.equal(y[:n], y[:1].expand(n, -1))
        assert first is None or all(torch.equal(a, b) for a, b in zip(first, ys))
        first = ys


@pytest.mark.gpu
def test_offsets_past_32_bits(gpu):
    """The last adapter of pools of more than 2^31 entries."""
    G, R, N, K, m = 300, 128, 65536, 65536, 3
    d = make(m, 1, R, [(N, K)], seed=8, none=0.0)
    t = d["t"][0]
    a = torch.zeros(G, R, K, dtype=torch.float16, device=gpu)
    b = torch.zeros(G, N, R, dtype=torch.float16, device=gpu)
    a[-1], b[-1] = t["a"][0].to(gpu), t["b"][0].to(gpu)
    y = t["base"].to(gpu)
    plan = capi.lora_plan_empty(m, G, gpu)
    capi.lora_plan(torch.full((m,), G - 1, dtype=torch.int32, device=gpu), plan)
    capi.lora(plan, [capi.lora_target(t["x"].to(gpu), a, b, y)])
    want, err = ref.lora(t["x"], t["a"], t["b"], t["base"], torch.zeros(m, dtype=torch.int32), None, False)
    assert ((y.cpu().double() - want).abs() <= err + HALF16 * (want.abs() + err) + 2.0 ** -25).all()


@pytest.mark.gpu
def test_rows_behind_the_plan_are_left(gpu):
    d = make(70, 3, 16, [(264, 72)], seed=9, none=0.3)
    t = d["t"][0]
    x, a, b = t["x"].to(gpu), t["a"].to(gpu), t["b"].to(gpu)
    plan = capi.lora_plan_empty(70, 3, gpu)
    for m in (41, 0, 1):
        y = t["base"].to(gpu)
        capi.lora_plan(d["ids"][:m].to(gpu), plan)
        capi.lora(plan, [capi.lora_target(x, a, b, y)], scale=d["scale"].to(gpu))
        assert torch.equal(y[m:].cpu(), t["base"][m:])
        want, err = ref.lora(t["x"][:m], t["a"], t["b"], t["base"][:m], d["ids"][:m], d["scale"], False)
        assert ((y[:m].cpu().double() - want).abs() <= err + HALF16 * (want.abs() + err) + 2.0 ** -25).all()
