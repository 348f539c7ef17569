"""Linear layers with 8-bit weights where the other tests do not go: scales near the end of fp32's range, rows up to the
largest K, and on the tile kernel many stages, every epilogue, several problems, and rows of zeros, infinities and NaN.

Tolerances as in test_linear_i8_gpu, whose formula in 64 bits is used here; results beyond fp16's range are infinities.
tanh and the sigmoid move by at most 0.45 of their argument's relative error (x / cosh(x)^2 <= 0.45), however large it is.
The sizes of ROUTES reach each kernel and tile on 256 CUs.
"""
import math

import pytest
import torch

from tests.test_linear_i8_gpu import EPI, close, expected, rand, weights
from vkwr_amd import capi

pytestmark = pytest.mark.gpu

# rows and outputs: one, three and eight rows (rounded where they are multiplied); streams of 16 x 16, 16 x 32,
# 32 x 32, 32 x 64, 64 x 64; tiles of 64 x 128, 128 x 128, 128 x 256, 192 x 256, 256 x 256
ROUTES = [(1, 45), (3, 77), (8, 77), (9, 501), (20, 2101), (40, 3005), (70, 3001), (130, 5003)]
TILE_ROUTES = [(250, 5003), (500, 5001), (1000, 5001), (2050, 5001), (2400, 5001)]


def close16(y, ref, tol, what):
    """As close(); where the result lies beyond fp16's largest value an infinity of its sign (either within
    2^-20 of 65520, from which on values round to it)."""
    if what in ("tanh", "sigmoid"):
        tol = torch.minimum(tol, ref.abs() * 2.0 ** -11 + 2.0 ** -25 + 2.0 ** -19)
    far, near = ref.abs() >= 65520.0 * (1 + 2.0 ** -20), ref.abs() < 65520.0 * (1 - 2.0 ** -20)
    want = torch.where(ref > 0, math.inf, -math.inf)
    assert torch.equal(y.cpu().double()[far], want[far]), what
    close(y.cpu()[near], ref[near], tol[near], what)


@pytest.mark.parametrize("epi", sorted(EPI))
@pytest.mark.parametrize("m,n", ROUTES + TILE_ROUTES)
def test_large_weight_scales(m, n, epi):
    """Scaled sums beyond fp32's range, of either sign, and sums of 0 under such a scale."""
    k = 72
    x, (wq, t) = rand(m, k, seed=m).half().cuda(), weights(n, k, seed=n)
    x[0] = 2.0 ** -24  # the smallest activations (q = 127, s = 2^-24 / 127)
    if m > 1:
        x[1] *= 2.0 ** 12  # a row whose scale alone takes the largest scales out of range
    wq[::5] = 0        # sums of 0, or of 1 and -1 times 127
    wq[5::10, 3] = 1
    wq[0::20, 3] = -1
    big = torch.tensor([1.0, -1.0, 2.0 ** 86, -2.0 ** 86, 2.0 ** 87, 1e30, 1e35, -1e36, 3e38, -3e38, 2.0 ** 40])
    t = torch.where(torch.arange(n) % 13 < 11, big[(torch.arange(n) % 13).clamp(max=10)], t)
    wq, t = wq.cuda(), t.cuda()
    bias = rand(n, seed=3).half().cuda() if epi == "bias" else None
    y = torch.empty(m, n, dtype=torch.float16, device="cuda")
    capi.linear_i8([capi.linear_i8_problem(x, capi.i8_weight(wq, t), y, EPI[epi], bias)])
    ref, tol = (v.cpu() for v in expected(x, wq, t, epi, bias))
    assert ref.isfinite().all() and (ref == 0).any() | (epi in ("bias", "sigmoid"))
    close16(y, ref, tol, epi)


# ---------------------------------------------------------------- the tile kernel's other uses

@pytest.mark.parametrize("epi", sorted(EPI))
@pytest.mark.parametrize("m,n", TILE_ROUTES)
def test_many_stages_and_every_epilogue(m, n, epi):
    """22 stages of 64 k, more than three times round a ring of 4 or 6 buffers and no multiple of either."""
    k = 1300
    x, (wq, t) = rand(m, k, seed=m).half().cuda(), weights(n, k, seed=n)
    wq, t = wq.cuda(), t.cuda()
    bias = rand(n, seed=3).half().cuda() if epi == "bias" else None
    out = torch.full((m * n + 64,), 5.0, dtype=torch.float16, device="cuda")
    y = out[:m * n].view(m, n)
    capi.linear_i8([capi.linear_i8_problem(x, capi.i8_weight(wq, t), y, EPI[epi], bias)])
    close(y, *(v.cpu() for v in expected(x, wq, t, epi, bias)), f"{m}x{n} {epi}")
    assert (out[m * n:] == 5).all()


def run_batch(sizes, shared=(0, 0)):
    """One call of problems (m, n, k, epilogue), the two of `shared` on the same activations."""
    ps, want = [], []
    xs = [rand(m, k, seed=i).half().cuda() for i, (m, n, k, epi) in enumerate(sizes)]
    xs[shared[1]] = xs[shared[0]]
    for i, (m, n, k, epi) in enumerate(sizes):
        wq, t = (v.cuda() for v in weights(n, k, seed=50 + i))
        bias = rand(n, seed=90 + i).half().cuda() if epi == "bias" else None
        y = torch.full((m, n), 7.0, dtype=torch.float16, device="cuda")
        ps.append(capi.linear_i8_problem(xs[i], capi.i8_weight(wq, t), y, EPI[epi], bias))
        if m:
            want.append((y, xs[i], wq, t, epi, bias))
    ws = torch.empty(capi.linear_i8_workspace_bytes(ps), dtype=torch.uint8, device="cuda")
    capi.linear_i8(ps, ws)
    for i, (y, *args) in enumerate(want):
        close(y, *(v.cpu() for v in expected(*args)), f"problem {i} of {sizes}")


@pytest.mark.parametrize("m", [300, 700, 1500, 2304])
def test_equal_problems_on_tiles(m):
    """r, k, v of a large step: tiles of 64 x 128, 128 x 256, 192 x 256 and 256 x 256 over three problems."""
    n = {300: 2048, 700: 2100, 1500: 2048, 2304: 4096}[m]
    run_batch([(m, n, 328, "none"), (m, n, 328, "relu2"), (m, n, 328, "sigmoid")])


@pytest.mark.parametrize("rows", [(500, 130, 900), (1000, 1500, 77), (2304, 2304, 2304)])
def test_different_problems_on_tiles(rows):
    """Problems of other sizes and epilogues, one of no rows and two on the same activations."""
    a, b, c = rows
    run_batch([(a, 2051, 200, "none"), (0, 64, 64, "tanh"), (b, 3000, 640, "relu2"), (1, 8, 40, "bias"),
               (a, 1030, 200, "tanh"), (c, 517, 1100, "bias")], shared=(0, 4))


@pytest.mark.parametrize("epi", ["none", "relu2", "bias"])
@pytest.mark.parametrize("m,n", TILE_ROUTES)
def test_zero_and_nonfinite_rows_on_tiles(m, n, epi):
    k = 200
    x, (wq, t) = rand(m, k, seed=4).half(), weights(n, k, seed=5)
    bias = rand(n, seed=6).half().cuda() if epi == "bias" else None
    bad = {1: math.inf, m // 2: math.nan, m - 1: -math.inf}
    x[[0, 33]] = 0.0
    for i, v in bad.items():
        x[i, i % k] = v
    y = torch.empty(m, n, dtype=torch.float16, device="cuda")
    wq, t = wq.cuda(), t.cuda()
    capi.linear_i8([capi.linear_i8_problem(x.cuda(), capi.i8_weight(wq, t), y, EPI[epi], bias)])
    rows = sorted(bad)
    assert y[rows].isnan().all()
    x[rows] = 0.0
    ref, tol = (v.cpu() for v in expected(x.cuda(), wq, t, epi, bias))
    keep = [i for i in range(m) if i not in bad]
    close(y.cpu()[keep], ref[keep], tol[keep], epi)


@pytest.mark.parametrize("m,n", TILE_ROUTES)
def test_largest_values_on_tiles(m, n):
    """All values at 127 over 22 stages: sums that fp32 does not hold exactly."""
    k = 1300
    x = torch.ones(m, k, dtype=torch.float16, device="cuda")
    x[:, 1::2] = -1.0
    x[m // 3] *= -1.0
    wq = torch.full((n, k), 127, dtype=torch.int8, device="cuda")
    wq[:, 1::2] = -127
    wq[5::7, 0] = 126
    t = torch.full((n,), 1.0 / 127 / k, device="cuda")
    y = torch.empty(m, n, dtype=torch.float16, device="cuda")
    capi.linear_i8([capi.linear_i8_problem(x, capi.i8_weight(wq, t), y)])
    close(y, *(v.cpu() for v in expected(x, wq, t, "none", None)), f"{m}")


@pytest.mark.parametrize("m,n,k", [(1, 40, 131072), (1, 40, 32769), (3, 40, 131071), (8, 100, 65536), (20, 2101, 131072),
                                   (40, 3005, 40000), (70, 3001, 33000), (130, 5003, 33000), (250, 5003, 33000), (9, 33, 131072)])
def test_longest_rows(m, n, k):
    """K up to 131072, the sums up to 127^2 K = 2^31 - 2^25, and among them ones of ordinary values."""
    x = rand(m, k, seed=1).half()
    x[0] = 1.0
    g = torch.Generator(device="cuda").manual_seed(2)
    wq = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8, device="cuda")
    wq[0] = 127
    wq[1] = -127
    x, t = x.cuda(), 2e-5 * (1.0 + torch.rand(n, generator=g, device="cuda"))
    y = torch.empty(m, n, dtype=torch.float16, device="cuda")
    capi.linear_i8([capi.linear_i8_problem(x, capi.i8_weight(wq, t), y)])
    close(y, *(v.cpu() for v in expected(x, wq, t, "none", None)), f"{m}x{n}x{k}")


@pytest.mark.parametrize("m,n", TILE_ROUTES)
def test_row_bits_on_tiles(m, n):
    """Rows among many have the bits that they have alone, among a few and on streams."""
    k = 1300
    x = rand(m, k, seed=7).half().cuda()
    wq, t = weights(n, k, seed=8)
    w, bias = capi.i8_weight(wq.cuda(), t.cuda()), rand(n, seed=9).half().cuda()
    for epi in sorted(EPI):
        def run(rows, y):
            capi.linear_i8([capi.linear_i8_problem(rows, w, y, EPI[epi], bias if epi == "bias" else None)])
            return y
        whole = run(x, torch.empty(m, n, dtype=torch.float16, device="cuda"))
        for a, b in [(m - 1, m), (3, 9), (100, 120), (63, 129), (7, 137)]:
            assert torch.equal(run(x[a:b].contiguous(), torch.empty(b - a, n, dtype=torch.float16, device="cuda")),
                               whole[a:b]), (epi, a, b)


@pytest.mark.parametrize("m,n", [(250, 5003), (1000, 5001), (2400, 5001)])
def test_captured_on_tiles(m, n):
    """Three problems, replayed three times with new inputs and eager work between."""
    k = 330
    xs = [rand(m, k, seed=i).half().cuda() for i in range(3)]
    ws8 = [tuple(v.cuda() for v in weights(n // 3, k, seed=10 + i)) for i in range(3)]
    ys = [torch.empty(m, n // 3, dtype=torch.float16, device="cuda") for _ in range(3)]
    ps = [capi.linear_i8_problem(x, capi.i8_weight(*w), y, capi.EPI_RELU_SQUARE) for x, w, y in zip(xs, ws8, ys)]
    ws = torch.empty(capi.linear_i8_workspace_bytes(ps), dtype=torch.uint8, device="cuda")
    capi.linear_i8(ps, ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        capi.linear_i8(ps, ws)
    for seed in (20, 30, 40):
        for i, x in enumerate(xs):
            x.copy_(rand(m, k, seed=seed + i).half())
            ys[i].zero_()
        g.replay()
        torch.cuda.synchronize()
        got = [y.clone() for y in ys]
        for x, w, y in zip(xs, ws8, got):
            close(y, *(v.cpu() for v in expected(x, *w, "relu2", None)), f"replay {seed}")
        capi.linear_i8(ps, ws)
        for a, b in zip(got, ys):
            assert torch.equal(a, b)


# ---------------------------------------------------------------- offsets past 32 bits

def part(w, a, b):
    """Outputs a..b of weights w (a a multiple of 32): their blocks of the packed matrix."""
    row = w.packed.numel() // (-(-w.n // 32))
    return capi.I8Weight(b - a, w.k, w.packed[a // 32 * row:-(-b // 32) * row], w.scale[a:b])


@pytest.mark.parametrize("m", [1, 5, 20, 130, 700])
def test_weights_past_32_bits(m):
    """70016 outputs of K 32768, 2.3 GB: the last outputs are those of their own block of the weights alone."""
    n, k = 70001, 32768
    g = torch.Generator(device="cuda").manual_seed(1)
    w = capi.I8Weight(n, k, torch.randint(-127, 128, (70016 * k,), generator=g, dtype=torch.int8, device="cuda"),
                      1e-5 * torch.rand(n, generator=g, device="cuda"))
    x = torch.randn(m, k, generator=g, device="cuda").half()
    y, tail = (torch.empty(m, c, dtype=torch.float16, device="cuda") for c in (n, n - 69600))
    capi.linear_i8([capi.linear_i8_problem(x, w, y)])
    capi.linear_i8([capi.linear_i8_problem(x, part(w, 69600, n), tail)])
    assert torch.equal(y[:, 69600:], tail) and (tail != 0).any()


@pytest.mark.parametrize("m,n,k", [(70001, 300, 32768), (131072, 16500, 40)])
def test_rows_past_32_bits(m, n, k):
    """Activations of 4.6 GB (2.3 GB in 8 bits), outputs of 4.3 GB: the last rows are those they give alone."""
    g = torch.Generator(device="cuda").manual_seed(2)
    w = capi.i8_weight(torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8, device="cuda"),
                       1e-5 * torch.rand(n, generator=g, device="cuda"))
    x = torch.empty(m, k, dtype=torch.float16, device="cuda")
    x[:] = torch.randn(k, generator=g, device="cuda").half()
    x[-150:] = torch.randn(150, k, generator=g, device="cuda").half()
    y, tail = (torch.empty(r, n, dtype=torch.float16, device="cuda") for r in (m, 150))
    capi.linear_i8([capi.linear_i8_problem(x, w, y)])
    capi.linear_i8([capi.linear_i8_problem(x[-150:].contiguous(), w, tail)])
    assert torch.equal(y[-150:], tail) and (tail != 0).any() and torch.equal(y[0], y[m // 2])


def test_packing_past_32_bits():
    """Weights of 2.3 GB packed from 8-bit and from fp16 values: the last rows' blocks are those they give alone."""
    n, k = 70001, 32768
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8, device="cuda")
    tail = q[69984:].contiguous()
    whole, alone = capi.i8_weight(q, torch.ones(n, device="cuda")), capi.i8_weight(tail, torch.ones(17, device="cuda"))
    assert torch.equal(whole.packed[69984 * k:], alone.packed)
    whole = capi.i8_quantize(q.half())
    alone = capi.i8_quantize(tail.half())
    used = lambda p: p.view(-1, 2, 32, 16)[:, :, :17]  # noqa: E731  (the block's pad rows are never used)
    assert torch.equal(used(whole.packed[69984 * k:]), used(alone.packed))
    assert torch.equal(whole.scale[69984:], alone.scale)


# ---------------------------------------------------------------- what 8 bits cost

@pytest.mark.parametrize("kind", ["normal", "channels", "relu2"])
def test_error_against_fp16_weights(kind):
    """Against the product of unrounded rows and weights: every output within the bound of its roundings, half a step
    of each factor.  Errors spread evenly over a step of max / 127 give a root mean square of sqrt(c_x^2 + c_w^2) /
    (127 sqrt 12) of the output's, c = max / rms of a row (zeros and values below half a step err less: at most that):
    2^-6.4 of normal rows, 2^-5.6 and 2^-5.9 of the others.  The sums have 2048 terms over 256 rows and 512 columns;
    a tenth leaves room for the statistics."""
    m, n, k = 256, 512, 2048
    x = rand(m, k, seed=1)
    x = {"normal": x, "channels": x * torch.exp(0.6 * rand(k, seed=2)), "relu2": torch.relu(x).square()}[kind].half()
    w = (0.02 * rand(n, k, seed=3) * torch.exp(0.3 * rand(n, 1, seed=4))).half()
    y = torch.empty(m, n, dtype=torch.float16, device="cuda")
    capi.linear_i8([capi.linear_i8_problem(x.cuda(), capi.i8_quantize(w.cuda()), y)])
    xd, wd = x.double(), w.double()
    ref = torch.matmul(xd, wd.t())
    err = y.cpu().double() - ref
    sx, sw = (v.abs().amax(1, keepdim=True) / 127.0 for v in (xd, wd))
    bound = sx / 2 * wd.abs().sum(1) + xd.abs().sum(1, keepdim=True) * sw.t() / 2 + sx * sw.t() * k / 4
    assert (err.abs() <= bound + y.cpu().double().abs() * 2.0 ** -10 + 2.0 ** -24).all()
    c2 = [((v.abs().amax(1) / v.square().mean(1).sqrt()) ** 2).mean() for v in (xd, wd)]
    want = float(((c2[0] + c2[1]) / 12).sqrt() / 127)
    got = float((err.square().mean(1) / ref.square().mean(1)).mean().sqrt())
    assert got < 1.1 * want and (kind == "relu2" or got > 0.9 * want)
    assert 2.0 ** -6.6 < got < 2.0 ** -5.4
