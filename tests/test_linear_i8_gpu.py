"""Linear layers with 8-bit weights against the same formula in 64 bits.

Tolerances count roundings.  y is rounded to fp16 once: 2^-11 of the value, 2^-25 below the normal
range.  Before that the exact sum is converted to fp32, multiplied with s t (s, s t and the product
rounded) and, with a bias, added: five roundings of 2^-24, of the product (`mag`) or of the result; the
square doubles them.  tanh and the sigmoid's exponential are within a few units of 2^-23 of their values,
and move by no more than their argument does: 2^-20 in all.
"""
import pytest
import torch

from vkwr_amd import capi

pytestmark = pytest.mark.gpu


def rand(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def rounded(x):
    """(q, s) of rows x in 64 bits; 127 x is exact, so a quotient that ends in .5 is too."""
    x = x.double()
    top = x.abs().amax(1, keepdim=True)
    return torch.round(127.0 * x / torch.where(top > 0, top, 1.0)), top / 127.0


def weights(n, k, seed):
    w = 0.05 * rand(n, k, seed=seed)
    q, t = rounded(w)
    return q.to(torch.int8), t[:, 0].float()


EPI = {"none": capi.EPI_NONE, "relu2": capi.EPI_RELU_SQUARE, "bias": capi.EPI_BIAS, "tanh": capi.EPI_TANH,
       "sigmoid": capi.EPI_SIGMOID}


def expected(x, wq, t, epi, bias):
    q, s = rounded(x)
    p = torch.matmul(q, wq.double().t()) * s * t.double()
    mag = p.abs()
    if epi == "bias":
        p = p + bias.double()
    y = {"relu2": lambda v: torch.clamp(v, min=0.0).square(), "tanh": torch.tanh, "sigmoid": torch.sigmoid}.get(epi, lambda v: v)(p)
    tol = y.abs() * 2.0 ** -11 + 2.0 ** -25
    tol += {"none": 5 * mag * 2.0 ** -24, "bias": 6 * (mag + y.abs()) * 2.0 ** -24, "relu2": 12 * y.abs() * 2.0 ** -24}.get(
        epi, torch.full_like(y, 2.0 ** -20) + 5 * mag * 2.0 ** -24)
    return y, tol


def close(y, ref, tol, what):
    err = (y.cpu().double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err - tol).max()):.3g} over"


SHAPES = [(1, 32, 128), (1, 1, 1), (2, 3, 5), (3, 64, 129), (4, 2048, 2048), (5, 1000, 257), (7, 96, 4096), (8, 768, 768),
          (16, 2048, 512), (17, 33, 31), (31, 65, 64), (32, 128, 8192), (33, 256, 1000), (64, 72, 640), (65, 4096, 256),
          (77, 1003, 2501), (96, 129, 2048), (127, 8, 8), (128, 512, 2048), (129, 320, 192), (200, 2051, 130),
          (256, 256, 256), (257, 1024, 1024), (300, 5, 7000), (433, 2048, 1024), (513, 520, 2560), (768, 2048, 384),
          (1000, 1000, 1000), (2304, 257, 320)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matches_formula(m, n, k):
    x, (wq, t) = rand(m, k, seed=m + n).half(), weights(n, k, seed=k)
    y = torch.empty(m, n, dtype=torch.float16, device="cuda")
    capi.linear_i8([capi.linear_i8_problem(x.cuda(), capi.i8_weight(wq.cuda(), t.cuda()), y)])
    close(y, *expected(x, wq, t, "none", None), f"{m}x{n}x{k}")


# one size for each tile on 256 CUs, from 16 x 16 to 256 x 256, with an odd last row and column tile each, and
# the largest rows that are rounded by the kernel that multiplies them
TILES = [(9, 501, 200), (20, 2101, 140), (40, 3005, 200), (70, 3001, 330), (130, 5003, 260), (250, 5003, 200), (500, 5001, 136),
         (1000, 5001, 130), (2050, 5001, 72), (2400, 5001, 72), (4100, 5001, 64), (8, 77, 4096), (5, 77, 4097), (4, 45, 8192),
         (3, 45, 8193), (2, 33, 16384), (1, 33, 32768), (6, 90, 640),
         (16, 77, 2048), (11, 45, 2040), (13, 100, 2049), (9, 2101, 140)]


@pytest.mark.parametrize("m,n,k", TILES)
def test_every_tile(m, n, k):
    x, (wq, t) = rand(m, k, seed=m).half(), weights(n, k, seed=n)
    bias = rand(n, seed=3).half()
    out = torch.full((m * n + 64,), 5.0, dtype=torch.float16, device="cuda")
    y = out[:m * n].view(m, n)
    capi.linear_i8([capi.linear_i8_problem(x.cuda(), capi.i8_weight(wq.cuda(), t.cuda()), y, capi.EPI_BIAS, bias.cuda())])
    close(y, *expected(x, wq, t, "bias", bias), f"{m}x{n}x{k}")
    assert (out[m * n:] == 5).all()


@pytest.mark.parametrize("epi", sorted(EPI))
@pytest.mark.parametrize("m,n,k", [(1, 2048, 512), (3, 37, 100), (40, 200, 384), (150, 1001, 260), (300, 640, 512)])
def test_epilogues(m, n, k, epi):
    x, (wq, t) = rand(m, k, seed=1).half(), weights(n, k, seed=2)
    bias = rand(n, seed=3).half() if epi == "bias" else None
    y = torch.empty(m, n, dtype=torch.float16, device="cuda")
    w = capi.i8_weight(wq.cuda(), t.cuda())
    capi.linear_i8([capi.linear_i8_problem(x.cuda(), w, y, epilogue=EPI[epi], bias=None if bias is None else bias.cuda())])
    close(y, *expected(x, wq, t, epi, bias), epi)


@pytest.mark.parametrize("m", [1, 6, 50, 700])
def test_batch_of_different_problems(m):
    """Different sizes, epilogues and rows in one call; two problems share their activations."""
    sizes = [(m, 256, 512, "none"), (m, 96, 512, "tanh"), (m, 256, 512, "relu2"), (3, 1000, 130, "none"),
             (m + 2, 64, 64, "sigmoid"), (0, 10, 10, "none"), (m, 33, 2048, "bias"), (1, 8, 40, "none")]
    ps, want = [], []
    shared = None
    for i, (r, n, k, epi) in enumerate(sizes):
        x, (wq, t) = rand(r, k, seed=i).half(), weights(n, k, seed=50 + i)
        if i == 0:
            shared, shared_gpu = x, x.cuda()
        x, xg = (shared, shared_gpu) if i in (0, 2) else (x, x.cuda())
        bias = rand(n, seed=90 + i).half() if epi == "bias" else None
        y = torch.full((r, n), 7.0, dtype=torch.float16, device="cuda")
        ps.append(capi.linear_i8_problem(xg, capi.i8_weight(wq.cuda(), t.cuda()), y, EPI[epi],
                                         None if bias is None else bias.cuda()))
        if r:
            want.append((y, *expected(x, wq, t, epi, bias), f"problem {i}"))
    ws = torch.empty(capi.linear_i8_workspace_bytes(ps), dtype=torch.uint8, device="cuda")
    capi.linear_i8(ps, ws)
    for w in want:
        close(*w)


def unpack(packed, rows, k):
    r, c = torch.meshgrid(torch.arange(rows), torch.arange(k), indexing="ij")
    steps = (k + 127) // 128 * 4
    at = ((r // 32) * steps + c // 32) * 1024 + (((c // 16) % 2) * 32 + r % 32) * 16 + c % 16
    return packed.cpu()[at]


@pytest.mark.parametrize("rows,k", [(1, 1), (3, 16), (8, 128), (33, 1000), (40, 1024), (9, 2048), (5, 8192), (2, 20000),
                                    (257, 333), (1, 131072)])
def test_rounding_is_exact(rows, k):
    """Every value, halves to even included: rows of small multiples of max / 254 hit them."""
    x = rand(rows, k, seed=rows).half()
    x[0, :] = torch.arange(k).remainder(255).half() - 127.0      # max 127 (or less): whole numbers and ties
    if rows > 1:
        x[1] = (torch.arange(k).remainder(509) - 254).half()     # 127 x / 254: every second one a tie
    if rows > 2:
        x[2] = 0.0
    if rows > 3:
        x[3] = x[3] * 2.0 ** -14                                 # subnormal fp16 values
    w = capi.i8_quantize(x.cuda())
    q, s = rounded(x)
    assert torch.equal(unpack(w.packed, rows, k).double(), q)
    assert torch.equal(w.scale.cpu(), (x.float().abs().amax(1) / 127.0))
    # and laid out from row-major values it is the same
    again = capi.i8_weight(q.to(torch.int8).cuda(), w.scale)
    assert torch.equal(unpack(again.packed, rows, k), unpack(w.packed, rows, k))


def test_padding_is_zero():
    """K is padded with zeros in both layouts, whatever the buffer held."""
    for rows, k in [(5, 130), (32, 1)]:
        q = torch.full((rows, k), 3, dtype=torch.int8, device="cuda")
        steps = (k + 127) // 128 * 4
        for packed in (capi.i8_weight(q, torch.ones(rows, device="cuda")).packed,
                       capi.i8_quantize(torch.ones(rows, k, dtype=torch.float16, device="cuda")).packed):
            whole = unpack(packed, rows, steps * 32)
            assert (whole[:, k:] == 0).all() and (whole[:, :k] != 0).all()


@pytest.mark.parametrize("m", [1, 4, 30, 300])
@pytest.mark.parametrize("epi", ["none", "relu2", "bias"])
def test_zero_and_nonfinite_rows(m, epi):
    """A row of zeros gives epilogue(0); one with an infinity or a NaN gives NaN; the others are untouched."""
    n, k = 72, 200
    x, (wq, t) = rand(m, k, seed=4).half(), weights(n, k, seed=5)
    bias = rand(n, seed=6).half() if epi == "bias" else None
    kinds = ["zero", "inf", "nan", "-inf"][:m]
    for i, kind in enumerate(kinds):
        if kind == "zero":
            x[i] = 0.0
        else:
            x[i, 17 * i] = float(kind)
    y = torch.empty(m, n, dtype=torch.float16, device="cuda")
    w = capi.i8_weight(wq.cuda(), t.cuda())
    capi.linear_i8([capi.linear_i8_problem(x.cuda(), w, y, EPI[epi], None if bias is None else bias.cuda())])
    y = y.cpu()
    clean = x.clone()
    for i, kind in enumerate(kinds):
        if kind != "zero":
            assert y[i].isnan().all(), kind
            clean[i] = 0.0
    ref, tol = expected(clean, wq, t, epi, bias)
    keep = [i for i in range(m) if i >= len(kinds) or kinds[i] == "zero"]
    close(y[keep], ref[keep], tol[keep], epi)


@pytest.mark.parametrize("k", [256, 16384])
def test_largest_sums(k):
    """All values at 127: 127^2 k does not fit fp32's 24 bits and has to be right all the same."""
    for m in (1, 40, 300):
        x = torch.ones(m, k).half()
        x[:, 1::2] *= -1.0
        wq = torch.full((64, k), 127, dtype=torch.int8)
        wq[:, 1::2] = -127
        wq[5, 0] = 126
        t = torch.full((64,), 1.0 / 127 / k)
        y = torch.empty(m, 64, dtype=torch.float16, device="cuda")
        capi.linear_i8([capi.linear_i8_problem(x.cuda(), capi.i8_weight(wq.cuda(), t.cuda()), y)])
        close(y, *expected(x, wq, t, "none", None), f"{m}")


@pytest.mark.parametrize("n,k", [(512, 512), (1003, 2501), (2048, 8192)])
def test_row_bits_do_not_depend_on_the_batch(n, k):
    """A row alone, among a few and among many has the same bits."""
    x = rand(700, k, seed=7).half().cuda()
    wq, t = weights(n, k, seed=8)
    w = capi.i8_weight(wq.cuda(), t.cuda())
    whole = torch.empty(700, n, dtype=torch.float16, device="cuda")
    capi.linear_i8([capi.linear_i8_problem(x, w, whole)])
    for a, b in [(0, 1), (699, 700), (3, 7), (100, 120), (31, 81), (5, 200), (64, 384)]:
        part = torch.empty(b - a, n, dtype=torch.float16, device="cuda")
        capi.linear_i8([capi.linear_i8_problem(x[a:b].contiguous(), w, part)])
        assert torch.equal(part, whole[a:b]), (a, b)


@pytest.mark.parametrize("m", [1, 3, 20, 200, 500])
def test_unaligned_tensors(m):
    """Tensors that start off 16 bytes; values before and behind y stay."""
    n, k = 104, 264
    x, (wq, t) = rand(m, k, seed=9).half(), weights(n, k, seed=10)
    flat = torch.zeros(m * k + 3, dtype=torch.float16, device="cuda")
    flat[3:] = x.reshape(-1).cuda()
    out = torch.full((m * n + 9,), 5.0, dtype=torch.float16, device="cuda")
    scale = torch.empty(n + 1, device="cuda")
    scale[1:] = t.cuda()
    w = capi.i8_weight(wq.cuda(), scale[1:])
    y = out[1:1 + m * n].view(m, n)
    capi.linear_i8([capi.linear_i8_problem(flat[3:].view(m, k), w, y)])
    close(y, *expected(x, wq, t, "none", None), "unaligned")
    assert (out[:1] == 5).all() and (out[1 + m * n:] == 5).all()


@pytest.mark.parametrize("m", [1, 24, 300])
def test_captured_and_other_stream(m):
    """Replayed three times with new inputs and eager work between; then on another stream."""
    n, k = 520, 1024
    x, (wq, t) = rand(m, k, seed=11).half().cuda(), weights(n, k, seed=12)
    w = capi.i8_weight(wq.cuda(), t.cuda())
    y = torch.empty(m, n, dtype=torch.float16, device="cuda")
    ps = [capi.linear_i8_problem(x, w, y, capi.EPI_RELU_SQUARE)]
    ws = torch.empty(capi.linear_i8_workspace_bytes(ps), dtype=torch.uint8, device="cuda")
    capi.linear_i8(ps, ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        capi.linear_i8(ps, ws)
    for seed in (20, 21, 22):
        new = rand(m, k, seed=seed).half()
        x.copy_(new)
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        got = y.clone()
        close(got, *expected(new, wq, t, "relu2", None), f"replay {seed}")
        capi.linear_i8(ps, ws)
        assert torch.equal(got, y)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y2 = torch.empty_like(y)
        capi.linear_i8([capi.linear_i8_problem(x, w, y2, capi.EPI_RELU_SQUARE)])
    s.synchronize()
    assert torch.equal(y2, y)
