"""Linear layers with 8-bit weights where the other tests do not go: scales near the end of fp32's range.

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
