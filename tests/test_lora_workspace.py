"""vkwr_lora_workspace_bytes: the most that any row count up to m takes, without going through them all."""
import time

import pytest

from vkwr_amd import capi


def targets(n, k, count):
    return (capi.LoraTarget * count)(*[capi.LoraTarget(None, None, None, None, None, n, k, 0) for _ in range(count)])


@pytest.mark.parametrize("n,k,G,R,count,want", [
    (2048, 2048, 16, 16, 1, {1: 1024, 65: 66560, 500: 512000, 2304: 1179648, 8000: 4096000, 40000: 8126208}),
    (2048, 8192, 300, 64, 3, {1: 12288, 65: 258048, 500: 384000, 2304: 1769472, 8000: 6144000, 39999: 30719232}),
    (64, 64, 1, 8, 1, {1: 128, 65: 8320, 500: 64000, 2304: 294912, 8000: 1024000, 40000: 5120000})])
def test_values(n, k, G, R, count, want):
    """As found by evaluating every row count; the first projection at 40000 rows (one part, 32 floats a row) needs
    less than 31743 rows of two parts do."""
    assert {m: capi._lora_ws(m, G, R, count, targets(n, k, count)) for m in want} == want
    assert capi._lora_ws(0, G, R, count, targets(n, k, count)) == 0


def test_many_rows_cost_no_more_than_few():
    """(`lora` asks at each call that is given no workspace; 32000 rows took 80 times as long as one.)"""
    t = targets(2048, 2048, 1)

    def least(m):
        best = 1.0
        for _ in range(50):
            start = time.perf_counter()
            for _ in range(20):
                capi._lora_ws(m, 16, 16, 1, t)
            best = min(best, time.perf_counter() - start)
        return best

    assert least(32000) < 10 * least(1)
