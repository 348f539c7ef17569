"""Arguments that the 8-bit layers and the beam operators refuse, on the host, before any GPU work."""
import ctypes

import pytest
import torch

from vkwr_amd import capi

L = capi._LIB


def at(i):
    """Device addresses far enough apart for every size below; never dereferenced."""
    return 0x100000000 * (i + 1)


def err():
    return L.vkwr_last_error().decode()


def problem(x=at(0), w=at(1), ws=at(2), bias=None, y=at(3), m=2, n=8, k=16, epilogue=0):
    return capi.I8Problem(x, w, ws, bias, y, m, n, k, epilogue)


def linear(*problems, workspace=at(9), nbytes=1 << 30, n=None):
    arr = (capi.I8Problem * max(len(problems), 1))(*problems)
    return capi._linear_i8(len(problems) if n is None else n, arr, workspace, nbytes, None)


@pytest.mark.parametrize("change,text", [
    ({"m": -1}, "sizes"), ({"n": 0}, "sizes"), ({"k": 0}, "sizes"), ({"k": 131073}, "sizes"), ({"m": 2 ** 22 + 1}, "sizes"),
    ({"n": 2 ** 22 + 1}, "sizes"), ({"epilogue": 2}, "epilogue"), ({"epilogue": 9}, "epilogue"), ({"x": None}, "null"),
    ({"w": None}, "null"), ({"ws": None}, "null"), ({"y": None}, "null"), ({"epilogue": 3}, "null"),
    ({"w": at(1) + 8}, "aligned"), ({"y": at(0) + 16}, "overlaps"), ({"y": at(1)}, "overlaps"), ({"y": at(2) + 4}, "overlaps"),
    ({"y": at(9)}, "workspace"), ({"x": at(9) + 16}, "workspace"), ({"w": at(9)}, "workspace"), ({"ws": at(9) + 4}, "workspace"),
    ({"epilogue": 3, "bias": at(9) + 2}, "workspace"), ({"epilogue": 3, "bias": at(3) + 2}, "overlaps")])
def test_linear_refuses(change, text):
    assert linear(problem(**change)) == 1 and text in err()


def test_linear_refuses_batches():
    assert linear() == 1 and "1 to 8" in err()
    assert linear(*[problem()] * 9) == 1 and "1 to 8" in err()
    assert linear(*[problem(m=2 ** 21)] * 3) == 1 and "rows together" in err()
    assert linear(problem(), workspace=None) == 1 and "workspace" in err()
    assert linear(problem(), workspace=at(9) + 4) == 1 and "workspace" in err()
    need = capi.linear_i8_workspace_bytes([problem()])
    assert linear(problem(), nbytes=need - 1) == 1 and "workspace" in err()
    assert linear(problem(), problem(x=at(4), w=at(5), ws=at(6))) == 1 and "overlaps" in err()  # the same y
    assert linear(problem(), problem(x=at(3), w=at(5), ws=at(6), y=at(7))) == 1 and "overlaps" in err()  # reads a y
    assert linear(problem(m=0, x=None, w=None, ws=None, y=None), nbytes=0, workspace=None) == 0


def test_linear_workspace_grows_with_rows():
    size = lambda m: capi.linear_i8_workspace_bytes([problem(m=m, k=300), problem(m=m, n=77, k=1000)])  # noqa: E731
    sizes = [size(m) for m in range(0, 300)]
    assert sizes == sorted(sizes) and sizes[0] == 0
    with pytest.raises(RuntimeError, match="sizes"):
        capi.linear_i8_workspace_bytes([problem(k=0)])


def test_packed_sizes():
    assert capi._i8_packed(1, 1) == 32 * 128 and capi._i8_packed(33, 129) == 64 * 256 and capi._i8_packed(0, 5) == 0
    for bad in ((-1, 8), (8, 0), (8, 131073), (2 ** 22 + 1, 8)):
        assert capi._i8_packed(*bad) == -1
    assert capi._i8_pack(4, 4, None, at(1), None) == 1 and "null" in err()
    assert capi._i8_pack(4, 4, at(0), at(1) + 8, None) == 1 and "aligned" in err()
    assert capi._i8_pack(4, 4, at(0), at(0), None) == 1 and "overlaps" in err()
    assert capi._i8_pack(4, 0, at(0), at(1), None) == 1 and "size" in err()
    assert capi._i8_pack(0, 4, None, None, None) == 0
    assert capi._i8_rows(4, 4, at(0), at(1), None, None) == 1 and "null" in err()
    assert capi._i8_rows(4, 4, at(0), at(1), at(1), None) == 1 and "overlap" in err()
    assert capi._i8_rows(4, 4, at(0), at(0), at(1), None) == 1 and "overlap" in err()


def select(B=2, W=3, V=8, logits=at(0), f16=1, ins=(at(1), at(2), at(3)), outs=tuple(at(i) for i in range(4, 9)), end=1,
           alpha=0.5, ws=at(9), nbytes=1 << 20):
    return capi._beam_select(B, W, V, logits, f16, *ins, *outs, end, alpha, ws, nbytes, None)


@pytest.mark.parametrize("change,text", [
    ({"B": -1}, "size"), ({"W": 0}, "size"), ({"W": 33}, "size"), ({"V": 0}, "size"), ({"V": 2 ** 20 + 1}, "size"),
    ({"alpha": -0.1}, "length penalty"), ({"alpha": float("nan")}, "length penalty"), ({"alpha": 17.0}, "length penalty"),
    ({"end": -2}, "end token"), ({"end": 8}, "end token"), ({"logits": None}, "null"), ({"ins": (at(1), None, at(3))}, "null"),
    ({"outs": (at(4), at(5), None, at(7), at(8))}, "null"), ({"ws": None}, "workspace"), ({"ws": at(9) + 8}, "workspace"),
    ({"nbytes": 100}, "workspace"), ({"outs": (at(1), at(5), at(6), at(7), at(8))}, "overlaps an input"),
    ({"outs": (at(4), at(4) + 8, at(6), at(7), at(8))}, "outputs overlap"),
    ({"outs": (at(4), at(5), at(9), at(7), at(8))}, "workspace"), ({"outs": (at(4), at(5), at(0), at(7), at(8))}, "logits"),
    ({"B": 4000, "W": 32, "nbytes": 1 << 40}, "rows")])
def test_select_refuses(change, text):
    assert select(**change) == 1 and text in err()


def test_select_sizes():
    assert select(B=0) == 0
    with pytest.raises(ValueError):
        capi.beam_workspace_bytes(1, 33, 100)
    assert capi.beam_workspace_bytes(0, 4, 100) == 0
    assert capi.beam_workspace_bytes(2, 4, 65536) == 2 * capi.beam_workspace_bytes(1, 4, 65536)
    with pytest.raises(TypeError):
        capi.beam_select(torch.zeros(1, 2, 8, dtype=torch.bfloat16), *[None] * 8)


def reorder(B=2, W=3, n_slots=9, slots=at(0), parents=at(1), skip=None, out=at(2), pools=((at(4), 2, 64),), n=None):
    arr = (capi.BeamPool * max(len(pools), 1))(*[capi.BeamPool(*p) for p in pools])
    return capi._beam_reorder(B, W, n_slots, slots, parents, skip, out, len(pools) if n is None else n, arr, None)


@pytest.mark.parametrize("change,text", [
    ({"B": -1}, "size"), ({"W": 0}, "size"), ({"W": 33}, "size"), ({"B": 2000}, "size"), ({"n_slots": -1}, "pools"),
    ({"pools": ((at(4), 2, 64),) * 9}, "pools"), ({"n": -1}, "pools"), ({"slots": None}, "null"), ({"parents": None}, "null"),
    ({"out": None}, "null"), ({"out": at(0) + 4}, "overlaps"), ({"out": at(1)}, "overlaps"), ({"skip": at(2)}, "overlaps"),
    ({"pools": ((at(4), 2, 60),)}, "multiple of 16"), ({"pools": ((at(4), -1, 64),)}, "layers"),
    ({"pools": ((None, 2, 64),)}, "null"), ({"pools": ((at(4) + 4, 2, 64),)}, "aligned"),
    ({"pools": ((at(4), 2, 64), (at(4) + 64, 2, 64))}, "overlap"), ({"pools": ((at(0), 2, 64),)}, "tables"),
    ({"pools": ((at(4), 2 ** 20, 2 ** 30), (at(4) + 2 ** 60, 2 ** 20, 2 ** 27))}, "large"),
    ({"pools": ((at(4), 2 ** 20, 2 ** 33),), "n_slots": 2 ** 31 - 1}, "large")])
def test_reorder_refuses(change, text):
    assert reorder(**change) == 1 and text in err()


def test_reorder_sizes():
    assert reorder(B=0) == 0
    slots = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="at most"):
        capi.beam_reorder(slots, None, None, [torch.zeros(2, 3, 4)] * 9)
    with pytest.raises(TypeError, match="pool"):
        capi.beam_reorder(slots, slots, slots, [torch.zeros(2, 3, 4)])


def test_python_refuses():
    for packed, scales in ((4095, 8), (4096, 7)):
        with pytest.raises(ValueError, match="packed bytes"):
            capi.I8Weight(8, 16, torch.zeros(packed, dtype=torch.int8), torch.zeros(scales))
    one = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="pool 0"):
        capi.beam_reorder(one, one, one, [torch.zeros(5)])
    w = capi.I8Weight(8, 16, torch.zeros(4096, dtype=torch.int8), torch.zeros(8))
    h = torch.zeros(2, 16, dtype=torch.float16)
    with pytest.raises(ValueError, match="linear_i8_problem"):
        capi.linear_i8_problem(h[:, :8], w, h)
    with pytest.raises(ValueError, match="epilogue"):
        capi.linear_i8_problem(h, w, h, epilogue=capi.EPI_VALUE_RESIDUAL)
    with pytest.raises(ValueError, match="epilogue"):
        capi.linear_i8_problem(h, w, h, epilogue=capi.EPI_BIAS)
    with pytest.raises((TypeError, ValueError)):
        capi.linear_i8_problem(h, w, h)  # not on a GPU
    with pytest.raises(ValueError, match="1 to 8"):
        capi.linear_i8([])
    with pytest.raises(ValueError, match="bad size"):
        capi.i8_quantize(torch.zeros(8, 131073, dtype=torch.float16))
