"""Which launches the mixed step's projections make, on the CPU: the engine's own lists, with the kernels' calls recorded."""
import types

import pytest
import torch

from vkwr.model_executor.mixed import MixedEngine
from vkwr_amd import capi

R, C = 3, 4


class Engine(MixedEngine):
    def __init__(self, int8=()):
        t = lambda: torch.zeros(R, C)  # noqa: E731
        self.mix = [t() for _ in range(6)]
        self.r, self.k, self.v, self.v_first, self.w1, self.a1, self.g1, self.v1 = (t() for _ in range(8))
        L = {n: n for n in ("Wr", "Wk", "Wv")}
        self.model = types.SimpleNamespace(layers=[L, L])
        self.lw, self.ws = [{n: n for n in ("w1", "a1", "g1", "v1")}] * 2, None
        self.eight, self.asked = [], 0
        self.int8 = types.SimpleNamespace(has=lambda n: n in int8, run=lambda l, items: self.eight.append([i[0] for i in items]))
        if not int8:
            self.int8 = None

    def _rkv(self, rows, first):
        self.asked += 1
        return super()._rkv(rows, first)


@pytest.fixture
def launches(monkeypatch):
    out = []
    monkeypatch.setattr(capi, "gemm_problem", lambda x, w, y, epilogue=capi.EPI_NONE: (w, epilogue))
    monkeypatch.setattr(capi, "gemm", lambda ps, ws: out.append([w for w, _ in ps]))
    return out


@pytest.mark.parametrize("layer", [0, 1])
def test_without_8_bit_weights_the_projections_are_listed_once(launches, layer):
    """Each list slices six tensors, 6 us of a layer's host time."""
    e = Engine()
    e._run_proj(layer, 2)
    assert launches == [["Wr", "Wk", "Wv", "w1", "a1", "g1"] + ["v1"] * layer]
    assert e.asked == 1


@pytest.mark.parametrize("names", [("Wk",), ("Wr", "Wk", "Wv"), ("key",)])
def test_with_8_bit_weights(launches, names):
    e = Engine(names)
    e._run_proj(1, 2)
    mine = [n for n in ("Wr", "Wk", "Wv") if n in names]
    assert e.eight == ([mine] if mine else [])
    assert launches == [[n for n in ("Wr", "Wk", "Wv") if n not in names] + ["w1", "a1", "g1", "v1"]]
    assert e.asked == 1
