"""Loading 8-bit weights into an engine's, on the CPU: a call that is refused leaves both values and scales as they were."""
import types

import pytest
import torch

from vkwr.model_executor import Int8Weights
from vkwr_amd import capi

N, K = 8, 16


class Weight:
    def __init__(self, n, k, packed, scale):
        self.n, self.k, self.packed, self.scale = n, k, packed, scale


@pytest.fixture
def weights(monkeypatch):
    monkeypatch.setattr(capi, "i8_quantize", lambda w: Weight(N, K, torch.zeros(N * K, dtype=torch.int8), torch.ones(N)))
    monkeypatch.setattr(capi, "i8_weight", lambda q, scale: Weight(N, K, q.reshape(-1).clone(), scale))
    return Int8Weights(types.SimpleNamespace(layers=[{"key": torch.zeros(N, K)}]), ("key",))


@pytest.mark.parametrize("shape", [(N, 1), (1, N), (N + 1,), ()])
def test_scales_of_another_shape(weights, shape):
    w = weights.layers[0]["key"]
    with pytest.raises(ValueError, match="scale"):
        weights.load(0, "key", torch.full((N, K), 3, dtype=torch.int8), torch.full(shape, 0.5))
    assert (w.packed == 0).all() and (w.scale == 1).all()


def test_loaded_in_place(weights):
    w = weights.layers[0]["key"]
    at = w.packed.data_ptr(), w.scale.data_ptr()
    weights.load(0, "key", torch.full((N, K), 3, dtype=torch.int8), torch.full((N,), 0.5))
    assert (w.packed == 3).all() and (w.scale == 0.5).all() and at == (w.packed.data_ptr(), w.scale.data_ptr())
