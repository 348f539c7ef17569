"""8-bit weights of a model's large projections, for MixedEngine(..., int8=weights).

`Int8Weights` holds the projections named (r, k, v, o of the time mix, key and value of the channel mix)
in 8 bits with a scale per output channel, laid out for vkwr_linear_i8_f16; the engine rounds each row
of activations to 8 bits as it multiplies.  The low-rank projections, which make the decay, the gates and
the learning rates, and the head stay fp16.  Half the weight bytes of a step and twice the matrix rate; the
error of a product has a root mean square of sqrt(c_x^2 + c_w^2) / 440 of the output's, with c = max / rms of a row
of activations and of weights: 2^-6.4 for normally distributed ones of 2048, 2^-5.5 where some channels are much larger than
others.  The model's fp16 matrices of these names are not read by such an engine and may be freed.
"""
import torch

from vkwr_amd import capi

PROJECTIONS = ("Wr", "Wk", "Wv", "Wo", "key", "value")


class Int8Weights:
    def __init__(self, model, names=PROJECTIONS):
        names = tuple(names)
        if not names or any(n not in PROJECTIONS for n in names) or len(set(names)) != len(names):
            raise ValueError(f"8-bit weights of {names}: expected some of {PROJECTIONS}")
        self.names = names
        self.layers = [{n: capi.i8_quantize(L[n]) for n in names} for L in model.layers]

    def load(self, layer, name, q, scale):
        """Replaces one projection by weights that are 8 bits already: q [N, K] int8 of -127..127, scale [N]
        fp32 (of a quantised checkpoint).  In place: captured steps see it."""
        w = self.layers[layer][name]
        if tuple(q.shape) != (w.n, w.k) or tuple(scale.shape) != (w.n,):
            raise ValueError(f"layer {layer}, {name}: q {tuple(q.shape)}, scale {tuple(scale.shape)}, expected [{w.n}, {w.k}] "
                             f"and [{w.n}]")
        new = capi.i8_weight(q, scale)
        w.packed.copy_(new.packed)
        w.scale.copy_(new.scale)

    @property
    def nbytes(self):
        return sum(w.nbytes for L in self.layers for w in L.values())


class Int8Step:
    """What an engine keeps to run 8-bit projections: scratch for any of its launches at any row count."""

    def __init__(self, weights, cfg, max_rows, device):
        self.weights = weights
        C, F = cfg.n_embd, cfg.dim_ffn
        shapes = {"key": (F, C), "value": (C, F)}
        if len(weights.layers) != cfg.n_layer or any((w.n, w.k) != shapes.get(n, (C, C)) for L in weights.layers
                                                     for n, w in L.items()):
            raise ValueError(f"8-bit weights of {len(weights.layers)} layers, of a model of other sizes than the engine's")
        # (sizes only: a launch has at most the three projections of the time mix, or one of the channel mix)
        need = max(3 * capi.linear_i8_scratch_bytes(max_rows, C), capi.linear_i8_scratch_bytes(max_rows, F))
        self.ws = torch.empty(need, dtype=torch.uint8, device=device)

    def has(self, name):
        return name in self.weights.names

    def run(self, layer, items, epilogue=capi.EPI_NONE):
        """items: (name, x, y) of one launch."""
        L = self.weights.layers[layer]
        capi.linear_i8([capi.linear_i8_problem(x, L[n], y, epilogue=epilogue) for n, x, y in items], self.ws)


__all__ = ["Int8Weights", "Int8Step", "PROJECTIONS"]
