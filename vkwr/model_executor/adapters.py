"""Low-rank adapters of many requests, served beside one model's weights.

An `AdapterPool` holds `n_adapters` adapters of the projections named: for each layer and name A
[n_adapters, rank, K] and B [n_adapters, N, rank], and a scale per adapter; row i of a step whose request
uses adapter g gets scale[g] (x_i A_g^T) B_g^T added to the projection's output (vkwr_lora_f16).  An
adapter of lower rank is padded with zeros, which add exact zeros; an adapter that holds nothing for a
projection is all zeros there.  `MixedEngine(..., adapters=pool)` and `DraftEngine(..., adapters=pool)`
take an adapter index per sequence and step.
"""
import torch

from vkwr_amd import capi

ADAPTED = ("Wr", "Wk", "Wv", "Wo", "key", "value")


class AdapterPool:
    def __init__(self, model, n_adapters, rank, names=ADAPTED):
        """rank: the largest of the adapters (rounded up to a multiple of 8, at most 128)."""
        names = tuple(names)
        if not names or any(n not in ADAPTED for n in names) or len(set(names)) != len(names):
            raise ValueError(f"adapters of {names}: expected some of {ADAPTED}")
        self.n_adapters, self.rank, self.names = n_adapters, -(-rank // 8) * 8, names
        if not 1 <= n_adapters <= 8192 or not 8 <= self.rank <= 128:
            raise ValueError(f"{n_adapters} adapters of rank {rank}: expected 1 to 8192, 1 to 128")
        dev = model.head.device
        self.layers = []
        for L in model.layers:
            d = {}
            for n in names:
                N, K = L[n].shape
                d[n] = (torch.zeros(n_adapters, self.rank, K, dtype=torch.float16, device=dev),
                        torch.zeros(n_adapters, N, self.rank, dtype=torch.float16, device=dev))
            self.layers.append(d)
        self.scale = torch.ones(n_adapters, dtype=torch.float32, device=dev)

    def load(self, index, weights, scale=1.0):
        """Sets adapter `index`: weights[layer][name] = (A [r, K], B [N, r]), r up to the pool's rank;
        projections that are not named are cleared."""
        if not 0 <= index < self.n_adapters or len(weights) != len(self.layers):
            raise ValueError(f"adapter {index} of {self.n_adapters}, {len(weights)} layers of {len(self.layers)}")
        for mine, given in zip(self.layers, weights):
            unknown = set(given) - set(self.names)
            if unknown:
                raise ValueError(f"adapter {index}: {sorted(unknown)} are not in the pool")
            for n, (a, b) in given.items():
                r = a.shape[0]
                if r > self.rank or a.shape[1] != mine[n][0].shape[2] or tuple(b.shape) != (mine[n][1].shape[1], r):
                    raise ValueError(f"adapter {index}, {n}: A {tuple(a.shape)} and B {tuple(b.shape)} do not fit")
        for mine, given in zip(self.layers, weights):
            for n in self.names:
                A, B = mine[n]
                A[index].zero_()
                B[index].zero_()
                if n in given:
                    a, b = given[n]
                    A[index, :a.shape[0]].copy_(a)
                    B[index, :, :a.shape[0]].copy_(b)
        self.scale[index] = scale


class AdapterStep:
    """What an engine keeps to run a pool's adapters: the rows' indices and their plan, and scratch for all
    the sets of projections that `targets` has described."""

    def __init__(self, pool, max_rows, device):
        self.pool, self.max_rows = pool, max_rows
        self.ids = torch.empty(max_rows, dtype=torch.int32, device=device)
        self.plan = capi.lora_plan_empty(max_rows, pool.n_adapters, device)
        self.ws = torch.empty(0, dtype=torch.uint8, device=device)

    def targets(self, layer, items, epilogue=capi.EPI_NONE):
        """The pool's projections among items (name, x, y): y, of the engine's full-size buffers, gets the
        adapters added in place.  Called while the engine is built, so that the scratch is never replaced
        under a captured step."""
        items = [it for it in items if it[0] in self.pool.names]
        if not items:
            return None
        L = self.pool.layers[layer]
        rows = min(t.shape[0] for _, x, y in items for t in (x, y))
        ts = [capi.lora_target(x[:rows], *L[n], y[:rows], epilogue=epilogue) for n, x, y in items]
        need = capi.lora_workspace_bytes(self.max_rows, self.pool.n_adapters, ts)
        if need > self.ws.numel():
            self.ws = torch.empty(need, dtype=torch.uint8, device=self.ids.device)
        return ts

    def begin(self, groups, adapter_ids):
        """groups: (B, T, first row, first sequence); adapter_ids int32 [sequences] on the device."""
        n = sum(B for B, _, _, _ in groups)
        if adapter_ids.dtype != torch.int32 or tuple(adapter_ids.shape) != (n,):
            raise ValueError(f"adapter_ids: expected int32 [{n}], got {adapter_ids.dtype} {tuple(adapter_ids.shape)}")
        rows = 0
        for B, T, r0, q0 in groups:
            self.ids[r0:r0 + B * T].view(B, T).copy_(adapter_ids[q0:q0 + B, None])
            rows = max(rows, r0 + B * T)
        capi.lora_plan(self.ids[:rows], self.plan)

    def add(self, targets):
        if targets is not None:
            capi.lora(self.plan, targets, scale=self.pool.scale, workspace=self.ws)


__all__ = ["AdapterPool", "AdapterStep", "ADAPTED"]
