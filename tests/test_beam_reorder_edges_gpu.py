"""States that follow their beams, in pools whose offsets pass 32 bits."""
import pytest
import torch

from oracle import beam_ref
from vkwr_amd import capi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layers,n_slots,slot", [(3, 1100, 2 ** 20), (70000, 9, 4096), (1, 5, 2 ** 30)])
def test_pools_past_32_bits(layers, n_slots, slot):
    """Layers of more than 2 GiB, layers that begin past 4 GiB, a slot of 1 GiB: copies where they belong, nothing else
    changed (`slot` in bytes)."""
    B, W = 1, min(4, n_slots)
    g = torch.Generator(device="cuda").manual_seed(1)
    pool = torch.randint(0, 2 ** 31, (layers, n_slots, slot // 4), generator=g, dtype=torch.int32, device="cuda")
    slots = torch.tensor([[n_slots - 1, 0, n_slots - 2, 1]], dtype=torch.int32)
    parents = torch.tensor([[2, 0, 0, 0]], dtype=torch.int32)
    want, _ = beam_ref.reorder(slots, parents, None, n_slots, [])
    keep = pool.clone()
    out = torch.empty(B, W, dtype=torch.int32, device="cuda")
    capi.beam_reorder(slots.cuda(), parents.cuda(), out, [pool])
    assert torch.equal(out.cpu(), want)
    moved = {}
    for c, to in enumerate(want[0].tolist()):
        moved[to] = int(slots[0, parents[0, c]])
    for i in range(n_slots):
        assert torch.equal(pool[:, i], keep[:, moved.get(i, i)]), i
