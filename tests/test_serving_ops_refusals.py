"""Arguments that the serving operators refuse, on the host, before any GPU work."""
import ctypes

import pytest
import torch

from vkwr_amd import capi

L = capi._LIB
P = ctypes.c_void_p(0x10000)


def err():
    return L.vkwr_last_error().decode()


def drafts(B=2, Pn=2, T=2, C=128, H=2, pool=P, n_slots=4, slots=P, kept=P, n_pending=2, rows=None, vec=P, y=P):
    return capi._wkv_drafts(B, Pn, T, C, H, pool, n_slots, slots, kept, n_pending, rows, *[vec] * 5, *[vec] * 6, y, None)


@pytest.mark.parametrize("change,text", [
    ({"B": -1}, "negative"), ({"Pn": -1, "kept": None}, "negative"), ({"C": 100}, "head size 64"),
    ({"kept": None}, "kept must be given"), ({"Pn": 0}, "kept must be given"), ({"pool": None}, "null"),
    ({"slots": None}, "null"), ({"vec": None}, "null"), ({"y": None}, "null"), ({"n_pending": 1}, "pending rows"),
    ({"pool": ctypes.c_void_p(0x10008)}, "aligned"), ({"vec": ctypes.c_void_p(0x10002)}, "aligned"),
    ({"B": 2 ** 20, "H": 2 ** 12, "C": 2 ** 18, "n_pending": 2 ** 20}, "too large")])
def test_wkv_drafts_refuses(change, text):
    assert drafts(**change) == 1 and text in err()


def test_wkv_drafts_refuses_too_many_tokens():
    assert drafts(B=1, H=1, C=64, T=2 ** 24) == 1 and "too large" in err()


def test_wkv_drafts_empty_work():
    assert drafts(B=0) == 0
    assert drafts(Pn=0, T=0, kept=None) == 0
    with pytest.raises(ValueError):
        capi.wkv_drafts_slots(1, 0, 64, 1, torch.empty(1, 1, 64, 64), None, *[None] * 7, kept=torch.zeros(1))


def verify(B=2, K=2, V=8, logits=P, f16=1, drafts=P, q=P, u=P, tokens=P, accepted=P, temperature=1.0, top_k=-1, top_p=1.0,
           ws=P, nbytes=1 << 20):
    return capi._verify(B, K, V, logits, f16, drafts, None, q, u, tokens, accepted, temperature, top_k, top_p, ws, nbytes,
                        None)


@pytest.mark.parametrize("change,text", [
    ({"B": -1}, "negative"), ({"K": -1}, "negative"), ({"V": 6}, "multiple of 4"), ({"V": 0}, "multiple of 4"),
    ({"V": 1 << 21}, "at most"), ({"temperature": 0.0}, "temperature"), ({"temperature": float("nan")}, "temperature"),
    ({"logits": None}, "null"), ({"drafts": None}, "null"), ({"u": None}, "null"), ({"tokens": None}, "null"),
    ({"accepted": None}, "null"), ({"logits": ctypes.c_void_p(0x10004)}, "aligned"),
    ({"logits": ctypes.c_void_p(0x10008), "f16": 0}, "aligned"), ({"q": ctypes.c_void_p(0x10004)}, "aligned"),
    ({"ws": None}, "workspace"), ({"nbytes": 191}, "workspace"), ({"B": 2 ** 30, "K": 7}, "too large")])
def test_verify_refuses(change, text):
    assert verify(**change) == 1 and text in err()


def test_verify_sizes():
    assert verify(B=0) == 0
    assert capi.verify_workspace_bytes(2, 2, 8) >= 192
    assert capi.verify_workspace_bytes(0, 2, 8) == 0


@pytest.mark.parametrize("V,rows", [(8, 1 << 20), (32768, 1 << 20), (65536, 1 << 19), (1 << 20, 1 << 15)])
def test_verify_launch_limits(V, rows):
    assert verify(B=rows, K=0, V=V) == 1 and "workspace" in err()  # the size itself is taken
    assert verify(B=rows + 1, K=0, V=V) == 1 and "too large" in err()
    assert capi.verify_workspace_bytes(rows, 0, V) > 0 and capi.verify_workspace_bytes(rows + 1, 0, V) == 0
    assert capi.verify_workspace_bytes(2 ** 30, 2 ** 30, V) == 0 and capi.verify_workspace_bytes(1, 1, 1 << 21) == 0


def target(n=64, k=64, x=0x10000, a=0x20000, b=0x30000, base=None, y=0x40000, epilogue=0):
    return capi.LoraTarget(x, a, b, base, y, n, k, epilogue)


def lora(m=4, G=2, rank=8, plan=P, targets=None, ws=P, nbytes=1 << 30):
    targets = [target()] if targets is None else targets
    arr = (capi.LoraTarget * max(len(targets), 1))(*targets)
    return capi._lora(m, G, rank, None, plan, len(targets), arr, ws, nbytes, None)


@pytest.mark.parametrize("change,text", [
    ({"m": -1}, "row count"), ({"G": 0}, "adapters"), ({"G": 8193}, "adapters"), ({"rank": 0}, "rank"),
    ({"rank": 12}, "rank"), ({"rank": 136}, "rank"), ({"targets": []}, "targets"), ({"targets": [target()] * 9}, "targets"),
    ({"targets": [target(n=12)]}, "multiples of 8"), ({"targets": [target(k=0)]}, "multiples of 8"),
    ({"targets": [target(epilogue=3)]}, "epilogue"), ({"plan": None}, "plan"), ({"ws": None}, "workspace"),
    ({"nbytes": 8}, "workspace"), ({"targets": [target(x=None)]}, "null"), ({"targets": [target(y=None)]}, "null"),
    ({"targets": [target(b=0x30008)]}, "aligned"), ({"targets": [target(y=0x10010)]}, "overlaps x"),
    ({"targets": [target(base=0x40010)]}, "base overlaps"),
    ({"targets": [target(), target(x=0x50000)]}, "overlaps y"),
    ({"targets": [target(), target(y=0x60000, base=0x40000)]}, "base of")])
def test_lora_refuses(change, text):
    assert lora(**change) == 1 and text in err()


def test_lora_plan_and_workspace_sizes():
    assert capi._lora_plan_bytes(-1, 2) == -1 and capi._lora_plan_bytes(4, 0) == -1
    assert capi._lora_plan(4, 2, P, P, 8, None) == 1 and "plan of" in err()
    assert capi._lora_plan(4, 2, None, P, 1 << 20, None) == 1 and "null" in err()
    assert capi._lora_plan_bytes(65535 * 64, 2) == -1 and capi._lora_plan_bytes(65531 * 64, 2) > 0
    assert capi._lora_plan(2 ** 31 - 100, 2, P, P, 2 ** 62, None) == 1 and "tiles" in err()
    sizes = [capi._lora_plan_bytes(m, 100) for m in range(0, 3000, 7)]
    assert sizes == sorted(sizes)
    arr = (capi.LoraTarget * 1)(target(n=2048, k=2048))
    need = [capi._lora_ws(m, 16, 16, 1, arr) for m in range(1, 600, 13)]
    assert need == sorted(need)
    assert capi._lora_ws(4, 16, 12, 1, arr) == -1 and "rank" in err()


def test_wrappers_refuse_cpu_tensors_and_wrong_types():
    x = torch.zeros(4, 64, dtype=torch.float16)
    with pytest.raises(TypeError):
        capi.lora_target(x, torch.zeros(2, 8, 64).half(), torch.zeros(2, 64, 8).half(), x.clone())
    with pytest.raises(ValueError):
        capi.lora_target(x, torch.zeros(2, 8, 64).half(), torch.zeros(2, 64, 16).half(), x.clone())
    with pytest.raises(TypeError):
        capi.verify_drafts(torch.zeros(1, 2, 8, dtype=torch.bfloat16), None, None, None, None)
    with pytest.raises(TypeError):
        capi.verify_drafts(torch.zeros(1, 2, 8), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, 2),
                           torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError):
        capi.lora_plan_empty(8, 0, "cpu")
