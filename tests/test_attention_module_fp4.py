"""Attention.forward over a 4-bit cache beside its e4m3 form: the slots it takes, and the kernel that a failure names."""
import pytest
import torch

from adallm_b200 import attention as A
from adallm_b200 import kvcache_fp4 as kv
from adallm_b200.context import reset_context, set_context

I32 = torch.int32


@pytest.fixture(autouse=True)
def no_context_left():
    yield
    reset_context()


def module(device="cpu"):
    m = A.Attention(4, 128, 0.1, 2)
    m.k_cache, m.v_cache = kv.empty_kvcache_fp4(3, 2, 16, device)
    return m


def test_slots_of_64_bits_reach_the_store_as_32(monkeypatch):
    seen = []
    monkeypatch.setattr(A.fp4, "store_kvcache_fp4", lambda k, v, kc, vc, slots, ks, vs: seen.append(slots))
    monkeypatch.setattr(A.fp4, "paged_decode_fp4", lambda q, *a: q)
    rows = torch.zeros((4, 2, 128), dtype=torch.bfloat16)
    for slots in (torch.tensor([3, -1, 2 ** 31 - 1, 7], dtype=I32), torch.tensor([3, -1, 2 ** 32 + 5, -2 ** 40])):
        set_context(False, slot_mapping=slots, context_lens=torch.ones(4, dtype=I32), block_tables=torch.zeros((4, 1), dtype=I32))
        module()(torch.zeros((4, 512), dtype=torch.bfloat16), rows, rows)
    assert all(s.dtype == I32 for s in seen)
    assert seen[0].tolist() == [3, -1, 2 ** 31 - 1, 7] and seen[1].tolist() == [3, -1, 2 ** 31 - 1, -1]


@pytest.mark.parametrize("bits", ["4-bit", "FP8"])
@pytest.mark.parametrize("prefill", [True, False])
def test_a_failure_names_the_kernel_that_ran(monkeypatch, bits, prefill):
    def fail(*args):
        raise RuntimeError("launch")

    where, tail = (A.fp4, "_fp4") if bits == "4-bit" else (A, "")
    monkeypatch.setattr(where, "paged_prefill" + tail, fail)
    monkeypatch.setattr(where, "paged_decode" + tail, fail)
    for name in ("store_kvcache_fp4", "store_kvcache"):
        monkeypatch.setattr(A.fp4 if name.endswith("4") else A, name, lambda *a: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    m = module()
    if bits == "FP8":
        m.k_cache = m.v_cache = torch.zeros((3, 16, 2, 128)).to(torch.float8_e4m3fn)
    one = torch.zeros(1, dtype=I32)
    set_context(prefill, one, one, 1, 0, one, one, one[None])
    with pytest.raises(RuntimeError, match=f"^{bits} {'paged prefill' if prefill else 'KV decode'} kernel failed"):
        m(torch.zeros((1, 512), dtype=torch.bfloat16), None, None)


@pytest.mark.gpu
def test_slots_of_64_bits_store_the_same_rows():
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn((5, h, 128), generator=g, device="cuda").to(torch.bfloat16) for h in (4, 2, 2))
    slots = torch.tensor([4, 17, -1, 40, 48])  # the last is behind the cache
    outs = []
    for dtype in (I32, torch.int64):
        m = module("cuda")
        set_context(False, slot_mapping=slots.to(dtype).cuda(), context_lens=torch.tensor([5, 2, 0, 9, 16], dtype=I32).cuda(),
                    block_tables=torch.tensor([[0], [1], [-1], [2], [0]], dtype=I32).cuda())
        outs.append((m(q.flatten(1), k, v), m.k_cache, m.v_cache))
    assert all(torch.equal(a, b) for a, b in zip(*outs)) and int((outs[0][1] != 0).sum()) > 0
