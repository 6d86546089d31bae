"""Shared-prefix decode, sampling and verification where calls meet: several threads on one stream,
calls of different size in turn, and inputs at the ends of their ranges.

Tolerances are those of the operators' own tests (tests/test_gpu_shared_prefix.py,
tests/test_gpu_sampling.py); where two runs of one call are compared they have to be equal."""
import functools
import threading

import numpy as np
import pytest
import torch

from adallm_b200.attention import paged_decode, paged_prefill
from adallm_b200.sampler import sample, verify_drafts
from adallm_b200.shared_prefix import shared_prefix_decode
from oracle import speculative as osp
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu


def _in_threads(*functions):
    """Runs each in a thread of its own, all at once; the first failure is raised."""
    failed = []

    def run(f):
        try:
            f()
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=run, args=(f,)) for f in functions]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if failed:
        raise failed[0]


@pytest.mark.parametrize("entry", ["shared", "decode", "prefill"])
def test_a_threads_first_cuda_call(entry):
    """Everything is allocated, so that the library's own calls are the first that need a context."""
    c = osp.make_shared_prefix_case(1, [96], [3], [20, 64, 7], [1, 1, 1], 32, 8, 16)
    c = {k: v.to(dev()) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    room = torch.empty(1 << 26, dtype=torch.uint8, device=dev())
    out = torch.empty_like(c["q"])
    cu_q = torch.arange(4, dtype=torch.int32, device=dev())
    cu_k = torch.tensor([0, 20, 84, 91], dtype=torch.int32, device=dev())
    call = {"shared": lambda: shared_prefix_decode(c["q"], c["k_cache"], c["v_cache"], c["prefix_tables"],
                                                   c["prefix_lens"], c["cu_groups"], c["block_tables"],
                                                   c["context_lens"], c["scale"], out=out, workspace=room),
            "decode": lambda: paged_decode(c["q"], c["k_cache"], c["v_cache"], c["block_tables"], c["context_lens"],
                                           c["scale"], out=out, workspace=room),
            "prefill": lambda: paged_prefill(c["q"], c["k_cache"], c["v_cache"], c["block_tables"], cu_q, cu_k, 1,
                                             c["scale"], out=out)}[entry]
    call()
    want = out.clone()
    out.zero_()
    torch.cuda.synchronize()
    _in_threads(call)
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def _attention(seed, prefix, n, rows, reach=0):
    c = osp.make_shared_prefix_case(seed, [prefix], [n], [3 + (7 * i) % 90 for i in range(n)], [rows] * n, 32, 8, 16)
    c = {k: v.to(dev()) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    if reach:  # a table of this many pages: enough rows then go to the tensor-core kernel
        c["prefix_tables"] = torch.nn.functional.pad(c["prefix_tables"], (0, reach), value=-1)
    return lambda: (shared_prefix_decode(c["q"], c["k_cache"], c["v_cache"], c["prefix_tables"], c["prefix_lens"],
                                         c["cu_groups"], c["block_tables"], c["context_lens"], c["scale"],
                                         cu_seqlens_q=c["cu_seqlens_q"]),)


def _verification(seed, batch, drafts, vocab):
    g = torch.Generator().manual_seed(seed)
    n = batch * (drafts + 1)
    target = 3 * torch.randn((n, vocab), generator=g)
    ids = target.roll(1, 0).argmax(-1)  # likely tokens: some are accepted
    a = [t.to(dev()) for t in (target, ids, torch.arange(0, n + 1, drafts + 1, dtype=torch.int32), torch.full((batch,), 0.3),
                               torch.rand((batch, drafts), generator=g),
                               torch.empty((batch, vocab)).exponential_(1.0, generator=g))]
    return lambda: verify_drafts(*a)


def _calls():
    return [_attention(1, 300, 5, 1), _verification(2, 3, 4, 5003), _attention(3, 900, 24, 3, reach=1 << 14),
            _verification(4, 40, 2, 1009), _attention(5, 64, 60, 2), _verification(6, 1, 1, 90001)]


def test_threads_on_one_stream_get_their_own_results():
    calls = _calls()
    alone = [tuple(t.clone() for t in f()) for f in calls]
    torch.cuda.synchronize()
    start, wrong = threading.Barrier(len(calls)), []

    def caller(i):
        start.wait(timeout=60)
        for _ in range(150):
            got = calls[i]()
            if not all(torch.equal(a, b) for a, b in zip(got, alone[i])):
                wrong.append(i)

    _in_threads(*(functools.partial(caller, i) for i in range(len(calls))))
    torch.cuda.synchronize()
    assert not wrong, wrong


def test_calls_of_different_sizes_in_turn():
    """No host wait between them: each one's launches follow the one's before on the stream."""
    calls = _calls()
    alone = [tuple(t.clone() for t in f()) for f in calls]
    torch.cuda.synchronize()
    order = np.random.default_rng(0).integers(0, len(calls), 400).tolist()
    got = [(i, calls[i]()) for i in order]
    torch.cuda.synchronize()
    for i, out in got:
        assert all(torch.equal(a, b) for a, b in zip(out, alone[i])), i


@pytest.mark.parametrize("reach", [0, 1 << 14])
@pytest.mark.parametrize("rows", [[1, 2], [40, 33], [3, 0]])
def test_windows_wider_than_all_positions(rows, reach):
    """Prefixes and contexts with fewer keys than rows; from the reach of the tables on a window cuts nothing."""
    c = osp.make_shared_prefix_case(7, [20], [2], [2, 30], rows, 32, 8, 16)
    c = {k: v.to(dev()) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    c["prefix_tables"] = torch.nn.functional.pad(c["prefix_tables"], (0, reach), value=-1)

    def run(window):
        return shared_prefix_decode(c["q"], c["k_cache"], c["v_cache"], c["prefix_tables"], c["prefix_lens"],
                                    c["cu_groups"], c["block_tables"], c["context_lens"], c["scale"],
                                    cu_seqlens_q=c["cu_seqlens_q"], window=window)

    want = run(0)
    reached = (c["prefix_tables"].shape[1] + c["block_tables"].shape[1]) * 16
    for window in (50, reached - 1, reached, 1 << 30, 2 ** 31 - 40, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 3, 1 << 62):
        got = run(window)
        assert float((got - want).float().abs().max()) <= 2 ** -8 * float(want.float().abs().max()), window
        if window >= reached:
            assert torch.equal(got, want), window


@pytest.mark.parametrize("cu", [[0, 5, 3, 8], [-3, 4, 6, 8], [0, 2 ** 31 - 1, -2 ** 31, 8], [8, 6, 2, 0], [5, 5, 9, 12]])
@pytest.mark.parametrize("temperature", [0.0, 0.7])
def test_verify_lists_that_do_not_ascend(cu, temperature):
    """Such a list has no meaning, but the call stays inside its tensors: tokens of the vocabulary or -1,
    whatever the workspace held before."""
    g = torch.Generator().manual_seed(3)
    v = 1003
    a = [t.to(dev()) for t in (torch.randn((8, v), generator=g), torch.randint(0, v, (8,), generator=g),
                               torch.tensor(cu, dtype=torch.int32), torch.full((3,), temperature),
                               torch.rand((3, 2), generator=g), torch.empty((3, v)).exponential_(1.0, generator=g))]
    for fill in (0x00, 0x7F, 0xFF):
        room = torch.full((1 << 16,), fill, dtype=torch.uint8, device=dev())
        tokens, accepted, _ = verify_drafts(*a, workspace=room)
        assert bool(((tokens >= -1) & (tokens < v)).all())
        assert bool(((accepted >= 0) & (accepted <= 2)).all())


@pytest.mark.parametrize("reach", [0, 1 << 14])
def test_attention_lists_that_do_not_ascend(reach):
    """Rows and sequences claimed several times over, or before and past all there are: the call stays inside
    its tensors, and lists in order give what they gave."""
    n = 12
    c = osp.make_shared_prefix_case(9, [100, 60], [7, 5], [5 + i for i in range(n)], [4] * n, 32, 8, 16)
    c = {k: v.to(dev()) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    c["prefix_tables"] = torch.nn.functional.pad(c["prefix_tables"], (0, reach), value=-1)

    def run(**kw):
        a = {**c, **kw}
        return shared_prefix_decode(a["q"], a["k_cache"], a["v_cache"], a["prefix_tables"], a["prefix_lens"],
                                    a["cu_groups"], a["block_tables"], a["context_lens"], a["scale"],
                                    cu_seqlens_q=a["cu_seqlens_q"])

    want = run()
    i32 = dict(dtype=torch.int32, device=dev())
    low, high = -2 ** 31, 2 ** 31 - 1
    for cu_q in ([0, 48] * 6 + [0], [48] * 6 + [0] * 7, [low, high] * 6 + [low], list(range(24, -2, -2))):
        assert run(cu_seqlens_q=torch.tensor(cu_q, **i32)).shape == want.shape
    for cu_g in ([0, 12, 0], [12, 0, 12], [low, high, low], [5, 5, 3]):
        assert run(cu_groups=torch.tensor(cu_g, **i32)).shape == want.shape
    torch.cuda.synchronize()
    assert torch.equal(run(), want)
