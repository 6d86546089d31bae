"""Shared-prefix decode, sampling and verification where calls meet and at the ends of their ranges.
Two runs of one call have to be equal."""
import threading

import pytest
import torch

from adallm_b200.attention import paged_decode, paged_prefill
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
