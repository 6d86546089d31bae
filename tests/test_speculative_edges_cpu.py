"""Shared-prefix decode and draft verification without a GPU: what a call keeps to itself, and models
of what the kernels do where a run on a GPU could not show it."""
import threading

import pytest
import torch

from adallm_b200 import _native as N
from adallm_b200 import build as B
from oracle import speculative as osp


class OnDevice(torch.Tensor):
    """A CPU tensor that says it is on a GPU: for the Python layer above a library that launches nothing."""
    is_cuda = property(lambda self: True)


class Library:
    """The sizes of the real library; its launching entries note the workspace and wait for each other."""

    def __init__(self, real, callers):
        self.real, self.inside, self.lock, self.seen = real, threading.Barrier(callers), threading.Lock(), []

    def __getattr__(self, name):
        return getattr(self.real, name)

    def _enter(self, address, nbytes):
        with self.lock:
            self.seen.append((address, nbytes))
        self.inside.wait(timeout=60)  # every caller is inside its call
        return 0

    def ada_verify_drafts(self, *a):
        return self._enter(a[-3], a[-2])

    def ada_fp8_shared_prefix_decode(self, *a):
        return self._enter(a[-4], a[-3])


def test_calls_of_several_threads_on_one_stream_have_workspaces_of_their_own(monkeypatch):
    """Both entries make several launches that talk through the workspace, and the foreign call lets other
    threads run: no byte of one call's workspace may be another's while both are inside."""
    from adallm_b200.sampler import verify_drafts
    from adallm_b200.shared_prefix import shared_prefix_decode
    B.build()
    library = Library(N.lib(), 4)
    monkeypatch.setattr(N, "lib", lambda: library)
    monkeypatch.setattr(N, "stream_ptr", lambda device=None: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    on = lambda t: t.as_subclass(OnDevice)  # noqa: E731

    def verify(rows):
        verify_drafts(on(torch.zeros((rows, 64))), on(torch.zeros(rows, dtype=torch.int64)),
                      on(torch.tensor([0, rows], dtype=torch.int32)), on(torch.ones(1)), on(torch.zeros((1, rows - 1))),
                      on(torch.ones((1, 64))))

    def attend(n):
        c = osp.make_shared_prefix_case(1, [40], [n], [5] * n, [1] * n, 8, 8, 16)
        c = {k: on(v) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
        shared_prefix_decode(c["q"], c["k_cache"], c["v_cache"], c["prefix_tables"], c["prefix_lens"], c["cu_groups"],
                             c["block_tables"], c["context_lens"], c["scale"])

    failed = []

    def caller(f, arg):
        try:
            f(arg)
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=caller, args=a) for a in ((verify, 3), (verify, 9), (attend, 2), (attend, 30))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed and len(library.seen) == 4
    spans = sorted((a, a + n) for a, n in library.seen)
    assert all(n > 0 for _, n in library.seen)
    assert all(end <= begin for (_, end), (begin, _) in zip(spans, spans[1:]))
