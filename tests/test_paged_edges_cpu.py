"""Edge cases of the paged cache's host side that need no GPU."""
import threading
import types

import torch

from anchor_attention_b200 import paged


def test_first_calls_of_two_threads_share_a_status_word(monkeypatch):
    """Both threads find no word for the device and make one; the interpreter lock is given up while they wait for their
    streams.  One word is kept, and both calls get that one: kernels write to its address."""
    meet = threading.Barrier(2, timeout=20)
    zeros = torch.zeros
    monkeypatch.setattr(paged, "_status", {})
    monkeypatch.setattr(paged.torch, "zeros", lambda *a, device=None, **k: zeros(*a, **k))
    monkeypatch.setattr(paged.torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(paged.torch.cuda, "current_stream", lambda device=None: types.SimpleNamespace(synchronize=meet.wait))
    words = [None, None]

    def first_call(i):
        words[i] = paged._new_status_word(3)

    threads = [threading.Thread(target=first_call, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(30)
    assert words[0] is not None and words[0] is words[1] and paged._status == {3: words[0]}
