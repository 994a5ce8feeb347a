"""Edge cases of the paged cache's host side that need no GPU."""
import sys
import threading
import types

import pytest
import torch

import anchor_attention_b200 as aa
from anchor_attention_b200 import build, paged


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


def _attend_args(B=2, H=4, Hkv=2):
    zeros = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    return dict(query=zeros(B, H, 128), k_pages=zeros(8, Hkv, 16, 128), v_pages=zeros(8, Hkv, 16, 128),
                block_table=torch.zeros(B, 3, dtype=torch.int32), seq_lens=torch.ones(B, dtype=torch.int32))


@pytest.mark.parametrize("out", [
    torch.zeros(1, 4, 128, dtype=torch.bfloat16).expand(2, 4, 128), torch.zeros(2, 1, 128, dtype=torch.bfloat16).expand(2, 4, 128)])
def test_an_output_whose_rows_share_memory_is_refused(lib, out):
    with pytest.raises(AssertionError, match="share memory"):
        aa.paged_decode_attention(**_attend_args(), out=out)


def test_an_output_that_overlaps_the_query_in_part_is_refused(lib):
    """The query itself may be the output: a row is read before it is written.  Shifted against it, it may not."""
    memory = torch.zeros(3, 4, 128, dtype=torch.bfloat16)
    args = _attend_args()
    args["query"] = memory[:2]
    with pytest.raises(AssertionError, match="overlap"):
        aa.paged_decode_attention(**args, out=memory[1:])
    for out in (memory[:2], torch.zeros(2, 4, 128, dtype=torch.bfloat16)):
        with pytest.raises(AssertionError, match="no CPU path"):
            aa.paged_decode_attention(**args, out=out)


@pytest.mark.parametrize("name", ["k_pages", "v_pages"])
def test_pools_whose_pages_share_memory_are_not_appended_to(lib, name):
    args = _attend_args()
    del args["query"]
    args["key"] = args["value"] = torch.zeros(2, 2, 128, dtype=torch.bfloat16)
    args[name] = torch.zeros(1, 2, 16, 128, dtype=torch.bfloat16).expand(8, 2, 16, 128)
    with pytest.raises(AssertionError, match="share memory"):
        aa.paged_kv_append(**args)


def test_the_library_builds_where_torch_is_missing(lib, monkeypatch, tmp_path, capsys):
    """The C interface needs neither torch nor Python: without torch the library is built and the Python entry points are left out."""
    monkeypatch.setattr(build, "BINDING", str(tmp_path / "_paged_binding.so"))
    monkeypatch.setitem(sys.modules, "torch", None)                         # importing it raises ImportError
    assert build.build_library() == build.LIB
    assert not (tmp_path / "_paged_binding.so").exists()
    assert "torch" in capsys.readouterr().err
