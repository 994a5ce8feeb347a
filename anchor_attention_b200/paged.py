"""Token generation behind an anchor-attention prefill: a paged key-value cache.

The reference's decode calls flash-attn on contiguous tensors
(anchor_attn/src/modules/llama/anchor_attention.py:101-113) and has no cache of its own; these
operators are this library's:

* ``paged_kv_append`` -- new keys and values into the pages of a cache, rotated by their positions
  on the way (queries too), with an 8-bit mean key kept for every page that fills up;
* ``paged_decode_attention`` -- attention of one or a few new tokens of every sequence over its pages,
  all of them or a list for each KV head;
* ``select_pages`` -- such lists: the pages whose mean key scores best against the queries, as the
  block-mean scores of ``block_sparse`` pick key blocks for a prefill.

The cache is plain tensors the caller owns: ``k_pages`` and ``v_pages`` [pages, Hkv, page_size, 128], bf16
or float8_e4m3fn (then ``k_scale`` and ``v_scale``, fp32 [Hkv]: a code of head h stands for
code * scale[h]); any strides whose rows of 128 values are contiguous and 16-byte aligned, so a
[pages, page_size, Hkv, 128] tensor is passed as its ``transpose(1, 2)``.  ``block_table`` int32 [B, width]
names the pages of every sequence in order, ``seq_lens`` int32 [B] counts its tokens, new ones included (0:
padding).  What follows a sequence's last page in its row of the table is not read.

All launches are asynchronous on the current stream of the tensors' device.  Nothing is synchronised, so page
numbers and lengths are checked on the device: a bad one is never used as an address, what it names is left
out, and ``check_paged_status`` raises for it afterwards.

The functions are for inference: no gradients flow through them.  They are not registered as torch operators, so
``torch.compile`` breaks its graph at a call (``fullgraph=True`` refuses it); CUDA graphs capture them.
"""
from __future__ import annotations

from typing import Dict, Optional, Tuple

import torch

from . import _lib

__all__ = ["paged_kv_append", "paged_decode_attention", "select_pages", "rotary_tables", "check_paged_status"]

HEAD_DIM = 128

_status: Dict[int, torch.Tensor] = {}
_binding = None


def _load():
    """The native half of these functions (argument checks, outputs, launches).  There is no fallback: a
    library or binding that has not been built raises."""
    global _binding
    _lib.load()
    try:
        from . import _paged_binding
    except ImportError as e:
        raise RuntimeError(f"_paged_binding.so is missing or does not load ({e}): build it with "
                           "`python -m anchor_attention_b200.build` (there is no fallback implementation)")
    _paged_binding.setup(_status, _new_status_word)
    _binding = _paged_binding
    return _binding


def _new_status_word(index: int) -> torch.Tensor:
    """The word of a device in which the kernels leave bad page numbers and lengths; made with the first call
    on the device, never cleared by one."""
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("paged cache: make one call on this device before capturing one into a CUDA graph")
    device = torch.device("cuda", index)
    word = torch.zeros(1, dtype=torch.int32, device=device)
    torch.cuda.current_stream(device).synchronize()          # whatever stream comes next sees the zero
    # Another thread's first call may have got here during the wait: its word is kept, and both calls use it.
    return _status.setdefault(index, word)


def check_paged_status(device=None) -> None:
    """Synchronises the current stream and raises if a call since the last check met a page number outside the
    pool, a list entry outside its sequence, or a sequence longer than its row of the block table (or than
    the rotary tables), or if a bounded wait of the attention kernel gave up.  The message names every kind that was met, and what it
    names is cleared.  Work of other streams is covered as far as it is done: wait for it first."""
    index = torch.device(device).index if device is not None else None
    index = torch.cuda.current_device() if index is None else index
    word = _status.get(index)
    if word is None:
        return
    check, met = _lib.load().aa_paged_check_status, {}
    with torch.cuda.device(index):
        for _ in range(3):                                   # the kinds there are, one a call
            rc = check(word.data_ptr(), torch.cuda.current_stream().cuda_stream)
            if rc == _lib.AA_OK:
                break
            met[rc] = _lib.error_text(rc)
            if rc == _lib.AA_ERR_CUDA:
                break
    if met:
        raise RuntimeError(f"paged cache: {'; '.join(met.values())}")


def rotary_tables(inv_freq: torch.Tensor, positions: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin), fp32 [positions, 64], of the angles position * inv_freq (64 frequencies, as a model's rotary
    embedding holds them), formed in 64 bits: at position 100000 a 32-bit angle is off by 0.004."""
    assert inv_freq.dim() == 1 and inv_freq.numel() == HEAD_DIM // 2, "inv_freq must hold 64 frequencies"
    angle = torch.arange(positions, dtype=torch.float64, device=inv_freq.device)[:, None] * inv_freq.double()
    return angle.cos().float(), angle.sin().float()


def paged_kv_append(key, value, k_pages, v_pages, block_table, seq_lens, cu_seqlens=None, query=None, cos=None, sin=None,
                    k_scale=None, v_scale=None, key_codes=None, key_code_scales=None, return_key: bool = False):
    """Append new tokens to a paged cache.  ``key``, ``value`` [T, Hkv, 128] bf16, in the order of the sequences:
    sequence b owns tokens ``cu_seqlens[b]`` .. ``cu_seqlens[b + 1] - 1`` (int32 [B + 1]), or T / B tokens where
    ``cu_seqlens`` is None; they take the positions ``seq_lens[b] - n`` .. ``seq_lens[b] - 1`` and must fall
    on pages no other sequence appends to.  Tokens that would take a negative position (all of a sequence of
    length 0) and tokens behind ``cu_seqlens[B]`` are padding: nothing of theirs is written.  ``cu_seqlens`` must ascend from 0
    or more to at most T; a range that does not is left out like padding, and not reported.

    With ``cos`` and ``sin`` (fp32 [positions, 64], see ``rotary_tables``) keys are rotated (rotate-half) by their
    position, in 32 bits with one rounding at the end.  ``query`` [T, H, 128] is rotated likewise.  With
    ``key_codes`` (int8 [pages, Hkv, 128]) and ``key_code_scales`` (fp32 [pages, Hkv]) every page whose last row this
    call writes gets its mean key in 8 bits, which ``select_pages`` reads.

    Returns ``(rotated query or None, rotated key if return_key else None)``, new [T, heads, 128] tensors; rows of
    padding tokens in them are undefined.  One launch; its result does not depend on how tokens are
    spread over calls."""
    return (_binding or _load()).append(key, value, k_pages, v_pages, block_table, seq_lens, cu_seqlens, query, cos, sin, k_scale,
                                        v_scale, key_codes, key_code_scales, return_key)


def paged_decode_attention(query, k_pages, v_pages, block_table, seq_lens, scaling: Optional[float] = None, k_scale=None,
                           v_scale=None, pages=None, page_counts=None, out: Optional[torch.Tensor] = None,
                           return_lse: bool = False):
    """Attention of the last tokens of every sequence over a paged cache that holds them already.  ``query``
    [B, H, 128] (one new token) or [B, n, H, 128] with n up to 16 (row j is position ``seq_lens[b] - n + j`` and sees
    positions up to its own); query head h reads KV head h // (H / Hkv); ``scaling`` defaults to 128 ** -0.5 (0 gives
    all keys the same weight).

    With ``pages`` (int32 [B, Hkv, width]) and ``page_counts`` (int32 [B, Hkv]), both contiguous, a KV head attends
    only the first ``page_counts`` logical pages of its list, in any order; a page listed twice counts twice.  Tables and lists
    may name up to 2^30 tokens a row, n * H / Hkv may be up to 65536 (the cache is read once for every 32 of these rows).

    Returns the output in the shape of ``query`` (``out``, if given: a strided view, or ``query`` itself, but not memory
    that overlaps it otherwise), and with ``return_lse`` also the natural logarithm of the softmax sums, fp32 of shape
    ``query.shape[:-1]``.  A row that sees nothing is 0, its logarithm -inf.  Scores, softmax and sums are 32-bit; the
    other lengths of the batch and the widths of table and lists change results only through the order of sums."""
    return (_binding or _load()).attend(query, k_pages, v_pages, block_table, seq_lens, scaling, k_scale, v_scale, pages,
                                        page_counts, out, return_lse)


def select_pages(query, key_codes, key_code_scales, block_table, seq_lens, top_k: int, page_size: int, keep_first: int = 1,
                 keep_last: int = 2):
    """The pages ``paged_decode_attention`` should read for every sequence and KV head: the first ``keep_first`` and
    the last ``keep_last`` pages of the sequence, then those whose mean key (``key_codes``, ``key_code_scales``, kept by
    ``paged_kv_append``) scores best against the head's query rows, ``top_k`` in all.  ``query`` as in
    ``paged_decode_attention``, rotated and finite.  A score is the maximum over the rows of the 8-bit dot product
    times both scales; a tie goes to the lower page.  ``keep_last`` must be at least 1: a last page that is not full has
    no mean yet.  The block table may be up to 40960 pages wide, and n * H / Hkv up to 256; more is refused.

    Returns ``(pages int32 [B, Hkv, top_k], counts int32 [B, Hkv])``: logical pages, ascending, -1 behind the
    counts."""
    return (_binding or _load()).select(query, key_codes, key_code_scales, block_table, seq_lens, top_k, page_size, keep_first,
                                        keep_last)
