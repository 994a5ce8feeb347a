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
"""
from __future__ import annotations

import ctypes
from typing import Dict, Optional, Tuple

import torch

from . import _lib

__all__ = ["paged_kv_append", "paged_decode_attention", "select_pages", "rotary_tables", "check_paged_status"]

HEAD_DIM = 128
MAX_NEW_TOKENS = 16          # tokens of one sequence a decode call takes; more belong to dense_causal_attention

_status: Dict[int, torch.Tensor] = {}
_workspace_bytes: Dict[tuple, int] = {}


def _status_word(device: torch.device) -> torch.Tensor:
    """The device word in which the kernels leave bad page numbers and lengths; one a device, never
    cleared by a call."""
    assert device.type == "cuda", "the tensors of a paged cache must be CUDA tensors (there is no CPU path)"
    word = _status.get(device.index)
    if word is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("paged cache: make one call on this device before capturing one into a CUDA graph")
        word = torch.zeros(1, dtype=torch.int32, device=device)
        torch.cuda.current_stream(device).synchronize()      # whatever stream comes next sees the zero
        _status[device.index] = word
    return word


def check_paged_status(device=None) -> None:
    """Synchronises the current stream and raises if a call since the last check met a page number outside the
    pool, a list entry outside its sequence, or a sequence longer than its row of the block table (or than
    the rotary tables)."""
    index = torch.device(device).index if device is not None else None
    index = torch.cuda.current_device() if index is None else index
    word = _status.get(index)
    if word is None:
        return
    with torch.cuda.device(index):
        rc = _lib.load().aa_paged_check_status(word.data_ptr(), torch.cuda.current_stream().cuda_stream)
    if rc != _lib.AA_OK:
        raise RuntimeError(f"paged cache: {_lib.error_text(rc)}")


def rotary_tables(inv_freq: torch.Tensor, positions: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin), fp32 [positions, 64], of the angles position * inv_freq (64 frequencies, as a model's rotary
    embedding holds them), formed in 64 bits: at position 100000 a 32-bit angle is off by 0.004."""
    assert inv_freq.dim() == 1 and inv_freq.numel() == HEAD_DIM // 2, "inv_freq must hold 64 frequencies"
    angle = torch.arange(positions, dtype=torch.float64, device=inv_freq.device)[:, None] * inv_freq.double()
    return angle.cos().float(), angle.sin().float()


def _int32(t, name: str, dim: int, device) -> None:
    assert t.dtype == torch.int32 and t.dim() == dim and t.device == device, \
        f"{name} must be a {dim}-dimensional int32 tensor on the device of the inputs"


def _rows(t, name: str, device) -> None:
    """A bf16 tensor whose last axis is a row of 128 values the kernels can read in 16-byte pieces."""
    assert t.dtype == torch.bfloat16 and t.device == device, f"{name} must be bfloat16 on the device of the other tensors"
    assert t.shape[-1] == HEAD_DIM, f"head dimension {t.shape[-1]} is not supported (128 only)"


def _usable(t):
    """``t``, or a copy where its rows are not contiguous or its strides or address not multiples of 16 bytes."""
    st = t.stride()
    ok = st[-1] == 1 and not t.data_ptr() & 15
    for s in st[:-1]:
        ok = ok and not s & 7
    return t if ok else t.contiguous()


def _cache(k_pages, v_pages, block_table, seq_lens, k_scale, v_scale):
    """The cache block of a call, its tensors checked; the status word is still missing."""
    device = k_pages.device
    shape = k_pages.shape
    assert len(shape) == 4 and v_pages.shape == shape and shape[3] == HEAD_DIM, \
        "k_pages and v_pages must both be [pages, Hkv, page_size, 128]"
    fp8 = k_pages.dtype == torch.float8_e4m3fn
    assert (fp8 or k_pages.dtype == torch.bfloat16) and v_pages.dtype == k_pages.dtype and v_pages.device == device, \
        "k_pages and v_pages must both be bfloat16 or both float8_e4m3fn, on one device"
    page = shape[2]
    assert 16 <= page <= 256 and not page & (page - 1), f"page size {page} is not a power of two from 16 to 256"
    ks, vs = k_pages.stride(), v_pages.stride()
    assert ks[3] == 1 and vs[3] == 1, "the rows of the pools must be contiguous"
    ksp = vsp = None
    if fp8:
        for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            assert t is not None and t.dtype == torch.float32 and t.shape == (shape[1],) and t.device == device \
                and t.is_contiguous(), f"{name} must be a contiguous fp32 [Hkv] tensor: the pools are float8_e4m3fn"
        ksp, vsp = k_scale.data_ptr(), v_scale.data_ptr()
    else:
        assert k_scale is None and v_scale is None, "k_scale and v_scale belong to float8_e4m3fn pools"
    B, width, table_stride = _table(block_table, seq_lens, device)
    return _lib.AAPagedCache(k_pages.data_ptr(), v_pages.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], ksp, vsp,
                             block_table.data_ptr(), table_stride, seq_lens.data_ptr(), None, shape[0], page, width, shape[1],
                             HEAD_DIM, _lib.AA_E4M3 if fp8 else _lib.AA_BF16, B)


def _table(block_table, seq_lens, device):
    _int32(block_table, "block_table", 2, device)
    _int32(seq_lens, "seq_lens", 1, device)
    B, width = block_table.shape
    assert seq_lens.shape[0] == B and (B < 2 or seq_lens.stride(0) == 1), "seq_lens must be a contiguous [B] tensor"
    assert width >= 1 and (width == 1 or block_table.stride(1) == 1), "the rows of block_table must be contiguous"
    return B, width, block_table.stride(0)


def _launch(fn, args, device, what: str) -> None:
    index = device.index
    stream = torch.cuda.current_stream(device).cuda_stream
    if index == torch.cuda.current_device():
        rc = fn(args, stream)
    else:
        with torch.cuda.device(index):
            rc = fn(args, stream)
    if rc != _lib.AA_OK:
        raise RuntimeError(f"{what}: {_lib.error_text(rc)}")


def paged_kv_append(key, value, k_pages, v_pages, block_table, seq_lens, cu_seqlens=None, query=None, cos=None, sin=None,
                    k_scale=None, v_scale=None, key_codes=None, key_code_scales=None, return_key: bool = False):
    """Append new tokens to a paged cache.  ``key``, ``value`` [T, Hkv, 128] bf16, in the order of the sequences:
    sequence b owns tokens ``cu_seqlens[b]`` .. ``cu_seqlens[b + 1] - 1`` (int32 [B + 1]), or T / B tokens where
    ``cu_seqlens`` is None; they take the positions ``seq_lens[b] - n`` .. ``seq_lens[b] - 1`` and must fall
    on pages no other sequence appends to.  Tokens that would take a negative position (all of a sequence of
    length 0) and tokens behind ``cu_seqlens[B]`` are padding: nothing of theirs is written.

    With ``cos`` and ``sin`` (fp32 [positions, 64], see ``rotary_tables``) keys are rotated (rotate-half) by their
    position, in 32 bits with one rounding at the end.  ``query`` [T, H, 128] is rotated likewise.  With
    ``key_codes`` (int8 [pages, Hkv, 128]) and ``key_code_scales`` (fp32 [pages, Hkv]) every page whose last row this
    call writes gets its mean key in 8 bits, which ``select_pages`` reads.

    Returns ``(rotated query or None, rotated key if return_key else None)``, new [T, heads, 128] tensors; rows of
    padding tokens in them are undefined.  One launch; its result does not depend on how tokens are
    spread over calls."""
    lib = _lib.load()
    device = k_pages.device
    c = _cache(k_pages, v_pages, block_table, seq_lens, k_scale, v_scale)
    _rows(key, "key", device)
    _rows(value, "value", device)
    assert key.dim() == 3 and value.shape == key.shape and key.shape[1] == c.Hkv, \
        "key and value must be [T, Hkv, 128] with the KV heads of the pools"
    T, B = key.shape[0], c.B
    if cu_seqlens is not None:
        _int32(cu_seqlens, "cu_seqlens", 1, device)
        assert cu_seqlens.shape[0] == B + 1 and cu_seqlens.stride(0) == 1, "cu_seqlens must be a contiguous [B + 1] tensor"
    else:
        assert B == 0 or T % B == 0, f"{T} tokens do not divide among {B} sequences: pass cu_seqlens"
    assert (cos is None) == (sin is None), "cos and sin go together"
    rope_rows = 0
    if cos is not None:
        for t in (cos, sin):
            assert t.dtype == torch.float32 and t.dim() == 2 and t.shape[1] == HEAD_DIM // 2 and t.is_contiguous() \
                and t.device == device, "cos and sin must be contiguous fp32 [positions, 64] tensors"
        rope_rows = min(cos.shape[0], sin.shape[0])
    assert (key_codes is None) == (key_code_scales is None), "key_codes and key_code_scales go together"
    if key_codes is not None:
        _check_codes(key_codes, key_code_scales, c.Hkv, device)
        assert key_codes.shape[0] == c.pages, "key_codes must have a row for every page of the pools"
    query_out = key_out = None
    H = 0
    if query is not None:
        _rows(query, "query", device)
        assert query.dim() == 3 and query.shape[0] == T and query.shape[1] % c.Hkv == 0 and query.shape[1] > 0, \
            "query must be [T, H, 128] with a multiple of the KV heads"
    c.status = _status_word(device).data_ptr()
    if query is not None:
        H = query.shape[1]
        query = _usable(query)
        query_out = torch.empty((T, H, HEAD_DIM), dtype=query.dtype, device=device)
    if return_key:
        key_out = torch.empty((T, c.Hkv, HEAD_DIM), dtype=key.dtype, device=device)
    if T == 0 or B == 0:
        return query_out, key_out
    key, value = _usable(key), _usable(value)
    kst, vst = key.stride(), value.stride()
    qst = query.stride() if query is not None else (0, 0)
    a = _lib.AAPagedAppend(
        c, key.data_ptr(), value.data_ptr(), None if query is None else query.data_ptr(),
        None if query_out is None else query_out.data_ptr(), None if key_out is None else key_out.data_ptr(),
        kst[0], kst[1], vst[0], vst[1], qst[0], qst[1], H * HEAD_DIM, HEAD_DIM, c.Hkv * HEAD_DIM, HEAD_DIM,
        None if cu_seqlens is None else cu_seqlens.data_ptr(), None if cos is None else cos.data_ptr(),
        None if sin is None else sin.data_ptr(), None if key_codes is None else key_codes.data_ptr(),
        None if key_code_scales is None else key_code_scales.data_ptr(), rope_rows, T, H, 0)
    _launch(lib.aa_paged_append, a, device, "paged_kv_append")
    return query_out, key_out


def _check_codes(key_codes, key_code_scales, Hkv, device) -> None:
    assert key_codes.dtype == torch.int8 and key_codes.dim() == 3 and key_codes.shape[1:] == (Hkv, HEAD_DIM) \
        and key_codes.is_contiguous() and key_codes.device == device, \
        "key_codes must be a contiguous int8 [pages, Hkv, 128] tensor"
    assert key_code_scales.dtype == torch.float32 and key_code_scales.shape == key_codes.shape[:2] \
        and key_code_scales.is_contiguous() and key_code_scales.device == device, \
        "key_code_scales must be a contiguous fp32 [pages, Hkv] tensor"


def _queries(query, Hkv: int, B: int):
    """``query`` as [B, new, H, 128] the kernels can read; its number of new tokens and heads."""
    q = query if query.dim() == 4 else query.unsqueeze(1)
    assert q.dim() == 4 and q.shape[0] == B, "query must be [B, H, 128] or [B, new tokens, H, 128]"
    new, H = q.shape[1], q.shape[2]
    assert 1 <= new <= MAX_NEW_TOKENS, \
        f"{new} new tokens: 1 to {MAX_NEW_TOKENS} are supported (dense_causal_attention takes longer chunks)"
    assert H % Hkv == 0 and H > 0, f"{Hkv} KV heads do not divide {H} query heads"
    return _usable(q), new, H


def paged_decode_attention(query, k_pages, v_pages, block_table, seq_lens, scaling: Optional[float] = None, k_scale=None,
                           v_scale=None, pages=None, page_counts=None, out: Optional[torch.Tensor] = None,
                           return_lse: bool = False):
    """Attention of the last tokens of every sequence over a paged cache that holds them already.  ``query``
    [B, H, 128] (one new token) or [B, n, H, 128] with n up to 16 (row j is position ``seq_lens[b] - n + j`` and sees
    positions up to its own); query head h reads KV head h // (H / Hkv); ``scaling`` defaults to 128 ** -0.5.

    With ``pages`` (int32 [B, Hkv, width]) and ``page_counts`` (int32 [B, Hkv]), both contiguous, a KV head attends
    only the first ``page_counts`` logical pages of its list, in any order; a page listed twice counts twice.

    Returns the output in the shape of ``query`` (``out``, which may be a strided view, if given), and with
    ``return_lse`` also the natural logarithm of the softmax sums, fp32 of shape ``query.shape[:-1]``.  A row that
    sees nothing is 0, its logarithm -inf.  Scores, softmax and sums are 32-bit; results depend on the lengths
    in the batch only through the order of sums."""
    lib = _lib.load()
    device = k_pages.device
    c = _cache(k_pages, v_pages, block_table, seq_lens, k_scale, v_scale)
    _rows(query, "query", device)
    q, new, H = _queries(query, c.Hkv, c.B)
    list_width = 0
    assert (pages is None) == (page_counts is None), "pages and page_counts go together"
    if pages is not None:
        _int32(pages, "pages", 3, device)
        _int32(page_counts, "page_counts", 2, device)
        list_width = pages.shape[2]
        assert pages.shape[:2] == (c.B, c.Hkv) and list_width >= 1 and pages.is_contiguous(), \
            "pages must be a contiguous [B, Hkv, width] tensor"
        assert page_counts.shape == (c.B, c.Hkv) and page_counts.is_contiguous(), \
            "page_counts must be a contiguous [B, Hkv] tensor"
    if out is not None:
        _rows(out, "out", device)
        assert out.shape == query.shape and _usable(out) is out, \
            "out must have the shape of query, contiguous rows and strides and address of 16-byte multiples"
    c.status = _status_word(device).data_ptr()
    if out is None:
        out = torch.empty(query.shape, dtype=query.dtype, device=device)
    lse = torch.empty(query.shape[:-1], dtype=torch.float32, device=device) if return_lse else None
    if c.B == 0:
        return (out, lse) if return_lse else out
    o = out if out.dim() == 4 else out.unsqueeze(1)
    qst, ost = q.stride(), o.stride()
    a = _lib.AAPagedAttend(c, q.data_ptr(), o.data_ptr(), None if lse is None else lse.data_ptr(), qst[0], qst[1], qst[2],
                           ost[0], ost[1], ost[2], None if pages is None else pages.data_ptr(),
                           None if page_counts is None else page_counts.data_ptr(), None, 0,
                           float(scaling) if scaling else 0.0, list_width, new, H, 0)
    # The workspace is this call's own (the allocator hands it out again in stream order): calls on other streams,
    # and graphs captured from different calls, never meet in one.
    key = (device.index, c.B, c.Hkv, H, new, c.table_width, c.page_size, list_width)
    nbytes = _workspace_bytes.get(key)
    if nbytes is None:
        need = ctypes.c_size_t(0)
        with torch.cuda.device(device.index):
            rc = lib.aa_paged_attend_workspace_bytes(ctypes.byref(a), ctypes.byref(need))
        if rc != _lib.AA_OK:
            raise RuntimeError(f"paged_decode_attention: {_lib.error_text(rc)}")
        if len(_workspace_bytes) > 4096:
            _workspace_bytes.clear()
        nbytes = _workspace_bytes[key] = need.value
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
    a.workspace, a.workspace_bytes = workspace.data_ptr(), nbytes
    _launch(lib.aa_paged_attend, a, device, "paged_decode_attention")
    return (out, lse) if return_lse else out


def select_pages(query, key_codes, key_code_scales, block_table, seq_lens, top_k: int, page_size: int, keep_first: int = 1,
                 keep_last: int = 2):
    """The pages ``paged_decode_attention`` should read for every sequence and KV head: the first ``keep_first`` and
    the last ``keep_last`` pages of the sequence, then those whose mean key (``key_codes``, ``key_code_scales``, kept by
    ``paged_kv_append``) scores best against the head's query rows, ``top_k`` in all.  ``query`` as in
    ``paged_decode_attention``, rotated and finite.  A score is the maximum over the rows of the 8-bit dot product
    times both scales; a tie goes to the lower page.  ``keep_last`` must be at least 1: a last page that is not full has
    no mean yet.

    Returns ``(pages int32 [B, Hkv, top_k], counts int32 [B, Hkv])``: logical pages, ascending, -1 behind the
    counts."""
    lib = _lib.load()
    device = query.device
    _rows(query, "query", device)
    assert key_codes.dim() == 3, "key_codes must be a contiguous int8 [pages, Hkv, 128] tensor"
    Hkv = key_codes.shape[1]
    _check_codes(key_codes, key_code_scales, Hkv, device)
    B, width, table_stride = _table(block_table, seq_lens, device)
    q, new, H = _queries(query, Hkv, B)
    assert 16 <= page_size <= 256 and not page_size & (page_size - 1), \
        f"page size {page_size} is not a power of two from 16 to 256"
    assert keep_first >= 0 and keep_last >= 1 and top_k >= keep_first + keep_last, \
        "keep_first must be at least 0, keep_last at least 1, and top_k hold both"
    status = _status_word(device).data_ptr()
    pages = torch.empty((B, Hkv, top_k), dtype=torch.int32, device=device)
    counts = torch.empty((B, Hkv), dtype=torch.int32, device=device)
    if B == 0:
        return pages, counts
    c = _lib.AAPagedCache(None, None, 0, 0, 0, 0, 0, 0, None, None, block_table.data_ptr(), table_stride, seq_lens.data_ptr(),
                          status, key_codes.shape[0], page_size, width, Hkv, HEAD_DIM, _lib.AA_BF16, B)
    st = q.stride()
    a = _lib.AAPageSelect(c, q.data_ptr(), st[0], st[1], st[2], key_codes.data_ptr(), key_code_scales.data_ptr(),
                          pages.data_ptr(), counts.data_ptr(), new, H, top_k, keep_first, keep_last, 0)
    _launch(lib.aa_page_select, a, device, "select_pages")
    return pages, counts
