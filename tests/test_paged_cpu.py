"""The paged-cache entry points without a GPU: refusals of the Python functions and of the C ABI, the layout of
the argument blocks, and the oracle against a second formulation."""
import ctypes
import math
import os
import re

import pytest
import torch

import anchor_attention_b200 as aa
from anchor_attention_b200 import _lib
from oracle import paged_oracle as oracle
from paged_util import make_pool, make_table

HEADER = os.path.join(os.path.dirname(__file__), "..", "include", "anchor_attn_b200.h")


def _tensors(B=2, Hkv=2, H=4, page=16, pages=8, T=2):
    return dict(
        key=torch.zeros(T, Hkv, 128, dtype=torch.bfloat16), value=torch.zeros(T, Hkv, 128, dtype=torch.bfloat16),
        query=torch.zeros(T, H, 128, dtype=torch.bfloat16),
        k_pages=torch.zeros(pages, Hkv, page, 128, dtype=torch.bfloat16),
        v_pages=torch.zeros(pages, Hkv, page, 128, dtype=torch.bfloat16),
        block_table=torch.zeros(B, 3, dtype=torch.int32), seq_lens=torch.ones(B, dtype=torch.int32))


APPEND = [
    (dict(k_pages=torch.zeros(8, 2, 16, 64, dtype=torch.bfloat16)), "page_size, 128"),
    (dict(k_pages=torch.zeros(8, 2, 24, 128, dtype=torch.bfloat16), v_pages=torch.zeros(8, 2, 24, 128, dtype=torch.bfloat16)),
     "power of two"),
    (dict(k_pages=torch.zeros(8, 2, 16, 128, dtype=torch.float16)), "both be bfloat16"),
    (dict(v_pages=torch.zeros(8, 2, 16, 128).to(torch.float8_e4m3fn)), "both be bfloat16"),
    (dict(k_scale=torch.ones(2)), "belong to float8"),
    (dict(key=torch.zeros(2, 2, 128)), "key must be bfloat16"),
    (dict(key=torch.zeros(2, 3, 128, dtype=torch.bfloat16), value=torch.zeros(2, 3, 128, dtype=torch.bfloat16)), "KV heads"),
    (dict(value=torch.zeros(2, 2, 64, dtype=torch.bfloat16)), "head dimension 64"),
    (dict(key=torch.zeros(3, 2, 128, dtype=torch.bfloat16), value=torch.zeros(3, 2, 128, dtype=torch.bfloat16)), "do not divide"),
    (dict(query=torch.zeros(2, 3, 128, dtype=torch.bfloat16)), "multiple of the KV heads"),
    (dict(block_table=torch.zeros(2, 3, dtype=torch.int64)), "block_table must be a 2-dimensional int32"),
    (dict(seq_lens=torch.ones(3, dtype=torch.int32)), "seq_lens must be"),
    (dict(cu_seqlens=torch.zeros(2, dtype=torch.int32)), "B \\+ 1"),
    (dict(cos=torch.zeros(4, 64)), "cos and sin go together"),
    (dict(cos=torch.zeros(4, 128), sin=torch.zeros(4, 128)), "positions, 64"),
    (dict(key_codes=torch.zeros(8, 2, 128, dtype=torch.int8)), "go together"),
    (dict(key_codes=torch.zeros(7, 2, 128, dtype=torch.int8), key_code_scales=torch.zeros(7, 2)), "every page"),
    (dict(), "no CPU path"),
]


@pytest.mark.parametrize("change,message", APPEND)
def test_append_refusals(lib, change, message):
    with pytest.raises(AssertionError, match=message):
        aa.paged_kv_append(**{**_tensors(), **change})


ATTEND = [
    (dict(query=torch.zeros(2, 17, 4, 128, dtype=torch.bfloat16)), "17 new tokens"),
    (dict(query=torch.zeros(2, 0, 4, 128, dtype=torch.bfloat16)), "0 new tokens"),
    (dict(query=torch.zeros(2, 3, 128, dtype=torch.bfloat16)), "do not divide"),
    (dict(query=torch.zeros(3, 4, 128, dtype=torch.bfloat16)), "new tokens, H, 128"),
    (dict(query=torch.zeros(2, 4, 128, dtype=torch.float16)), "query must be bfloat16"),
    (dict(pages=torch.zeros(2, 2, 3, dtype=torch.int32)), "go together"),
    (dict(pages=torch.zeros(2, 4, 3, dtype=torch.int32), page_counts=torch.zeros(2, 2, dtype=torch.int32)), "B, Hkv, width"),
    (dict(pages=torch.zeros(2, 2, 3, dtype=torch.int32), page_counts=torch.zeros(2, 3, dtype=torch.int32)), "page_counts must be"),
    (dict(out=torch.zeros(2, 4, 129, dtype=torch.bfloat16)[..., 1:]), "out must have"),
    (dict(k_pages=torch.zeros(8, 2, 16, 128).to(torch.float8_e4m3fn), v_pages=torch.zeros(8, 2, 16, 128).to(torch.float8_e4m3fn)),
     "k_scale must be"),
    (dict(), "no CPU path"),
]


@pytest.mark.parametrize("change,message", ATTEND)
def test_attend_refusals(lib, change, message):
    t = _tensors()
    args = dict(query=torch.zeros(2, 4, 128, dtype=torch.bfloat16), **{n: t[n] for n in ("k_pages", "v_pages", "block_table", "seq_lens")})
    with pytest.raises(AssertionError, match=message):
        aa.paged_decode_attention(**{**args, **change})


SELECT = [
    (dict(page_size=48), "power of two"),
    (dict(top_k=2), "top_k hold both"),
    (dict(keep_last=0), "keep_last at least 1"),
    (dict(key_codes=torch.zeros(8, 2, 64, dtype=torch.int8)), "key_codes must be"),
    (dict(key_code_scales=torch.zeros(8, 3)), "key_code_scales must be"),
    (dict(query=torch.zeros(2, 5, 128, dtype=torch.bfloat16)), "do not divide"),
    (dict(), "no CPU path"),
]


@pytest.mark.parametrize("change,message", SELECT)
def test_select_refusals(lib, change, message):
    t = _tensors()
    args = dict(query=torch.zeros(2, 4, 128, dtype=torch.bfloat16), key_codes=torch.zeros(8, 2, 128, dtype=torch.int8),
                key_code_scales=torch.zeros(8, 2), block_table=t["block_table"], seq_lens=t["seq_lens"], top_k=4, page_size=16)
    with pytest.raises(AssertionError, match=message):
        aa.select_pages(**{**args, **change})


def _cache_block():
    c = _lib.AAPagedCache()
    c.k_pages = c.v_pages = c.block_table = c.seq_lens = c.status = 4096
    c.k_stride_row = c.v_stride_row = 128
    c.table_stride = c.table_width = 4
    c.pages, c.page_size, c.Hkv, c.D, c.B = 8, 16, 2, 128, 2
    return c


@pytest.mark.parametrize("field,value,code", [
    ("B", 0, -2), ("D", 64, -3), ("page_size", 8, -15), ("page_size", 96, -15), ("page_size", 512, -15), ("pages", 0, -15),
    ("table_width", 0, -15), ("block_table", None, -1), ("status", None, -1), ("table_width", 1 << 27, -12),
])
def test_abi_refuses_a_bad_cache(lib, field, value, code):
    c = _cache_block()
    setattr(c, field, value)
    for block, fn in ((_lib.AAPagedAppend(), lib.aa_paged_append), (_lib.AAPagedAttend(), lib.aa_paged_attend),
                      (_lib.AAPageSelect(), lib.aa_page_select)):
        block.cache = c
        assert fn(ctypes.byref(block), None) == code
        assert len(lib.aa_strerror(code)) > 10 and lib.aa_strerror(code) != b"unknown error"


@pytest.mark.parametrize("fields,code", [
    (dict(key=None), -1), (dict(T=0), -2), (dict(T=3), -2), (dict(query=4096, H=3), -2), (dict(query=4096, H=4), -1),
    (dict(key_stride_t=4), -8), (dict(key=4100), -8), (dict(cos=4096), -1), (dict(key_codes=4096), -1),
    (dict(cos=4096, sin=4096), -2),
])
def test_abi_refuses_a_bad_append(lib, fields, code):
    a = _lib.AAPagedAppend()
    a.cache, a.key, a.value, a.T, a.H = _cache_block(), 4096, 4096, 2, 4
    for n, v in fields.items():
        setattr(a, n, v)
    assert lib.aa_paged_append(ctypes.byref(a), None) == code


def test_abi_refuses_bad_pools(lib):
    for field, value, code in (("k_pages", None, -1), ("cache_dtype", 2, -9), ("cache_dtype", 1, -1), ("v_stride_row", 68, -8),
                               ("k_pages", 4104, -8)):
        a = _lib.AAPagedAppend()
        a.cache, a.key, a.value, a.T, a.H = _cache_block(), 4096, 4096, 2, 4
        setattr(a.cache, field, value)
        assert lib.aa_paged_append(ctypes.byref(a), None) == code


@pytest.mark.parametrize("fields,code", [
    (dict(H=3), -2), (dict(Nq=0), -2), (dict(Nq=17), -16), (dict(pages=4096, list_width=4), -1),
    (dict(pages=4096, page_counts=4096, list_width=0), -2), (dict(pages=4096, page_counts=4096, list_width=1 << 28), -12),
])
def test_abi_refuses_a_bad_attend(lib, fields, code):
    a = _lib.AAPagedAttend()
    a.cache, a.q, a.out, a.Nq, a.H = _cache_block(), 4096, 4096, 1, 4
    for n, v in fields.items():
        setattr(a, n, v)
    assert lib.aa_paged_attend(ctypes.byref(a), None) == code
    need = ctypes.c_size_t()
    assert lib.aa_paged_attend_workspace_bytes(ctypes.byref(a), ctypes.byref(need)) == code


@pytest.mark.parametrize("fields,code", [
    (dict(top=0), -2), (dict(keep_last=0), -2), (dict(keep_first=4), -2), (dict(Nq=17), -16), (dict(H=130, Nq=4), -16),
    (dict(key_codes=None), -1), (dict(q=4104), -8),
])
def test_abi_refuses_a_bad_select(lib, fields, code):
    a = _lib.AAPageSelect()
    a.cache, a.q, a.key_codes, a.key_code_scales, a.out, a.counts = _cache_block(), 4096, 4096, 4096, 4096, 4096
    a.Nq, a.H, a.top, a.keep_first, a.keep_last = 1, 4, 4, 1, 2
    for n, v in fields.items():
        setattr(a, n, v)
    assert lib.aa_page_select(ctypes.byref(a), None) == code
    a.cache.table_width = 50000
    assert lib.aa_page_select(ctypes.byref(a), None) in (code, -12)


def test_null_blocks(lib):
    for fn in (lib.aa_paged_append, lib.aa_paged_attend, lib.aa_page_select):
        assert fn(None, None) == -1
    assert lib.aa_paged_check_status(None, None) == -1


@pytest.mark.parametrize("name,struct", [("aa_paged_cache", _lib.AAPagedCache), ("aa_paged_append", _lib.AAPagedAppend),
                                         ("aa_paged_attend", _lib.AAPagedAttend), ("aa_page_select", _lib.AAPageSelect)])
def test_argument_blocks_mirror_the_header(name, struct):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, flags=re.S).group(1)
    fields = []
    for line in body.split(";"):
        for part in line.replace("\n", " ").split(","):
            words = re.findall(r"\w+", part)
            if words:
                fields.append(words[-1])
    assert fields == [f[0] for f in struct._fields_]


def test_rotary_tables():
    inv = 500000.0 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128)
    cos, sin = aa.rotary_tables(inv.float(), 131072)
    assert cos.shape == sin.shape == (131072, 64) and cos.dtype == torch.float32
    for at, d in ((0, 0), (131071, 0), (100003, 7), (77, 63)):
        angle = at * float(inv.float()[d])
        assert abs(float(cos[at, d]) - math.cos(angle)) <= 2 ** -24 and abs(float(sin[at, d]) - math.sin(angle)) <= 2 ** -24
    with pytest.raises(AssertionError, match="64 frequencies"):
        aa.rotary_tables(inv[:32], 8)


@pytest.mark.parametrize("picked", [False, True])
def test_oracle_against_dense_formulation(picked):
    """The per-sequence oracle against one masked softmax over the gathered cache."""
    g = torch.Generator().manual_seed(0)
    lens, page, H, Hkv, n = [37, 0, 16, 3], 16, 6, 2, 4
    table, total = make_table(lens, page, g)
    k, v, _, _ = make_pool(total, Hkv, page, g, False)
    q = torch.randn(4, n, H, 128, generator=g).bfloat16()
    kw = {}
    if picked:
        kw = dict(pages=torch.tensor([[[0, 2], [1, 1]]] * 4, dtype=torch.int32), page_counts=torch.tensor([[2, 1]] * 4, dtype=torch.int32))
        kw["page_counts"][1:] = 0
    out, lse, weight, _ = oracle.attend(q, k.double(), v.double(), table, lens, **kw)
    for b, length in enumerate(lens):
        for h in range(H):
            at = torch.arange(table.shape[1] * page)
            if picked:
                rows = kw["pages"][b, h // 3, :int(kw["page_counts"][b, h // 3])].long()
                at = (rows[:, None] * page + torch.arange(page)).flatten()
            phys = table[b][at // page].long().clamp(min=0)
            K, V = k[phys, h // 3, at % page].double(), v[phys, h // 3, at % page].double()
            for j in range(n):
                s = K @ q[b, j, h].double() / math.sqrt(128)
                s[at > length - n + j] = -math.inf
                if torch.isinf(s).all():
                    assert lse[b, j, h] == -math.inf and (out[b, j, h] == 0).all()
                    continue
                p = (s - s.max()).exp()
                assert torch.allclose(out[b, j, h], (p / p.sum()) @ V, atol=1e-12)
                assert abs(float(lse[b, j, h]) - float(s.max() + p.sum().log())) < 1e-12


def test_oracle_selection_keeps_ends_and_breaks_ties_low():
    codes = torch.zeros(10, 1, 128, dtype=torch.int8)
    codes[:, 0, 0] = torch.tensor([0, 5, 9, 9, 9, 1, 9, 2, 0, 0])
    table = torch.arange(10, dtype=torch.int32)[None]
    q = torch.zeros(1, 1, 1, 128)
    q[..., 0] = 1.0
    lists, counts = oracle.select(q.bfloat16(), codes, torch.ones(10, 1), table, [150], 5, 16)
    assert counts.item() == 5 and lists[0, 0].tolist() == [0, 2, 3, 8, 9]
    lists, counts = oracle.select(q.bfloat16(), codes, torch.ones(10, 1), table, [33], 5, 16)
    assert counts.item() == 3 and lists[0, 0].tolist() == [0, 1, 2, -1, -1]


class _NoTruth:
    def __bool__(self):
        raise ValueError("no truth value")


def test_flags_without_a_truth_value(lib):
    t = _tensors()
    with pytest.raises(ValueError, match="no truth value"):
        aa.paged_kv_append(**t, return_key=_NoTruth())
    attend = {n: t[n] for n in ("query", "k_pages", "v_pages", "block_table", "seq_lens")}
    with pytest.raises(ValueError, match="no truth value"):
        aa.paged_decode_attention(**attend, return_lse=_NoTruth())
