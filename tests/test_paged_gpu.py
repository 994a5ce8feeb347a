"""The paged key-value cache on the GPU against the 64-bit oracle: append with rotation, decode attention over all
pages and over picked ones, page selection; then the three together behind a prefill."""
import math

import pytest
import torch

import anchor_attention_b200 as aa
from oracle import paged_oracle as oracle
from paged_util import assert_decode, make_pool, make_table

pytestmark = pytest.mark.gpu

HEADS = [(32, 8), (28, 4), (4, 4), (8, 1), (6, 2)]


@pytest.fixture(autouse=True)
def _clean_status(lib):
    aa.check_paged_status()
    yield
    aa.check_paged_status()


def _decode_case(seed, lens, page, H, Hkv, n, fp8, nhd=False, width=None):
    g = torch.Generator().manual_seed(seed)
    table, total = make_table(lens, page, g, width=width)
    k, v, ks, vs = make_pool(total, Hkv, page, g, fp8, nhd)
    q = (torch.randn(len(lens), n, H, 128, generator=g) * 1.5).bfloat16()
    return q, k, v, ks, vs, table, torch.tensor(lens, dtype=torch.int32)


def _cuda(*ts):
    """The same memory layout on the GPU (``Tensor.cuda`` keeps strides of dense views)."""
    return [None if t is None else t.cuda() for t in ts]


def _run(q, k, v, ks, vs, table, lens, **kw):
    q, k, v, ks, vs, table, lens = _cuda(q, k, v, ks, vs, table, lens)
    return aa.paged_decode_attention(q, k, v, table, lens, k_scale=ks, v_scale=vs, return_lse=True, **kw)


# ---------------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("H,Hkv", HEADS)
def test_decode_lengths(H, Hkv, page, fp8):
    lens = [1, 15, 16, 17, 63, 64, 65, 0, 129, 1000, 511]
    case = _decode_case(H + page, lens, page, H, Hkv, 1, fp8)
    out, lse = _run(*case)
    q, k, v, ks, vs, table, lens = case
    assert out.shape == q.shape and lse.shape == q.shape[:3]
    assert_decode(out, lse, q, oracle.dequantised(k, ks), oracle.dequantised(v, vs), table, lens, fp8)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n,H,Hkv", [(2, 32, 8), (5, 32, 8), (16, 4, 4), (3, 28, 4), (16, 8, 1), (7, 6, 2), (16, 64, 1)])
def test_several_new_tokens(n, H, Hkv, fp8):
    """Rows from 3 to 1024, in one to many tiles; sequences shorter than the new tokens leave rows empty."""
    lens = [n, 0, 1, n + 15, 200, 77, n - 1]
    case = _decode_case(n, lens, 16, H, Hkv, n, fp8)
    out, lse = _run(*case)
    q, k, v, ks, vs, table, lens = case
    assert_decode(out, lse, q, oracle.dequantised(k, ks), oracle.dequantised(v, vs), table, lens, fp8)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("lens,H,Hkv", [([20000], 8, 1), ([9001, 1, 12000], 8, 2), ([4097] * 40, 4, 4)])
def test_split_over_many_blocks(lens, H, Hkv, fp8):
    """One long sequence cut into hundreds of parts, and many entries with a few cuts."""
    case = _decode_case(3, lens, 64, H, Hkv, 1, fp8)
    out, lse = _run(*case)
    q, k, v, ks, vs, table, lens = case
    assert_decode(out, lse, q, oracle.dequantised(k, ks), oracle.dequantised(v, vs), table, lens, fp8)
    again, _ = _run(*case)
    assert torch.equal(out, again)


@pytest.mark.parametrize("fp8", [False, True])
def test_picked_pages(fp8):
    """Lists of different lengths for each head, unsorted, one page twice, the partial last page in the middle, an
    empty list, a list of the whole sequence."""
    lens, page, H, Hkv, n = [300, 90, 16, 512], 32, 12, 3, 2
    q, k, v, ks, vs, table, lens = _decode_case(5, lens, page, H, Hkv, n, fp8)
    pages = torch.full((4, Hkv, 16), -1, dtype=torch.int32)
    picks = [[[0, 9, 3], [9], [4, 4, 0, 9]], [[2, 0, 1], [], [1]], [[0], [0, 0], []], [[15, 0, 7, 8], list(range(16)), [15]]]
    counts = torch.tensor([[len(x) for x in row] for row in picks], dtype=torch.int32)
    for b, row in enumerate(picks):
        for h, x in enumerate(row):
            pages[b, h, :len(x)] = torch.tensor(x, dtype=torch.int32)
    out, lse = _run(q, k, v, ks, vs, table, lens, pages=pages.cuda(), page_counts=counts.cuda())
    assert_decode(out, lse, q, oracle.dequantised(k, ks), oracle.dequantised(v, vs), table, lens, fp8, pages=pages, page_counts=counts)


@pytest.mark.parametrize("fp8", [False, True])
def test_strided_views(fp8):
    """[pages, page, heads, 128] pools, queries that are a slice of a fused projection, a table that is a slice, an
    output that is a view of other memory; a query whose strides do not fit is copied."""
    lens, page, H, Hkv = [100, 33, 260], 32, 8, 2
    q, k, v, ks, vs, table, lens = _decode_case(6, lens, page, H, Hkv, 3, fp8, nhd=True)
    k_d, v_d, ks_d, vs_d, lens_d = _cuda(k, v, ks, vs, lens)
    assert not k_d.is_contiguous()
    fused = torch.randn(3, 3, 12, 128, device="cuda").bfloat16()
    fused[:, :, 2:10] = q.cuda()
    wide = torch.full((3, 20), 1 << 20, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table.cuda()
    memory = torch.full((3, 3, 10, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    out = memory[:, :, 1:9]
    same, lse = aa.paged_decode_attention(fused[:, :, 2:10], k_d, v_d, wide[:, :table.shape[1]], lens_d, k_scale=ks_d, v_scale=vs_d,
                                          out=out, return_lse=True)
    assert same is out
    assert_decode(out, lse, q, oracle.dequantised(k, ks), oracle.dequantised(v, vs), table, lens, fp8)
    assert bool((memory[:, :, 0] == 7).all()) and bool((memory[:, :, 9] == 7).all())
    odd = torch.zeros(3, 3, 8, 129, device="cuda", dtype=torch.bfloat16)
    odd[..., 1:] = q.cuda()
    again = aa.paged_decode_attention(odd[..., 1:], k_d, v_d, wide[:, :table.shape[1]], lens_d, k_scale=ks_d, v_scale=vs_d)
    assert torch.equal(again, out)


@pytest.mark.parametrize("fp8", [False, True])
def test_non_finite_values_in_masked_places(fp8):
    """NaN and infinities behind the end of a sequence, in pages nobody names, and -- for all but the tokens that may see
    them -- at the newest positions, keys and values."""
    lens, page, n = [21, 45], 16, 4
    q, k, v, ks, vs, table, lens = _decode_case(7, lens, page, 4, 2, n, fp8)
    clean = _run(q, k, v, ks, vs, table, lens)
    k2, v2 = k.float(), v.float()
    used = set(table[0, :2].tolist()) | set(table[1, :3].tolist())
    for p in set(range(k.shape[0])) - used:
        k2[p], v2[p] = math.nan, math.nan
    k2[table[0, 1], :, 5:], v2[table[0, 1], :, 5:] = math.nan, math.nan
    k2[table[1, 2], :, 13:], v2[table[1, 2], :, 13:] = math.nan, math.nan
    dirty = _run(q, k2.to(k.dtype), v2.to(v.dtype), ks, vs, table, lens)
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])
    # the last position of sequence 0 (page 1, row 4): only its last new token sees it
    v2[table[0, 1], :, 4] = math.nan
    k3 = k2.clone()
    out, lse = _run(q, k3.to(k.dtype), v2.to(v.dtype), ks, vs, table, lens)
    assert torch.equal(out[0, :3], clean[0][0, :3]) and torch.equal(out[1], clean[0][1])
    assert bool(out[0, 3].isnan().all()) and torch.equal(lse, clean[1])
    k3[table[0, 1], :, 4] = math.nan
    out, lse = _run(q, k3.to(k.dtype), v2.to(v.dtype), ks, vs, table, lens)
    assert torch.equal(out[0, :3], clean[0][0, :3]) and bool(lse[0, 3].isnan().all()) and torch.equal(lse[0, :3], clean[1][0, :3])
    if not fp8:
        v2[table[0, 1], :, 4] = math.inf
        k3[table[0, 1], :, 4] = k.float()[table[0, 1], :, 4]
        out, _ = _run(q, k3.to(k.dtype), v2.to(v.dtype), ks, vs, table, lens)
        assert bool((out[0, 3] == math.inf).all()) and torch.equal(out[0, :3], clean[0][0, :3])


@pytest.mark.parametrize("magnitude", [2.0 ** -100, 2.0 ** -20, 64.0, 2.0 ** 60])
def test_query_magnitudes_over_an_e4m3_cache(magnitude):
    """Queries whose values f16 could not hold as they are."""
    q, k, v, ks, vs, table, lens = _decode_case(8, [70, 5], 16, 4, 2, 1, True)
    q = (q.float() * magnitude).bfloat16()
    scaling = 128 ** -0.5 / magnitude
    out, lse = _run(q, k, v, ks, vs, table, lens, scaling=scaling)
    assert_decode(out, lse, q, oracle.dequantised(k, ks), oracle.dequantised(v, vs), table, lens, True, scaling=scaling)


@pytest.mark.parametrize("scaling", [0.02, 1.0, -0.1])
def test_scaling(scaling):
    q, k, v, ks, vs, table, lens = _decode_case(9, [400, 31], 64, 8, 2, 1, False)
    out, lse = _run(q, k, v, ks, vs, table, lens, scaling=scaling)
    assert_decode(out, lse, q, oracle.dequantised(k, ks), oracle.dequantised(v, vs), table, lens, False, scaling=scaling)


def test_three_dimensional_query_and_no_lse():
    q, k, v, ks, vs, table, lens = _decode_case(10, [50, 7], 16, 8, 2, 1, False)
    full, _ = _run(q, k, v, ks, vs, table, lens)
    q, k, v, table, lens = _cuda(q, k, v, table, lens)
    out = aa.paged_decode_attention(q[:, 0], k, v, table, lens)
    assert out.shape == (2, 8, 128) and torch.equal(out, full[:, 0])


def test_bad_pages_and_lengths_are_left_out_and_reported():
    """Page numbers outside the pool, list entries outside the sequence, a length beyond the table row: nothing is read
    through them, the rest is attended, and the check raises once."""
    q, k, v, ks, vs, table, lens = _decode_case(11, [100, 100, 64], 16, 4, 2, 1, False)
    table[0, 2], table[1, 0], table[2, 3] = -5, 1 << 30, k.shape[0]
    out, lse = _run(q, k, v, ks, vs, table, lens)
    assert_decode(out, lse, q, k.double(), v.double(), table, lens, False)
    with pytest.raises(RuntimeError, match="outside the pool"):
        aa.check_paged_status()
    aa.check_paged_status()
    q, k, v, ks, vs, table, lens = _decode_case(12, [100, 40], 16, 4, 2, 1, False)
    lens[1] = 100000
    table[1] = table[0]
    out, lse = _run(q, k, v, ks, vs, table, lens)
    lens[1] = table.shape[1] * 16
    assert_decode(out, lse, q, k.double(), v.double(), table, lens, False)
    with pytest.raises(RuntimeError, match="longer than its row"):
        aa.check_paged_status()
    lens[1] = 40
    pages = torch.tensor([[[0, 7, -3, 2]] * 2, [[0, 3, 1 << 28, 1]] * 2], dtype=torch.int32)      # 7 and 3 are behind the ends
    counts = torch.tensor([[4, 9], [-2, 4]], dtype=torch.int32)
    out, lse = _run(q, k, v, ks, vs, table, lens, pages=pages.cuda(), page_counts=counts.cuda())
    good = torch.tensor([[[0, 2]] * 2, [[0, 1]] * 2], dtype=torch.int32)
    assert_decode(out, lse, q, k.double(), v.double(), table, lens, False, pages=good,
                  page_counts=torch.tensor([[2, 2], [0, 2]], dtype=torch.int32))
    with pytest.raises(RuntimeError, match="outside the pool"):
        aa.check_paged_status()


def test_offsets_beyond_32_bits():
    """A pool of 5 GB: pages whose bytes and whose elements lie beyond 2^32 and 2^31."""
    page, Hkv, total = 64, 8, 40000
    k = torch.empty((total, Hkv, page, 128), dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    table = torch.tensor([[39999, 17000, 33000, 0]], dtype=torch.int32)
    g = torch.Generator().manual_seed(1)
    k_small, v_small, _, _ = make_pool(4, Hkv, page, g, False)
    for i, p in enumerate(table[0].tolist()):
        k[p], v[p] = k_small[i].cuda(), v_small[i].cuda()
    q = torch.randn(1, 1, 32, 128, generator=g).bfloat16()
    lens = torch.tensor([250], dtype=torch.int32)
    out, lse = _run(q, k, v, None, None, table, lens)
    assert_decode(out, lse, q, k_small.double(), v_small.double(), torch.arange(4, dtype=torch.int32)[None], lens, False)
    key = torch.randn(1, Hkv, 128, generator=g).bfloat16().cuda()
    aa.paged_kv_append(key, key, k, v, table.cuda(), torch.tensor([40], dtype=torch.int32).cuda())
    assert torch.equal(k[39999, :, 39], key[0]) and torch.equal(v[39999, :, 39], key[0])


# ------------------------------------------------------------------------------------------------------- append
def _append_case(seed, new, cached, page, H, Hkv, fp8, ragged=True, extra=0, nhd=False):
    g = torch.Generator().manual_seed(seed)
    lens = [a + b for a, b in zip(new, cached)]
    table, total = make_table(lens, page, g)
    k, v, ks, vs = make_pool(total, Hkv, page, g, fp8, nhd)
    tokens = sum(new) + extra
    fused = torch.randn(tokens, H + 2 * Hkv, 128, generator=g).bfloat16()
    cu = torch.tensor([0] + new).cumsum(0).int() if ragged else None
    inv = 10000.0 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128)
    cos, sin = aa.rotary_tables(inv, max(lens) + 1)
    return dict(query=fused[:, :H], key=fused[:, H:H + Hkv], value=fused[:, H + Hkv:], k=k, v=v, ks=ks, vs=vs, table=table,
                lens=torch.tensor(lens, dtype=torch.int32), cu=cu, cos=cos, sin=sin, new=new, cached=cached, page=page)


def _append(c, rotate=True, codes=True, return_key=True, query=True):
    d = {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in c.items()}
    P, Hkv = c["k"].shape[:2]
    kc = torch.full((P, Hkv, 128), 55, dtype=torch.int8, device="cuda") if codes else None
    kcs = torch.full((P, Hkv), 5.0, device="cuda") if codes else None
    q, key = aa.paged_kv_append(d["key"], d["value"], d["k"], d["v"], d["table"], d["lens"], cu_seqlens=d["cu"],
                                query=d["query"] if query else None, cos=d["cos"] if rotate else None, sin=d["sin"] if rotate else None,
                                k_scale=d["ks"], v_scale=d["vs"], key_codes=kc, key_code_scales=kcs, return_key=return_key)
    return dict(q=q, key=key, k=d["k"], v=d["v"], codes=kc, scales=kcs)


def _check_append(c, r, rotate=True):
    """Rotation: two products and a sum rounded in 32 bits (3 * 2^-24 of |a cos| + |b sin|), then one rounding: 2^-8 for
    bf16, 2^-4 or half a subnormal step of 2^-9 for e4m3 (and 2^-24 for the division).  Values: one rounding, none in
    bf16.  Everything else of the pools is untouched.  Codes: exact."""
    fp8, page = c["ks"] is not None, c["page"]
    k, v = (t.float().double() for t in (c["k"], c["v"]))
    touched = torch.zeros(k.shape[0], page, dtype=torch.bool)
    full = []
    got = {n: t.cpu() for n, t in r.items() if t is not None}
    at = 0
    for b, (n, before) in enumerate(zip(c["new"], c["cached"])):
        pos = torch.arange(before, before + n)
        where, row = c["table"][b][pos // page].long(), pos % page
        x = slice(at, at + n)
        at += n
        touched[where, row] = True
        full += where[row == page - 1].tolist()
        cos, sin = (c["cos"][pos], c["sin"][pos]) if rotate else (torch.ones(n, 64), torch.zeros(n, 64))
        for src, name in ((c["query"], "q"), (c["key"], "key")):
            if name not in got:
                continue
            want = oracle.rotate(src[x], cos, sin)
            size = oracle.rotate(src[x].abs(), cos.abs(), -sin.abs()).abs()[..., :64].repeat(1, 1, 2) + src[x].double().abs()
            tol = 2.0 ** -8 * want.abs() + (3 * 2.0 ** -24 * 2 * size if rotate else 0)
            assert ((got[name][x].double() - want).abs() <= tol).all()
        want = oracle.rotate(c["key"][x], cos, sin)
        size = src_size = c["key"][x].double().abs()
        size = src_size + torch.cat([src_size[..., 64:], src_size[..., :64]], -1)
        for pool, name, y, s, loose in ((got["k"], "k", want, c["ks"], 3 * 2.0 ** -24 * size if rotate else 0 * size),
                                        (got["v"], "v", c["value"][x].double(), c["vs"], 0 * size)):
            stored = pool[where, :, row].float().double()
            if fp8:
                y, loose = y / s.double()[:, None], loose / s.double()[:, None]
                tol = 2.0 ** -4 * y.abs() + 2.0 ** -10 + 2.0 ** -23 * y.abs() + 2 * loose
                y = y.clamp(-448, 448)
            else:
                tol = 2.0 ** -8 * y.abs() + 2 * loose if name == "k" and rotate else 0 * y
            assert ((stored - y).abs() <= tol).all(), name
        # the 32-bit formula, step by step, gives the very codes
        a, b2 = c["key"][x][..., :64].float(), c["key"][x][..., 64:].float()
        co, si = cos[:, None], sin[:, None]
        rot = torch.cat([a * co - b2 * si, b2 * co + a * si], -1) if rotate else c["key"][x].float()
        if fp8:
            rot, val = ((y / s[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn) for y, s in ((rot, c["ks"]), (c["value"][x].float(), c["vs"])))
        else:
            rot, val = rot.bfloat16(), c["value"][x]
        assert torch.equal(got["k"][where, :, row].float(), rot.float()) and torch.equal(got["v"][where, :, row].float(), val.float())
    rest = ~touched[:, None, :, None].expand_as(k)
    assert torch.equal(got["k"].float()[rest], c["k"].float()[rest]) and torch.equal(got["v"].float()[rest], c["v"].float()[rest])
    if "codes" in got:
        others = torch.ones(k.shape[0], dtype=torch.bool)
        others[full] = False
        assert (got["codes"][others] == 55).all() and (got["scales"][others] == 5).all()
        for p in full:
            codes, scale = oracle.page_summary(got["k"], p, c["ks"])
            assert torch.equal(got["codes"][p], codes) and torch.equal(got["scales"][p], scale)
    return full


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("new,cached", [
    ([1, 1, 1, 1], [0, 15, 63, 255]), ([7, 0, 300, 1, 64], [9, 40, 0, 63, 64]), ([33] * 3, [0, 31, 500]), ([1], [1000])])
def test_append_rotates_writes_and_summarises(new, cached, page, fp8):
    c = _append_case(page + len(new), new, cached, page, 12, 4, fp8)
    full = _check_append(c, _append(c))
    if cached == [0, 15, 63, 255]:
        assert len(full) == {16: 3, 64: 2, 256: 1}[page]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n", [1, 5, 130])
def test_append_without_offsets(n, fp8):
    """T / B tokens each, no rotation, no queries, no codes, [pages, page, heads, 128] pools."""
    c = _append_case(n, [n] * 3, [12, 0, 130], 32, 4, 2, fp8, ragged=False, nhd=True)
    r = _append(c, rotate=False, codes=False, query=False)
    _check_append(c, r, rotate=False)
    assert r["q"] is None and torch.equal(r["key"].cpu(), c["key"])


@pytest.mark.parametrize("fp8", [False, True])
def test_append_many_sequences(fp8):
    """More sequences than a warp looks at in one go, most of them with nothing new."""
    new = [0] * 100
    new[3], new[31], new[32], new[64], new[99] = 5, 1, 40, 2, 17
    c = _append_case(4, new, [i % 23 for i in range(100)], 16, 4, 2, fp8)
    _check_append(c, _append(c))


@pytest.mark.parametrize("fp8", [False, True])
def test_append_in_pieces_gives_the_same_cache(fp8):
    """A prompt at once, and the same prompt in chunks of odd sizes with the codes kept along."""
    c = _append_case(8, [150, 70], [0, 0], 16, 8, 2, fp8)
    whole = _append(c)
    d = {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in c.items()}
    P, Hkv = c["k"].shape[:2]
    kc, kcs = torch.full((P, Hkv, 128), 55, dtype=torch.int8, device="cuda"), torch.full((P, Hkv), 5.0, device="cuda")
    done, starts = [0, 0], [0, 150]
    for chunk in ([1, 0], [15, 3], [17, 29], [1, 1], [90, 30], [26, 7]):
        rows = torch.cat([torch.arange(s + a, s + a + n) for s, a, n in zip(starts, done, chunk)])
        done = [a + n for a, n in zip(done, chunk)]
        q, key = aa.paged_kv_append(d["key"][rows], d["value"][rows], d["k"], d["v"], d["table"],
                                    torch.tensor(done, dtype=torch.int32, device="cuda"),
                                    cu_seqlens=torch.tensor([0, chunk[0], sum(chunk)], dtype=torch.int32, device="cuda"),
                                    query=d["query"][rows], cos=d["cos"], sin=d["sin"], k_scale=d["ks"], v_scale=d["vs"],
                                    key_codes=kc, key_code_scales=kcs, return_key=True)
        assert torch.equal(q, whole["q"][rows]) and torch.equal(key, whole["key"][rows])
    assert done == [150, 70]
    for a, b in ((d["k"], whole["k"]), (d["v"], whole["v"]), (kc, whole["codes"]), (kcs, whole["scales"])):
        assert torch.equal(a.float(), b.float())


def test_append_padding_is_left_out():
    """Sequences of length 0 in a decode batch, tokens behind the last sequence: no page is written, nothing is reported."""
    c = _append_case(2, [1, 1, 1], [4, 0, 16], 16, 4, 2, False, ragged=False)
    c["lens"][1] = 0
    before = c["k"].clone(), c["v"].clone()
    r = _append(c)
    written = torch.zeros_like(before[0], dtype=torch.bool)
    written[c["table"][0, 0], :, 4] = True
    written[c["table"][2, 1], :, 0] = True
    assert torch.equal(r["k"].cpu()[~written], before[0][~written]) and torch.equal(r["v"].cpu()[~written], before[1][~written])
    assert torch.equal(r["v"].cpu()[c["table"][2, 1], :, 0], c["value"][2])
    aa.check_paged_status()
    c = _append_case(3, [20, 3], [0, 9], 16, 4, 2, False, extra=6)
    _check_append(c, _append(c))


def test_append_bad_pages_and_lengths():
    """A page number outside the pool, a sequence beyond its table row, positions beyond the rotary tables, token ranges
    outside the inputs: nothing is written through them."""
    c = _append_case(5, [40, 3], [0, 9], 16, 4, 2, False)
    good = _append(c)
    c["table"][0, 1] = 1 << 20
    r = _append(c)
    lost = _append_case(5, [40, 3], [0, 9], 16, 4, 2, False)["table"][0, 1]
    keep = torch.arange(c["k"].shape[0]) != lost
    assert torch.equal(r["k"].cpu()[keep], good["k"].cpu()[keep]) and torch.equal(r["k"].cpu()[lost], c["k"][lost])
    assert torch.equal(r["q"], good["q"]) and torch.equal(r["key"], good["key"])
    with pytest.raises(RuntimeError, match="outside the pool"):
        aa.check_paged_status()
    c = _append_case(6, [5, 3], [0, 0], 16, 4, 2, False)
    before = c["k"].clone()
    c["lens"][0] = 2 ** 31 - 1
    c["cos"], c["sin"] = c["cos"][:2].contiguous(), c["sin"][:2].contiguous()
    r = _append(c)
    changed = (r["k"].cpu() != before).any(-1).any(1)
    assert changed.sum() == 2 and bool(changed[c["table"][1, 0], :2].all())
    with pytest.raises(RuntimeError, match="longer"):
        aa.check_paged_status()
    c = _append_case(7, [5, 3], [0, 0], 16, 4, 2, False)
    before = c["k"].clone()
    c["cu"] = torch.tensor([-7, 2 ** 31 - 1, 3], dtype=torch.int32)
    r = _append(c)
    assert torch.equal(r["k"].cpu(), before)


def test_append_codes_over_all_magnitudes():
    """e4m3 codes of values from 2^-126 to 2^126, near and on the ties between codes, for scales of any mantissa and far from
    1: those of the 32-bit quotient."""
    g = torch.Generator().manual_seed(1)
    T, Hkv = 2048, 16
    scale = torch.cat([torch.tensor([1.0, 0.5, 3e-30, 7e25, 1.9999999, 2.0 ** -60, 2.0 ** 60, 448.0 ** -1]),
                       0.01 + torch.rand(8, generator=g)])
    x = torch.randn(T, Hkv, 128, generator=g) * 2.0 ** torch.randint(-12, 10, (T, Hkv, 128), generator=g)
    ties = (torch.randint(8, 16, (T, Hkv, 64), generator=g) + 0.5) * 2.0 ** torch.randint(-9, 5, (T, Hkv, 64), generator=g)
    x[..., :64] = ties * (1 + torch.randint(-2, 3, (T, Hkv, 64), generator=g) * 2.0 ** -8)
    x = (x * scale[:, None]).bfloat16()
    x[:32] = (torch.randn(32, Hkv, 128, generator=g) * 2.0 ** torch.randint(-126, 126, (32, Hkv, 128), generator=g)).bfloat16()
    k = torch.zeros(T // 16, Hkv, 16, 128, device="cuda").to(torch.float8_e4m3fn)
    v = torch.zeros_like(k)
    table = torch.arange(T // 16, dtype=torch.int32, device="cuda")[None]
    s = scale.cuda()
    aa.paged_kv_append(x.cuda(), x.flip(0).cuda(), k, v, table, torch.tensor([T], dtype=torch.int32, device="cuda"),
                       cu_seqlens=torch.tensor([0, T], dtype=torch.int32, device="cuda"), k_scale=s, v_scale=s)
    for pool, y in ((k, x), (v, x.flip(0))):
        want = (y.float() / scale[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
        got = pool.cpu().transpose(1, 2).reshape(T, Hkv, 128)
        assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))


def test_append_non_finite_keys_and_saturation():
    """NaN and infinities are stored as they are (an e4m3 code saturates at 448), and leave their page without a score."""
    c = _append_case(9, [16], [0], 16, 4, 2, False)
    key = c["key"].clone()
    key[3, 0, 5], key[4, 1, 6] = math.nan, math.inf
    c["key"] = key
    r = _append(c, rotate=False)
    page = c["table"][0, 0]
    assert r["k"][page, 0, 3, 5].isnan() and r["k"][page, 1, 4, 6] == math.inf
    assert (r["codes"][page] == 0).all() and (r["scales"][page] == 0).all()
    c = _append_case(10, [1], [0], 16, 4, 2, True)
    key = c["key"].clone()
    key[0, 0, 0], key[0, 0, 1], key[0, 1, 0] = 1e6, -1e6, math.nan
    c["key"] = key
    r = _append(c, rotate=False)
    stored = r["k"].float()[c["table"][0, 0], :, 0]
    assert stored[0, 0] == 448 and stored[0, 1] == -448 and stored[1, 0].isnan()


# ------------------------------------------------------------------------------------------------------- select
@pytest.mark.parametrize("H,Hkv,n", [(32, 8, 1), (28, 4, 3), (4, 4, 1), (16, 1, 16)])
@pytest.mark.parametrize("page,top,first,last", [(16, 8, 1, 2), (64, 5, 0, 1), (32, 40, 3, 4)])
def test_select(H, Hkv, n, page, top, first, last):
    g = torch.Generator().manual_seed(H + page)
    lens = [0, 1, page * top, page * top + 1, 3001, 5000]
    table, total = make_table(lens, page, g)
    codes = torch.randint(-127, 128, (total, Hkv, 128), generator=g, dtype=torch.int8)
    scales = torch.rand(total, Hkv, generator=g) / 100
    q = torch.randn(len(lens), n, H, 128, generator=g).bfloat16()
    q[4, 0, 0] = 0
    lens = torch.tensor(lens, dtype=torch.int32)
    got = aa.select_pages(*_cuda(q, codes, scales, table, lens), top, page, first, last)
    want = oracle.select(q, codes, scales, table, lens, top, page, first, last)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_select_ties():
    """Pages with the same score, and scores of +0 and -0: the lower ones get in."""
    pages = 3000
    codes = torch.zeros(pages, 1, 128, dtype=torch.int8)
    codes[:, 0, 0] = torch.arange(pages).remainder(3).to(torch.int8) - 1
    table = torch.arange(pages, dtype=torch.int32)[None]
    q = torch.zeros(1, 2, 128)
    q[..., 0] = torch.tensor([1.0, -0.0])
    lens = torch.tensor([pages * 16 - 5], dtype=torch.int32)
    scales = torch.ones(pages, 1)
    for top in (10, 999, 1002, 1500, 2500):
        got = aa.select_pages(*_cuda(q.bfloat16(), codes, scales, table, lens), top, 16)
        want = oracle.select(q.bfloat16()[:, None], codes, scales, table, lens, top, 16)
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_select_the_longest_table():
    pages = 40960
    g = torch.Generator().manual_seed(2)
    codes = torch.randint(-127, 128, (pages, 1, 128), generator=g, dtype=torch.int8)
    table = torch.randperm(pages, generator=g).int()[None]
    q = torch.randn(1, 4, 128, generator=g).bfloat16()
    lens = torch.tensor([pages * 16], dtype=torch.int32)
    scales = torch.rand(pages, 1, generator=g)
    got = aa.select_pages(*_cuda(q, codes, scales, table, lens), 700, 16)
    want = oracle.select(q[:, None], codes, scales, table, lens, 700, 16)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    with pytest.raises(RuntimeError, match="too large"):
        aa.select_pages(*_cuda(q, codes, scales, torch.zeros(1, 40961, dtype=torch.int32), lens), 700, 16)


def test_select_bad_page():
    table = torch.arange(20, dtype=torch.int32)[None].clone()
    table[0, 7] = -1
    g = torch.Generator().manual_seed(3)
    codes = torch.randint(-127, 128, (20, 1, 128), generator=g, dtype=torch.int8)
    q = torch.randn(1, 4, 128, generator=g).bfloat16()
    pages, counts = aa.select_pages(*_cuda(q, codes, torch.ones(20, 1), table, torch.tensor([320], dtype=torch.int32)), 19, 16)
    assert counts.item() == 19 and pages[0, 0].tolist() == [i for i in range(20) if i != 7]
    with pytest.raises(RuntimeError, match="outside the pool"):
        aa.check_paged_status()


# --------------------------------------------------------------------------------------- streams, graphs, together
def test_two_streams_at_once():
    """Calls in flight on two streams do not meet in a workspace."""
    cases = [_decode_case(i, [6000 + 700 * i, 900], 64, 32, 8, 1, False) for i in range(2)]
    alone = [_run(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    data = [_cuda(*c) for c in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        outs = []
        for s, (q, k, v, ks, vs, table, lens) in zip(streams, data):
            with torch.cuda.stream(s):
                outs.append(aa.paged_decode_attention(q, k, v, table, lens))
        torch.cuda.synchronize()
        for o, a in zip(outs, alone):
            assert torch.equal(o, a[0])


def test_captured_decode_step_replays_with_growing_lengths():
    """Append, selection and attention captured once; lengths grow in place between the replays, across page ends.  Every
    replay equals the eager calls.  Two such graphs replayed on two streams at once keep apart."""
    def build(seed):
        c = _append_case(seed, [1, 1], [140, 30], 16, 8, 2, False, ragged=False)
        c["cos"], c["sin"] = aa.rotary_tables(10000.0 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128), 400)
        g = torch.Generator().manual_seed(seed)
        c["table"], total = make_table([400, 400], 16, g)
        c["k"], c["v"], _, _ = make_pool(total, 2, 16, g, False)
        d = {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in c.items()}
        d["codes"] = torch.zeros(total, 2, 128, dtype=torch.int8, device="cuda")
        d["scales"] = torch.zeros(total, 2, device="cuda")
        return d

    def step(d):
        q, _ = aa.paged_kv_append(d["key"], d["value"], d["k"], d["v"], d["table"], d["lens"], query=d["query"], cos=d["cos"],
                                  sin=d["sin"], key_codes=d["codes"], key_code_scales=d["scales"])
        pages, counts = aa.select_pages(q, d["codes"], d["scales"], d["table"], d["lens"], 6, 16)
        return aa.paged_decode_attention(q, d["k"], d["v"], d["table"], d["lens"], pages=pages, page_counts=counts), pages, counts

    both, graphs = [build(1), build(2)], []
    for d in both:
        lens0, k0, v0 = d["lens"].clone(), d["k"].clone(), d["v"].clone()
        step(d)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(d)
        d["lens"].copy_(lens0), d["k"].copy_(k0), d["v"].copy_(v0), d["codes"].zero_(), d["scales"].zero_()
        graphs.append((graph, outs))
    eager = [build(1), build(2)]
    streams = [torch.cuda.Stream() for _ in both]
    torch.cuda.synchronize()
    for i in range(40):
        for d, e, (graph, _), s in zip(both, eager, graphs, streams):
            with torch.cuda.stream(s):
                g = torch.Generator(device="cuda").manual_seed(i)
                for n in ("key", "value", "query"):
                    d[n].copy_(torch.randn(d[n].shape, generator=g, device="cuda"))
                    e[n].copy_(d[n])
                graph.replay()
        torch.cuda.synchronize()
        for d, e, (_, outs) in zip(both, eager, graphs):
            want = step(e)
            for a, b in zip(outs, want):
                assert torch.equal(a, b)
            d["lens"] += 1
            e["lens"] += 1
        torch.cuda.synchronize()
    for d, e in zip(both, eager):
        for n in ("k", "v", "codes", "scales"):
            assert torch.equal(d[n], e[n])


def test_prefill_then_generation():
    """A prompt through append and the prefill operator, then generated tokens over the cache: the first layer's attention
    as a user runs it.  Every decode output is checked against the 64-bit oracle on what the cache holds, and the
    sparse step with every page picked equals the full one up to rounding."""
    H, Hkv, page, N, steps = 8, 2, 64, 4096, 70
    g = torch.Generator().manual_seed(0)
    table, total = make_table([N + steps], page, g)
    k = torch.zeros(total, Hkv, page, 128, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    codes = torch.zeros(total, Hkv, 128, dtype=torch.int8, device="cuda")
    scales = torch.zeros(total, Hkv, device="cuda")
    table = table.cuda()
    cos, sin = aa.rotary_tables(500000.0 ** (-torch.arange(0, 128, 2, dtype=torch.float64, device="cuda") / 128), N + steps)
    fused = torch.randn(N + steps, H + 2 * Hkv, 128, generator=g).bfloat16().cuda()

    def append(lo, hi):
        x = fused[lo:hi]
        lens = torch.tensor([hi], dtype=torch.int32, device="cuda")
        q, key = aa.paged_kv_append(x[:, H:H + Hkv], x[:, H + Hkv:], k, v, table, lens, query=x[:, :H], cos=cos, sin=sin,
                                    key_codes=codes, key_code_scales=scales, return_key=True)
        return q, key, lens

    q, key, lens = append(0, N)
    Q, K, V = (x[None].transpose(1, 2) for x in (q, key, fused[:N, H + Hkv:]))
    out = aa.anchor_attn(Q, K, V, difference=12, return_computational_ratio=False)
    assert out.shape == (1, H, N, 128) and bool(out.isfinite().all())
    # the prompt's last rows by the decode kernel and by the dense prefill kernel: same keys, both rounded to bf16
    tail = aa.dense_causal_attention(Q[:, :, -16:], K, V)
    decode = aa.paged_decode_attention(q[None, -16:], k, v, table, lens)
    assert (decode.transpose(1, 2).float() - tail.float()).abs().max() <= 2.0 ** -7 * tail.float().abs().max()
    for i in range(steps):
        q, _, lens = append(N + i, N + i + 1)
        full, lse = aa.paged_decode_attention(q, k, v, table, lens, return_lse=True)
        if i % 23 == 0 or i == steps - 1:
            assert_decode(full, lse, q[None].cpu(), k.cpu().double(), v.cpu().double(), table.cpu(), lens.cpu(), False)
            pages, counts = aa.select_pages(q, codes, scales, table, lens, 16, page)
            want = oracle.select(q[None].cpu(), codes.cpu(), scales.cpu(), table.cpu(), lens.cpu(), 16, page)
            assert torch.equal(pages.cpu(), want[0]) and torch.equal(counts.cpu(), want[1])
            part, lse = aa.paged_decode_attention(q, k, v, table, lens, pages=pages, page_counts=counts, return_lse=True)
            assert_decode(part, lse, q[None].cpu(), k.cpu().double(), v.cpu().double(), table.cpu(), lens.cpu(), False,
                          pages=pages.cpu(), page_counts=counts.cpu())
            pages, counts = aa.select_pages(q, codes, scales, table, lens, 80, page)
            every = aa.paged_decode_attention(q, k, v, table, lens, pages=pages, page_counts=counts)
            assert (every.float() - full.float()).abs().max() <= 2.0 ** -7 * full.float().abs().max()


def test_empty_batches():
    q, k, v, ks, vs, table, lens = _cuda(*_decode_case(1, [5], 16, 4, 2, 1, False))
    out, lse = aa.paged_decode_attention(q[:0], k, v, table[:0], lens[:0], return_lse=True)
    assert out.shape == (0, 1, 4, 128) and lse.shape == (0, 1, 4)
    q2, _ = aa.paged_kv_append(k[:0, :, 0], v[:0, :, 0], k, v, table, lens, query=q[0][:0])
    assert q2.shape == (0, 4, 128)


def test_first_call_inside_a_capture_is_refused():
    from anchor_attention_b200 import paged
    q, k, v, ks, vs, table, lens = _cuda(*_decode_case(1, [5], 16, 4, 2, 1, False))
    aa.paged_decode_attention(q, k, v, table, lens)
    kept = dict(paged._status)
    paged._status.clear()
    try:
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="before capturing"):
            with torch.cuda.graph(graph):
                aa.paged_decode_attention(q, k, v, table, lens)
    finally:
        paged._status.update(kept)
    torch.cuda.synchronize()
    aa.paged_decode_attention(q, k, v, table, lens)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("page,n,H,Hkv", [(16, 1, 8, 2), (256, 1, 8, 2), (16, 6, 8, 2), (64, 16, 4, 2), (128, 9, 8, 2)])
def test_picked_pages_of_all_sizes_and_rows(page, n, H, Hkv, fp8):
    """Lists over pages smaller and larger than a step of the kernel, for one to many tiles of rows, long enough to be cut."""
    g = torch.Generator().manual_seed(page + n)
    lens = [40 * page - 3, 7 * page + 1, 150 * 16]
    q, k, v, ks, vs, table, lens = _decode_case(page, lens, page, H, Hkv, n, fp8)
    live = -(-lens // page)
    width = int(live.max())
    pages = torch.full((3, Hkv, width), -1, dtype=torch.int32)
    counts = torch.zeros((3, Hkv), dtype=torch.int32)
    for b in range(3):
        for h in range(Hkv):
            c = int(torch.randint(1, int(live[b]) + 1, (1,), generator=g))
            pages[b, h, :c] = torch.randperm(int(live[b]), generator=g)[:c].int()
            counts[b, h] = c
    out, lse = _run(q, k, v, ks, vs, table, lens, pages=pages.cuda(), page_counts=counts.cuda())
    assert_decode(out, lse, q, oracle.dequantised(k, ks), oracle.dequantised(v, vs), table, lens, fp8, pages=pages, page_counts=counts)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n,H,Hkv", [(16, 8, 1), (3, 20, 2), (11, 4, 4), (5, 16, 4)])
def test_many_rows_over_long_sequences(n, H, Hkv, fp8):
    """Several tiles of rows of sequences that are cut into parts."""
    case = _decode_case(n, [5000, 777], 32, H, Hkv, n, fp8)
    out, lse = _run(*case)
    q, k, v, ks, vs, table, lens = case
    assert_decode(out, lse, q, oracle.dequantised(k, ks), oracle.dequantised(v, vs), table, lens, fp8)


def test_many_short_sequences():
    """More sequences and heads than the kernel keeps at hand of a range, most of one unit."""
    lens = [(i * 37) % 90 for i in range(700)]
    case = _decode_case(5, lens, 16, 8, 4, 1, False)
    out, lse = _run(*case)
    q, k, v, ks, vs, table, lens = case
    assert_decode(out, lse, q, k.double(), v.double(), table, lens, False)


def test_attention_in_place_of_the_query():
    """``out`` may be the query itself."""
    case = _decode_case(6, [3000, 50, 700], 16, 8, 2, 2, False)
    want, _ = _run(*case)
    q, k, v, ks, vs, table, lens = _cuda(*case)
    assert aa.paged_decode_attention(q, k, v, table, lens, out=q) is q
    assert torch.equal(q, want)


@pytest.mark.parametrize("ragged", [False, True])
def test_append_at_the_largest_length(ragged):
    """Positions up to 2^31 - 2, whose page ends at 2^31: the keys lie beyond the table and are left out, the queries (not
    rotated, so no position is beyond the tables) are copied."""
    n = 1 if not ragged else 3
    c = _append_case(8, [n], [0], 16, 4, 2, False, ragged=ragged)
    c["lens"][0] = 2 ** 31 - 1
    r = _append(c, rotate=False)
    assert torch.equal(r["q"].cpu(), c["query"]) and torch.equal(r["k"].cpu(), c["k"]) and torch.equal(r["v"].cpu(), c["v"])
    assert (r["codes"] == 55).all()
    with pytest.raises(RuntimeError, match="longer"):
        aa.check_paged_status()
