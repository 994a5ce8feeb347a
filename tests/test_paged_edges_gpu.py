"""Edge cases of the paged cache on the GPU: arguments and cache contents at the borders of what the functions accept."""
import ctypes
import math

import pytest
import torch

import anchor_attention_b200 as aa
from anchor_attention_b200 import _lib
from oracle import paged_oracle as oracle
from paged_util import assert_decode, make_pool, make_table

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean_status(lib):
    aa.check_paged_status()
    yield
    aa.check_paged_status()


def _case(seed, lens, page, H, Hkv, n, fp8, width=None):
    g = torch.Generator().manual_seed(seed)
    table, total = make_table(lens, page, g, width=width)
    k, v, ks, vs = make_pool(total, Hkv, page, g, fp8)
    q = (torch.randn(len(lens), n, H, 128, generator=g) * 1.5).bfloat16()
    return q, k, v, ks, vs, table, torch.tensor(lens, dtype=torch.int32)


def _run(q, k, v, ks, vs, table, lens, **kw):
    q, k, v, ks, vs, table, lens = [None if t is None else t.cuda() for t in (q, k, v, ks, vs, table, lens)]
    return aa.paged_decode_attention(q, k, v, table, lens, k_scale=ks, v_scale=vs, return_lse=True, **kw)


# ---------------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("scaling", [0.0, -0.0, 0])
def test_a_scale_of_zero_weighs_all_keys_alike(scaling, fp8):
    """Every weight is 1 and every product exact.  32-bit sums of L terms are off by 2^-23 L of the sum of their sizes at most
    (tensor cores may truncate); a bf16 weight's second part and the scale add 2^-21; then one rounding of the output."""
    lens = [400, 31, 0]
    q, k, v, ks, vs, table, lens_t = _case(1, lens, 64, 8, 2, 1, fp8)
    out, lse = _run(q, k, v, ks, vs, table, lens_t, scaling=scaling)
    out, lse = out.double().cpu(), lse.double().cpu()
    values = oracle.dequantised(v, vs)
    for b, n in enumerate(lens):
        if not n:
            assert (out[b] == 0).all() and (lse[b] == -math.inf).all()
            continue
        V = oracle.gather(values, table[b], torch.arange(n)).repeat_interleave(4, 0)           # [H, n, 128]
        want, size = V.mean(1), V.abs().mean(1)
        assert ((out[b, 0] - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -23 * n + 2.0 ** -21) * size).all()
        assert ((lse[b] - math.log(n)).abs() <= 2.0 ** -20 + 2.0 ** -22 * math.log(n)).all()
    ref = oracle.attend(q, oracle.dequantised(k, ks), values, table, lens_t, scaling=scaling)
    assert (ref[1][0] - math.log(400)).abs().max() < 1e-12


def _own_key_bounds(query, out, lse, weight, spread, lens, v):
    """decode_bounds of an e4m3 cache with the part that does not scale with a row's values taken from the sequence's own
    keys: a weight is held in f16 relative to 2^15 at its lane's largest, so what rounds to nothing is below 2^-40 of it.
    A score is off by 128 * 2^-23 of its sum of sizes (128 exact products added in 32 bits), a query's f16 copy by 2^-33 of its
    row's largest value an element; scale, exponential and its argument add 2^-15; a weight in f16 2^-11; the output 2^-8."""
    d = 128 * 2.0 ** -23 * spread + 2.0 ** -15 + 128 * 2.0 ** -33 * spread
    nothing = 2.0 ** -40 * lens.double() * v.abs().max()
    tol_out = 2.0 ** -8 * out.abs() + (2 * d + 2.0 ** -11)[..., None] * weight + nothing[:, None, None, None] + 1e-30
    return tol_out, d + 2.0 ** -20 + 2.0 ** -22 * torch.where(lse.isfinite(), lse.abs(), torch.zeros_like(lse))


def test_e4m3_tail_behind_strong_keys():
    """A few strong keys at the front and thousands of others at 2^-17 to 2^-25 of their weight, one level for each KV head;
    some values come from the others alone, so what is lost of their weights shows at full size.  37 sequences of 8 heads
    (all on the same pages) leave every entry whole, so that the strong keys' lanes see most of the others."""
    Hkv, page, n = 8, 64, 16384
    g = torch.Generator().manual_seed(4)
    k = torch.zeros(n // page, Hkv, page, 128)
    k[..., 0] = -2.0 - torch.arange(Hkv).float()[None, :, None]
    k[:2, :, ::16, 0] = 16.0                                # every 16th of the first 128 positions
    v = (torch.randint(4, 13, k.shape, generator=g) / 8).float()
    v[..., :64] = 0.0
    v[:2, :, ::16] = 0.0
    v[:2, :, ::16, :64] = 1.0
    k, v = k.to(torch.float8_e4m3fn), v.to(torch.float8_e4m3fn)
    ones = torch.ones(Hkv)
    q = torch.zeros(37, 1, Hkv, 128)
    q[..., 0] = 1.0
    q = q.bfloat16()
    table = torch.arange(n // page, dtype=torch.int32)[None].repeat(37, 1)
    lens = torch.full((37,), n, dtype=torch.int32)
    scaling = 0.97 * math.log(2)
    got, got_lse = _run(q, k, v, ones, ones, table, lens, scaling=scaling)
    out, lse, weight, spread = oracle.attend(q[:1], k.double(), v.double(), table[:1], lens[:1], scaling=scaling)
    tol_out, tol_lse = _own_key_bounds(q[:1], out, lse, weight, spread, lens[:1], v.double())
    assert bool((out[..., 64:] > 2.0 ** -16).all())
    for b in range(37):
        assert ((got[b].double().cpu() - out[0]).abs() <= tol_out[0]).all()
        assert ((got_lse[b].double().cpu() - lse[0]).abs() <= tol_lse[0]).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("exponent", list(range(16, 36)) + [60, 90, 110])
def test_scores_so_large_that_one_key_has_all_weight(exponent, fp8):
    """Scores of 2^exponent and more, where 32 bits hold no small differences: the best key's value comes out, rounded once (the
    weight's two bf16 parts add 2^-22), and the logarithm is its score (three roundings: scale, product, conversion)."""
    n, page = 700, 16
    g = torch.Generator().manual_seed(exponent)
    level = torch.randint(8, 15, (n,), generator=g).float()
    best = int(torch.randint(0, n, (1,), generator=g))
    level[best] = 15.0
    k = torch.zeros(44, 1, page, 128)
    k.view(-1, 128)[:n, 0] = level
    v = (torch.randint(-15, 16, k.shape, generator=g) / 8).float()
    dtype = torch.float8_e4m3fn if fp8 else torch.bfloat16
    k, v = k.to(dtype), v.to(dtype)
    one = torch.ones(1) if fp8 else None
    q = torch.zeros(1, 1, 4, 128)
    q[0, 0, :, 0] = torch.tensor([1.0, 1.25, 1.5, 1.75])
    scaling = 2.0 ** exponent
    out, lse = _run(q.bfloat16(), k, v, one, one, torch.arange(44, dtype=torch.int32)[None], torch.tensor([n], dtype=torch.int32),
                    scaling=scaling)
    want = v.float().view(-1, 128)[best].double()
    assert ((out[0, 0].double().cpu() - want).abs() <= (2.0 ** -8 + 2.0 ** -22) * want.abs()).all()
    score = 15.0 * scaling * q[0, 0, :, 0].double()
    assert ((lse[0, 0].double().cpu() - score).abs() <= 4 * 2.0 ** -24 * score).all()


@pytest.mark.parametrize("lens,H,Hkv", [([20000], 8, 1), ([9001, 1, 12000], 8, 2), ([4097] * 40, 4, 4)])
def test_e4m3_within_the_bounds_of_the_sequences_own_keys(lens, H, Hkv):
    q, k, v, ks, vs, table, lens = _case(3, lens, 64, H, Hkv, 1, True)
    got, got_lse = _run(q, k, v, ks, vs, table, lens)
    values = oracle.dequantised(v, vs)
    out, lse, weight, spread = oracle.attend(q, oracle.dequantised(k, ks), values, table, lens)
    tol_out, tol_lse = _own_key_bounds(q, out, lse, weight, spread, lens, values)
    assert ((got.double().cpu() - out).abs() <= tol_out).all()
    assert ((got_lse.double().cpu() - lse).abs() <= tol_lse).all()


# ------------------------------------------------------------------------------------------------ bounded waits
def _attend_block(q, k, v, ks, vs, table, lens, out, lse, status):
    a = _lib.AAPagedAttend()
    c = a.cache
    c.k_pages, c.v_pages, c.block_table, c.seq_lens, c.status = (t.data_ptr() for t in (k, v, table, lens, status))
    for name, t in (("k", k), ("v", v)):
        for axis, stride in zip(("page", "head", "row"), t.stride()):
            setattr(c, f"{name}_stride_{axis}", stride)
    if ks is not None:
        c.k_scale, c.v_scale, c.cache_dtype = ks.data_ptr(), vs.data_ptr(), _lib.AA_E4M3
    c.table_stride, c.table_width = table.stride(0), table.shape[1]
    c.pages, c.Hkv, c.page_size, c.D, c.B = k.shape[0], k.shape[1], k.shape[2], 128, table.shape[0]
    a.q, a.out, a.lse, a.Nq, a.H = q.data_ptr(), out.data_ptr(), lse.data_ptr(), q.shape[1], q.shape[2]
    a.q_stride_b, a.q_stride_n, a.q_stride_h, _ = q.stride()
    a.o_stride_b, a.o_stride_n, a.o_stride_h, _ = out.stride()
    need = ctypes.c_size_t()
    assert _lib.load().aa_paged_attend_workspace_bytes(ctypes.byref(a), ctypes.byref(need)) == 0
    workspace = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = workspace.data_ptr(), need.value
    return a, workspace


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("lens,H,Hkv,n", [
    ([5], 8, 2, 1),                 # one unit: the producer has issued everything before anyone gives up
    ([200, 90, 0], 8, 2, 1),        # fewer units than stages
    ([30000], 8, 1, 1),             # more units than stages, cut into parts
    ([9000] * 40, 8, 8, 1),         # many units a block
    ([4000, 17], 8, 2, 5), ([4000, 17], 8, 1, 4),
])
def test_a_computing_warp_that_gives_up_is_reported(lens, H, Hkv, n, fp8):
    """The self-test's computing warps give up on every copy: the call ends, its copies have landed before its blocks do, the status says
    so, and the same call with ordinary limits is right afterwards."""
    q, k, v, ks, vs, table, lens_t = [None if t is None else t.cuda() for t in _case(5, lens, 16, H, Hkv, n, fp8)]
    want, want_lse = aa.paged_decode_attention(q, k, v, table, lens_t, k_scale=ks, v_scale=vs, return_lse=True)
    out, lse = torch.empty_like(want), torch.empty_like(want_lse)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    a, workspace = _attend_block(q, k, v, ks, vs, table, lens_t, out, lse, status)
    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
    for _ in range(3):
        assert lib.aa_selftest_paged_wait(ctypes.byref(a), stream) == 0
        assert lib.aa_paged_check_status(status.data_ptr(), stream) == -11
        assert lib.aa_paged_attend(ctypes.byref(a), stream) == 0
        assert lib.aa_paged_check_status(status.data_ptr(), stream) == 0
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


# ------------------------------------------------------------------------------------------------------- append
def test_e4m3_codes_of_negative_zeros():
    """-0 / scale is -0, whose code is 0x80; for scales the kernel multiplies by the reciprocal of and for one it divides by."""
    scales = torch.tensor([1.0, 0.37, 3e-30])
    x = torch.zeros(16, 3, 128)
    x[:, :, ::2] = -0.0
    x[:, :, 1::4] = torch.tensor([-1e-38, 2.0 ** -40])[None, None].repeat(16, 3, 16) * scales[:, None].clamp(min=1.0)
    x = x.bfloat16()
    k = torch.full((1, 3, 16, 128), 1.0, device="cuda").to(torch.float8_e4m3fn)
    v = k.clone()
    one = torch.tensor([16], dtype=torch.int32, device="cuda")
    aa.paged_kv_append(x.cuda(), x.flip(0).cuda(), k, v, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), one,
                       cu_seqlens=torch.tensor([0, 16], dtype=torch.int32, device="cuda"), k_scale=scales.cuda(), v_scale=scales.cuda())
    for pool, y in ((k, x), (v, x.flip(0))):
        want = (y.float() / scales[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
        assert (want[:, :, ::2].view(torch.uint8) == 0x80).all()
        assert torch.equal(pool[0].transpose(0, 1).cpu().view(torch.uint8), want.view(torch.uint8))


# ------------------------------------------------------------------------------------------------------- status
def test_the_check_reports_every_kind_and_clears_what_it_reports():
    """A bad page and a length beyond the table in one call: both are named.  The C entry point clears the bit that it reports and
    no other, so nothing that comes up beside it is lost."""
    q, k, v, ks, vs, table, lens = _case(2, [40, 33], 16, 4, 2, 1, False)
    table[0, 1], lens[1] = -7, 1 << 20
    _run(q, k, v, ks, vs, table, lens)
    with pytest.raises(RuntimeError, match="outside the pool.*longer than its row"):
        aa.check_paged_status()
    aa.check_paged_status()
    word = torch.tensor([7], dtype=torch.int32, device="cuda")
    check, stream = _lib.load().aa_paged_check_status, torch.cuda.current_stream().cuda_stream
    for code, left in ((-11, 3), (-17, 2), (-18, 0), (0, 0)):
        assert check(word.data_ptr(), stream) == code and word.item() == left


# ------------------------------------------------------------------------------------------- tables of any width
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("lens,H,Hkv,n", [([5], 8, 2, 1), ([120, 0, 64, 1], 32, 8, 1), ([380], 8, 2, 1), ([250] * 16, 32, 8, 1),
                                          ([130, 40], 8, 2, 5), ([90], 8, 1, 4), ([4000, 33], 4, 4, 16)])
def test_attention_with_a_table_wider_than_the_sequences(lens, H, Hkv, n, fp8):
    """Entries are cut by a rule on the table's width: whole with a narrow table, cut with a wide one.  Both are right."""
    for width in (None, 8192):
        q, k, v, ks, vs, table, lens_t = _case(7, lens, 16, H, Hkv, n, fp8, width=width)
        got, got_lse = _run(q, k, v, ks, vs, table, lens_t)
        assert_decode(got, got_lse, q, oracle.dequantised(k, ks), oracle.dequantised(v, vs), table[:, :256], lens_t, fp8)


@pytest.mark.parametrize("width", [13, 129, 513, 20000])
def test_selection_with_a_table_wider_than_the_sequences(width):
    """The blocks of a sequence are chosen by the table's width."""
    g = torch.Generator().manual_seed(width)
    lens = [200, 0, 16, 199]
    table, total = make_table(lens, 16, g, width=width)
    codes = torch.randint(-127, 128, (total, 2, 128), generator=g, dtype=torch.int8)
    scales = torch.rand(total, 2, generator=g) / 100
    q = torch.randn(4, 2, 8, 128, generator=g).bfloat16()
    lens = torch.tensor(lens, dtype=torch.int32)
    got = aa.select_pages(*[t.cuda() for t in (q, codes, scales, table, lens)], 6, 16)
    want = oracle.select(q, codes, scales, table, lens, 6, 16)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_selection_of_the_most_rows():
    """256 rows a KV head (16 new tokens on a group of 16) are the most that the selection takes; the attention takes more."""
    g = torch.Generator().manual_seed(1)
    table, total = make_table([900], 16, g)
    codes = torch.randint(-127, 128, (total, 1, 128), generator=g, dtype=torch.int8)
    scales = torch.rand(total, 1, generator=g)
    lens = torch.tensor([900], dtype=torch.int32)
    q = torch.randn(1, 16, 16, 128, generator=g).bfloat16()
    got = aa.select_pages(*[t.cuda() for t in (q, codes, scales, table, lens)], 9, 16)
    want = oracle.select(q, codes, scales, table, lens, 9, 16)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    q = torch.randn(1, 16, 17, 128, generator=g).bfloat16()
    with pytest.raises(RuntimeError, match="too many new tokens"):
        aa.select_pages(*[t.cuda() for t in (q, codes, scales, table, lens)], 9, 16)
