"""Edge cases of the paged cache on the GPU: arguments and cache contents at the borders of what the functions accept."""
import math

import pytest
import torch

import anchor_attention_b200 as aa
from oracle import paged_oracle as oracle
from paged_util import make_pool, make_table

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
