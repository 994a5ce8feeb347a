"""Inputs and error bounds shared by the tests of the paged key-value cache."""
import math

import torch

from oracle import paged_oracle as oracle


def make_table(lens, page, g, spare=3, width=None):
    """Shuffled pages for sequences of these lengths: (block_table on the CPU, pages of the pool)."""
    need = [-(-max(n, 0) // page) for n in lens]
    total = sum(need) + spare
    ids = torch.randperm(total, generator=g).int()
    table = torch.full((len(lens), width or max(1, max(need, default=1))), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    return table, total


def make_pool(total, kv_heads, page, g, fp8, nhd=False):
    """(k, v, k_scale, v_scale) on the CPU; nhd: [pages, page, heads, 128] memory."""
    def pool():
        shape = (total, page, kv_heads, 128) if nhd else (total, kv_heads, page, 128)
        x = torch.randn(shape, generator=g).bfloat16()
        return x.transpose(1, 2) if nhd else x
    k, v = pool(), pool()
    if not fp8:
        return k, v, None, None
    ks, vs = (0.02 + 0.02 * torch.rand(kv_heads, generator=g) for _ in range(2))
    return tuple((x.float() / s[None, :, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn) for x, s in ((k, ks), (v, vs))) + (ks, vs)


def decode_bounds(query, k, v, out, lse, weight, spread, fp8):
    """How far a 32-bit evaluation may be from the 64-bit one.

    A score is a dot product of 128 exact products added in 32 bits: off by at most 128 * 2^-23 * sum |q k| scale (a
    tensor core may truncate instead of rounding, hence 2^-23); with e4m3 pages the query's f16 copy is off by
    2^-33 of its row's largest value per element.  Scaling, the exponential (2^-22) and its argument (2^-24 of a
    score below 2^8 in log2 units) add 2^-15 at most.  A weight's relative error d makes an output error of 2 d sum p |v|
    (numerator and denominator).  A probability is held in two bf16 values: the upper one is cut off, which leaves a rest
    below 2^-7 of it, and the rest is rounded, 2^-8 of 2^-7, plus a last bit of 32-bit arithmetic: 2^-15 + 2^-22.  For
    e4m3 pages it is rounded to f16: 2^-11, and 2^-25 absolute.  The output is rounded to bf16 once: 2^-8 of its value."""
    d = 128 * 2.0 ** -23 * spread + 2.0 ** -15
    absolute = 0.0
    if fp8:
        d = d + 128 ** 0.5 * 2.0 ** -33 * query.double().abs().amax(-1) * k.abs().max() * 128 ** 0.5
        absolute = 2.0 ** -25 * k.shape[0] * k.shape[2] * v.abs().max()
    held = 2.0 ** -11 if fp8 else 2.0 ** -15 + 2.0 ** -22
    tol_out = 2.0 ** -8 * out.abs() + (2 * d + held)[..., None] * weight + absolute + 1e-30
    tol_lse = d + 2.0 ** -20 + 2.0 ** -22 * torch.where(lse.isfinite(), lse.abs(), torch.zeros_like(lse))
    return tol_out, tol_lse


def assert_decode(got, got_lse, query, k, v, table, lens, fp8, **kw):
    """The kernel's outputs (any device) against the 64-bit ones; k, v 64-bit pools on the CPU."""
    out, lse, weight, spread = oracle.attend(query, k, v, table, lens, **kw)
    tol_out, tol_lse = decode_bounds(query, k, v, out, lse, weight, spread, fp8)
    got, got_lse = got.double().cpu().view(out.shape), got_lse.double().cpu().view(lse.shape)
    empty = lse == -math.inf
    assert torch.equal(got_lse == -math.inf, empty)
    assert bool((got[empty] == 0).all())
    over = ((got - out).abs() / tol_out).amax()
    assert over <= 1, f"output {float(over):.3g} times its bound"
    over = ((got_lse - lse)[~empty].abs() / tol_lse[~empty]).amax() if (~empty).any() else 0
    assert over <= 1, f"lse {float(over):.3g} times its bound"
    return out, lse
