"""The paged key-value cache in plain torch, 64 bits, on the CPU (test infrastructure): what the operators of
``anchor_attention_b200.paged`` compute, written from their formulas one sequence at a time."""
import math

import torch

INV_127 = torch.tensor(1.0) / 127            # in 32 bits


def dequantised(pool, scale):
    """A pool [pages, Hkv, page, 128] as 64-bit values."""
    x = pool.float().double()
    return x if scale is None else x * scale.double()[None, :, None, None]


def rotate(x, cos, sin):
    """Rotate-half in 64 bits: x [n, heads, 128], cos / sin [n, 64]."""
    a, b = x[..., :64].double(), x[..., 64:].double()
    c, s = cos.double()[:, None], sin.double()[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def gather(pool, table_row, positions):
    """Rows of a [pages, Hkv, page, 128] pool at the positions of one sequence: [Hkv, n, 128]."""
    page = pool.shape[2]
    return pool[table_row[positions // page].long(), :, positions % page].transpose(0, 1)


def attend(query, k, v, block_table, seq_lens, scaling=None, pages=None, page_counts=None):
    """query [B, n, H, 128]; k, v 64-bit pools.  Returns (out, lse, weight, spread): the 64-bit output, the natural
    logarithm of the softmax sums, sum p |v| and the largest |q| . |k| of a row -- what rounding errors scale with."""
    B, n, H, _ = query.shape
    Hkv, page = k.shape[1], k.shape[2]
    group = H // Hkv
    scaling = 128 ** -0.5 if scaling is None else scaling
    out = torch.zeros(query.shape, dtype=torch.float64)
    weight = torch.zeros(query.shape, dtype=torch.float64)
    lse = torch.full(query.shape[:3], -math.inf, dtype=torch.float64)
    spread = torch.zeros(query.shape[:3], dtype=torch.float64)
    for b in range(B):
        length = min(max(int(seq_lens[b]), 0), block_table.shape[1] * page)
        for h in range(Hkv):
            if pages is None:
                positions = torch.arange(length)
            else:
                listed = pages[b, h, :int(page_counts[b, h])].long()
                positions = (listed[:, None] * page + torch.arange(page)).flatten()
                positions = positions[positions < length]
            keep = (block_table[b][positions // page] >= 0) & (block_table[b][positions // page] < k.shape[0])
            positions = positions[keep]
            if positions.numel() == 0:
                continue
            K, V = gather(k, block_table[b], positions)[h], gather(v, block_table[b], positions)[h]
            for j in range(n):
                seen = positions <= length - n + j
                if not seen.any():
                    continue
                heads = slice(h * group, (h + 1) * group)
                q = query[b, j, heads].double()
                s = q @ K[seen].T * scaling
                p = s.softmax(-1)
                out[b, j, heads] = p @ V[seen]
                weight[b, j, heads] = p @ V[seen].abs()
                lse[b, j, heads] = s.logsumexp(-1)
                spread[b, j, heads] = (q.abs() @ K[seen].abs().T).amax(-1) * abs(scaling)
    return out, lse, weight, spread


def page_summary(k_pool, page, k_scale=None):
    """(codes int8 [Hkv, 128], scales fp32 [Hkv]) of one stored page; the mean in 64 bits, then the 32-bit steps
    of the definition."""
    mean = k_pool[page].float().double().mean(1).float()
    if k_scale is not None:
        mean = mean * k_scale[:, None]
    scale = mean.abs().amax(-1) * INV_127
    codes = torch.where(scale[:, None] > 0, (mean / scale[:, None]).round(), torch.zeros_like(mean))
    return codes.to(torch.int8), scale


def select(query, codes, code_scales, block_table, seq_lens, top, page, keep_first=1, keep_last=2):
    """(lists, counts) by the definition: whole-number dot products, 32-bit scale products, ties to the lower page."""
    B, n, H, _ = query.shape
    Hkv = codes.shape[1]
    group = H // Hkv
    q = query.float()
    q_scale = q.abs().amax(-1) * INV_127
    q_code = torch.where(q_scale[..., None] > 0, (q / q_scale[..., None]).round().clamp(-127, 127), torch.zeros_like(q)).long()
    out = torch.full((B, Hkv, top), -1, dtype=torch.int32)
    counts = torch.zeros((B, Hkv), dtype=torch.int32)
    for b in range(B):
        live = -(-max(int(seq_lens[b]), 0) // page)
        where = block_table[b, :live].long()
        for h in range(Hkv):
            heads = slice(h * group, (h + 1) * group)
            dots = torch.einsum('nhd,pd->nhp', q_code[b, :, heads], codes[where, h].long())
            score = (dots.float() * q_scale[b, :, heads, None]).flatten(0, 1).amax(0) * code_scales[where, h]
            forced = (torch.arange(live) < keep_first) | (torch.arange(live) >= live - keep_last)
            order = sorted(range(live), key=lambda i: (not forced[i], -float(score[i]), i))[:top]
            counts[b, h] = len(order)
            out[b, h, :len(order)] = torch.tensor(sorted(order), dtype=torch.int32)
    return out, counts
