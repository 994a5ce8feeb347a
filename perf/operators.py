"""The serving operators of the paged key-value cache, as workloads with a plain form.

Three operators carry token generation behind an anchor-attention prefill:

* ``append``  rotate the new keys (and queries) by their positions and write keys and values into the pages of
  a cache, bf16 or e4m3, with an 8-bit mean key kept for every page that fills up;
* ``select``  the pages of a long cache that a cheap score (8-bit query against 8-bit page mean) picks for
  every sequence and key head;
* ``attend``  attention of one or a few new tokens over the cached ones, over all pages or over picked ones.

Layouts: pages [pages, key heads, page size, 128]; new tokens [tokens, heads, 128]; queries of an attention
[sequences, new tokens, heads, 128]; a block table [sequences, width] names the pages of every sequence in order,
and ``seq_lens`` counts the tokens of every sequence, the new ones included.  Query head h belongs to key head
h // (heads / key heads).  Page numbers behind a sequence's end are -1.
"""
import math

import torch

own = False

DIM = 128
HALF = DIM // 2
DEVICE = "cuda"
HEADS = [(32, 8), (28, 4), (16, 16), (8, 1), (64, 8)]


# ----------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one chat turn of a short sequence: nothing but latency
        dict(name="attend_one_short", op="attend", heads=32, kv_heads=8, page=16, batch=1, longest=577, shortest=1.0, new=1,
             fp8=False, picked=0),
        # a small server batch of mixed lengths, one slot of the batch empty (padding of a captured graph)
        dict(name="attend_batch", op="attend", heads=28, kv_heads=4, page=32, batch=16, longest=4001, shortest=0.02, new=1,
             fp8=False, picked=0, empty=1),
        # one user on a whole-context prompt, the length of the repository's benchmark
        dict(name="attend_one_long", op="attend", heads=32, kv_heads=8, page=64, batch=1, longest=131072, shortest=1.0, new=1,
             fp8=False, picked=0),
        # a full server batch of long prompts of mixed lengths: the largest cache that is read
        dict(name="attend_batch_long", op="attend", heads=32, kv_heads=8, page=64, batch=32, longest=32768, shortest=0.1, new=1,
             fp8=False, picked=0),
        # the same kind of batch on a cache kept in 8 bits
        dict(name="attend_fp8", op="attend", heads=32, kv_heads=8, page=64, batch=32, longest=32768, shortest=0.1, new=1,
             fp8=True, picked=0),
        # five drafted tokens a sequence are checked at once
        dict(name="attend_drafts", op="attend", heads=32, kv_heads=8, page=16, batch=8, longest=16001, shortest=0.25, new=5,
             fp8=False, picked=0),
        # long prompts read through the 64 pages that were picked for each key head
        dict(name="attend_picked", op="attend", heads=32, kv_heads=8, page=64, batch=16, longest=65536, shortest=0.5, new=1,
             fp8=False, picked=64),
        # every sequence of a server batch adds its token
        dict(name="append_tokens", op="append", heads=32, kv_heads=8, page=64, batch=64, longest=1, cached=8192, fp8=False,
             keys_back=False),
        # prompts of mixed lengths enter the cache; the rotated keys are wanted for the prefill attention too
        dict(name="append_prompts", op="append", heads=32, kv_heads=8, page=64, batch=5, longest=8191, cached=0, fp8=False,
             keys_back=True),
        # later chunks of prompts enter an 8-bit cache
        dict(name="append_prompts_fp8", op="append", heads=28, kv_heads=4, page=32, batch=3, longest=6143, cached=1001, fp8=True,
             keys_back=False),
        # pages for one user on a whole-context prompt
        dict(name="select_one", op="select", heads=32, kv_heads=8, page=64, batch=1, longest=131072, shortest=1.0, new=1, top=64),
        # pages for a server batch, small pages
        dict(name="select_batch", op="select", heads=32, kv_heads=8, page=32, batch=32, longest=65536, shortest=0.25, new=1, top=128),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    heads, kv_heads = rng.choice(HEADS)
    page = rng.choice([16, 32, 64, 128])
    op = rng.choice(["attend", "attend", "attend", "append", "select"])
    fp8 = rng.random() < 0.35
    if op == "append":
        longest = 1 if rng.random() < 0.4 else _log_int(rng, 2, 8192)
        batch = _log_int(rng, 1, max(1, min(64, 24576 // longest)))
        return dict(op=op, heads=heads, kv_heads=kv_heads, page=page, batch=batch, longest=longest,
                    cached=_log_int(rng, 1, 2048) - 1, fp8=fp8, keys_back=longest > 1 and rng.random() < 0.5)
    new = 1 if rng.random() < 0.7 else rng.randint(2, 8)
    budget = 400000 * 8 // kv_heads                                # cached tokens: no more than attend_batch_long reads
    batch = _log_int(rng, 1, 64)
    longest = _log_int(rng, new, max(new, min(131072, budget // batch)))
    shortest = round(rng.uniform(0.05, 1.0), 2)
    if op == "select":
        return dict(op=op, heads=heads, kv_heads=kv_heads, page=page, batch=batch, longest=longest, shortest=shortest, new=new,
                    top=_log_int(rng, 4, 256))
    picked = _log_int(rng, 4, 128) if longest > 8 * page and rng.random() < 0.3 else 0
    return dict(op=op, heads=heads, kv_heads=kv_heads, page=page, batch=batch, longest=longest, shortest=shortest, new=new, fp8=fp8,
                picked=picked)


def _lengths(case):
    """The lengths of a case's sequences, longest first: spread between shortest * longest and longest, and empty ones."""
    n, longest, low = case["batch"], case["longest"], case.get("shortest", 0.2)
    least = case.get("new", 1)
    lens = [max(least, round(longest * (1 - (1 - low) * ((i * 0.6180339887) % 1)))) for i in range(n)]
    for i in range(case.get("empty", 0)):
        lens[n - 1 - i] = 0
    return lens


def _cached(case):
    """Tokens that an append's sequences hold already."""
    return [round(case["cached"] * (1 - 0.7 * ((i * 0.4142135624) % 1))) for i in range(case["batch"])]


def _picked_counts(case):
    return [min(case["picked"], -(-n // case["page"])) for n in _lengths(case)]


# ---------------------------------------------------------------------------------------------------- inputs
def _order(n, seed):
    return torch.randperm(n, generator=torch.Generator().manual_seed(seed)).tolist()


def _table(lens, page, g):
    """A block table of shuffled pages for sequences of these lengths, and the number of pages of the pool."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + 3
    ids = torch.randperm(total, generator=g, device=DEVICE).int()
    table = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    return table, total


def _channel_scales(g):
    """Keys have a few strong channels."""
    s = 0.5 + torch.rand(DIM, generator=g, device=DEVICE)
    s[torch.randperm(DIM, generator=g, device=DEVICE)[:4]] *= 3.0
    return s


def _normal(shape, g):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=torch.bfloat16)


def _to_pages(x, scale):
    """bf16 [pages, heads, page, 128] -> e4m3 codes of x / scale[head]."""
    return (x / scale.to(x.dtype)[None, :, None, None]).clamp_(-448, 448).to(torch.float8_e4m3fn)


def prepare(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)
    heads, kv_heads, page, batch = case["heads"], case["kv_heads"], case["page"], case["batch"]
    order = _order(batch, seed)
    if case["op"] == "append":
        return _prepare_append(case, g, order)
    lens = [_lengths(case)[i] for i in order]
    table, total = _table(lens, page, g)
    channel = _channel_scales(g)
    query = (_normal((batch, case["new"], heads, DIM), g) * (2.0 / channel.square().mean().sqrt())).bfloat16()
    state = dict(case=dict(case), query=query, table=table, lens=torch.tensor(lens, dtype=torch.int32, device=DEVICE))
    if case["op"] == "select":
        state["codes"] = torch.randint(-127, 128, (total, kv_heads, DIM), generator=g, device=DEVICE, dtype=torch.int8)
        state["code_scales"] = (0.2 + torch.rand((total, kv_heads), generator=g, device=DEVICE)) / 127
        return state
    k = _normal((total, kv_heads, page, DIM), g).mul_(channel.bfloat16())
    v = _normal((total, kv_heads, page, DIM), g).add_((0.3 * torch.randn(DIM, generator=g, device=DEVICE)).bfloat16())
    state["k_scale"] = state["v_scale"] = None
    if case["fp8"]:
        state["k_scale"] = (0.02 + 0.02 * torch.rand(kv_heads, generator=g, device=DEVICE))
        state["v_scale"] = (0.01 + 0.01 * torch.rand(kv_heads, generator=g, device=DEVICE))
        k, v = _to_pages(k, state["k_scale"]), _to_pages(v, state["v_scale"])
    state["k"], state["v"] = k, v
    state["pages"] = state["counts"] = None
    if case["picked"]:
        counts = torch.tensor([[c] * kv_heads for c in [_picked_counts(case)[i] for i in order]], dtype=torch.int32, device=DEVICE)
        live = -(-state["lens"].long() // page)
        rank = torch.rand((batch, kv_heads, table.shape[1]), generator=g, device=DEVICE)
        index = torch.arange(table.shape[1], device=DEVICE)
        rank.masked_fill_(index >= live[:, None, None], 9.0)
        rank.masked_fill_((index == 0) | (index == live[:, None, None] - 1), -1.0)   # the first and the last page always
        best = rank.argsort(-1)[..., :case["picked"]]
        slot = torch.arange(best.shape[-1], device=DEVICE)
        best = best.masked_fill(slot >= counts[..., None], 1 << 30).sort(-1).values
        state["pages"] = best.masked_fill(best == 1 << 30, -1).int()
        state["counts"] = counts
    return state


def _prepare_append(case, g, order):
    heads, kv_heads, page = case["heads"], case["kv_heads"], case["page"]
    new = [_lengths(case)[i] for i in order]
    lens = [n + c for n, c in zip(new, [_cached(case)[i] for i in order])]
    table, total = _table(lens, page, g)
    tokens = sum(new)
    fused = _normal((tokens, heads + 2 * kv_heads, DIM), g)          # one projection's output: queries, keys, values
    fused[:, heads:heads + kv_heads].mul_(_channel_scales(g).bfloat16())
    state = dict(case=dict(case), query=fused[:, :heads], key=fused[:, heads:heads + kv_heads], value=fused[:, heads + kv_heads:],
                 table=table, lens=torch.tensor(lens, dtype=torch.int32, device=DEVICE), k_scale=None, v_scale=None)
    state["cu"] = None
    if case["longest"] > 1:
        state["cu"] = torch.tensor([0] + new, device=DEVICE).cumsum(0).int()
    angle = torch.arange(max(lens), dtype=torch.float64, device=DEVICE)[:, None] * 500000.0 ** (
        -torch.arange(0, DIM, 2, dtype=torch.float64, device=DEVICE) / DIM)
    state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    k, v = _normal((total, kv_heads, page, DIM), g), _normal((total, kv_heads, page, DIM), g)
    if case["fp8"]:
        state["k_scale"] = (0.02 + 0.02 * torch.rand(kv_heads, generator=g, device=DEVICE))
        state["v_scale"] = (0.01 + 0.01 * torch.rand(kv_heads, generator=g, device=DEVICE))
        k, v = _to_pages(k, state["k_scale"]), _to_pages(v, state["v_scale"])
    state["k"], state["v"] = k, v
    state["codes"] = torch.zeros((total, kv_heads, DIM), dtype=torch.int8, device=DEVICE)
    state["code_scales"] = torch.zeros((total, kv_heads), device=DEVICE)
    return state


# ------------------------------------------------------------------------------------------------------- run
def run(state):
    op = state["case"]["op"]
    if own:
        import anchor_attention_b200 as aa
        if op == "append":
            query, key = aa.paged_kv_append(
                state["key"], state["value"], state["k"], state["v"], state["table"], state["lens"], cu_seqlens=state["cu"],
                query=state["query"], cos=state["cos"], sin=state["sin"], k_scale=state["k_scale"], v_scale=state["v_scale"],
                key_codes=state["codes"], key_code_scales=state["code_scales"], return_key=state["case"]["keys_back"])
            return _append_outputs(state, query, key)
        if op == "select":
            pages, counts = aa.select_pages(state["query"], state["codes"], state["code_scales"], state["table"], state["lens"],
                                            state["case"]["top"], state["case"]["page"])
            return dict(pages=pages, counts=counts)
        out, lse = aa.paged_decode_attention(
            state["query"], state["k"], state["v"], state["table"], state["lens"], k_scale=state["k_scale"], v_scale=state["v_scale"],
            pages=state["pages"], page_counts=state["counts"], return_lse=True)
        return dict(out=out, lse=lse)
    return {"append": _append, "select": _select, "attend": _attend}[op](state)


def _append_outputs(state, query, key):
    outputs = dict(query=query, k=state["k"], v=state["v"], codes=state["codes"], code_scales=state["code_scales"])
    if state["case"]["keys_back"]:
        outputs["key"] = key
    return outputs


def _rotate(x, cos, sin):
    """Rotate-half by the tables' rows, in 32 bits: x [tokens, heads, 128], cos and sin [tokens, 64]."""
    a, b = x[..., :HALF].float(), x[..., HALF:].float()
    c, s = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def _places(state):
    """The sequence, position, page and row of every new token."""
    tokens, batch = state["key"].shape[0], state["table"].shape[0]
    page = state["case"]["page"]
    token = torch.arange(tokens, device=state["key"].device)
    if state["cu"] is None:
        seq, position = token, state["lens"].long() - 1
    else:
        cu = state["cu"].long()
        seq = torch.searchsorted(cu, token, right=True) - 1
        position = state["lens"].long()[seq] - cu[seq + 1] + token
    return position, state["table"][seq, position // page].long(), position % page


def _append(state):
    case = state["case"]
    position, where, row = _places(state)
    cos, sin = state["cos"][position], state["sin"][position]
    query = _rotate(state["query"], cos, sin).bfloat16()
    rotated = _rotate(state["key"], cos, sin)
    k, v = state["k"], state["v"]
    if case["fp8"]:
        codes = [(x / s[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
                 for x, s in ((rotated, state["k_scale"]), (state["value"].float(), state["v_scale"]))]
        k.view(torch.uint8)[where, :, row] = codes[0]
        v.view(torch.uint8)[where, :, row] = codes[1]
    else:
        k[where, :, row] = rotated.bfloat16()
        v[where, :, row] = state["value"]
    full = where[row == case["page"] - 1]                            # the pages that are complete now
    mean = k[full].double().mean(2).float()                          # in 64 bits: the sum's order does not show
    if case["fp8"]:
        mean = mean * state["k_scale"][:, None]
    scale = mean.abs().amax(-1) / 127
    state["codes"][full] = torch.where(scale[..., None] > 0, (mean / scale[..., None]).round(), 0.0).to(torch.int8)
    state["code_scales"][full] = scale
    return _append_outputs(state, query, rotated.bfloat16())


def _select(state):
    case = state["case"]
    batch, new, heads, _ = state["query"].shape
    kv_heads, table, top = case["kv_heads"], state["table"], case["top"]
    q = state["query"].float()
    q_scale = q.abs().amax(-1, keepdim=True) / 127
    q_code = torch.where(q_scale > 0, (q / q_scale).round().clamp(-127, 127), 0.0)
    rows = new * heads // kv_heads

    def by_head(x):
        return x.view(batch, new, kv_heads, heads // kv_heads, -1).transpose(1, 2).reshape(batch, kv_heads, rows, -1)

    k_code = state["codes"][table.long()].permute(0, 2, 1, 3).float()             # [batch, kv_heads, width, 128]
    dots = by_head(q_code) @ k_code.transpose(-1, -2)                            # whole numbers below 2^24: exact in any order
    score = (dots * by_head(q_scale)).amax(2) * state["code_scales"][table.long()].transpose(1, 2)
    live = -(-state["lens"].long() // case["page"])[:, None, None]
    index = torch.arange(table.shape[1], device=table.device)
    score = score.masked_fill((index < 1) | (index >= live - 2), math.inf)        # the first page and the last two are kept
    score = score.masked_fill(index >= live, -math.inf)
    best = score.sort(dim=-1, descending=True, stable=True).indices[..., :top]
    counts = live[..., 0].clamp(max=top).expand(batch, kv_heads).int()
    slot = torch.arange(best.shape[-1], device=table.device)
    best = best.masked_fill(slot >= counts[..., None], 1 << 30).sort(-1).values
    pages = torch.full((batch, kv_heads, top), -1, dtype=torch.int32, device=table.device)
    pages[..., :best.shape[-1]] = best.masked_fill(best == 1 << 30, -1).int()
    return dict(pages=pages, counts=counts.contiguous())


def _attend(state):
    case = state["case"]
    query, table = state["query"], state["table"]
    batch, new, heads, _ = query.shape
    kv_heads, page = case["kv_heads"], case["page"]
    group = heads // kv_heads
    lens = state["lens"].long()
    if state["pages"] is None:
        index = torch.arange(table.shape[1], device=table.device)[None, None].expand(batch, 1, -1)
        here = index >= 0
    else:
        index = state["pages"].long()
        here = index >= 0
        index = index.clamp(min=0)
    position = (index[..., None] * page + torch.arange(page, device=table.device)).flatten(2)     # [batch, 1 or kv_heads, keys]
    here = here.repeat_interleave(page, dim=-1)
    where = table.long()[torch.arange(batch, device=table.device)[:, None, None], index]
    head = torch.arange(kv_heads, device=table.device)[None, :, None]

    def cached(pool, scale):
        if pool.dtype != torch.bfloat16:
            x = pool.view(torch.uint8)[where, head].view(pool.dtype).float() * scale[:, None, None, None]
        else:
            x = pool[where, head].float()
        return x.reshape(batch, kv_heads, -1, DIM)

    q = query.float().view(batch, new, kv_heads, group, DIM).transpose(1, 2).reshape(batch, kv_heads, new * group, DIM)
    score = q @ cached(state["k"], state["k_scale"]).transpose(-1, -2) * DIM ** -0.5
    last = lens[:, None] - new + torch.arange(new, device=table.device)                          # a row's own position
    last = last.repeat_interleave(group, dim=1)[:, None, :, None]
    score.masked_fill_(~here[:, :, None] | (position[:, :, None] > last), -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    out = p @ cached(state["v"], state["v_scale"])
    out = torch.where(total > 0, out / total, 0.0)
    lse = (top + total.log())[..., 0]

    def by_token(x):
        return x.view(batch, kv_heads, new, group, -1).transpose(1, 2).reshape(batch, new, heads, -1)

    return dict(out=by_token(out).bfloat16(), lse=by_token(lse[..., None])[..., 0])


# ----------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    if case["op"] == "select":
        return None                                                  # whole numbers only
    state = prepare(case, seed)
    return _exact_append(state) if case["op"] == "append" else _exact_attend(state)


def _exact_attend(state):
    query, k, v = state["query"].double(), state["k"], state["v"]
    batch, new, heads, _ = query.shape
    kv_heads, page = k.shape[1], k.shape[2]
    out = torch.zeros(query.shape, dtype=torch.float64, device=query.device)
    lse = torch.full(query.shape[:3], -math.inf, dtype=torch.float64, device=query.device)
    lens, table = state["lens"].tolist(), state["table"].tolist()
    picked = None if state["pages"] is None else state["pages"].tolist()
    for b in range(batch):
        for h in range(kv_heads):
            index = list(range(-(-lens[b] // page))) if picked is None else [i for i in picked[b][h] if i >= 0]
            if not index:
                continue
            where = torch.tensor([table[b][i] for i in index], device=query.device)
            keys, values = k[:, h][where].double().flatten(0, 1), v[:, h][where].double().flatten(0, 1)
            if state["k_scale"] is not None:
                keys, values = keys * state["k_scale"][h].double(), values * state["v_scale"][h].double()
            at = torch.tensor(index, device=query.device).repeat_interleave(page) * page + torch.arange(
                page, device=query.device).repeat(len(index))
            first, last = h * heads // kv_heads, (h + 1) * heads // kv_heads
            for j in range(new):
                seen = at <= lens[b] - new + j
                s = query[b, j, first:last] @ keys[seen].T / math.sqrt(DIM)
                if s.shape[1]:
                    lse[b, j, first:last] = s.logsumexp(-1)
                    out[b, j, first:last] = s.softmax(-1) @ values[seen]
    return dict(out=out, lse=lse)


def _exact_append(state):
    case = state["case"]
    page, batch = case["page"], len(state["lens"])
    k, v = state["k"].double(), state["v"].double()
    query = torch.zeros(state["query"].shape, dtype=torch.float64, device=k.device)
    key = torch.zeros(state["key"].shape, dtype=torch.float64, device=k.device)
    begins = list(range(batch + 1)) if state["cu"] is None else state["cu"].tolist()
    turn = torch.complex(state["cos"].double(), state["sin"].double())[:, None]
    for b, end in enumerate(state["lens"].tolist()):
        lo, hi = begins[b], begins[b + 1]
        at = torch.arange(end - (hi - lo), end, device=k.device)
        for x, y in ((state["query"], query), (state["key"], key)):
            z = torch.complex(x[lo:hi, :, :HALF].double(), x[lo:hi, :, HALF:].double()) * turn[at]
            y[lo:hi] = torch.cat([z.real, z.imag], -1)
        where = state["table"][b].long()[at // page]
        if case["fp8"]:
            k[where, :, at % page] = key[lo:hi] / state["k_scale"].double()[:, None]
            v[where, :, at % page] = state["value"][lo:hi].double() / state["v_scale"].double()[:, None]
        else:
            k[where, :, at % page] = key[lo:hi]
            v[where, :, at % page] = state["value"][lo:hi].double()
    # the codes and their scales are those of the keys as they were rounded for the pages: no value in 64 bits
    outputs = dict(query=query, k=k, v=v, codes=None, code_scales=None)
    if case["keys_back"]:
        outputs["key"] = key
    return outputs


# ------------------------------------------------------------------------------------------------------ work
def work(case):
    heads, kv_heads, page, batch = case["heads"], case["kv_heads"], case["page"], case["batch"]
    lens = _lengths(case)
    if case["op"] == "append":
        tokens, size = sum(lens), 1 if case["fp8"] else 2
        ends = [(c, c + n) for c, n in zip(_cached(case), lens)]
        full = sum(e // page - s // page for s, e in ends)
        old = sum(min(s % page, s) for s, e in ends if e // page > s // page)       # cached rows of the pages that fill up
        moved = tokens * DIM * (2 * (heads + 2 * kv_heads) + 2 * heads + 2 * size * kv_heads + (2 * kv_heads if case["keys_back"] else 0))
        moved += 4 * DIM * max(e for _, e in ends) if case["longest"] > 1 else 4 * DIM * tokens
        moved += full * kv_heads * (DIM + 4) + old * kv_heads * DIM * size
        return {"bytes": moved, "flops": tokens * (heads + kv_heads) * DIM * 3}
    rows = batch * case["new"] * heads
    if case["op"] == "select":
        live = [-(-n // page) for n in lens]
        found = sum(min(case["top"], n) for n in live) * kv_heads
        return {"bytes": sum(live) * (kv_heads * (DIM + 4) + 4) + rows * DIM * 2 + found * 4 + 4 * batch * (1 + kv_heads),
                "flops": 2 * DIM * case["new"] * heads * sum(live)}
    keys = [min(n, c * page) for n, c in zip(lens, _picked_counts(case))] if case["picked"] else lens
    pages = sum(-(-n // page) for n in keys)
    moved = sum(keys) * kv_heads * 2 * DIM * (1 if case["fp8"] else 2) + rows * (4 * DIM + 4) + 4 * batch + 4 * pages
    moved += 4 * pages * kv_heads if case["picked"] else 0
    return {"bytes": moved, "flops": 4 * DIM * case["new"] * heads * sum(keys)}
