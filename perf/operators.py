"""What the serving operators around a cache in 4 bits are measured on: block tables and slot maps built on the GPU,
keys and values written into pages of 4 bits and read back, attention over such pages, and the log probabilities of
given tokens.

The cache of 4 bits, as the operators define it: a head's key or value is cut into groups of 32 elements; a group with
the largest magnitude ``a`` has the scale ``2^e``, ``e = floor(log2 a) - 2`` (at least -125), held as the byte
``e + 127``, and every element the code of ``x / 2^e`` rounded to the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6 (ties to
the even code), sign in the fourth bit.  Pages:

    key codes     [pages, kv heads, tokens, d/2]            two elements a byte, the lower one in the low half
    key scales    [pages, kv heads, tokens, d/32]
    value codes   [pages, kv heads, tokens/4, d/8, 4, 4]    (four tokens, eight elements): four bytes a token
    value scales  [pages, kv heads, tokens/4, d/32, 4]
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


# -- cases ---------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a decode step of a serving engine: a token for each of 64 requests of up to 4,096 tokens
        {"name": "tables_decode", "op": "tables", "requests": 64, "longest": 4096, "new": 1, "page": 16},
        # a step that packs prompts: 256 requests bring some 32 thousand tokens, the block tables reach 32,768 tokens
        {"name": "tables_prompts", "op": "tables", "requests": 256, "longest": 32768, "new": 257, "page": 32},
        # keys and values of a decode step (the 8-head cache of the Qwen3 models)
        {"name": "append_decode", "op": "append", "tokens": 64, "kv_heads": 8, "dim": 128, "page": 16, "type": "bfloat16"},
        # keys and values of a packed step of prompts, in the float32 path, ragged
        {"name": "append_prompt", "op": "append", "tokens": 8209, "kv_heads": 8, "dim": 128, "page": 16, "type": "float32"},
        # decoding at batch 8 behind 512-token prompts (the default benchmark's step, 0.6B head counts)
        {"name": "decode_short", "op": "attention", "requests": 8, "longest": 532, "ragged": False, "new": 1, "heads": 16,
         "kv_heads": 8, "dim": 128, "page": 16, "window": 0, "type": "bfloat16"},
        # decoding at batch 64, requests of every length up to 8,192 (8B head counts)
        {"name": "decode_batch", "op": "attention", "requests": 64, "longest": 8192, "ragged": True, "new": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "window": 0, "type": "bfloat16"},
        # a few very long contexts
        {"name": "decode_long", "op": "attention", "requests": 4, "longest": 131071, "ragged": False, "new": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "type": "bfloat16"},
        # portions of prompts behind what is held already
        {"name": "prompt_portions", "op": "attention", "requests": 4, "longest": 8192, "ragged": True, "new": 2048,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "window": 0, "type": "bfloat16"},
        # the float32 path, a window, small heads, odd lengths
        {"name": "portions_window", "op": "attention", "requests": 7, "longest": 1511, "ragged": True, "new": 129,
         "heads": 12, "kv_heads": 4, "dim": 64, "page": 8, "window": 500, "type": "float32"},
        # the tokens a decode step picked, with five alternatives (vocabulary of the Qwen3 models)
        {"name": "logprobs_decode", "op": "logprobs", "rows": 8, "vocab": 151936, "top": 5, "type": "float32"},
        # scoring prompts: every row's next token, twenty alternatives
        {"name": "logprobs_score", "op": "logprobs", "rows": 1024, "vocab": 151936, "top": 20, "type": "bfloat16"},
        # an odd vocabulary, no alternatives
        {"name": "logprobs_odd", "op": "logprobs", "rows": 501, "vocab": 50001, "top": 0, "type": "float32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("tables", "append", "attention", "attention", "logprobs"))
    if op == "tables":
        requests = _log(rng, 1, 700)
        return {"op": op, "requests": requests, "longest": _log(rng, 16, 40000), "new": _log(rng, 1, max(1, 60000 // requests)),
                "page": rng.choice((8, 16, 32, 64, 128))}
    if op == "append":
        return {"op": op, "tokens": _log(rng, 1, 9000), "kv_heads": rng.choice((1, 2, 4, 8)),
                "dim": rng.choice((32, 64, 96, 128, 256)), "page": rng.choice((8, 16, 32, 64, 128)),
                "type": rng.choice(("float32", "bfloat16"))}
    if op == "logprobs":
        vocab = _log(rng, 100, 260000)
        return {"op": op, "rows": _log(rng, 1, max(1, 150_000_000 // vocab)), "vocab": vocab,
                "top": min(rng.choice((0, 1, 5, 20, 32)), vocab), "type": rng.choice(("float32", "bfloat16"))}
    kv_heads = rng.choice((1, 2, 4, 8))
    case = {"op": op, "kv_heads": kv_heads, "heads": kv_heads * rng.choice((1, 2, 3, 4, 8, 16)),
            "dim": rng.choice((32, 64, 96, 128, 256)), "page": rng.choice((8, 16, 32, 64, 128)),
            "ragged": rng.random() < 0.7, "type": rng.choice(("float32", "bfloat16", "bfloat16"))}
    if rng.random() < 0.5:      # decoding
        case["longest"] = _log(rng, 1, 60000)
        case["requests"] = _log(rng, 1, max(1, min(128, 200_000 // case["longest"])))
        case["new"] = rng.choice((1, 1, 1, 2, 4))
    else:                       # prompts
        case["longest"] = _log(rng, 32, 6000)
        case["new"] = _log(rng, 2, min(1500, case["longest"]))
        case["requests"] = _log(rng, 1, max(1, min(16, 12_000_000 // (case["new"] * case["longest"]))))
    case["new"] = min(case["new"], case["longest"])
    case["window"] = 0 if rng.random() < 0.6 else _log(rng, 1, case["longest"])
    return case


# -- inputs --------------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed) * 2654435761 % (1 << 31) + 17)


def _integers(g, lo, hi, n):
    return torch.randint(lo, hi + 1, (n,), generator=g, device=DEVICE, dtype=torch.int32)


def _news(case, seed):
    """New tokens of every request: always as many in all, another request each seed."""
    rng = random.Random(case["requests"] * 65537 + case["new"])
    news = [case["new"]] + [rng.randint(max(1, case["new"] // 2), case["new"]) for _ in range(case["requests"] - 1)]
    turn = seed % case["requests"]
    return news[turn:] + news[:turn]


def prepare(case, seed):
    g = _generator(seed)
    return {"tables": _prepare_tables, "append": _prepare_append, "attention": _prepare_attention,
            "logprobs": _prepare_logprobs}[case["op"]](case, seed, g)


def _prepare_tables(case, seed, g):
    b, page = case["requests"], case["page"]
    columns = -(-(case["longest"] + case["new"]) // page)
    lengths = _integers(g, 0, case["longest"], b)
    host_new = _news(case, seed)
    news = torch.tensor(host_new, dtype=torch.int32, device=DEVICE)
    pool = b * columns
    order = torch.randperm(pool, generator=g, device=DEVICE).to(torch.int32)
    held = (lengths + page - 1) // page
    table = torch.full((b, columns), -1, dtype=torch.int32, device=DEVICE)
    mapped = torch.arange(columns, device=DEVICE)[None, :] < held[:, None]
    total_held = int(mapped.sum())
    table[mapped] = order[:total_held]
    free = torch.sort(order[total_held:]).values if total_held < pool else order[:0]
    tokens = sum(host_new)
    return {"case": case, "lengths": lengths, "news": news, "table": table, "free": free.contiguous(),
            "cursor": torch.zeros(1, dtype=torch.int32, device=DEVICE), "tokens": tokens}


def _random_rows(g, rows, width):
    """Rows as keys and values have them: every channel with a spread of its own, a few of them large."""
    spread = torch.exp(0.5 * torch.randn(width, generator=g, device=DEVICE))
    return torch.randn((rows, width), generator=g, device=DEVICE) * spread


def _empty_pages(pages, kv_heads, page, dim):
    shapes = ((pages, kv_heads, page, dim // 2), (pages, kv_heads, page, dim // 32),
              (pages, kv_heads, page // 4, dim // 8, 4, 4), (pages, kv_heads, page // 4, dim // 32, 4))
    return tuple(torch.zeros(s, dtype=torch.uint8, device=DEVICE) for s in shapes)


def _prepare_append(case, seed, g):
    t, h, d, page = case["tokens"], case["kv_heads"], case["dim"], case["page"]
    dtype = TYPES[case["type"]]
    pages = -(-t // page) + 1
    k = _random_rows(g, t, h * d).to(dtype)
    v = _random_rows(g, t, h * d).to(dtype)
    # runs of neighbouring tokens on pages in any order
    order = torch.randperm(pages, generator=g, device=DEVICE)
    at = torch.arange(t, device=DEVICE)
    slots = (order[at // page] * page + at % page).to(torch.int32)
    every = torch.arange(pages * page, dtype=torch.int32, device=DEVICE)
    return {"case": case, "k": k, "v": v, "slots": slots, "every": every, "pages": _empty_pages(pages, h, page, d)}


def _prepare_attention(case, seed, g):
    b, d, h, page = case["requests"], case["dim"], case["kv_heads"], case["page"]
    longest, new = case["longest"], case["new"]
    host_new = _news(case, seed) if case["ragged"] else [new] * b
    news = torch.tensor(host_new, dtype=torch.int32, device=DEVICE)
    if case["ragged"]:
        lengths = torch.maximum(_integers(g, max(1, longest // 8), longest, b), news)
        lengths[0] = longest
    else:
        lengths = torch.full((b,), longest, dtype=torch.int32, device=DEVICE)
    host_lengths = lengths.tolist()
    columns = -(-longest // page)
    held = (lengths + page - 1) // page
    pages = sum(-(-n // page) for n in host_lengths)
    table = torch.full((b, columns), -1, dtype=torch.int32, device=DEVICE)
    table[torch.arange(columns, device=DEVICE)[None, :] < held[:, None]] = (
        torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32))
    cache = _empty_pages(pages, h, page, d)
    step = max(1, (1 << 26) // (h * page * d))
    spread = 0.5 * torch.exp(0.3 * torch.randn((h, 1, d), generator=g, device=DEVICE))
    for lo in range(0, pages, step):       # pages of the pool, filled a run at a time
        hi = min(pages, lo + step)
        for which in (0, 2):
            x = torch.randn((hi - lo, h, page, d), generator=g, device=DEVICE) * spread
            codes, scales = _quantise(x)
            if which == 0:
                cache[0][lo:hi], cache[1][lo:hi] = _pack(codes), scales
            else:
                packed = _pack(codes).view(hi - lo, h, page // 4, 4, d // 8, 4)
                cache[2][lo:hi] = packed.transpose(3, 4)
                cache[3][lo:hi] = scales.view(hi - lo, h, page // 4, 4, d // 32).transpose(3, 4)
    offsets = torch.zeros(b + 1, dtype=torch.int32, device=DEVICE)
    offsets[1:] = torch.cumsum(news, 0)
    q = torch.randn((sum(host_new), case["heads"] * d), generator=g, device=DEVICE).to(TYPES[case["type"]])
    return {"case": case, "q": q, "pages": cache, "table": table, "offsets": offsets, "lengths": lengths,
            "host_lengths": host_lengths, "host_new": host_new, "longest": max(host_lengths), "most": max(host_new)}


def _prepare_logprobs(case, seed, g):
    n, vocab = case["rows"], case["vocab"]
    logits = torch.randn((n, vocab), generator=g, device=DEVICE) * 2.5
    # a model is surer of a few tokens of every row than of the rest
    some = torch.randint(0, vocab, (n, 8), generator=g, device=DEVICE)
    logits.scatter_add_(1, some, 6.0 * torch.rand((n, 8), generator=g, device=DEVICE))
    tokens = torch.where(torch.rand(n, generator=g, device=DEVICE) < 0.7, some[:, 0],
                         torch.randint(0, vocab, (n,), generator=g, device=DEVICE)).to(torch.int32)
    return {"case": case, "logits": logits.to(TYPES[case["type"]]), "tokens": tokens}


# -- the number format, plain -----------------------------------------------------------------------------------------
def _quantise(x):
    """Codes (uint8, one an element) and scale bytes of the groups of 32 along the last dimension."""
    x = x.to(torch.float32)
    groups = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    largest = groups.abs().amax(-1)
    exponent = torch.frexp(largest).exponent - 1 - 2            # frexp's mantissa lies in [1/2, 1)
    exponent = torch.where(largest > 0, exponent, torch.full_like(exponent, -125)).clamp(min=-125)
    y = torch.ldexp(groups, -exponent[..., None])
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = (code + 8 * (y < 0)).to(torch.uint8)
    return code.reshape(x.shape), (exponent + 127).to(torch.uint8)


def _pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _values(packed, scales):
    """float32 values of packed codes ``[..., d/2]`` with scales ``[..., d/32]``."""
    levels = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=torch.float32, device=packed.device)
    low, high = levels[(packed & 15).int()], levels[(packed >> 4).int()]
    x = torch.stack((low, high), -1).reshape(*packed.shape[:-1], packed.shape[-1] // 16, 32)
    return torch.ldexp(x, (scales.to(torch.int32) - 127)[..., None]).reshape(*packed.shape[:-1], 2 * packed.shape[-1])


def _value_rows(codes, scales):
    """Value pages with the tokens in order: (codes [..., tokens, d/2], scales [..., tokens, d/32])."""
    p, h, blocks, octets = codes.shape[:4]
    return (codes.transpose(3, 4).reshape(p, h, blocks * 4, octets * 4),
            scales.transpose(3, 4).reshape(p, h, blocks * 4, scales.shape[3]))


# -- one pass ------------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        from lockstep_amd.ops import Fp4Pages, kernels

        return {"tables": _own_tables, "append": _own_append, "attention": _own_attention,
                "logprobs": _own_logprobs}[op](state, kernels(), Fp4Pages)
    return {"tables": _plain_tables, "append": _plain_append, "attention": _plain_attention,
            "logprobs": _plain_logprobs}[op](state)


def _table_outputs(state):
    b, t = state["lengths"].shape[0], state["tokens"]
    make = lambda n: torch.empty(n, dtype=torch.int32, device=DEVICE)  # noqa: E731
    return {"slots": make(t), "tok_seq": make(t), "tok_pos": make(t), "offsets": make(b + 1), "new_lengths": make(b),
            "progress": make(2)}


def _own_tables(state, k, _):
    out = _table_outputs(state)
    k.step_tables(state["lengths"], state["news"], state["table"], state["case"]["page"], state["free"], state["cursor"],
                  out["slots"], out["tok_seq"], out["tok_pos"], out["offsets"], out["new_lengths"], out["progress"])
    return {"table": state["table"], **out}


def _plain_tables(state):
    lengths, news, table, free = state["lengths"].long(), state["news"].long(), state["table"], state["free"]
    page, (b, columns) = state["case"]["page"], table.shape
    cursor = state["cursor"].long()
    held = (lengths + page - 1) // page
    fits = (lengths >= 0) & (news >= 0) & (lengths + news <= columns * page)
    need = torch.where(fits, (lengths + news + page - 1) // page - held, 0)
    first = torch.cumsum(need, 0) - need + cursor          # where the request's pages begin in the free list
    taken = fits & ((need == 0) | (first + need <= free.shape[0]))
    news, need = torch.where(taken, news, 0), torch.where(taken, need, 0)
    offsets = torch.cat((news.new_zeros(1), torch.cumsum(news, 0)))
    # the block tables: column c of a request that is to get pages
    column = torch.arange(columns, device=DEVICE)[None, :]
    fresh = (column >= held[:, None]) & (column < (held + need)[:, None])
    source = (first[:, None] + column - held[:, None]).clamp(0, max(0, free.shape[0] - 1))
    if free.shape[0]:
        table.copy_(torch.where(fresh, free[source.reshape(-1)].view(b, columns), table))
    # the new tokens
    at = torch.arange(state["tokens"], device=DEVICE)
    request = torch.searchsorted(offsets, at, right=True) - 1
    inside = at < offsets[b]
    request = torch.where(inside, request, 0)
    position = lengths[request] + at - offsets[request]
    page_id = table[request, (position // page).clamp(0, columns - 1)].long()
    slot = torch.where(page_id >= 0, page_id * page + position % page, -1)
    some = lambda x: torch.where(inside, x, -1).to(torch.int32)  # noqa: E731
    progress = torch.stack((cursor[0] + need.sum(), (~taken).sum()))
    return {"table": table, "slots": some(slot), "tok_seq": some(request), "tok_pos": some(position),
            "offsets": offsets.to(torch.int32), "new_lengths": (lengths + news).to(torch.int32),
            "progress": progress.to(torch.int32)}


def _own_append(state, k, pages):
    case, cache = state["case"], pages(*state["pages"])
    n, width = state["every"].shape[0], case["kv_heads"] * case["dim"]
    k.fp4_write(state["k"], state["v"], state["slots"], cache)
    keys = torch.empty((n, width), dtype=torch.bfloat16, device=DEVICE)
    values = torch.empty_like(keys)
    k.fp4_read(cache, state["every"], keys, values)
    return keys, values


def _plain_append(state):
    case = state["case"]
    t, h, d, page = case["tokens"], case["kv_heads"], case["dim"], case["page"]
    k_codes, k_scales, v_codes, v_scales = state["pages"]
    slots = state["slots"].long()
    page_id, place = slots // page, slots % page
    codes, scales = _quantise(state["k"].view(t, h, d))
    k_codes[page_id, :, place] = _pack(codes)
    k_scales[page_id, :, place] = scales
    codes, scales = _quantise(state["v"].view(t, h, d))
    v_codes[page_id, :, place // 4, :, place % 4] = _pack(codes).view(t, h, d // 8, 4)
    v_scales[page_id, :, place // 4, :, place % 4] = scales
    rows = lambda x: x.transpose(1, 2).reshape(-1, h * d).to(torch.bfloat16)  # noqa: E731
    return rows(_values(k_codes, k_scales)), rows(_values(*_value_rows(v_codes, v_scales)))


def _own_attention(state, k, pages):
    case = state["case"]
    out = torch.empty_like(state["q"])
    k.fp4_attention(state["q"], case["heads"], case["kv_heads"], case["dim"], pages(*state["pages"]), state["table"],
                    state["offsets"], state["lengths"], state["most"], state["longest"], out, case["dim"] ** -0.5,
                    window=case["window"])
    return out


def _plain_attention(state):
    case = state["case"]
    h, d, page, window = case["kv_heads"], case["dim"], case["page"], case["window"]
    group = case["heads"] // h
    q, table = state["q"], state["table"]
    k_codes, k_scales, v_codes, v_scales = state["pages"]
    out = torch.empty_like(q)
    row = 0
    for i, (length, new) in enumerate(zip(state["host_lengths"], state["host_new"])):
        start = length - new
        first = max(0, start - window + 1) // page if window else 0        # no row sees a page before this one
        ids = table[i, first:-(-length // page)].long()
        keys = _values(k_codes[ids], k_scales[ids]).transpose(0, 1).reshape(h, -1, d)
        values = _values(*_value_rows(v_codes[ids], v_scales[ids])).transpose(0, 1).reshape(h, -1, d)
        at = torch.arange(first * page, first * page + keys.shape[1], device=DEVICE)
        for lo in range(0, new, 512):
            n = min(512, new - lo)
            x = q[row + lo:row + lo + n].to(torch.float32).view(n, h, group, d).permute(1, 2, 0, 3).reshape(h, group * n, d)
            scores = torch.matmul(x, keys.transpose(1, 2).contiguous()) * d ** -0.5
            position = start + lo + torch.arange(n, device=DEVICE)
            seen = at[None, :] <= position[:, None]
            if window:
                seen &= at[None, :] > position[:, None] - window
            scores = scores.view(h, group, n, -1).masked_fill(~seen, float("-inf"))
            weights = torch.exp(scores - scores.amax(-1, keepdim=True))
            weights = weights / weights.sum(-1, keepdim=True)
            y = torch.matmul(weights.view(h, group * n, -1), values)
            out[row + lo:row + lo + n] = y.view(h, group, n, d).permute(2, 0, 1, 3).reshape(n, -1).to(out.dtype)
        row += new
    return out


def _own_logprobs(state, k, _):
    case = state["case"]
    n, top = case["rows"], case["top"]
    f = lambda *s: torch.empty(s, dtype=torch.float32, device=DEVICE)  # noqa: E731
    i = lambda *s: torch.empty(s, dtype=torch.int32, device=DEVICE)  # noqa: E731
    out = {"logprob": f(n), "entropy": f(n), "rank": i(n), "top_ids": i(n, top), "top_logprobs": f(n, top)}
    k.token_logprobs(state["logits"], state["tokens"], out["logprob"], out["entropy"], out["rank"], out["top_ids"],
                     out["top_logprobs"])
    return out


def _plain_logprobs(state):
    case, tokens = state["case"], state["tokens"].long()
    x = state["logits"].to(torch.float32)
    n, vocab = x.shape
    shifted = x - x.amax(-1, keepdim=True)
    weights = torch.exp(shifted)
    total = weights.sum(-1)
    log_total = torch.log(total)
    mine = x.gather(1, tokens[:, None])
    at = torch.arange(vocab, device=DEVICE)
    rank = ((x > mine) | ((x == mine) & (at[None, :] < tokens[:, None]))).sum(-1)
    entropy = log_total - (weights * shifted).sum(-1) / total
    # the order of the alternatives: larger first, then the lower id, as one whole number
    bits = (x + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64)
    key = order * (1 << 32) + (vocab - 1 - at)[None, :]
    ids = vocab - 1 - (torch.topk(key, case["top"], dim=-1).values & 0xFFFFFFFF)
    return {"logprob": shifted.gather(1, tokens[:, None])[:, 0] - log_total, "entropy": entropy, "rank": rank.to(torch.int32),
            "top_ids": ids.to(torch.int32), "top_logprobs": shifted.gather(1, ids) - log_total[:, None]}


# -- the least work, and the values in 64 bits -------------------------------------------------------------------------
def _size(name):
    return 4 if name == "float32" else 2


def _pairs(case):
    """Keys read and (query, key) pairs of one attention pass, for the average drawn lengths of a ragged case."""
    news = _news(case, 0) if case["ragged"] else [case["new"]] * case["requests"]
    lengths = [max(news[i], case["longest"] * (1.0 if not case["ragged"] or i == 0 else 9.0 / 16.0))
               for i in range(case["requests"])]
    keys = pairs = 0.0
    for length, new in zip(lengths, news):
        window = case["window"] or length
        keys += min(length, window + new - 1)
        pairs += new * max(1.0, min(window, length - (new - 1) / 2))
    return keys, pairs, sum(news)


def work(case):
    op = case["op"]
    if op == "tables":
        tokens = sum(_news(case, 0))
        return {"bytes": 4 * (3 * case["requests"] + 3 * tokens + 2 * tokens / case["page"]), "flops": 0}
    if op == "append":
        values = case["tokens"] * case["kv_heads"] * case["dim"] * 2
        pool = (-(-case["tokens"] // case["page"]) + 1) * case["page"] * case["kv_heads"] * case["dim"] * 2
        return {"bytes": values * (_size(case["type"]) + 17 / 32) + pool * (2 + 17 / 32), "flops": 4 * values}
    if op == "attention":
        keys, pairs, rows = _pairs(case)
        return {"bytes": keys * case["kv_heads"] * case["dim"] * 2 * 17 / 32
                + 2 * rows * case["heads"] * case["dim"] * _size(case["type"]),
                "flops": 4 * pairs * case["heads"] * case["dim"]}
    entries = case["rows"] * case["vocab"]
    return {"bytes": entries * _size(case["type"]) + case["rows"] * (16 + 8 * case["top"]), "flops": 6 * entries}


def exact(case, seed):
    state = prepare(case, seed)
    return {"tables": _exact_tables, "append": _exact_append, "attention": _exact_attention,
            "logprobs": _exact_logprobs}[case["op"]](state)


def _exact_tables(state):
    """A request at a time, as a program on the host would go about it."""
    page = state["case"]["page"]
    table, free = state["table"].cpu(), state["free"].tolist()
    columns = table.shape[1]
    at = state["cursor"].item()
    short, refused = False, 0
    slots, owner, places, offsets, lengths = [], [], [], [0], []
    for i, (length, new) in enumerate(zip(state["lengths"].tolist(), state["news"].tolist())):
        ok = length >= 0 and new >= 0 and length + new <= columns * page
        if ok:
            need = (length + new + page - 1) // page - (length + page - 1) // page
            short = short or (need > 0 and at + need > len(free))
            ok = need == 0 or not short
        if not ok:
            refused += 1
            new = 0
        else:
            for c in range(need):
                table[i, (length + page - 1) // page + c] = free[at]
                at += 1
            ids = table[i].tolist()
            for p in range(length, length + new):
                slots.append(ids[p // page] * page + p % page if ids[p // page] >= 0 else -1)
                owner.append(i)
                places.append(p)
        offsets.append(offsets[-1] + new)
        lengths.append(length + new)
    fill = [-1] * (state["tokens"] - len(slots))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEVICE)  # noqa: E731
    return {"table": table.to(DEVICE), "slots": i32(slots + fill), "tok_seq": i32(owner + fill), "tok_pos": i32(places + fill),
            "offsets": i32(offsets), "new_lengths": i32(lengths), "progress": i32([at, refused])}


def _nearest(x):
    """Every group of 32 held in 4 bits, as values in 64 bits: the level with the smallest distance, by comparison."""
    shape = x.shape
    groups = x.double().reshape(-1, 32)
    largest = groups.abs().amax(-1, keepdim=True)
    exponent = torch.floor(torch.log2(largest))
    exponent = torch.where(torch.exp2(exponent) > largest, exponent - 1, exponent)       # a logarithm that rounded up
    exponent = torch.where(torch.exp2(exponent + 1) <= largest, exponent + 1, exponent)   # or down
    scale = torch.exp2(torch.where(largest > 0, exponent - 2, -125.0).clamp(min=-125.0))
    magnitude = groups.abs() / scale
    best = torch.zeros_like(magnitude)
    distance = magnitude.clone()
    for place, level in enumerate(LEVELS[1:], 1):
        d = (magnitude - level).abs()
        closer = (d < distance) | ((d == distance) & (place % 2 == 0))
        best = torch.where(closer, torch.full_like(best, level), best)
        distance = torch.minimum(d, distance)
    return (best * scale * torch.where(groups < 0, -1.0, 1.0)).reshape(shape)


def _exact_append(state):
    pool = state["every"].shape[0]
    found = []
    for x in (state["k"], state["v"]):
        rows = torch.zeros((pool, x.shape[1]), dtype=torch.float64, device=DEVICE)
        rows[state["slots"].long()] = _nearest(x)
        found.append(rows)
    return tuple(found)


def _held(pages, ids, value):
    """Keys or values of the pages ``ids`` in 64 bits, [kv heads, tokens, d]."""
    levels = torch.tensor(LEVELS, dtype=torch.float64, device=DEVICE)
    codes, scales = pages[2 if value else 0][ids], pages[3 if value else 1][ids]
    n, h = codes.shape[:2]
    if value:
        codes = codes.permute(1, 0, 2, 4, 3, 5).reshape(h, -1, codes.shape[3] * 4)
        scales = scales.permute(1, 0, 2, 4, 3).reshape(h, -1, scales.shape[3])
    else:
        codes = codes.transpose(0, 1).reshape(h, -1, codes.shape[3])
        scales = scales.transpose(0, 1).reshape(h, -1, scales.shape[3])
    x = torch.empty((h, codes.shape[1], codes.shape[2] * 2), dtype=torch.float64, device=DEVICE)
    for half in (0, 1):
        nibble = (codes >> (4 * half)).long() & 15
        x[..., half::2] = levels[nibble & 7] * (1.0 - 2.0 * (nibble >> 3))
    return x * torch.exp2(scales.double() - 127.0).repeat_interleave(32, -1)


def _exact_attention(state):
    case = state["case"]
    h, d, page, window = case["kv_heads"], case["dim"], case["page"], case["window"]
    keys, pairs, _ = _pairs(case)
    if pairs * case["heads"] * d > 1.5e11:
        return None                         # minutes in 64 bits
    group = case["heads"] // h
    result = torch.zeros(state["q"].shape, dtype=torch.float64, device=DEVICE)
    row = 0
    for i, (length, new) in enumerate(zip(state["host_lengths"], state["host_new"])):
        ids = state["table"][i, :-(-length // page)].long()
        k, v = (_held(state["pages"], ids, value)[:, :length] for value in (False, True))
        for lo in range(0, new, 128):
            n = min(128, new - lo)
            for head in range(case["heads"]):
                x = state["q"][row + lo:row + lo + n, head * d:(head + 1) * d].double()
                scores = (x @ k[head // group].T) / math.sqrt(d)
                distance = (length - new + lo + torch.arange(n, device=DEVICE))[:, None] - torch.arange(length, device=DEVICE)
                hidden = (distance < 0) | (distance >= window) if window else distance < 0
                weights = torch.softmax(scores.masked_fill(hidden, float("-inf")), -1)
                result[row + lo:row + lo + n, head * d:(head + 1) * d] = weights @ v[head // group]
        row += new
    return result


def _exact_logprobs(state):
    top, tokens = state["case"]["top"], state["tokens"].long()
    found = {"logprob": [], "entropy": [], "rank": [], "top_ids": [], "top_logprobs": []}
    for lo in range(0, tokens.shape[0], 64):
        x = state["logits"][lo:lo + 64].double()
        t = tokens[lo:lo + 64]
        log_p = x - torch.logsumexp(x, -1, keepdim=True)
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices
        found["logprob"].append(log_p.gather(1, t[:, None])[:, 0])
        found["entropy"].append(-(log_p.exp() * log_p).sum(-1))
        found["rank"].append((order == t[:, None]).int().argmax(-1).to(torch.int32))
        found["top_ids"].append(order[:, :top].to(torch.int32))
        found["top_logprobs"].append(log_p.gather(1, order[:, :top]))
    return {name: torch.cat(parts) for name, parts in found.items()}
