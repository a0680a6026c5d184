"""Plain implementations, in 64 bits on the host, of what stands around a step: block tables and slot maps, keys and
values held in 4 bits, attention over them, log probabilities of given tokens."""

from __future__ import annotations

import math

import torch

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def step_tables(lengths, news, table, page_size, free_pages, cursor, room):
    """Lists in, a dict of lists out (``table``: a list of lists, changed in place)."""
    columns = len(table[0]) if table else 0
    used, row, refused = cursor, 0, 0
    no_pages = no_rows = False
    slots, seqs, places, offsets, after = [], [], [], [], []
    for i, (length, new) in enumerate(zip(lengths, news)):
        offsets.append(row)
        ok = length >= 0 and new >= 0 and length + new <= columns * page_size
        need = -(-(length + new) // page_size) + (-length // page_size) if ok else 0
        if ok and need and (no_pages or cursor < 0 or used + need > len(free_pages)):
            no_pages, ok = True, False
        if ok and new and (no_rows or row + new > room):
            no_rows, ok = True, False
            no_pages = no_pages or need > 0
        if not ok:
            refused += 1
            after.append(length)
            continue
        for c in range(need):
            table[i][-(-length // page_size) + c] = free_pages[used + c]
        used += need
        for p in range(length, length + new):
            page = table[i][p // page_size]
            slots.append(page * page_size + p % page_size if page >= 0 else -1)
            seqs.append(i)
            places.append(p)
        row += new
        after.append(length + new)
    offsets.append(row)
    pad = [-1] * (room - row)
    return {"slots": slots + pad, "tok_seq": seqs + pad, "tok_pos": places + pad, "offsets": offsets, "new_lengths": after,
            "progress": [used, refused], "table": table}


def held(x: torch.Tensor) -> torch.Tensor:
    """What the groups of 32 along the last dimension read as once they are held in 4 bits (float64)."""
    groups = x.to(torch.float64).reshape(-1, 32)
    out = torch.empty_like(groups)
    for i, g in enumerate(groups):
        largest = g.abs().max()
        if not bool(torch.isfinite(g).all()):
            out[i] = float("nan")
            continue
        e = -125 if float(largest) == 0 else max(-125, math.frexp(float(largest))[1] - 1 - 2)
        scale = math.ldexp(1.0, e)
        y = (g.abs() / scale)[:, None] - LEVELS[None, :]
        d = y.abs()
        d = torch.where(torch.arange(8) % 2 == 0, d * (1 - 1e-15), d)       # ties go to the even code
        out[i] = LEVELS[d.argmin(1)] * scale * torch.where(g < 0, -1.0, 1.0)
    return out.reshape(x.shape)


def values_of_pages(pages):
    """(keys, values) [pages, kv heads, tokens, d] in float64 of the four page tensors (on the host)."""
    k_codes, k_scales, v_codes, v_scales = (t.cpu() for t in pages)
    p, h, n, half = k_codes.shape
    v_codes = v_codes.permute(0, 1, 2, 4, 3, 5).reshape(p, h, n, half)
    v_scales = v_scales.permute(0, 1, 2, 4, 3).reshape(p, h, n, half // 16)
    out = []
    for codes, scales in ((k_codes, k_scales), (v_codes, v_scales)):
        both = torch.stack((codes & 15, codes >> 4), -1).reshape(p, h, n, 2 * half).long()
        x = LEVELS[both & 7] * torch.where(both >= 8, -1.0, 1.0)
        factor = torch.exp2(scales.double() - 127.0)
        factor = torch.where(scales == 255, float("nan"), factor)
        out.append(x * factor.repeat_interleave(32, -1))
    return out


def attention(q, nq, nkv, d, keys, values, table, offsets, lengths, page_size, scale, window):
    """(out, spread, reach) in float64, rows of no request NaN: ``spread`` is sum p |v|, ``reach`` the largest
    |scale| sum |q| |k| of the row, for error bounds."""
    pages = keys.shape[0]
    out = torch.full((q.shape[0], nq * d), float("nan"), dtype=torch.float64)
    spread, reach = torch.zeros_like(out), torch.zeros_like(out)
    q = q.double().cpu()
    for i, length in enumerate(lengths):
        first, end = offsets[i], offsets[i + 1]
        at = torch.arange(max(length, 0))
        ids = torch.tensor([table[i][int(p) // page_size] for p in at], dtype=torch.long)
        good = (ids >= 0) & (ids < pages)
        ids = torch.where(good, ids, 0)
        k, v = keys[ids, :, at % page_size], values[ids, :, at % page_size]        # [length, nkv, d]
        for r in range(first, end):
            position = length - (end - r)
            seen = good & (at <= position)
            if window:
                seen &= at > position - window
            for h in range(nq):
                cols = slice(h * d, (h + 1) * d)
                if not bool(seen.any()):
                    out[r, cols] = 0.0
                    continue
                kk, vv = k[seen][:, h // (nq // nkv)], v[seen][:, h // (nq // nkv)]
                p = torch.softmax(scale * (kk @ q[r, cols]), 0)
                out[r, cols] = p @ vv
                spread[r, cols] = p @ vv.abs()
                reach[r, cols] = abs(scale) * (kk.abs() @ q[r, cols].abs()).max()
    return out, spread, reach


def logit_order(row: torch.Tensor) -> list:
    """Token ids, larger logits first, then lower ids; NaN before everything."""
    values = row.tolist()
    return sorted(range(len(values)), key=lambda i: (0, 0.0, i) if math.isnan(values[i]) else (1, -values[i], i))


def token_logprobs(logits, tokens, top):
    """By the formula: with m the largest logit, log p = (x - m) - log sum e^(x - m), so a row with an infinity has NaN."""
    x = logits.double().cpu()
    shifted = x - x.amax(-1, keepdim=True)
    log_p = shifted - torch.log(shifted.exp().sum(-1, keepdim=True))
    orders = [logit_order(row) for row in x]
    n, vocab = x.shape
    valid = [0 <= t < vocab for t in tokens]
    p = log_p.exp()
    terms = torch.where(p == 0, 0.0, p * log_p)
    return {
        "logprob": torch.tensor([float(log_p[i, t]) if valid[i] else float("nan") for i, t in enumerate(tokens)], dtype=torch.float64),
        "entropy": -terms.sum(-1),
        "rank": [orders[i].index(t) if valid[i] else -1 for i, t in enumerate(tokens)],
        "top_ids": [o[:top] for o in orders],
        "top_logprobs": torch.stack([log_p[i, o[:top]] for i, o in enumerate(orders)]) if top else torch.empty((n, 0)),
        "log_sum": torch.log(shifted.exp().sum(-1)),
    }
