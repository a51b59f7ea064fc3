"""Plain implementations, in 64 bits and one row at a time, of the operators for requests
that branch: attention over pages, and drafted tokens against the target."""

from __future__ import annotations

import torch


def attention_rows(q, key_pool, value_pool, block_table, query_start, context_lens, scale):
    """For every token of every sequence ``(out, weight of |v|, bound of the scores)``,
    float64 ``[N, heads, head_dim]`` twice and ``[N, heads]``: the attention over the
    sequence's own table, the same with the values' magnitudes (what rounding a weight can
    move), and the largest ``sum_d |q_d k_d| * scale`` over the keys.  All zero where a token
    sees no key, or behind the last sequence."""

    q, key_pool, value_pool = q.double().cpu(), key_pool.double().cpu(), value_pool.double().cpu()
    n, heads, dim = q.shape
    kv_heads, page = key_pool.shape[1], key_pool.shape[2]
    group = heads // kv_heads
    out, spread, score = torch.zeros(n, heads, dim).double(), torch.zeros(n, heads, dim).double(), torch.zeros(n, heads).double()
    start = [int(x) for x in query_start]
    for s, context in enumerate(int(x) for x in context_lens):
        tokens = start[s + 1] - start[s]
        for t in range(tokens):
            seen = torch.arange(context - tokens + t + 1) if context - tokens + t >= 0 else torch.arange(0)
            if seen.numel() == 0:
                continue
            pages = block_table[s].cpu()[seen // page].long()
            keys = key_pool[pages, :, seen % page, :].repeat_interleave(group, 1)          # [L, heads, D]
            values = value_pool[pages, :, :, seen % page].repeat_interleave(group, 1)
            row = q[start[s] + t]
            scores = (keys * row).sum(-1) * scale
            weights = torch.softmax(scores, 0)
            out[start[s] + t] = (weights[..., None] * values).sum(0)
            spread[start[s] + t] = (weights[..., None] * values.abs()).sum(0)
            score[start[s] + t] = ((keys * row).abs().sum(-1) * abs(scale)).amax(0)
    return out, spread, score


def attention_bound(out, spread, score, dtype, head_dim, longest):
    """How far a right kernel may be from :func:`attention_rows`, value by value.

    Scores: a sum of ``head_dim`` products in 32 bits, the scale and the maximum taken off:
    each of those roundings is at most ``2**-24`` of the sum of magnitudes, which moves a
    weight, relative to the others, by ``e = (head_dim + 8) * 2**-24 * score``, and the sums
    over the keys add at most ``longest + 16`` roundings; numerator and denominator both
    carry it.  bfloat16: every weight is rounded (half a step, ``2**-8``) before it meets its
    value, and the output is rounded once."""

    e = (head_dim + 8) * 2.0**-24 * score[..., None] + (longest + 16) * 2.0**-24
    bound = 2 * e * spread + 2.0**-24 * out.abs()
    if dtype == torch.bfloat16:
        bound = bound + 2.0**-8 * spread + 2.0**-8 * (out.abs() + 2.0**-8 * spread)
    return bound * (1 + 2.0**-7) + 1e-30


def verify(logits, row_start, draft_tokens, draft_probs, accept_uniform, draw_uniform, temperature):
    """(tokens, accepted) as lists, one request after the other; every argument a CPU tensor,
    list or None as ``ops.verify_drafts`` takes them."""

    tokens, accepted = [-1] * logits.shape[0], []
    draft = 0
    for r in range(len(row_start) - 1):
        first, drafts = int(row_start[r]), int(row_start[r + 1]) - int(row_start[r]) - 1
        t = 0.0 if temperature is None else float(temperature[r])
        for i in range(drafts + 1):
            row = logits[first + i].double()
            if not bool(torch.isfinite(row).all()):
                chosen = -1
                break
            x = int(draft_tokens[draft + i]) if i < drafts else -1
            if t == 0.0:
                chosen = int((row == row.max()).nonzero()[0])
                if i < drafts and x == chosen:
                    tokens[first + i] = x
                    continue
                break
            p = torch.softmax(row / t, 0)
            q = None if draft_probs is None or i == drafts else draft_probs[draft + i].double()
            if i < drafts:
                inside = 0 <= x < row.numel()
                if inside and float(accept_uniform[draft + i]) * (1.0 if q is None else float(q[x])) < float(p[x]):
                    tokens[first + i] = x
                    continue
                w = p.clone()
                if q is not None:
                    w = torch.clamp(p - q, min=0)
                elif inside:
                    w[x] = 0
                if float(w.sum()) > 0:
                    p = w
            running = p.cumsum(0)
            above = (running > float(draw_uniform[r]) * running[-1]).nonzero()
            chosen = int(above[0]) if above.numel() else int((p > 0).nonzero()[-1])
            break
        tokens[first + i] = chosen
        accepted.append(i)
        draft += drafts
    return tokens, accepted
