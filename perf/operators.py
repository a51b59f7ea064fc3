"""Operators for requests that branch: what is measured of them.

``attention_shared_prefix``  attention of a batch whose sequences share a long prefix of their cache;
``copy_pages``               copies of cache pages in all layers (a fork's last page, a compaction);
``verify_drafts``            drafted tokens against the target's probabilities, from given random numbers.

A case is a dict of sizes; ``prepare`` makes its inputs on the GPU, ``run`` makes one pass, in plain torch or, with
``own``, through this framework's entry points.
"""

from __future__ import annotations

import random

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    attention = {"op": "attention", "page": 16, "head_dim": 128, "dtype": "bfloat16", "tokens": 1, "ragged": False}
    copy = {"op": "copy", "page": 16, "kv_heads": 8, "head_dim": 128, "dtype": "bfloat16"}
    verify = {"op": "verify", "vocab": 151936, "ragged": False, "temperature": 0.8}
    return [
        # two answers to one short prompt on a small model: latency
        dict(attention, name="two answers, 512 shared", sequences=2, groups=1, shared=512, behind=40, heads=16, kv_heads=8),
        # eight answers to one prompt of a usual length
        dict(attention, name="eight answers, 2048 shared", sequences=8, groups=1, shared=2048, behind=128, heads=32, kv_heads=8),
        # a served batch of conversations that begin with one of seven system prompts, all lengths odd
        dict(attention, name="seven prompts, 45 rows, ragged", sequences=45, groups=7, shared=5000, behind=700, heads=32, kv_heads=8,
             ragged=True),
        # sixteen answers that each bring a token and four drafted ones
        dict(attention, name="sixteen answers, 5 tokens each", sequences=16, groups=1, shared=4096, behind=200, tokens=5, heads=16,
             kv_heads=8),
        # a large batch over one long document
        dict(attention, name="64 rows, 30000 shared", sequences=64, groups=1, shared=30000, behind=200, heads=64, kv_heads=8),
        # the 32-bit path
        dict(attention, name="eight answers, 1024 shared, f32", sequences=8, groups=1, shared=1024, behind=64, heads=16, kv_heads=8,
             head_dim=64, dtype="float32"),
        # one request forked in two: its last page in every layer
        dict(copy, name="fork, one page", layers=28, pages=64, moves=1, kind="fork"),
        # sixteen requests forked into four each
        dict(copy, name="fork, 48 pages", layers=36, pages=512, moves=48, kind="fork"),
        # a pool with holes made dense, the pages in use moved to its front
        dict(copy, name="compaction, 1000 pages", layers=28, pages=4096, moves=1000, kind="compact"),
        # one request with four drafted tokens
        dict(verify, name="one request, 4 drafts", requests=1, drafts=4, probs=True),
        # drafts from a table (no probabilities of their own) for a few requests, some of them with none
        dict(verify, name="nine requests, 0 to 6 drafts", requests=9, drafts=6, probs=False, ragged=True),
        # a large batch with the draft model's probabilities
        dict(verify, name="64 requests, 8 drafts", requests=64, drafts=8, probs=True),
    ]


def _spread(rng, low, high):
    """A whole number between the two, its logarithm evenly spread."""
    return min(high, max(low, round(low * (high / low) ** rng.random())))


def draw(rng):
    op = rng.choice(["attention", "attention", "copy", "verify"])
    if op == "attention":
        sequences = _spread(rng, 1, 64)
        tokens = rng.choice([1, 1, 1, rng.randint(2, 8)])
        heads, kv_heads = rng.choice([(16, 8), (32, 8), (64, 8), (8, 8), (12, 4), (24, 2), (9, 1)])
        # no more work than the largest listed case has
        longest = min(30000, 64 * 30000 // (sequences * tokens), 64 * 64 * 30000 // (sequences * tokens * heads))
        return {"op": op, "sequences": sequences, "groups": rng.randint(1, min(sequences, 9)), "shared": _spread(rng, 16, longest),
                "behind": tokens + _spread(rng, 1, 600), "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
                "head_dim": rng.choice([64, 80, 96, 128, 128]), "page": rng.choice([16, 16, 32, 64]),
                "dtype": rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"]), "ragged": rng.random() < 0.6}
    if op == "copy":
        kv_heads, dim, page, dtype = rng.choice([1, 4, 8]), rng.choice([64, 80, 128]), rng.choice([5, 16, 32]), rng.choice(list(DTYPES))
        moves = _spread(rng, 1, 1000)
        # no more bytes than the largest listed case has
        layers = _spread(rng, 1, max(1, min(48, 28 * 1000 * 16 * 1024 // (moves * kv_heads * dim * page * DTYPES[dtype].itemsize // 2))))
        return {"op": op, "layers": layers, "kv_heads": kv_heads, "head_dim": dim, "page": page, "dtype": dtype, "moves": moves,
                "pages": moves * rng.randint(2, 4) + rng.randint(1, 50), "kind": rng.choice(["fork", "compact"])}
    return {"op": op, "requests": _spread(rng, 1, 64), "drafts": _spread(rng, 1, 8),
            "vocab": rng.choice([151936, 32000 + rng.randint(0, 70000), _spread(rng, 50, 30000)]), "probs": rng.random() < 0.6,
            "ragged": rng.random() < 0.5, "temperature": rng.choice([0.0, 0.6, 0.8, 1.0, 1.3])}


# ---- sizes that follow from a case ----------------------------------------------------------------------------------------------------------


def _rng(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _attention_sizes(case):
    """Sequences of each group, the length each group shares, and for every sequence its tokens and what it has behind the shared part."""
    rng, groups, sequences, tokens = _rng(case), case["groups"], case["sequences"], case["tokens"]
    if not case["ragged"]:
        sizes = [sequences // groups + (g < sequences % groups) for g in range(groups)]
        return sizes, [case["shared"] // case["page"] * case["page"]] * groups, [tokens] * sequences, [case["behind"]] * sequences
    cuts = sorted(rng.sample(range(1, sequences), groups - 1))
    sizes = [b - a for a, b in zip([0, *cuts], [*cuts, sequences])]
    # whole pages are shared; a group of one shares with nobody, and may share nothing at all
    shared = [rng.randint(0 if size == 1 else 1, max(1, case["shared"] // case["page"])) * case["page"] for size in sizes]
    brings = [rng.randint(1, tokens) for _ in range(sequences)]
    return sizes, shared, brings, [max(t, rng.randint(1, case["behind"])) for t in brings]


def _verify_sizes(case):
    """Drafted tokens of every request."""
    rng = _rng(case)
    return [rng.randint(0, case["drafts"]) if case["ragged"] else case["drafts"] for _ in range(case["requests"])]


def work(case):
    if case["op"] == "attention":
        sizes, shared, brings, behind = _attention_sizes(case)
        item = DTYPES[case["dtype"]].itemsize
        group_of = [g for g, size in enumerate(sizes) for _ in range(size)]
        keys = sum(shared) + sum(behind)
        seen = sum(t * (shared[g] + b) - t * (t - 1) // 2 for g, t, b in zip(group_of, brings, behind))
        rows = 2 * sum(brings) * case["heads"] * case["head_dim"] * item
        return {"bytes": keys * 2 * case["kv_heads"] * case["head_dim"] * item + rows, "flops": 4 * case["heads"] * case["head_dim"] * seen}
    if case["op"] == "copy":
        page = case["kv_heads"] * case["page"] * case["head_dim"] * DTYPES[case["dtype"]].itemsize
        read = len(set(_moves(case)[0]))
        return {"bytes": (read + case["moves"]) * 2 * case["layers"] * page, "flops": 0}
    drafts = _verify_sizes(case)
    rows = sum(drafts) + case["requests"]
    # every row of the target; of the draft's probabilities the row at which a request's drafts end
    extra = case["requests"] if case["probs"] else 0
    return {"bytes": 4 * case["vocab"] * (rows + extra), "flops": 4 * case["vocab"] * (rows + extra)}


def _moves(case):
    """Pages and where they are copied to. A fork copies one page to up to three others; a compaction moves pages from behind to the front."""
    rng, moves, pages = _rng(case), case["moves"], case["pages"]
    if case["kind"] == "fork":
        ids = rng.sample(range(pages), moves + -(-moves // 3))
        return [ids[moves + i // 3] for i in range(moves)], ids[:moves]
    return sorted(rng.sample(range(pages // 2, pages), moves), reverse=True), sorted(rng.sample(range(pages // 2), moves))


# ---- inputs ---------------------------------------------------------------------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    return {"attention": _prepare_attention, "copy": _prepare_copy, "verify": _prepare_verify}[case["op"]](case, gen)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _prepare_attention(case, gen):
    sizes, shared, brings, behind = _attention_sizes(case)
    page, dtype, dim, kv_heads = case["page"], DTYPES[case["dtype"]], case["head_dim"], case["kv_heads"]
    group_of = [g for g, size in enumerate(sizes) for _ in range(size)]
    own_pages = [-(-b // page) for b in behind]
    shared_pages = [s // page for s in shared]
    width = max(shared_pages[g] + n for g, n in zip(group_of, own_pages))
    total = sum(shared_pages) + sum(own_pages)
    # the pages of a request lie anywhere in the pool, as they do in a pool that has been in use
    ids = torch.randperm(total, generator=gen, device=DEVICE).int()
    table = torch.zeros((len(group_of), width), dtype=torch.int32, device=DEVICE)
    starts, at = [], 0
    for n in shared_pages:
        starts.append(at)
        at += n
    for s, (g, n) in enumerate(zip(group_of, own_pages)):
        table[s, : shared_pages[g]] = ids[starts[g] : starts[g] + shared_pages[g]]
        table[s, shared_pages[g] : shared_pages[g] + n] = ids[at : at + n]
        at += n
    query_start, group_start = [0], [0]
    for t in brings:
        query_start.append(query_start[-1] + t)
    for size in sizes:
        group_start.append(group_start[-1] + size)
    context = [shared[g] + b for g, b in zip(group_of, behind)]
    randn = lambda *shape: torch.randn(*shape, generator=gen, device=DEVICE)  # noqa: E731
    return {
        "op": "attention",
        # normed heads: queries are a few times as long as keys, so that some keys carry most of the weight
        "q": (2.5 * randn(query_start[-1], case["heads"], dim)).to(dtype),
        "key_pool": randn(total, kv_heads, page, dim).to(dtype),
        "value_pool": randn(total, kv_heads, dim, page).to(dtype),
        "block_table": table,
        "query_start": _ints(query_start),
        "context_lens": _ints(context),
        "group_start": _ints(group_start),
        "shared_lens": _ints(shared),
        "scale": dim**-0.5,
        "max_shared": max(shared),
        "max_own": max(behind),
        "max_query": max(brings),
    }


def _prepare_copy(case, gen):
    dtype, source, destination = DTYPES[case["dtype"]], *_moves(case)
    shape = (case["layers"], case["pages"], case["kv_heads"])
    return {
        "op": "copy",
        "keys": torch.randn(*shape, case["page"], case["head_dim"], generator=gen, device=DEVICE, dtype=dtype),
        "values": torch.randn(*shape, case["head_dim"], case["page"], generator=gen, device=DEVICE, dtype=dtype),
        "source": source,              # the cache manager's page numbers, which live on the host
        "destination": destination,
    }


def _prepare_verify(case, gen):
    drafts, vocab = _verify_sizes(case), case["vocab"]
    starts = [0]
    for n in drafts:
        starts.append(starts[-1] + n + 1)
    rows = starts[-1]
    logits = 3 * torch.randn(rows, vocab, generator=gen, device=DEVICE)
    draft_rows = [start + i for start, n in zip(starts, drafts) for i in range(n)]
    # the draft model nearly agrees with the target: its tokens are drawn from its own probabilities
    guess = logits[draft_rows] + 0.4 * torch.randn(len(draft_rows), vocab, generator=gen, device=DEVICE)
    guess = guess / (case["temperature"] or 1.0)
    if case["temperature"]:
        noise = torch.rand(guess.shape, generator=gen, device=DEVICE).clamp_(1e-20, 1 - 1e-7)
        tokens = (guess - torch.log(-torch.log(noise))).argmax(-1)
    else:
        tokens = guess.argmax(-1)
    uniform = torch.rand(len(draft_rows) + len(drafts), generator=gen, device=DEVICE)
    return {
        "op": "verify",
        "logits": logits,
        "row_start": _ints(starts),
        "draft_tokens": tokens.int(),
        "draft_probs": torch.softmax(guess, -1) if case["probs"] else None,
        "accept_uniform": uniform[: len(draft_rows)].clone(),
        "draw_uniform": uniform[len(draft_rows) :].clone(),
        "temperature": torch.full((len(drafts),), case["temperature"], device=DEVICE),
        "max_drafts": max(drafts),
    }


# ---- one pass -------------------------------------------------------------------------------------------------------------------------------


def run(state):
    op = state["op"]
    if own:
        from miniserve_amd import ops

        if op == "attention":
            return ops.attention_shared_prefix(
                state["q"], state["key_pool"], state["value_pool"], block_table=state["block_table"], query_start=state["query_start"],
                context_lens=state["context_lens"], group_start=state["group_start"], shared_lens=state["shared_lens"],
                scale=state["scale"], max_shared=state["max_shared"], max_own=state["max_own"], max_query=state["max_query"])
        if op == "copy":
            ops.copy_pages([state["keys"], state["values"]], state["source"], state["destination"])
            return state["keys"], state["values"]
        return ops.verify_drafts(state["logits"], state["row_start"], state["draft_tokens"], draft_probs=state["draft_probs"],
                                 accept_uniform=state["accept_uniform"], draw_uniform=state["draw_uniform"],
                                 temperature=state["temperature"])
    if op == "attention":
        return _plain_attention(state)
    if op == "copy":
        source = torch.tensor(state["source"], device=DEVICE)
        destination = torch.tensor(state["destination"], device=DEVICE)
        state["keys"][:, destination] = state["keys"][:, source]
        state["values"][:, destination] = state["values"][:, source]
        return state["keys"], state["values"]
    return _plain_verify(state)


def _plain_attention(state):
    """softmax(q . k * scale) . v over the keys 0 .. position of every token's sequence, in 32 bits."""
    q, keys, values, table = state["q"], state["key_pool"], state["value_pool"], state["block_table"].long()
    n, heads, dim = q.shape
    kv_heads, page = keys.shape[1], keys.shape[2]
    sequences, width = table.shape
    start = state["query_start"].long()
    seq = torch.repeat_interleave(torch.arange(sequences, device=q.device), start[1:] - start[:-1], output_size=n)
    position = state["context_lens"].long()[seq] - start[seq + 1] + torch.arange(n, device=q.device)
    k = keys[table].float().permute(0, 2, 4, 1, 3).reshape(sequences, kv_heads, dim, width * page)
    scores = torch.matmul(q.float().view(n, kv_heads, heads // kv_heads, dim), k[seq] if n > sequences else k) * state["scale"]
    hidden = torch.arange(width * page, device=q.device) > position[:, None]
    scores = scores.masked_fill_(hidden[:, None, None, :], float("-inf"))
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    weights = weights / weights.sum(-1, keepdim=True)
    v = values[table].float().permute(0, 2, 1, 4, 3).reshape(sequences, kv_heads, width * page, dim)
    return torch.matmul(weights, v[seq] if n > sequences else v).view(n, heads, dim).to(q.dtype)


def _plain_verify(state):
    """Draft i of a request is taken while u_i q_i(x_i) < p_i(x_i) (greedy: while it is the best token); then one token of
    max(p - q, 0), or of p behind the last draft. 64 bits: a token hangs on which side of a border a number lies."""
    logits, start, drafts, temperature = state["logits"], state["row_start"].long(), state["draft_tokens"].long(), state["temperature"]
    rows, vocab = logits.shape
    requests, most, count = start.numel() - 1, state["max_drafts"], start[1:] - start[:-1] - 1
    row = torch.arange(rows, device=logits.device)
    request = torch.repeat_interleave(torch.arange(requests, device=logits.device), count + 1, output_size=rows)
    greedy = temperature == 0
    best = logits.argmax(-1)
    x = logits.double() / torch.where(greedy, 1.0, temperature)[request].double()[:, None]
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    is_draft = row - start[request] < count[request]
    draft_of_row = torch.clamp(row - request, max=max(drafts.numel() - 1, 0))
    if drafts.numel():
        token = drafts[draft_of_row]
        q_token = state["draft_probs"][draft_of_row, token].double() if state["draft_probs"] is not None else torch.ones_like(p[:, 0])
        taken = state["accept_uniform"].double()[draft_of_row] * q_token < p.gather(1, token[:, None])[:, 0]
        taken = torch.where(greedy[request], token == best, taken) & is_draft
    else:
        token, taken = torch.zeros_like(row), torch.zeros_like(is_draft)
    place = torch.arange(most + 1, device=logits.device)
    at = torch.clamp(start[:-1, None] + place, max=rows - 1)
    accepted = ((taken[at] & (place < count[:, None])).long().cumprod(-1)).sum(-1)
    end = start[:-1] + accepted
    weight = p[end]
    if drafts.numel():
        rejected = (accepted < count)[:, None]
        if state["draft_probs"] is not None:
            less = torch.clamp(weight - state["draft_probs"][draft_of_row[end]].double(), min=0.0)
        else:
            less = weight.scatter(1, token[end][:, None], 0.0)
        less = torch.where(less.sum(-1, keepdim=True) > 0, less, weight)
        weight = torch.where(rejected, less, weight)
    running = weight.cumsum(-1)
    drawn = (running <= state["draw_uniform"].double()[:, None] * running[:, -1:]).sum(-1).clamp(max=vocab - 1)
    drawn = torch.where(greedy, best[end], drawn)
    local = row - start[request]
    tokens = torch.where(local < accepted[request], token, torch.where(local == accepted[request], drawn[request], -1))
    return tokens.int(), accepted.int()


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(state)
    if case["op"] == "copy":
        for pool in (state["keys"], state["values"]):
            for a, b in zip(state["source"], state["destination"]):
                pool[:, b].copy_(pool[:, a])
        return state["keys"], state["values"]
    return None      # whole numbers


def _exact_attention(state):
    """Sequence by sequence."""
    q, start, context = state["q"], state["query_start"].tolist(), state["context_lens"].tolist()
    kv_heads, dim = state["key_pool"].shape[1], q.shape[2]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    for s, length in enumerate(context):
        pages = state["block_table"][s, : -(-length // state["key_pool"].shape[2])].long()
        k = state["key_pool"][pages].double().transpose(0, 1).reshape(kv_heads, -1, dim)[:, :length]
        v = state["value_pool"][pages].double().transpose(2, 3).transpose(0, 1).reshape(kv_heads, -1, dim)[:, :length]
        for t in range(start[s], start[s + 1]):
            seen = length - (start[s + 1] - 1 - t)
            rows = q[t].double().view(kv_heads, -1, dim)
            out[t] = (torch.softmax(rows @ k[:, :seen].transpose(1, 2) * state["scale"], -1) @ v[:, :seen]).view(-1, dim)
    return out
