"""Workloads of the uncompressed paged cache: prompt attention, attention weights, decode, eviction.

Four operators, each over the range of sizes that serving spans:

    prompt   causal attention of several packed sequences, each possibly behind a history
             (``inquant.prompt.prompt_attention``)
    weights  the attention weight that every key of the packed sequences received from their last
             queries (``inquant.prompt.prompt_weights``)
    token    attention of one new token per request over a paged cache, with the store of its key
             and value and the accumulated weights where the case asks for them
             (``inquant.dense_paged.paged_attention``)
    evict    the tokens of least accumulated weight leave the cache
             (``inquant.dense_paged.evict_tokens``)

Head shapes are those of the repository's benchmark and tests (28 query heads over 4 KV heads, 32 over
8, head dimension 128) and their small relatives; pages hold 16 to 256 tokens.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
QWEN = {"q_heads": 28, "heads": 4, "dim": 128}       # the benchmark's shapes
MISTRAL = {"q_heads": 32, "heads": 8, "dim": 128}


def listed():
    return [
        # a short question to an idle server: latency counts (odd length)
        {"name": "prompt 301", "kind": "prompt", "requests": 1, "low": 301, "high": 301, "past_low": 0, "past_high": 0, "mix": 1,
         "dtype": "bf16", **QWEN},
        # the prompts that arrived since the last step, one launch (ragged)
        {"name": "prompts 16 to 2000", "kind": "prompt", "requests": 16, "low": 17, "high": 2000, "past_low": 0, "past_high": 0,
         "mix": 2, "dtype": "bf16", **MISTRAL},
        # chunks of prompts whose beginning is in the cache already (small heads, an empty request among them)
        {"name": "chunks behind 7000", "kind": "prompt", "requests": 4, "low": 0, "high": 700, "past_low": 2500, "past_high": 7000,
         "mix": 3, "dtype": "fp16", "q_heads": 32, "heads": 8, "dim": 64},
        # one long document: the largest
        {"name": "prompt 8192", "kind": "prompt", "requests": 1, "low": 8192, "high": 8192, "past_low": 0, "past_high": 0, "mix": 4,
         "dtype": "bf16", **QWEN},
        # which tokens of a prompt to keep, judged by all of its queries
        {"name": "weights 4096", "kind": "weights", "requests": 1, "low": 4096, "high": 4096, "window": 0, "mix": 5, "dtype": "bf16",
         **QWEN},
        # the same for a batch of long prompts, judged by the last 64 queries of each
        {"name": "weights 8 by 64 of 16000", "kind": "weights", "requests": 8, "low": 900, "high": 16000, "window": 64, "mix": 6,
         "dtype": "fp16", **MISTRAL},
        # one token of a short conversation: latency counts
        {"name": "token at 700", "kind": "token", "requests": 1, "low": 700, "high": 700, "page": 16, "append": False, "weights": False,
         "mix": 7, "dtype": "bf16", **QWEN},
        # one request with the longest context of the benchmark
        {"name": "token at 131072", "kind": "token", "requests": 1, "low": 131072, "high": 131072, "page": 64, "append": False,
         "weights": False, "mix": 8, "dtype": "bf16", **QWEN},
        # a full batch, the new rows stored by the same call
        {"name": "tokens of 64 requests", "kind": "token", "requests": 64, "low": 1, "high": 8192, "page": 16, "append": True,
         "weights": False, "mix": 9, "dtype": "bf16", **MISTRAL},
        # a batch whose cache is under a budget: the weights are kept up
        {"name": "tokens with weights", "kind": "token", "requests": 16, "low": 1000, "high": 16384, "page": 64, "append": True,
         "weights": True, "mix": 10, "dtype": "fp16", **QWEN},
        # a step of a batch that has outgrown its budget again
        {"name": "evict 256 of 2304", "kind": "evict", "requests": 32, "low": 2304, "high": 2304, "budget": 2048, "sink": 4,
         "recent": 128, "page": 16, "fresh": False, "mix": 11, "dtype": "bf16", **MISTRAL},
        # a long prompt and some shorter ones cut down to their budget
        {"name": "evict to 8192 of 32768", "kind": "evict", "requests": 4, "low": 7000, "high": 32768, "budget": 8192, "sink": 4,
         "recent": 512, "page": 64, "fresh": True, "mix": 12, "dtype": "bf16", **QWEN},
    ]


def _spread(rng, low, high):
    """An integer spread over the logarithm of the range."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "weights", "token", "token", "token", "evict", "evict"])
    heads, q_heads, dim = rng.choice([(4, 28, 128), (8, 32, 128), (2, 14, 64), (8, 32, 64), (4, 4, 128), (1, 16, 128), (2, 10, 128)])
    case = {"kind": kind, "requests": 1, "dtype": rng.choice(["bf16", "bf16", "fp16"]), "q_heads": q_heads, "heads": heads, "dim": dim,
            "mix": rng.randrange(1 << 20)}
    if kind in ("prompt", "weights"):
        # the plain form's scores (requests x heads x longest queries x longest keys) stay below the largest listed case's
        room = 28 * 8192 * 8192 // q_heads
        case["requests"] = _spread(rng, 1, 24)
        if kind == "weights" and rng.random() < 0.6:
            case["window"] = _spread(rng, 16, 256)
            case["high"] = _spread(rng, 60, min(16000, room // (case["requests"] * case["window"]), 100000 // case["requests"]))
        else:
            past = _spread(rng, 60, 7000) if kind == "prompt" and rng.random() < 0.4 else 0
            side = int(math.sqrt(room // case["requests"] + past * past / 4) - past / 2)
            case["high"] = _spread(rng, 30, max(31, min(side, 8192)))
            case.update({"past_low": past // 3, "past_high": past} if kind == "prompt" else {"window": 0})
        case["low"] = rng.randint(1, case["high"])
    else:
        total = 32768 * 8 // heads      # tokens of the batch
        case["requests"] = _spread(rng, 1, 96)
        case["page"] = rng.choice([16, 16, 32, 64, 256, 24])
        case["high"] = _spread(rng, 50, min(131072, max(64, total // case["requests"])))
        case["low"] = rng.randint(1, case["high"])
        if kind == "token":
            case.update(append=rng.random() < 0.6, weights=rng.random() < 0.4)
        else:
            case["budget"] = rng.randint(case["high"] // 4 + 8, case["high"] + 8)
            case.update(sink=rng.choice([0, 4, 4]), recent=rng.randint(0, case["budget"] // 2), fresh=rng.random() < 0.5)
    return case


def _lengths(case):
    """Tokens of every request: spread evenly over the case's range, the longest always among them."""
    rng = random.Random(case["mix"])
    got = [rng.randint(case["low"], case["high"]) for _ in range(case["requests"])]
    got[rng.randrange(len(got))] = case["high"]
    if case["low"] == 0 and len(got) > 1:
        got[got.index(min(got))] = 0
    return got


def _past(case):
    rng = random.Random(case["mix"] + 1)
    return [rng.randint(case.get("past_low", 0), case.get("past_high", 0)) for _ in range(case["requests"])]


def _pairs(queries, keys, window=0):
    """Visible (query, key) pairs of one sequence."""
    queries_seen = min(queries, window) if window else queries
    return queries_seen * keys - queries_seen * (queries_seen - 1) // 2


def _starts(lengths):
    total, got = 0, [0]
    for n in lengths:
        total += n
        got.append(total)
    return got


def prepare(case, seed):
    torch.manual_seed(seed)
    device = torch.device("cuda")
    dtype, dim, heads, q_heads = DTYPES[case["dtype"]], case["dim"], case["heads"], case["q_heads"]
    lengths = _lengths(case)
    state = {"case": case, "scale": dim ** -0.5, "longest": max(lengths)}

    def rows(*shape):
        """N(0, 1) rows with a few channels of larger spread, as keys and queries have them."""
        x = torch.randn(*shape, dim, device=device)
        x[..., ::37] *= 2.5
        return x.to(dtype)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=device)

    if case["kind"] in ("prompt", "weights"):
        past = _past(case)
        keys = [n + p for n, p in zip(lengths, past)]
        state.update(query=rows(sum(lengths), q_heads), key=rows(sum(keys), heads), cu=ints(_starts(lengths)), cu_k=ints(_starts(keys)),
                     longest_k=max(keys))
        if case["kind"] == "prompt":
            state["value"] = torch.randn(sum(keys), heads, dim, device=device).to(dtype)
        else:
            state["window"] = case["window"]
            state["lse"] = _prompt_lse(state)
        return state
    page, budget = case["page"], case.get("budget", 0)
    capacity = max(-(-(n + 1) // page) for n in lengths) * page
    per_request = [-(-(n + 1) // page) for n in lengths]
    order = torch.randperm(sum(per_request) + 3, device=device).to(torch.int32)
    starts = _starts(per_request)
    column = torch.arange(capacity // page, device=device)
    first, count = ints(starts[:-1]).long(), ints(per_request).long()
    state["block_table"] = order[first[:, None] + torch.minimum(column[None], count[:, None] - 1)].contiguous()
    shape = (sum(per_request) + 3, heads, page)
    state.update(key_pages=rows(*shape), value_pages=torch.randn(*shape, dim, device=device).to(dtype), lengths=ints(lengths),
                 longest=max(lengths), capacity=capacity)
    accumulated = torch.exp(2 * torch.randn(len(lengths), heads, capacity, device=device) - 3)
    if case["kind"] == "token":
        state["query"] = rows(len(lengths), q_heads)
        if case["append"]:
            state.update(new_key=rows(len(lengths), heads), new_value=torch.randn(len(lengths), heads, dim, device=device).to(dtype))
        if case["weights"]:
            state.update(weights=accumulated, out_weights=torch.zeros_like(accumulated))
        return state
    # some tokens have received nothing at all: their weights tie
    accumulated = torch.where(torch.rand_like(accumulated) < 0.2, torch.zeros_like(accumulated), accumulated)
    if case["fresh"]:
        seen = list(lengths)
        positions = torch.arange(capacity, device=device, dtype=torch.int32).expand(len(lengths), heads, capacity).contiguous()
    else:
        # tokens that survived earlier evictions, in the order these left, and the newest behind them
        seen = [3 * n + 5 for n in lengths]
        here, n = torch.arange(capacity, device=device), ints(lengths)[:, None, None].long()
        old = torch.where(here < n, torch.rand(len(lengths), heads, capacity, device=device), 2.0).argsort(-1) * 2 + 1
        newest = n // 4
        positions = torch.where(here < n - newest, old, ints(seen)[:, None, None] - n + here).to(torch.int32)
    state.update(weights=accumulated, positions=positions, seen=ints(seen), budget=budget, sink=case["sink"],
                 recent=min(case["recent"], budget - case["sink"]))
    return state


# ---------------------------------------------------------------- plain forms
def _unpack(x, first, last, longest):
    """[tokens, heads, dim] packed -> [requests, heads, longest, dim] in 32 bits, and the packed row of every place."""
    row = first[:, None].long() + torch.arange(longest, device=x.device)
    row = torch.where(row < last[:, None], row, x.shape[0])
    return x[row.clamp_max(x.shape[0] - 1)].transpose(1, 2).float(), row


def _scores(state):
    """Scaled products of all queries and keys, -inf where a key is not visible: [requests, heads, group, queries, keys]."""
    window = state.get("window") or state["longest"]
    first, last = state["cu"][:-1], state["cu"][1:]
    first = torch.maximum(first, last - window)      # with a window the last queries of every sequence alone
    q, q_row = _unpack(state["query"], first, last, min(window, state["longest"]))
    k, k_row = _unpack(state["key"], state["cu_k"][:-1], state["cu_k"][1:], state["longest_k"])
    n, m = (last - first).long(), state["cu_k"].diff().long()
    q = q.reshape(q.shape[0], k.shape[1], -1, q.shape[2], q.shape[3])
    s = torch.matmul(q, k.unsqueeze(2).transpose(-1, -2)).mul_(state["scale"])
    i, j = torch.arange(s.shape[3], device=s.device), torch.arange(s.shape[4], device=s.device)
    limit = (m - n)[:, None] + i            # the last key that a query sees
    dark = (j > limit[..., None]) | (i[:, None] >= n[:, None, None]) | (j >= m[:, None, None])
    return s.masked_fill_(dark[:, None, None], float("-inf")), q_row, k_row


def _prompt_lse(state):
    s, q_row, _ = _scores(state)
    top = s.amax(-1).clamp_min(-1e30)
    lse = top + s.sub_(top.unsqueeze(-1)).exp_().sum(-1).log()
    out = torch.zeros(lse.shape[1] * lse.shape[2], state["query"].shape[0] + 1, device=s.device)
    out[:, q_row] = lse.flatten(1, 2).transpose(0, 1)
    return out[:, :-1].contiguous()


def _plain_prompt(state):
    s, q_row, _ = _scores(state)
    v, _ = _unpack(state["value"], state["cu_k"][:-1], state["cu_k"][1:], state["longest_k"])
    top = s.amax(-1, keepdim=True).clamp_min(-1e30)
    total = s.sub_(top).exp_().sum(-1, keepdim=True)
    o = torch.matmul(s, v.unsqueeze(2)) / total.clamp_min(1e-37)
    lse = (top + total.log()).squeeze(-1)
    tokens = state["query"].shape[0]
    out = torch.zeros(tokens + 1, *state["query"].shape[1:], dtype=state["query"].dtype, device=s.device)
    out[q_row] = o.flatten(1, 2).transpose(1, 2).to(out.dtype)
    packed_lse = torch.zeros(out.shape[1], tokens + 1, device=s.device)
    packed_lse[:, q_row] = lse.flatten(1, 2).transpose(0, 1)
    return {"out": out[:-1], "lse": packed_lse[:, :-1]}


def _plain_weights(state):
    s, q_row, k_row = _scores(state)
    lse = state["lse"][:, q_row.clamp_max(state["query"].shape[0] - 1)].transpose(0, 1).reshape(s.shape[:4])
    w = s.sub_(lse.unsqueeze(-1)).exp_().sum((2, 3))
    out = torch.zeros(w.shape[1], state["key"].shape[0] + 1, device=w.device)
    out[:, k_row] = w.transpose(0, 1)
    return {"weights": out[:, :-1]}


def _plain_token(state):
    k_pages, v_pages, table, lengths = state["key_pages"], state["value_pages"], state["block_table"], state["lengths"].long()
    page, requests, longest = k_pages.shape[2], table.shape[0], state["longest"] + ("new_key" in state)
    if "new_key" in state:
        at = table.gather(1, (lengths // page)[:, None])[:, 0].long()
        k_pages[at, :, lengths % page] = state["new_key"]
        v_pages[at, :, lengths % page] = state["new_value"]
        seen = lengths + 1
    else:
        seen = lengths
    used = table[:, :-(-longest // page)].long()
    k = k_pages[used].transpose(1, 2).flatten(2, 3)[:, :, :longest].float()      # [requests, heads, tokens, dim]
    q = state["query"].float().reshape(requests, k.shape[1], -1, k.shape[3])
    s = torch.matmul(q, k.transpose(-1, -2)) * state["scale"]
    lit = torch.arange(longest, device=s.device) < seen[:, None]
    s = s.masked_fill(~lit[:, None, None], float("-inf"))
    p = (s - s.amax(-1, keepdim=True)).exp_()
    p /= p.sum(-1, keepdim=True)
    v = v_pages[used].transpose(1, 2).flatten(2, 3)[:, :, :longest].float()
    got = {"out": torch.matmul(p, v).reshape(state["query"].shape).to(state["query"].dtype)}
    if "new_key" in state:
        got.update(key_pages=k_pages, value_pages=v_pages)
    if "weights" in state:
        old = torch.where((torch.arange(longest, device=s.device) < lengths[:, None])[:, None], state["weights"][:, :, :longest], 0.0)
        state["out_weights"][:, :, :longest] = torch.where(lit[:, None], old + p.sum(2), state["out_weights"][:, :, :longest])
        got["weights"] = state["out_weights"]
    return got


def _plain_evict(state):
    w, pos, budget = state["weights"], state["positions"], state["budget"]
    lengths, seen = state["lengths"].long()[:, None, None], state["seen"][:, None, None]
    here = torch.arange(w.shape[2], device=w.device).expand(w.shape)
    lit = here < lengths
    kept_for_position = (pos < state["sink"]) | (pos >= seen - state["recent"])
    worth = torch.where(kept_for_position, float("inf"), w).masked_fill(~lit, float("-inf"))
    rank = worth.sort(dim=-1, descending=True, stable=True).indices.argsort(-1)
    left = lengths.clamp_max(budget)
    kept = lit & (rank < left)
    source = torch.where(kept & (here >= left), here, w.shape[2]).sort(-1).values
    hole = (here < left) & ~kept
    origin = torch.where(hole, source.gather(-1, (hole.cumsum(-1) - 1).clamp_min(0)), here)[:, :, :min(budget, w.shape[2])]
    place = here[:, :, :origin.shape[2]]
    filled = place < left
    out_w, out_p = w.new_zeros(*w.shape[:2], budget), pos.new_full((*w.shape[:2], budget), -1)
    out_w[:, :, :origin.shape[2]] = torch.where(filled, w.gather(2, origin), 0.0)
    out_p[:, :, :origin.shape[2]] = torch.where(filled, pos.gather(2, origin), -1)
    # rows go by (page, head, token in the page); what stays is written over itself
    table, page = state["block_table"].long(), state["key_pages"].shape[2]
    request = torch.arange(w.shape[0], device=w.device)[:, None, None].expand(place.shape)
    head = torch.arange(w.shape[1], device=w.device)[None, :, None].expand(place.shape)
    origin = torch.where(filled, origin, 0)
    place = torch.where(filled, place, 0)
    # a place that no token fills repeats the first one, with the same row
    start = torch.where(hole[:, :, :1], source[:, :, :1], 0)
    origin = torch.where(filled, origin, start)
    for pages in (state["key_pages"], state["value_pages"]):
        moved = pages[table[request, origin // page], head, origin % page]
        pages[table[request, place // page], head, place % page] = moved
    return {"key_pages": state["key_pages"], "value_pages": state["value_pages"], "weights": out_w, "positions": out_p,
            "lengths": state["lengths"].clamp_max(budget)}


# ---------------------------------------------------------------- the framework's calls
def _own_run(state):
    package = os.path.join(os.getcwd(), "inquant-open-source_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    kind = state["case"]["kind"]
    if kind == "prompt":
        from inquant.prompt import prompt_attention
        out, lse = prompt_attention(state["query"], state["key"], state["value"], state["cu"], state["cu_k"], scale=state["scale"])
        return {"out": out, "lse": lse}
    if kind == "weights":
        from inquant.prompt import prompt_weights
        return {"weights": prompt_weights(state["query"], state["key"], state["lse"], state["cu"], state["cu_k"], scale=state["scale"],
                                          window=state["window"] or None)}
    if kind == "token":
        from inquant.dense_paged import paged_attention
        got = paged_attention(state["query"], state["key_pages"], state["value_pages"], state["block_table"], state["lengths"],
                              scale=state["scale"], new_key=state.get("new_key"), new_value=state.get("new_value"),
                              weights=state.get("weights"), out_weights=state.get("out_weights"))
        got = {"out": got} if "weights" not in state else {"out": got[0], "weights": got[1]}
        if "new_key" in state:
            got.update(key_pages=state["key_pages"], value_pages=state["value_pages"])
        return got
    from inquant.dense_paged import evict_tokens
    lengths, weights, positions = evict_tokens(state["key_pages"], state["value_pages"], state["block_table"], state["lengths"],
                                               state["weights"], state["positions"], state["seen"], state["budget"], sink=state["sink"],
                                               recent=state["recent"])
    return {"key_pages": state["key_pages"], "value_pages": state["value_pages"], "weights": weights, "positions": positions,
            "lengths": lengths}


@torch.no_grad()
def run(state):
    if own:
        return _own_run(state)
    return {"prompt": _plain_prompt, "weights": _plain_weights, "token": _plain_token, "evict": _plain_evict}[state["case"]["kind"]](state)


def work(case):
    lengths, heads, q_heads, dim = _lengths(case), case["heads"], case["q_heads"], case["dim"]
    if case["kind"] in ("prompt", "weights"):
        keys = [n + p for n, p in zip(lengths, _past(case))]
        window = case.get("window", 0)
        pairs = q_heads * sum(_pairs(n, m, window) for n, m in zip(lengths, keys))
        if case["kind"] == "prompt":
            return {"bytes": sum(lengths) * q_heads * (4 * dim + 4) + 4 * sum(keys) * heads * dim, "flops": 4 * dim * pairs}
        queries = sum(min(n, window or n) for n in lengths)
        return {"bytes": queries * q_heads * (2 * dim + 4) + sum(keys) * heads * (2 * dim + 4), "flops": 2 * dim * pairs}
    tokens = sum(lengths) * heads
    if case["kind"] == "token":
        size = 4 * dim * tokens + 4 * dim * len(lengths) * q_heads
        size += 8 * dim * len(lengths) * heads if case["append"] else 0
        size += 8 * tokens if case["weights"] else 0
        return {"bytes": size, "flops": 4 * dim * sum(lengths) * q_heads}
    budget, sink = case["budget"], case["sink"]
    moved = 0
    for n in lengths:
        if n > budget:
            recent = min(case["recent"], budget - sink)
            far = max(0, n - budget - recent)           # places behind the budget that are not protected
            spare = max(1, n - sink - recent)
            moved += min(recent, n - budget) + far * (budget - sink - recent) // spare
    return {"bytes": 8 * tokens + 8 * heads * len(lengths) * budget + 8 * dim * heads * moved, "flops": 0}


# ---------------------------------------------------------------- from the definition, in 64 bits
def _exact_sequences(case, state):
    """Per sequence: its rows of the packed queries and of the packed keys."""
    lengths, past = _lengths(case), _past(case)
    keys = [n + p for n, p in zip(lengths, past)]
    starts, starts_k = _starts(lengths), _starts(keys)
    return [(slice(starts[b], starts[b + 1]), slice(starts_k[b], starts_k[b + 1])) for b in range(len(lengths))]


@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    group, scale = case["q_heads"] // case["heads"], state["scale"]
    if case["kind"] in ("prompt", "weights"):
        out = torch.zeros_like(state["query"], dtype=torch.float64)
        lse = torch.zeros(case["q_heads"], out.shape[0], dtype=torch.float64, device=out.device)
        weights = torch.zeros(case["heads"], state["key"].shape[0], dtype=torch.float64, device=out.device)
        for queries, keys in _exact_sequences(case, state):
            n, m = queries.stop - queries.start, keys.stop - keys.start
            if n == 0:
                continue
            visible = torch.ones(n, m, dtype=torch.bool, device=out.device).tril(m - n)
            if case.get("window"):
                visible[:max(0, n - case["window"])] = False
            for h in range(case["q_heads"]):
                logits = (state["query"][queries, h].double() @ state["key"][keys, h // group].double().T) * scale
                logits[~visible] = float("-inf")
                if case["kind"] == "prompt":
                    lse[h, queries] = torch.logsumexp(logits, -1)
                    out[queries, h] = torch.softmax(logits, -1) @ state["value"][keys, h // group].double()
                else:
                    weights[h // group, keys] += torch.exp(logits - state["lse"][h, queries].double()[:, None]).sum(0)
        return {"out": out, "lse": lse} if case["kind"] == "prompt" else {"weights": weights}
    lengths, page = _lengths(case), case["page"]
    keys, values = state["key_pages"].double(), state["value_pages"].double()
    tables = state["block_table"].tolist()

    def places(b, tokens):
        """Pages and offsets of the given tokens of request b."""
        t = tokens if isinstance(tokens, torch.Tensor) else torch.tensor(tokens, device=keys.device)
        return torch.tensor(tables[b], device=keys.device)[t // page], t % page

    if case["kind"] == "token":
        out = torch.zeros_like(state["query"], dtype=torch.float64)
        weights = torch.zeros(len(lengths), case["heads"], state["capacity"], dtype=torch.float64, device=out.device)
        for b, n in enumerate(lengths):
            total = n
            if case["append"]:
                at, offset = places(b, [n])
                keys[at[0], :, offset[0]] = state["new_key"][b].double()
                values[at[0], :, offset[0]] = state["new_value"][b].double()
                total = n + 1
            at, offset = places(b, torch.arange(total, device=keys.device))
            for h in range(case["heads"]):
                logits = state["query"][b, h * group:(h + 1) * group].double() @ keys[at, h, offset].T * scale
                share = torch.softmax(logits, -1)
                out[b, h * group:(h + 1) * group] = share @ values[at, h, offset]
                if case["weights"]:
                    weights[b, h, :total] = share.sum(0)
                    weights[b, h, :n] += state["weights"][b, h, :n].double()
        got = {"out": out}
        if case["append"]:
            got.update(key_pages=keys, value_pages=values)
        if case["weights"]:
            got["weights"] = weights
        return got
    budget = case["budget"]
    out_w = torch.zeros(len(lengths), case["heads"], budget, dtype=torch.float64)
    out_p = torch.full(out_w.shape, -1, dtype=torch.int64)
    all_w, all_p, seen = state["weights"].cpu().numpy(), state["positions"].cpu().numpy(), state["seen"].tolist()
    for b, n in enumerate(lengths):
        left = min(n, budget)
        for h in range(case["heads"]):
            w, p = all_w[b, h, :n], all_p[b, h, :n]
            safe = (p < state["sink"]) | (p >= seen[b] - state["recent"])
            # the protected first, then by falling weight, then by place: numpy's sort by several keys takes the last key first
            worth = torch.tensor(w).double().masked_fill(torch.tensor(safe), float("inf")).numpy()
            best = (-worth).argsort(kind="stable")[:left]
            best.sort()
            stays = set(best[best < left].tolist())
            new = list(range(left))
            moving = iter(best[best >= left].tolist())
            for place in range(left):
                if place not in stays:
                    new[place] = next(moving)
            out_w[b, h, :left], out_p[b, h, :left] = torch.tensor(w[new]).double(), torch.tensor(p[new]).long()
            moves = [(place, origin) for place, origin in enumerate(new) if place != origin]
            if moves:
                to_page, to_offset = places(b, [m[0] for m in moves])
                from_page, from_offset = places(b, [m[1] for m in moves])
                keys[to_page, h, to_offset] = keys[from_page, h, from_offset]
                values[to_page, h, to_offset] = values[from_page, h, from_offset]
    return {"key_pages": keys, "value_pages": values, "weights": out_w, "positions": out_p,
            "lengths": torch.tensor([min(n, budget) for n in lengths])}
