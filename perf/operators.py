"""Attention over keys and values in memory or in a paged cache, as cases that can be timed and compared.

A case is a dict of plain values; its "family" says which operator it is:

    prompt   Attention: the queries of whole sequences against their own keys and values, causal or not, with or without a
             sliding window and first tokens that stay visible; one sequence, several packed behind one another ("lengths" holds
             their number of tokens, "packed" is true) or a padded batch ("packed" is false: "lengths" are its valid keys)
    append   PagedAppend: the keys and values of new tokens written to their slots of a paged cache
    decode   PagedAttention: one or a few new tokens per sequence against a paged cache

`run` computes them in elementary operations in 32 bits, or, where `own` is true, by the library's operators, each prepared
once and submitted on every pass.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
SIZE = {"bf16": 2, "f16": 2, "e4m3": 1}
E4M3_LARGEST = 448.0


def listed():
    return [
        # a long prompt at the benchmark's head shape: the largest matrix products
        {"name": "prompt_8192", "family": "prompt", "lengths": "8192", "packed": True, "queries": 16, "heads": 4, "depth": 128,
         "dtype": "bf16", "causal": True, "window": 0, "sinks": 0, "log_sum": False},
        # a longer one through a layer with a sliding window whose first tokens stay visible
        {"name": "prompt_window_sinks", "family": "prompt", "lengths": "16384", "packed": True, "queries": 8, "heads": 2, "depth": 128,
         "dtype": "f16", "causal": True, "window": 1024, "sinks": 4, "log_sum": False},
        # what a server has waiting: prompts of any length behind one another, one of a single token
        {"name": "prompts_ragged", "family": "prompt", "lengths": "1037,1,250,2003,64,511,1137", "packed": True, "queries": 20, "heads": 5,
         "depth": 80, "dtype": "f16", "causal": True, "window": 0, "sinks": 0, "log_sum": False},
        # an encoder's padded batch: every token sees every valid one
        {"name": "encoder_batch", "family": "prompt", "lengths": "777,512,300,776,41,600,777,129", "packed": False, "queries": 12, "heads": 12,
         "depth": 64, "dtype": "bf16", "causal": False, "window": 0, "sinks": 0, "log_sum": False},
        # wide heads, with the logarithms of the sums that a later pass over other keys joins by
        {"name": "prompt_wide_heads", "family": "prompt", "lengths": "2048", "packed": True, "queries": 16, "heads": 2, "depth": 256,
         "dtype": "bf16", "causal": True, "window": 0, "sinks": 0, "log_sum": True},
        # the new token of every stream of a batch: what each layer writes per step
        {"name": "append_step", "family": "append", "tokens": 64, "heads": 8, "depth": 128, "dtype": "bf16", "cache": "bf16", "page": 16,
         "pages": 1024, "skipped": 3},
        # a prompt's keys and values into a cache of 8 bits
        {"name": "append_prompt_e4m3", "family": "append", "tokens": 8192, "heads": 8, "depth": 128, "dtype": "bf16", "cache": "e4m3",
         "page": 64, "pages": 160, "skipped": 0},
        # the first tokens of a few chats: the smallest call
        {"name": "decode_short", "family": "decode", "sequences": 4, "shortest": 9, "longest": 100, "new": 1, "queries": 16, "heads": 4,
         "depth": 128, "dtype": "bf16", "cache": "bf16", "page": 16, "window": 0, "sinks": 0, "log_sum": False},
        # one user with a long document, wide heads: few rows, a long axis
        {"name": "decode_one_long", "family": "decode", "sequences": 1, "shortest": 32751, "longest": 32751, "new": 1, "queries": 16, "heads": 2,
         "depth": 256, "dtype": "bf16", "cache": "bf16", "page": 16, "window": 0, "sinks": 0, "log_sum": True},
        # a batch of streams of every age
        {"name": "decode_batch_ragged", "family": "decode", "sequences": 64, "shortest": 30, "longest": 16384, "new": 1, "queries": 32, "heads": 8,
         "depth": 128, "dtype": "bf16", "cache": "bf16", "page": 16, "window": 0, "sinks": 0, "log_sum": False},
        # long streams over a cache of 8 bits: the most bytes
        {"name": "decode_e4m3", "family": "decode", "sequences": 16, "shortest": 20000, "longest": 32768, "new": 1, "queries": 32, "heads": 8,
         "depth": 128, "dtype": "bf16", "cache": "e4m3", "page": 64, "window": 0, "sinks": 0, "log_sum": False},
        # four drafted tokens per stream through a layer with a window and first tokens that stay visible
        {"name": "decode_drafts_window", "family": "decode", "sequences": 12, "shortest": 500, "longest": 9000, "new": 4, "queries": 20, "heads": 5,
         "depth": 80, "dtype": "f16", "cache": "f16", "page": 24, "window": 2048, "sinks": 4, "log_sum": False},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    family = rng.choice(["prompt", "prompt", "prompt", "append", "decode", "decode", "decode"])
    heads = rng.choice([1, 2, 3, 4, 5, 8])
    depth = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if family == "append":
        page, tokens = rng.choice([1, 8, 16, 16, 24, 64, 256]), _log(rng, 1, 8192)
        return {"family": family, "tokens": tokens, "heads": heads, "depth": depth, "dtype": dtype, "cache": rng.choice([dtype, dtype, "e4m3"]),
                "page": page, "pages": -(-tokens // page) + rng.randint(1, 64), "skipped": rng.choice([0, 0, tokens // 7])}
    queries = heads * rng.choice([1, 2, 4, 4, 5, 8])
    window, sinks = rng.choice([(0, 0), (0, 0), (_log(rng, 16, 4096), rng.choice([0, 1, 4]))])
    if family == "prompt":
        most = math.isqrt(16 * 8192 * 8192 * 64 // (queries * max(depth, 128)))
        total = min(_log(rng, 1, 8192), most)
        causal = window > 0 or rng.random() < 0.8
        count = rng.choice([1, 1, 2, 5, 9])
        if rng.random() < 0.75:  # packed behind one another
            cuts = sorted(rng.randint(0, total) for _ in range(count - 1))
            lengths = [b - a for a, b in zip([0] + cuts, cuts + [total])]
            packed = True
        else:
            longest = max(1, total // count)
            lengths = [longest] + [rng.randint(0, longest) for _ in range(count - 1)]
            packed = False
        return {"family": family, "lengths": ",".join(str(n) for n in lengths), "packed": packed, "queries": queries, "heads": heads,
                "depth": depth, "dtype": dtype, "causal": causal, "window": window, "sinks": sinks, "log_sum": rng.random() < 0.3}
    sequences = _log(rng, 1, 128)
    longest = max(1, min(_log(rng, 1, 65536), (3 << 26) // (sequences * heads * depth)))
    return {"family": family, "sequences": sequences, "shortest": rng.randint(1, longest), "longest": longest,
            "new": rng.choice([1, 1, 1, 2, 3, 4, 8]), "queries": queries, "heads": heads, "depth": depth, "dtype": dtype,
            "cache": rng.choice([dtype, dtype, "e4m3"]), "page": rng.choice([8, 16, 16, 24, 64, 256]), "window": window, "sinks": sinks,
            "log_sum": rng.random() < 0.3}


def _prompt_lengths(case):
    return [int(n) for n in case["lengths"].split(",")]


def _decode_lengths(case):
    """Lengths between the shortest and the longest, evenly over their logarithm and in no order."""
    low, high = case["shortest"], case["longest"]
    return [round(low * (high / low) ** ((1 + 0.6180339887 * i) % 1 if i else 1)) for i in range(case["sequences"])]


class _Make:
    """Inputs on the GPU from one seed."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEVICE)
        self.g.manual_seed(seed)

    def normal(self, shape, dtype, std=1.0):
        if dtype == "e4m3":
            return torch.empty(shape, dtype=torch.bfloat16, device=DEVICE).normal_(0.0, std, generator=self.g).to(TYPES[dtype])
        return torch.empty(shape, dtype=TYPES[dtype], device=DEVICE).normal_(0.0, std, generator=self.g)

    def order(self, count):
        return torch.randperm(count, device=DEVICE, generator=self.g)


def prepare(case, seed):
    """Queries of normed heads (their products with the keys spread over a few units once scaled), values near one, caches
    whose pages are handed out in no order and whose free slots hold what was there before."""
    make = _Make(seed)
    heads, depth, dtype = case["heads"], case["depth"], case["dtype"]
    state = {"case": case}
    if case["family"] == "append":
        page, pages, tokens = case["page"], case["pages"], case["tokens"]
        state["key"], state["value"] = make.normal((tokens, heads, depth), dtype, 1.5), make.normal((tokens, heads, depth), dtype)
        slots = make.order(pages * page)[:tokens].to(torch.int32)
        slots[make.order(tokens)[:case["skipped"]]] = -1  # tokens that keep no place
        state["slots"] = slots
        state["buffer"] = make.normal((pages + 1, 2, heads, page, depth), case["cache"])  # the last page takes what has no place
        state["cache"] = state["buffer"][:pages]
    elif case["family"] == "prompt":
        lengths = _prompt_lengths(case)
        shape = (sum(lengths),) if case["packed"] else (len(lengths), max(lengths))
        state["query"] = make.normal((*shape, case["queries"], depth), dtype, 1.5)
        state["key"], state["value"] = make.normal((*shape, heads, depth), dtype), make.normal((*shape, heads, depth), dtype)
        marks = [sum(lengths[:i]) for i in range(len(lengths) + 1)] if case["packed"] else lengths
        state["marks"] = torch.tensor(marks, dtype=torch.int32, device=DEVICE)
    else:
        lengths, page = _decode_lengths(case), case["page"]
        held = [-(-n // page) for n in lengths]
        pages, most = sum(held) + 3, max(held)
        state["cache"] = make.normal((pages, 2, heads, page, depth), case["cache"])
        state["query"] = make.normal((len(lengths), case["new"], case["queries"], depth), dtype, 1.5)
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
        starts = torch.tensor([sum(held[:i]) for i in range(len(held))], device=DEVICE)[:, None]
        column = torch.arange(most, device=DEVICE)[None]
        has = column < torch.tensor(held, device=DEVICE)[:, None]
        state["table"] = torch.where(has, make.order(pages)[(starts + column).clamp(max=pages - 1)], -1).to(torch.int32)
    if own:
        state["submit"], state["outputs"] = _bound(case, state)
    return state


def _bound(case, state):
    """The library's operator for a case, its inputs bound to it, and the tensors it writes."""
    from hyle_amd import compute as hc
    from hyle_amd import torch_io as tio
    if case["family"] == "append":
        operation = hc.PagedAppend(case["pages"], case["page"], tio.desc_of(state["cache"]).data_type)
        inputs = [state["key"], state["value"], state["slots"]]
    elif case["family"] == "prompt":
        operation = hc.Attention(scale=case["depth"] ** -0.5, causal=case["causal"], window=case["window"], sinks=case["sinks"],
                                 return_log_sum=case["log_sum"])
        inputs = [state["query"], state["key"], state["value"], state["marks"]]
    else:
        operation = hc.PagedAttention(scale=case["depth"] ** -0.5, window=case["window"], sinks=case["sinks"], return_log_sum=case["log_sum"])
        inputs = [state["query"], state["cache"], state["table"], state["lengths"]]
    bound = tio.Bound(hc.Context.create(0), operation, [tio.desc_of(t) for t in inputs])
    outputs = [state["cache"]] if case["family"] == "append" else bound.outputs()
    return (lambda: bound.submit(inputs, outputs)), outputs


def run(state):
    """One pass through an operator; its outputs."""
    if own:
        state["submit"]()
        return state["outputs"]
    return {"prompt": _prompt, "append": _append, "decode": _decode}[state["case"]["family"]](state)


def _attend(case, query, key, value, visible):
    """Softmax attention in 32 bits: query [n, q, queries, d], key and value [n, k, heads, d], visible [n, q, k]; rows that see
    nothing come out as zeros, with the logarithm of an empty sum."""
    n, rows, queries, depth = query.shape
    keys, heads = key.shape[1], key.shape[2]
    shared = queries // heads
    q = query.float().view(n, rows, heads, shared, depth).permute(0, 2, 3, 1, 4).reshape(n * heads, shared * rows, depth)
    k = key.float().permute(0, 2, 3, 1).reshape(n * heads, depth, keys).contiguous()
    v = value.float().permute(0, 2, 1, 3).reshape(n * heads, keys, depth).contiguous()
    scores = torch.matmul(q, k).view(n, heads, shared, rows, keys).mul_(depth ** -0.5)
    scores.masked_fill_(~visible[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.view(n * heads, shared * rows, keys), v).view(n, heads, shared, rows, depth) / total.masked_fill(total == 0, 1.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(n, rows, queries, depth).to(query.dtype)
    if not case["log_sum"]:
        return [out]
    logs = (top + total.log()).squeeze(-1).masked_fill(total.squeeze(-1) == 0, -math.inf)
    return [out, logs.permute(0, 3, 1, 2).reshape(n, rows, queries)]


def _window(case, position, place):
    """Which of the keys at `place` a query at `position` sees, by the window and the first tokens."""
    seen = place <= position
    if case["window"]:
        seen = seen & ((place > position - case["window"]) | (place < case["sinks"]))
    return seen


def _prompt(state):
    case, query, key, value, marks = state["case"], state["query"], state["key"], state["value"], state["marks"]
    if not case["packed"]:
        place = torch.arange(query.shape[1], device=DEVICE)
        seen = (place[None, :] < marks[:, None])[:, None, :].expand(-1, query.shape[1], -1)
        if case["causal"]:
            seen = seen & _window(case, place[:, None], place[None, :])
        return _attend(case, query, key, value, seen)
    token = torch.arange(query.shape[0], device=DEVICE)
    sequence = torch.searchsorted(marks, token.to(torch.int32), right=True)
    place = token - marks[sequence - 1]
    seen = sequence[:, None] == sequence[None, :]
    if case["causal"]:
        seen = seen & _window(case, place[:, None], place[None, :])
    return [out[0] for out in _attend(case, query[None], key[None], value[None], seen[None])]


def _append(state):
    case, buffer = state["case"], state["buffer"]
    slots = state["slots"].long()
    page = torch.where(slots < 0, case["pages"], slots // case["page"])
    at = torch.where(slots < 0, 0, slots % case["page"])
    rows = torch.stack((state["key"], state["value"]), dim=1)
    if case["cache"] == "e4m3":
        rows = rows.float().clamp(-E4M3_LARGEST, E4M3_LARGEST).to(torch.float8_e4m3fn).view(torch.uint8)
        buffer = buffer.view(torch.uint8)
    buffer[page[:, None, None], torch.arange(2, device=DEVICE)[None, :, None], torch.arange(case["heads"], device=DEVICE)[None, None, :],
           at[:, None, None]] = rows
    return [state["cache"]]


def _decode(state):
    case, query, cache, table, lengths = state["case"], state["query"], state["cache"], state["table"], state["lengths"]
    sequences, columns = table.shape
    page, heads, depth = case["page"], case["heads"], case["depth"]
    if case["cache"] == "e4m3":
        cache = cache.to(torch.bfloat16)
    rows = cache[table.clamp(min=0).long()].permute(2, 0, 1, 4, 3, 5).reshape(2, sequences, columns * page, heads, depth)
    place = torch.arange(columns * page, device=DEVICE)[None, None, :]
    position = (lengths[:, None] - case["new"] + torch.arange(case["new"], device=DEVICE)[None])[:, :, None]
    return _attend(case, query, rows[0], rows[1], _window(case, position, place))


def _pairs(case, position, keys):
    """How many of the first `keys` keys a query at `position` sees."""
    most = min(keys, position + 1) if case["causal"] else keys
    if most <= 0 or not case["window"]:
        return max(0, most)
    low = max(0, position - case["window"] + 1)
    return max(0, most - low) + min(case["sinks"], low, most)


def work(case):
    """Every input and output once, of the keys those that some query sees; two products of `depth` for every pair seen."""
    heads, depth, size = case["heads"], case["depth"], SIZE[case["dtype"]]
    if case["family"] == "append":
        kept = case["tokens"] - case["skipped"]
        row = heads * depth
        return {"bytes": kept * 2 * row * (size + SIZE[case["cache"]]) + 4 * case["tokens"], "flops": kept * 2 * row}
    if case["family"] == "prompt":
        lengths = _prompt_lengths(case)
        tokens = sum(lengths) if case["packed"] else len(lengths) * max(lengths)
        pairs = sum(_pairs(case, i, n) for n in lengths for i in range(n if case["packed"] else max(lengths)))
        moved = tokens * 2 * case["queries"] * depth * size + sum(lengths) * 2 * heads * depth * size + 4 * len(lengths)
    else:
        lengths, new = _decode_lengths(case), case["new"]
        tokens = new * len(lengths)
        known = {**case, "causal": True}
        pairs = sum(_pairs(known, n - new + i, n) for n in lengths for i in range(new))
        window = case["window"] + new - 1 if case["window"] else 1 << 40
        seen = sum(min(n, window) + min(case["sinks"], max(0, n - window)) for n in lengths)
        moved = tokens * 2 * case["queries"] * depth * size + seen * 2 * heads * depth * SIZE[case["cache"]]
        moved += 4 * (len(lengths) + sum(-(-n // case["page"]) for n in lengths))
    return {"bytes": moved + (4 * tokens * case["queries"] if case["log_sum"] else 0), "flops": 4 * depth * case["queries"] * pairs}


def exact(case, seed):
    """What `run` returns, from the definition in 64 bits: a head and a sequence at a time, each query's row of weights over the
    keys that it may see."""
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    if case["family"] == "append":
        cache = state["cache"].double()
        kept = [(token, slot) for token, slot in enumerate(state["slots"].tolist()) if slot >= 0]
        token = torch.tensor([t for t, _ in kept], dtype=torch.int64, device=DEVICE)
        slot = torch.tensor([s for _, s in kept], dtype=torch.int64, device=DEVICE)
        for side, rows in enumerate((state["key"], state["value"])):
            rows = rows.double()[token]
            if case["cache"] == "e4m3":
                rows = _nearest_e4m3(rows)
            for head in range(case["heads"]):
                cache[slot // case["page"], side, head, slot % case["page"]] = rows[:, head]
        return [cache]
    if case["family"] == "decode":
        lengths, new = _decode_lengths(case), case["new"]
        spans = []
        for i, n in enumerate(lengths):
            place = torch.arange(n, device=DEVICE)
            where = state["table"][i].long()[place // case["page"]], place % case["page"]
            spans.append((state["query"][i], state["cache"][where[0], 0, :, where[1]], state["cache"][where[0], 1, :, where[1]], n - new, True))
    else:
        spans, first = [], 0
        for i, n in enumerate(_prompt_lengths(case)):
            if case["packed"]:
                spans.append(tuple(state[t][first:first + n] for t in ("query", "key", "value")) + (0, case["causal"]))
            else:
                spans.append((state["query"][i], state["key"][i, :n], state["value"][i, :n], 0, case["causal"]))
            first += n
    done = [_rows_exactly(case, *span) for span in spans]
    join = torch.cat if case["family"] == "prompt" and case["packed"] else torch.stack
    out = [join([d[0] for d in done])]
    return out + [join([d[1] for d in done])] if case["log_sum"] else out


def _rows_exactly(case, query, key, value, first, causal):
    """One sequence: query i stands at position first + i, key j at position j."""
    rows, queries, depth = query.shape
    keys = key.shape[0]
    out = torch.zeros((rows, queries, depth), dtype=torch.float64, device=DEVICE)
    logs = torch.full((rows, queries), -math.inf, dtype=torch.float64, device=DEVICE)
    if not keys:
        return out, logs
    for begin in range(0, rows, 2048):
        end = min(rows, begin + 2048)
        distance = torch.arange(first + begin, first + end, device=DEVICE)[:, None] - torch.arange(keys, device=DEVICE)[None, :]
        hidden = torch.zeros_like(distance, dtype=torch.bool)
        if causal:
            hidden |= distance < 0
            if case["window"]:
                far = distance >= case["window"]
                far[:, :case["sinks"]] = False
                hidden |= far
        empty = hidden.all(dim=1)
        for head in range(queries):
            shared = head // (queries // case["heads"])
            logits = query[begin:end, head].double() @ key[:, shared].double().t().contiguous() / math.sqrt(depth)
            logits = torch.where(hidden, -math.inf, logits)
            log_sum = torch.logsumexp(logits, dim=1)
            weights = torch.where(hidden, 0.0, torch.exp(logits - torch.where(empty, 0.0, log_sum)[:, None]))
            out[begin:end, head] = weights @ value[:, shared].double().contiguous()
            logs[begin:end, head] = log_sum
    return out, logs


def _nearest_e4m3(x):
    """The nearest number of three mantissa bits and exponents from -6 to 8, ties to the even mantissa, at most 448."""
    size = x.abs().clamp(max=E4M3_LARGEST)
    exponent = torch.floor(torch.log2(size.clamp(min=2.0 ** -6)))
    step = torch.exp2(exponent - 3)
    return torch.copysign((torch.round(size / step) * step).clamp(max=E4M3_LARGEST), x)
