"""What a decoding step does to a paged cache, as cases that can be timed and compared.

A case is a dict of plain values; its "family" says which operator it is:

    append   RotaryAppend: the fused projection of new tokens to rotated queries and to their slots of a cache
    decode4  PagedAttention over a cache in 4 bits
    bounds   PageBounds: the least and largest key of every channel of the pages that changed
    select   PagedSelect: the pages that a score by those bounds finds for each key head
    sparse   PagedAttention over the pages that were selected for each key head

"mx4" is a cache of bytes [pages, 2, heads, page, 17 depth / 32]: a head's side of a page is the codes [page, depth / 2] of its rows, two
to a byte, the first in the low bits, then their scales [page, depth / 32], one to 32 elements: a sign, two exponent bits and one of
mantissa times a power of two whose exponent is the byte less 127.

`run` computes them in elementary operations in 32 bits (the selection's scores in 64: which page comes first is decided by the last of
them), or, where `own` is true, by the library's operators, each prepared once and submitted on every pass.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
SIZE = {"bf16": 2.0, "f16": 2.0, "e4m3": 1.0, "mx4": 17 / 32}
E4M3_LARGEST = 448.0
BASE = 1.0e6  # of the rotation's frequencies
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # of a code without its sign
TIES = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)     # between them


def listed():
    return [
        # the new token of every stream of a batch: what each layer does per step before it attends
        {"name": "append_step", "family": "append", "tokens": 64, "queries": 32, "heads": 8, "depth": 128, "rotary": 128, "half_split": True,
         "dtype": "bf16", "cache": "bf16", "page": 16, "pages": 256, "skipped": 3, "prompt": False},
        # a prompt's queries, and its keys and values into a cache of 8 bits
        {"name": "append_prompt_e4m3", "family": "append", "tokens": 8192, "queries": 32, "heads": 8, "depth": 128, "rotary": 128,
         "half_split": True, "dtype": "bf16", "cache": "e4m3", "page": 64, "pages": 160, "skipped": 0, "prompt": True},
        # prompts of a batch that add up to any number of tokens, part of each head rotated, into 4 bits (given back as values, which takes
        # most of the pass on both sides)
        {"name": "append_ragged_mx4", "family": "append", "tokens": 1037, "queries": 20, "heads": 5, "depth": 96, "rotary": 64,
         "half_split": False, "dtype": "f16", "cache": "mx4", "page": 16, "pages": 80, "skipped": 40, "prompt": True},
        # a batch of streams of every age
        {"name": "decode4_batch_ragged", "family": "decode4", "sequences": 64, "shortest": 30, "longest": 16384, "new": 1, "queries": 32,
         "heads": 8, "depth": 128, "dtype": "bf16", "cache": "mx4", "page": 16, "window": 0, "sinks": 0, "log_sum": False},
        # one user with a very long document, wide heads: few rows, a long axis
        {"name": "decode4_one_long", "family": "decode4", "sequences": 1, "shortest": 131055, "longest": 131055, "new": 1, "queries": 16,
         "heads": 2, "depth": 256, "dtype": "bf16", "cache": "mx4", "page": 16, "window": 0, "sinks": 0, "log_sum": True},
        # four drafted tokens per stream through a layer with a window and first tokens that stay visible
        {"name": "decode4_drafts_window", "family": "decode4", "sequences": 12, "shortest": 500, "longest": 9000, "new": 4, "queries": 20,
         "heads": 5, "depth": 96, "dtype": "f16", "cache": "mx4", "page": 32, "window": 2048, "sinks": 4, "log_sum": False},
        # after every step, the page that each stream wrote to: the smallest call
        {"name": "bounds_step", "family": "bounds", "sequences": 64, "shortest": 100, "longest": 8192, "newest": 1, "heads": 8, "depth": 128,
         "cache": "bf16", "page": 16},
        # after prompts were read, all of their pages
        {"name": "bounds_prompts_e4m3", "family": "bounds", "sequences": 5, "shortest": 9001, "longest": 32768, "newest": 0, "heads": 8,
         "depth": 128, "cache": "e4m3", "page": 64},
        # a sixteenth of the pages of long streams
        {"name": "select_batch", "family": "select", "sequences": 16, "shortest": 20000, "longest": 32768, "new": 1, "queries": 32, "heads": 8,
         "depth": 128, "dtype": "bf16", "page": 16, "count": 128},
        # two drafted tokens of one user with a very long document
        {"name": "select_one_long", "family": "select", "sequences": 1, "shortest": 131055, "longest": 131055, "new": 2, "queries": 16,
         "heads": 2, "depth": 256, "dtype": "f16", "page": 32, "count": 200},
        # the attention over what was selected
        {"name": "sparse_batch", "family": "sparse", "sequences": 16, "shortest": 20000, "longest": 32768, "new": 1, "queries": 32, "heads": 8,
         "depth": 128, "dtype": "bf16", "cache": "bf16", "page": 16, "count": 128, "log_sum": False},
        # drafted tokens over a cache in 4 bits, some streams shorter than what may be selected
        {"name": "sparse_drafts_mx4", "family": "sparse", "sequences": 7, "shortest": 700, "longest": 30000, "new": 3, "queries": 20, "heads": 5,
         "depth": 128, "dtype": "f16", "cache": "mx4", "page": 32, "count": 48, "log_sum": True},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    family = rng.choice(["append", "append", "decode4", "decode4", "bounds", "select", "sparse"])
    heads = rng.choice([1, 2, 3, 4, 5, 8])
    queries = heads * rng.choice([1, 2, 4, 4, 5, 8])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    cache = "mx4" if family == "decode4" else rng.choice([dtype, dtype, "e4m3", "mx4"])
    depth = rng.choice([64, 96, 128, 128, 128, 256] if cache == "mx4" else [64, 80, 96, 128, 128, 128, 256])
    page = rng.choice([8, 16, 16, 32, 64, 256])
    if family == "append":
        tokens = _log(rng, 1, 8192)
        return {"family": family, "tokens": tokens, "queries": queries, "heads": heads, "depth": depth,
                "rotary": rng.choice([depth, depth, depth // 2, 16]), "half_split": rng.random() < 0.7, "dtype": dtype, "cache": cache, "page": page,
                "pages": -(-tokens // page) + rng.randint(1, 64), "skipped": rng.choice([0, 0, tokens // 7]), "prompt": rng.random() < 0.5}
    sequences = _log(rng, 1, 64)
    longest = max(1, min(_log(rng, 1, 131072), (3 << 26) // (sequences * heads * depth)))
    ages = {"sequences": sequences, "shortest": rng.randint(1, longest), "longest": longest, "heads": heads, "depth": depth, "page": page}
    if family == "bounds":
        return {"family": family, **ages, "newest": rng.choice([0, 0, 1, 1, 4, 500]), "cache": cache}
    ages.update({"new": rng.choice([1, 1, 1, 2, 3, 4, 8]), "queries": queries, "dtype": dtype})
    if family == "decode4":
        window, sinks = rng.choice([(0, 0), (0, 0), (_log(rng, 16, 4096), rng.choice([0, 1, 4]))])
        return {"family": family, **ages, "cache": cache, "window": window, "sinks": sinks, "log_sum": rng.random() < 0.3}
    ages["count"] = 1 + _always(ages) + _log(rng, 1, 256)
    return {"family": family, **ages} if family == "select" else {"family": family, **ages, "cache": cache, "log_sum": rng.random() < 0.3}


def _always(case):
    """The most pages that a sequence's newest tokens lie in."""
    return (case["new"] + case["page"] - 2) // case["page"] + 1


def _lengths(case):
    """Lengths between the shortest and the longest, evenly over their logarithm and in no order."""
    low, high = case["shortest"], case["longest"]
    return [round(low * (high / low) ** ((1 + 0.6180339887 * i) % 1 if i else 1)) for i in range(case["sequences"])]


class _Make:
    """Inputs on the GPU from one seed."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEVICE)
        self.g.manual_seed(seed)

    def normal(self, shape, dtype, std=1.0):
        made = torch.empty(shape, dtype=torch.bfloat16 if dtype == "e4m3" else TYPES.get(dtype, torch.float32), device=DEVICE)
        made.normal_(0.0, std, generator=self.g)
        return made.to(TYPES[dtype]) if dtype == "e4m3" else made

    def uniform(self, shape):
        return torch.empty(shape, dtype=torch.float32, device=DEVICE).uniform_(generator=self.g)

    def order(self, count):
        return torch.randperm(count, device=DEVICE, generator=self.g)

    def cache(self, pages, heads, page, depth, kind):
        """A cache whose every row holds something: in 4 bits codes of every kind and scales around those of numbers near one."""
        if kind != "mx4":
            return self.normal((pages, 2, heads, page, depth), kind)
        codes = torch.randint(0, 256, (pages, 2, heads, page * depth // 2), dtype=torch.uint8, device=DEVICE, generator=self.g)
        scales = torch.randint(124, 128, (pages, 2, heads, page * depth // 32), dtype=torch.uint8, device=DEVICE, generator=self.g)
        return torch.cat((codes, scales), dim=-1).view(pages, 2, heads, page, depth * 17 // 32)


def prepare(case, seed):
    """Queries of normed heads, values near one, caches whose pages are handed out in no order and whose free slots hold what was
    there before."""
    make = _Make(seed)
    heads, depth, page = case["heads"], case["depth"], case["page"]
    state = {"case": case}
    if case["family"] == "append":
        pages, tokens, rotary = case["pages"], case["tokens"], case["rotary"]
        state["projected"] = make.normal((tokens, case["queries"] + 2 * heads, depth), case["dtype"], 1.25)
        # a prompt's tokens stand behind one another, new tokens of streams anywhere
        state["positions"] = (torch.arange(tokens, device=DEVICE) + 77 if case["prompt"] else make.order(131072)[:tokens]).to(torch.int32)
        state["frequencies"] = torch.tensor([BASE ** (-2 * i / rotary) for i in range(rotary // 2)], dtype=torch.float32, device=DEVICE)
        slots = make.order(pages * page)[:tokens].to(torch.int32)
        slots[make.order(tokens)[:case["skipped"]]] = -1  # tokens that keep no place
        state["slots"] = slots
        state["buffer"] = make.cache(pages + 1, heads, page, depth, case["cache"])  # the last page takes what has no place
        state["cache"] = state["buffer"][:pages]
    else:
        lengths = _lengths(case)
        held = [-(-n // page) for n in lengths]
        pages, most = sum(held) + 3, max(held)
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
        starts = torch.tensor([sum(held[:i]) for i in range(len(held))], device=DEVICE)[:, None]
        column = torch.arange(most, device=DEVICE)[None]
        columns = torch.tensor(held, device=DEVICE)[:, None]
        has = column < columns
        state["table"] = torch.where(has, make.order(pages)[(starts + column).clamp(max=pages - 1)], -1).to(torch.int32)
        if case["family"] != "bounds":
            state["query"] = make.normal((len(lengths), case["new"], case["queries"], depth), case["dtype"], 1.5)
        if case["family"] == "select":
            # pages whose keys lie round a center of their own
            center, width = make.normal((pages, heads, depth), "f32", 0.5), make.normal((pages, heads, depth), "f32", 0.4).abs() + 1.3
            state["bounds"] = torch.stack((center - width, center + width), dim=1).to(torch.bfloat16)
        else:
            state["cache"] = make.cache(pages, heads, page, depth, case["cache"])
        if case["family"] == "bounds":
            state["bounds"] = torch.zeros((pages, 2, heads, depth), dtype=torch.bfloat16, device=DEVICE)
        if case["family"] == "sparse":
            # any pages of each key head, the first and the newest tokens' among them, in order
            count = case["count"]
            chance = make.uniform((len(lengths), heads, most))
            chance.masked_fill_(((column == 0) | (column >= columns - _always(case)))[:, None], -1.0)
            chance.masked_fill_(~has[:, None], 2.0)
            first = torch.argsort(chance, dim=-1)[..., :count]
            kept = torch.where(torch.gather(chance, -1, first) < 1.5, first, most).sort(dim=-1).values
            there = kept < most
            physical = torch.gather(state["table"][:, None].expand(-1, heads, -1), -1, kept.clamp(max=most - 1))
            state["selected"] = torch.where(there, physical, -1).to(torch.int32)
            state["seen"] = (state["lengths"][:, None] - page * (columns - there.sum(-1))).to(torch.int32)
    if own:
        state["submit"], state["outputs"] = _bound(case, state)
    return state


def _bound(case, state):
    """The library's operator for a case, its inputs bound to it, and the tensors it writes."""
    from hyle_amd import compute as hc
    from hyle_amd import torch_io as tio
    family = case["family"]
    if family == "append":
        operation = hc.RotaryAppend(case["pages"], case["page"], tio.desc_of(state["cache"]).data_type, case["heads"],
                                    hc.RopeLayout.kHalfSplit if case["half_split"] else hc.RopeLayout.kInterleaved)
        inputs = [state[t] for t in ("projected", "positions", "frequencies", "slots")]
    elif family == "bounds":
        operation, inputs = hc.PageBounds(newest=case["newest"]), [state["cache"], state["table"], state["lengths"]]
    elif family == "select":
        operation = hc.PagedSelect(count=case["count"], page_size=case["page"])
        inputs = [state["query"], state["bounds"], state["table"], state["lengths"]]
    else:
        operation = hc.PagedAttention(scale=case["depth"] ** -0.5, window=case.get("window", 0), sinks=case.get("sinks", 0),
                                      return_log_sum=case["log_sum"])
        named = ("query", "cache", "selected", "seen") if family == "sparse" else ("query", "cache", "table", "lengths")
        inputs = [state[t] for t in named]
    bound = tio.Bound(hc.Context.create(0), operation, [tio.desc_of(t) for t in inputs])
    outputs = [state["bounds"]] if family == "bounds" else bound.outputs()
    if family == "append":
        outputs[0] = state["cache"]
    return (lambda: bound.submit(inputs, outputs)), outputs


def run(state):
    """One pass through an operator; its outputs."""
    case = state["case"]
    if own:
        state["submit"]()
        outputs = state["outputs"]
    else:
        outputs = {"append": _append, "decode4": _decode, "bounds": _page_bounds, "select": _select, "sparse": _sparse}[case["family"]](state)
    if case["family"] == "append" and case["cache"] == "mx4":
        return [_values(outputs[0], case["depth"]), *outputs[1:]]
    return outputs


# ---- plain forms ----

def _planes(cache, depth):
    """A 4-bit cache's codes [.., page, depth / 2] and scales [.., page, depth / 32]."""
    page = cache.shape[-2]
    flat = cache.view(*cache.shape[:-2], page * depth * 17 // 32)
    codes, scales = flat[..., :page * depth // 2], flat[..., page * depth // 2:]
    return codes.unflatten(-1, (page, depth // 2)), scales.unflatten(-1, (page, depth // 32))


_pairs_of_levels = {}


def _values(cache, depth):
    """The bf16 numbers that a 4-bit cache stands for, [.., page, depth]."""
    codes, scales = _planes(cache, depth)
    if not _pairs_of_levels:
        level = torch.tensor([*LEVELS, *(-v for v in LEVELS)], dtype=torch.bfloat16, device=DEVICE)
        byte = torch.arange(256, device=DEVICE)
        _pairs_of_levels["bf16"] = torch.stack((level[byte % 16], level[byte // 16]), dim=-1).view(torch.int32).view(256)
    pairs = torch.index_select(_pairs_of_levels["bf16"], 0, codes.reshape(-1).int()).view(torch.bfloat16)
    factor = torch.exp2(scales.float() - 127.0).to(torch.bfloat16)
    return (pairs.view(*factor.shape, 32) * factor[..., None]).view(*cache.shape[:-1], depth)


def _to_mx4(x):
    """Rows of f32 as codes [.., depth / 2] and scales [.., depth / 32]: the largest's exponent less two, one more where its significand
    is over 1.75, so that nothing is further from its code than half a step; nearest codes, ties to the even one."""
    blocks = x.unflatten(-1, (x.shape[-1] // 32, 32))
    exponent = (blocks.abs().amax(-1).view(torch.int32) + 0x1FFFFF) >> 23
    byte = (exponent - 2).clamp(0, 252)
    scaled = blocks * torch.exp2((127 - byte).float())[..., None]
    size = scaled.abs()
    code = torch.zeros_like(size, dtype=torch.uint8)
    for i, tie in enumerate(TIES):
        code += (size > tie) if i % 2 == 0 else (size >= tie)
    code = (code + 8 * torch.signbit(scaled).to(torch.uint8)).flatten(-2)
    return code[..., 0::2] + 16 * code[..., 1::2], byte.to(torch.uint8)


def _append(state):
    case, buffer, projected = state["case"], state["buffer"], state["projected"]
    queries, heads, depth, page, rotary = case["queries"], case["heads"], case["depth"], case["page"], case["rotary"]
    # phases in f32, as RoPE has them; the functions of far ones in 64 bits
    phase = (state["frequencies"][None, :] * state["positions"].float()[:, None]).double()
    c, s = torch.cos(phase).float()[:, None], torch.sin(phase).float()[:, None]
    x = projected.float()
    turned = x[:, :queries + heads].clone()
    first = slice(0, rotary // 2) if case["half_split"] else slice(0, rotary, 2)
    second = slice(rotary // 2, rotary) if case["half_split"] else slice(1, rotary, 2)
    a, b = x[:, :queries + heads, first], x[:, :queries + heads, second]
    turned[..., first] = a * c - b * s
    turned[..., second] = a * s + b * c
    rows = torch.stack((turned[:, queries:], x[:, queries + heads:]), dim=1)  # [tokens, 2, heads, depth]
    slots = state["slots"].long()
    at_page = torch.where(slots < 0, case["pages"], slots // page)
    at = torch.where(slots < 0, 0, slots % page)
    place = (at_page[:, None, None], torch.arange(2, device=DEVICE)[None, :, None], torch.arange(heads, device=DEVICE)[None, None, :],
             at[:, None, None])
    if case["cache"] == "mx4":
        codes, scales = _planes(buffer, depth)
        codes[place], scales[place] = _to_mx4(rows)
    elif case["cache"] == "e4m3":
        buffer.view(torch.uint8)[place] = rows.clamp(-E4M3_LARGEST, E4M3_LARGEST).to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        buffer[place] = rows.to(buffer.dtype)
    return [state["cache"], turned[:, :queries].to(projected.dtype)]


def _attend(query, key, value, visible, log_sum):
    """Softmax attention in 32 bits: query [n, q, heads, shared, depth], key and value [n, k, heads, depth], visible [n, heads or 1, q, k];
    rows that see nothing come out as zeros, with the logarithm of an empty sum."""
    n, rows, heads, shared, depth = query.shape
    keys = key.shape[1]
    q = query.float().permute(0, 2, 3, 1, 4).reshape(n * heads, shared * rows, depth)
    k = key.float().permute(0, 2, 3, 1).reshape(n * heads, depth, keys).contiguous()
    v = value.float().permute(0, 2, 1, 3).reshape(n * heads, keys, depth).contiguous()
    scores = torch.matmul(q, k).view(n, heads, shared, rows, keys).mul_(depth ** -0.5)
    scores.masked_fill_(~visible[:, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.view(n * heads, shared * rows, keys), v).view(n, heads, shared, rows, depth) / total.masked_fill(total == 0, 1.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(n, rows, heads * shared, depth).to(query.dtype)
    if not log_sum:
        return [out]
    logs = (top + total.log()).squeeze(-1).masked_fill(total.squeeze(-1) == 0, -math.inf)
    return [out, logs.permute(0, 3, 1, 2).reshape(n, rows, heads * shared)]


def _numbers(cache, depth):
    return _values(cache, depth) if cache.dtype == torch.uint8 else cache.to(torch.bfloat16) if cache.dtype == torch.float8_e4m3fn else cache


def _grouped(case, query):
    return query.view(query.shape[0], query.shape[1], case["heads"], case["queries"] // case["heads"], case["depth"])


def _decode(state):
    case, table, lengths = state["case"], state["table"], state["lengths"]
    sequences, columns = table.shape
    page, heads, depth = case["page"], case["heads"], case["depth"]
    rows = _numbers(state["cache"], depth)[table.clamp(min=0).long()].permute(2, 0, 1, 4, 3, 5).reshape(2, sequences, columns * page, heads, depth)
    place = torch.arange(columns * page, device=DEVICE)[None, None, :]
    position = (lengths[:, None] - case["new"] + torch.arange(case["new"], device=DEVICE)[None])[:, :, None]
    seen = place <= position
    if case["window"]:
        seen = seen & ((place > position - case["window"]) | (place < case["sinks"]))
    return _attend(_grouped(case, state["query"]), rows[0], rows[1], seen[:, None], case["log_sum"])


def _sparse(state):
    case, selected, seen = state["case"], state["selected"], state["seen"]
    sequences, heads, columns = selected.shape
    page, depth = case["page"], case["depth"]
    head = torch.arange(heads, device=DEVICE)[None, :, None]
    rows = _numbers(state["cache"], depth)[selected.clamp(min=0).long(), :, head]  # [sequences, heads, columns, 2, page, depth]
    rows = rows.permute(3, 0, 2, 4, 1, 5).reshape(2, sequences, columns * page, heads, depth)
    place = torch.arange(columns * page, device=DEVICE)
    position = seen[:, :, None] - case["new"] + torch.arange(case["new"], device=DEVICE)
    visible = (place <= position[..., None]) & (selected >= 0).repeat_interleave(page, dim=-1)[:, :, None]
    return _attend(_grouped(case, state["query"]), rows[0], rows[1], visible, case["log_sum"])


def _changed(case, table, lengths):
    """[sequences, columns]: the pages that hold some of the newest tokens (or any token)."""
    page, column = case["page"], torch.arange(table.shape[1], device=DEVICE)[None]
    since = (lengths[:, None] - case["newest"]).clamp(min=0) if case["newest"] else torch.zeros_like(lengths[:, None])
    return (column * page < lengths[:, None]) & ((column + 1) * page > since)


def _page_bounds(state):
    case, table, lengths, bounds = state["case"], state["table"], state["lengths"], state["bounds"]
    page = case["page"]
    sequence, column = torch.nonzero(_changed(case, table, lengths), as_tuple=True)
    pages = table[sequence, column].long()
    if state["cache"].dtype == torch.float8_e4m3fn:
        held = state["cache"].view(torch.uint8)[pages, 0].view(torch.float8_e4m3fn).float()
    else:
        held = state["cache"][pages, 0]
        held = _values(held, case["depth"]).float() if held.dtype == torch.uint8 else held.float()
    # [pages, heads, page, depth], of them the sequence's own keys
    there = (column[:, None] * page + torch.arange(page, device=DEVICE)[None] < lengths[sequence][:, None])[:, None, :, None]
    low = held.masked_fill(~there, math.inf).amin(2).view(torch.int32)
    high = held.masked_fill(~there, -math.inf).amax(2).view(torch.int32)
    # the nearest bf16 below and above
    low = torch.where(low < 0, (low + 0xFFFF), low) & -0x10000
    high = torch.where(high < 0, high, (high + 0xFFFF)) & -0x10000
    bounds[pages] = torch.stack((low.view(torch.float32), high.view(torch.float32)), dim=1).to(torch.bfloat16)
    return [bounds]


def _select(state):
    case, table, lengths, query = state["case"], state["table"], state["lengths"], state["query"]
    sequences, columns = table.shape
    heads, page, count = case["heads"], case["page"], case["count"]
    column = torch.arange(columns, device=DEVICE)[None]
    filled = (lengths[:, None] + page - 1) // page
    bounds = state["bounds"][table.clamp(min=0).long()].double().permute(0, 3, 2, 4, 1)  # [sequences, heads, 2, depth, columns]
    bounds = bounds.reshape(sequences * heads, 2 * case["depth"], columns).contiguous()
    q = _grouped(case, query).double().permute(0, 2, 3, 1, 4).reshape(sequences * heads, -1, case["depth"])
    scores = torch.matmul(torch.cat((q.clamp(max=0.0), q.clamp(min=0.0)), dim=-1), bounds).amax(1).float().view(sequences, heads, columns)
    always = (column == 0) | ((column + 1) * page > lengths[:, None] - case["new"])
    scores = scores.masked_fill(always[:, None], math.inf).masked_fill((column >= filled)[:, None], -math.inf)
    best = torch.sort(scores, dim=-1, descending=True, stable=True).indices[..., :count]
    kept = torch.where(best < filled[:, :, None], best, columns).sort(dim=-1).values
    kept = torch.nn.functional.pad(kept, (0, count - kept.shape[-1]), value=columns)
    there = kept < columns
    pages = torch.gather(table[:, None].expand(-1, heads, -1), -1, kept.clamp(max=columns - 1))
    seen = lengths[:, None] - page * (filled - there.sum(-1))
    return [torch.where(there, pages, -1).to(torch.int32), seen.to(torch.int32)]


# ---- work ----

def work(case):
    """Every input and output once, of the cache what some row sees; two products of `depth` for every pair seen."""
    heads, depth, family = case["heads"], case["depth"], case["family"]
    if family == "append":
        tokens, queries, kept = case["tokens"], case["queries"], case["tokens"] - case["skipped"]
        size = SIZE[case["dtype"]]
        moved = tokens * 2 * queries * depth * size + kept * 2 * heads * depth * (size + SIZE[case["cache"]])
        return {"bytes": int(moved + 8 * tokens + 2 * case["rotary"]), "flops": (tokens * queries + kept * heads) * case["rotary"] * 3}
    lengths, page = _lengths(case), case["page"]
    if family == "bounds":
        spans = [(0 if not case["newest"] else max(0, n - case["newest"]) // page * page, n) for n in lengths]
        keys, pages = sum(n - first for first, n in spans), sum(-(-(n - first) // page) for first, n in spans)
        return {"bytes": int(keys * heads * depth * SIZE[case["cache"]] + pages * (4 * heads * depth + 4) + 4 * len(lengths)),
                "flops": 2 * keys * heads * depth}
    new, tokens = case["new"], case["new"] * len(lengths)
    columns = [-(-n // page) for n in lengths]
    moved = tokens * case["queries"] * depth * SIZE[case["dtype"]] + 4 * len(lengths)
    if family == "select":
        scored = sum(columns)
        return {"bytes": int(moved + scored * (4 + 4 * heads * depth) + len(lengths) * heads * 4 * (case["count"] + 1)),
                "flops": 2 * depth * case["queries"] * new * scored}
    moved *= 2
    if family == "sparse":
        lengths = [n - page * (c - min(c, case["count"])) for n, c in zip(lengths, columns)]
    window = case.get("window", 0)
    pairs, keys = 0, 0
    for n in lengths:
        for i in range(new):
            most = max(0, n - new + i + 1)
            low = max(0, most - window) if window else 0
            pairs += most - low + min(case["sinks"], low) if window else most
        low = max(0, n - new + 1 - window) if window else 0
        keys += n - low + (min(case["sinks"], low) if window else 0)
    tables = 4 * sum(-(-n // page) for n in lengths) * (heads if family == "sparse" else 1)
    moved += keys * 2 * heads * depth * SIZE[case["cache"]] + tables + (4 * tokens * case["queries"] if case["log_sum"] else 0)
    return {"bytes": int(moved), "flops": 4 * depth * case["queries"] * pairs}


# ---- the definitions in 64 bits ----

def exact(case, seed):
    """What `run` returns, from the definition in 64 bits."""
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    if case["family"] == "append":
        return _append_exactly(case, state)
    if case["family"] == "bounds":
        return [_bounds_exactly(case, state)]
    if case["family"] == "select":
        return _select_exactly(case, state)
    outs, logs = [], []
    for i, n in enumerate(_lengths(case)):
        for head in range(case["heads"]):
            if case["family"] == "sparse":
                table, length = state["selected"][i, head].long(), int(state["seen"][i, head])
            else:
                table, length = state["table"][i].long(), n
            place = torch.arange(length, device=DEVICE)
            key, value = (_rows_exactly(case, state["cache"], table[place // case["page"]], place % case["page"], side, head) for side in (0, 1))
            out, log = _softmax_exactly(case, state["query"][i], key, value, head)
            outs.append(out)
            logs.append(log)
    out = torch.stack(outs).unflatten(0, (len(_lengths(case)), case["heads"]))  # [sequences, heads, new, shared, depth]
    log = torch.stack(logs).unflatten(0, (len(_lengths(case)), case["heads"]))
    answers = [out.permute(0, 2, 1, 3, 4).flatten(2, 3)]
    return answers + [log.permute(0, 2, 1, 3).flatten(2, 3)] if case["log_sum"] else answers


def _rows_exactly(case, cache, page, at, side, head):
    """Rows of one head in 64 bits, [rows, depth]."""
    if case["cache"] != "mx4":
        return cache[page, side, head, at].double()
    depth = case["depth"]
    flat = cache[page, side, head].flatten(1)
    byte = torch.arange(depth, device=DEVICE) // 2
    held = torch.gather(flat, 1, at[:, None] * (depth // 2) + byte[None])
    code = torch.where(torch.arange(depth, device=DEVICE) % 2 == 0, held & 15, held >> 4).long()
    power = (code >> 1) & 3
    size = torch.where(power == 0, 0.5 * (code & 1), (1.0 + 0.5 * (code & 1)) * torch.exp2(power.double() - 1))
    scale = torch.gather(flat, 1, case["page"] * (depth // 2) + at[:, None] * (depth // 32) + (torch.arange(depth, device=DEVICE) // 32)[None])
    return torch.where(code >= 8, -size, size) * torch.exp2(scale.double() - 127)


def _softmax_exactly(case, query, key, value, head):
    new, shared, depth = case["new"], case["queries"] // case["heads"], case["depth"]
    q = query[:, head * shared:(head + 1) * shared].double().reshape(new * shared, depth)
    position = key.shape[0] - new + torch.arange(new, device=DEVICE).repeat_interleave(shared)[:, None]
    place = torch.arange(key.shape[0], device=DEVICE)[None]
    hidden = place > position
    window = case.get("window", 0)
    if window:
        hidden = hidden | ((place <= position - window) & (place >= case["sinks"]))
    logits = torch.where(hidden, -math.inf, q @ key.t().contiguous() / math.sqrt(depth))
    log = torch.logsumexp(logits, dim=1)
    weights = torch.where(hidden, 0.0, torch.exp(logits - torch.where(torch.isfinite(log), log, 0.0)[:, None]))
    return (weights @ value).view(new, shared, depth), log.view(new, shared)


def _append_exactly(case, state):
    queries, heads, depth, rotary = case["queries"], case["heads"], case["depth"], case["rotary"]
    x = state["projected"].double()
    phase = torch.outer(state["positions"].float(), state["frequencies"]).double()  # (an f32 product: the operator's phase)
    turn = torch.polar(torch.ones_like(phase), phase)[:, None]
    rotated = x[..., :rotary]
    pair = rotated.unflatten(-1, (2, rotary // 2)).transpose(-1, -2) if case["half_split"] else rotated.unflatten(-1, (rotary // 2, 2))
    pair = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
    pair = pair.transpose(-1, -2).flatten(-2) if case["half_split"] else pair.flatten(-2)
    y = torch.cat((pair, x[..., rotary:]), dim=-1)
    if case["cache"] == "mx4":
        pages, page = torch.meshgrid(torch.arange(case["pages"], device=DEVICE), torch.arange(case["page"], device=DEVICE), indexing="ij")
        cache = torch.stack([torch.stack([_rows_exactly(case, state["cache"], pages.flatten(), page.flatten(), side, head)
                                          .view(case["pages"], case["page"], depth) for head in range(heads)], dim=1) for side in (0, 1)], dim=1)
    else:
        cache = state["cache"].double()
    kept = [(token, slot) for token, slot in enumerate(state["slots"].tolist()) if slot >= 0]
    token = torch.tensor([t for t, _ in kept], dtype=torch.int64, device=DEVICE)
    slot = torch.tensor([s for _, s in kept], dtype=torch.int64, device=DEVICE)
    for side, rows in enumerate((y[:, queries:queries + heads], x[:, queries + heads:])):
        rows = rows[token]
        if case["cache"] == "mx4":
            rows = _nearest_mx4(rows)
        elif case["cache"] == "e4m3":
            rows = _nearest(rows, torch.exp2(_exponent(rows).clamp(min=-6) - 3), E4M3_LARGEST)
        for head in range(heads):
            cache[slot // case["page"], side, head, slot % case["page"]] = rows[:, head]
    return [cache, y[:, :queries]]


def _exponent(x):
    return torch.floor(torch.log2(x.abs().clamp(min=1e-300)))


def _nearest(x, step, largest):
    """The nearest multiple of `step`, ties to the even one, no larger than `largest`."""
    size = (torch.round(x.abs() / step) * step).clamp(max=largest)
    return torch.copysign(size, x)


def _nearest_mx4(x):
    blocks = x.unflatten(-1, (-1, 32))
    most = blocks.abs().amax(-1, keepdim=True)
    power = _exponent(most)
    scale = torch.exp2(power + (most > 1.75 * torch.exp2(power)).double() - 2)
    y = blocks / scale
    return (_nearest(y, torch.exp2(_exponent(y).clamp(min=0) - 1), 6.0) * scale).flatten(-2)


def _select_exactly(case, state):
    pages = torch.full((case["sequences"], case["heads"], case["count"]), -1, dtype=torch.int32, device=DEVICE)
    seen = torch.zeros((case["sequences"], case["heads"]), dtype=torch.int32, device=DEVICE)
    shared, page = case["queries"] // case["heads"], case["page"]
    for i, n in enumerate(_lengths(case)):
        filled = -(-n // page)
        newest = max(0, n - case["new"]) // page  # the first page of the newest tokens
        for head in range(case["heads"]):
            low, high = state["bounds"][state["table"][i, :filled].long(), :, head].double().unbind(1)
            score = torch.full((filled,), -math.inf, device=DEVICE)
            for q in state["query"][i, :, head * shared:(head + 1) * shared].double().flatten(0, 1):
                score = torch.maximum(score, (q * torch.where(q >= 0, high, low)).sum(-1).float())
            score[0], score[newest:] = math.inf, math.inf
            kept = torch.sort(torch.argsort(-score, stable=True)[:case["count"]]).values
            pages[i, head, :len(kept)] = state["table"][i, kept]
            seen[i, head] = n - page * (filled - len(kept))
    return [pages, seen]


def _bounds_exactly(case, state):
    bounds = state["bounds"].double()
    for i, n in enumerate(_lengths(case)):
        first = 0 if not case["newest"] else max(0, n - case["newest"]) // case["page"] * case["page"]
        place = torch.arange(first, n, device=DEVICE)
        for head in range(case["heads"]):
            key = _rows_exactly(case, state["cache"], state["table"][i].long()[place // case["page"]], place % case["page"], 0, head)
            lacks = -len(place) % case["page"]
            whole = torch.cat((key, key[-1:].expand(lacks, -1))).view(-1, case["page"], case["depth"])
            pages = state["table"][i, first // case["page"]:first // case["page"] + whole.shape[0]].long()
            for side, (edge, to) in enumerate(((whole.amin(1), torch.floor), (whole.amax(1), torch.ceil))):
                step = torch.exp2(_exponent(edge).clamp(min=-126) - 7)
                bounds[pages, side, head] = to(edge / step) * step
    return bounds
