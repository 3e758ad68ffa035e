"""PagedAppend where several tokens have one slot: its elements are some token's at that place, and nothing else changes."""
from __future__ import annotations

import pytest
import torch

from hyle_amd import compute as hc
from hyle_amd import torch_io as tio

from gpu_support import DEVICE, context, note

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}


@pytest.mark.parametrize("tag,cache_tag", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "e4m3")])
@pytest.mark.parametrize("tokens,heads,depth", [(2, 1, 8), (40, 2, 128), (40, 3, 80), (700, 8, 128), (130, 2, 63)])
def test_a_slot_of_several_tokens_holds_their_elements(tag, cache_tag, tokens, heads, depth):
    make = torch.Generator(DEVICE).manual_seed(depth + tokens)
    keys, values = (torch.empty((tokens, heads, depth), device=DEVICE).normal_(0.0, 2.0, generator=make).to(TYPES[tag]) for _ in range(2))
    pages, page = 6, 4
    cache = torch.empty((pages, 2, heads, page, depth), device=DEVICE).normal_(0.0, 1.0, generator=make).to(TYPES[cache_tag])
    before = cache.float()
    slots = torch.randint(5, 8, (tokens,), device=DEVICE, generator=make).to(torch.int32)  # three of the 24 slots
    slots[:2] = 5
    note(f"append of {tokens} tokens to three slots {tag} -> {cache_tag} depth {depth}")
    bound = tio.Bound(context(), hc.PagedAppend(pages, page, tio.desc_of(cache).data_type), [tio.desc_of(t) for t in (keys, values, slots)])
    bound.submit([keys, values, slots], [cache])
    torch.cuda.synchronize()
    kept = (torch.stack((keys, values), 1).float().clamp(-448, 448) if cache_tag == "e4m3" else torch.stack((keys, values), 1)).to(TYPES[cache_tag]).float()
    after = cache.float()
    for slot in range(pages * page):
        mine, got = kept[slots == slot], after[slot // page, :, :, slot % page]
        if mine.shape[0] == 0:
            assert torch.equal(got, before[slot // page, :, :, slot % page])
        else:
            assert (mine == got).any(0).all()
