"""The attention of beams where a shared page has the lowest number there is, and where the products of queries and keys are huge."""
import math

import pytest
import torch

from test_gpu_beams import K, _attention, _beams, _near  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 8), (128, 64), (64, 5), (48, 16)])
@pytest.mark.parametrize("bad", [-(1 << 31), -(1 << 31) + 1, (1 << 31) - 1])
def test_shared_pages_of_the_numbers_at_the_ends(K, dim, page, bad):  # noqa: F811
    """A page of zeros in a group's shared keys, whatever the number outside the cache; what the stages held before is no number."""
    heads, kv_heads, beams = 4, 2, 3
    q, cache, table, kv_len, sh = _beams(2, beams, heads, kv_heads, dim, page, [310, 200], [[40, 33, 21], [5, 1, 30]], seed=dim + page)
    zeros = int((set(range(cache.shape[0])) - set(table[table >= 0].tolist())).pop())
    cache[zeros] = 0
    table[:3, 64 // page + 1] = bad
    table[:3, 200 // page] = bad
    table[3:, 0] = bad
    used = torch.arange(table.shape[1], device="cuda")[None] * page < kv_len[:, None]
    want_table = torch.where((table < 0) | (table >= cache.shape[0]), zeros, table)
    want = _attention(q, cache, want_table, kv_len, heads, kv_heads, dim, 0.125, None)
    out = torch.empty_like(q)
    for hints in ((310, 40), (1, 1)):                      # ranges of a tile or two, and one of all tiles
        # CTAs whose stages hold no numbers, then the call
        nan = torch.full_like(cache, math.nan)
        K.attention_decode_beams(q, out, nan, table.clamp(min=0, max=cache.shape[0] - 1), kv_len, sh, beams, heads, kv_heads, dim, 0.125, None, 310, 40)
        K.attention_decode_beams(q, out, cache, torch.where(used, table, 0), kv_len, sh, beams, heads, kv_heads, dim, 0.125, None, *hints)
        _near(out, *want, dim, 360)


@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (16, 2, 128), (8, 8, 48)])
@pytest.mark.parametrize("size", [2.0 ** 4, 2.0 ** 12, 2.0 ** 20, 2.0 ** 26, 2.0 ** 30, -2.0 ** 26])
def test_products_of_any_size(K, heads, kv_heads, dim, size):  # noqa: F811
    """Keys that are multiples of one row of signs and queries that are one too, so that every product is a whole number times `size` and is exact;
    the largest stands `size` * dim * scale >= 16 * 48 / 8 = 96 above the next, whose weight is then below 2^-126: the output is the
    largest key's value, as it is stored."""
    beams, shared, mine = 3, [200, 70], [[10, 4, 7], [30, 31, 1]]
    q, cache, table, kv_len, sh = _beams(2, beams, heads, kv_heads, dim, 16, shared, mine, seed=dim)
    signs = torch.where(torch.arange(dim, device="cuda") % 3 == 0, -1.0, 1.0)
    q[:] = (size * signs).repeat(heads).bfloat16()
    order = torch.randperm(256, generator=torch.Generator(device="cuda").manual_seed(dim), device="cuda").tolist()
    for i in range(2):                                     # a number of its own for every key of the longest row; the shared ones are alike
        for r in range(3 * i, 3 * i + 3):
            for t in range(int(kv_len[r])):
                cache[int(table[r, t // 16]), 0, :, t % 16] = (order[t] * signs).bfloat16()
    table = table.clamp(min=0)
    out = torch.empty_like(q)
    K.attention_decode_beams(q, out, cache, table, kv_len, sh, beams, heads, kv_heads, dim, 0.125, None, 200, 30)
    for r, n in enumerate(kv_len.tolist()):
        t = (max if size > 0 else min)(range(n), key=lambda t: order[t])
        want = cache[int(table[r, t // 16]), 1, :, t % 16].repeat_interleave(heads // kv_heads, 0).reshape(-1)
        assert torch.equal(out[r], want), r
