"""The operators of beam search against their formulas in 64 bits, and the calls they refuse."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from rustinfer_b200.ops import kernels
    return kernels


def _refused(call):
    from rustinfer_b200.ops.library import KernelError
    with pytest.raises(KernelError):
        call()


# ----------------------------------------------------------------------------------------------- the choice
def _best(logits, scores, beams, picks):
    """score, row, token of the best continuations, by numpy in 64 bits; what is no number has score -inf."""
    x = np.asarray(logits, dtype=np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max(1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore"):
        inf = np.isposinf(top)
        weights = np.where(inf, np.isposinf(x), np.exp(x - np.where(np.isfinite(top), top, 0)))
        lp = np.where(inf, np.where(np.isposinf(x), 0.0, -np.inf), x - np.where(np.isfinite(top), top, 0)) - np.log(weights.sum(1, keepdims=True))
        s = np.asarray(scores, dtype=np.float64)[:, None] + lp
    s = np.where(np.isnan(s), -np.inf, s)
    groups, vocab = len(scores) // beams, x.shape[1]
    out = []
    for g in range(groups):
        flat = s[g * beams: (g + 1) * beams].reshape(-1)
        order = np.lexsort((np.arange(flat.size), -flat))[:picks]
        out.append((flat[order], g * beams + order // vocab, order % vocab))
    return [np.stack(c) for c in zip(*out)]


def _select(K, logits, scores, beams, picks):
    groups = scores.numel() // beams
    out = (torch.full((groups, picks), 7.0, device="cuda"), torch.full((groups, picks), -7, dtype=torch.int32, device="cuda"),
           torch.full((groups, picks), -7, dtype=torch.int32, device="cuda"))
    K.beam_select(logits, scores, beams, *out)
    return [t.cpu().numpy() for t in out]


def _agree(got, want, vocab):
    """Rows and tokens are equal.  A score is rounded once (2^-24 of itself); its log-sum is put together from 32-bit
    exponentials: a weight is off by its argument's roundings (2 of 2^-24 of at most 1.45 * 40, since e^-40 of 2^17 weights is
    below 2^-40) and by its own 2 ulp, so the sum and its logarithm are off by no more than 2 * 2^-24 * 58 + 2^-22."""
    np.testing.assert_array_equal(got[1], want[1])
    np.testing.assert_array_equal(got[2], want[2])
    np.testing.assert_array_equal(np.isneginf(got[0]), np.isneginf(want[0]))
    live = ~np.isneginf(want[0])
    assert np.all(np.abs(got[0][live] - want[0][live]) <= 2.0 ** -24 * np.abs(want[0][live]) + 2 * 2.0 ** -24 * 58 + 2.0 ** -22)


@pytest.mark.parametrize("groups,beams,vocab,picks", [
    (1, 1, 1, 1), (1, 1, 2, 2), (3, 2, 3, 6), (2, 4, 7, 28), (1, 64, 5, 128), (1, 1, 257, 128), (2, 3, 1000, 6), (5, 8, 2049, 16), (2, 1, 4096, 64),
    (1, 4, 128256, 8), (3, 5, 50021, 15), (40, 8, 32000, 16), (2, 64, 9001, 128), (148, 2, 16385, 4)])
def test_choice(K, groups, beams, vocab, picks):
    g = torch.Generator(device="cuda").manual_seed(vocab + beams)
    logits = 3 * torch.randn((groups * beams, vocab), generator=g, device="cuda")
    scores = -10 * torch.rand(groups * beams, generator=g, device="cuda")
    _agree(_select(K, logits, scores, beams, picks), _best(logits.cpu().numpy(), scores.cpu().numpy(), beams, picks), vocab)


@pytest.mark.parametrize("vocab", [5, 300, 5000, 40000])
@pytest.mark.parametrize("kind", ["equal", "few values", "equal rows", "zeros of both signs", "one allowed", "a few allowed", "none allowed", "dead rows",
                                  "dead and equal", "no numbers", "wide"])
def test_choice_among_equals_and_masks(K, kind, vocab):
    beams, groups = 4, 3
    picks = min(12, vocab * beams)
    g = torch.Generator(device="cuda").manual_seed(vocab)
    logits = torch.randn((groups * beams, vocab), generator=g, device="cuda")
    scores = -torch.rand(groups * beams, generator=g, device="cuda")
    if kind == "equal":
        logits.fill_(1.25)
        scores.fill_(-3.0)
    elif kind == "few values":
        logits = torch.round(logits)
    elif kind == "equal rows":                             # the beams of a request that has not branched yet
        logits = logits[::beams].repeat_interleave(beams, 0).contiguous()
        scores.fill_(-1.0)
    elif kind == "zeros of both signs":
        logits = torch.where(torch.rand(logits.shape, generator=g, device="cuda") < 0.5, 0.0, -0.0)
        scores.zero_()
    elif kind == "one allowed":
        keep = torch.randint(0, vocab, (groups * beams, 1), generator=g, device="cuda")
        logits = torch.full_like(logits, -math.inf).scatter(1, keep, logits.gather(1, keep))
    elif kind == "a few allowed":
        logits.masked_fill_(torch.rand(logits.shape, generator=g, device="cuda") > 7 / vocab, -math.inf)
    elif kind == "none allowed":
        logits[::2] = -math.inf
    elif kind == "dead rows":
        scores[1::4] = -math.inf
        scores[2::4] = math.nan
    elif kind == "dead and equal":
        scores.fill_(-math.inf)
    elif kind == "no numbers":
        logits.masked_fill_(torch.rand(logits.shape, generator=g, device="cuda") < 0.5, math.nan)
        logits[1] = math.nan
    elif kind == "wide":                                   # a row of one certain word, and one whose logits are huge
        logits[0, vocab // 2] = 200.0
        logits[1] *= 1e30
    _agree(_select(K, logits, scores, beams, picks), _best(logits.cpu().numpy(), scores.cpu().numpy(), beams, picks), vocab)


@pytest.mark.parametrize("kind", ["random", "equal", "two values", "one group of equals", "mostly forbidden", "large"])
def test_choice_from_long_slices(K, kind):
    """So many rows that a slice is a whole row of thirteen chunks; the rows start at every offset from a 16-byte boundary."""
    beams, groups, vocab, picks = 4, 50, 50021, 24
    g = torch.Generator(device="cuda").manual_seed(len(kind))
    logits = torch.randn((groups * beams, vocab), generator=g, device="cuda")
    scores = -5 * torch.rand(groups * beams, generator=g, device="cuda")
    if kind == "equal":
        logits.fill_(-2.5)
    elif kind == "two values":                             # half of all words reach any threshold
        logits = torch.where(logits > 0, 1.0, 0.0)
    elif kind == "one group of equals":
        logits[8:12] = 0.5
        scores[8:12] = -1.0
    elif kind == "mostly forbidden":
        logits.masked_fill_(torch.rand(logits.shape, generator=g, device="cuda") > 20 / vocab, -math.inf)
        logits[5] = -math.inf
    elif kind == "large":                                  # weights by differences
        logits[::3] *= 1e6
    _agree(_select(K, logits, scores, beams, picks), _best(logits.cpu().numpy(), scores.cpu().numpy(), beams, picks), vocab)


def test_choice_with_infinite_logits(K):
    logits = torch.randn((2, 9000), device="cuda")
    logits[0, [17, 8000]] = math.inf
    got = _select(K, logits, torch.tensor([-1.0, -50.0], device="cuda"), 2, 4)
    assert got[1][0, :2].tolist() == [0, 0] and got[2][0, :2].tolist() == [17, 8000]
    assert np.allclose(got[0][0, :2], -1.0 - math.log(2), rtol=2 ** -23) and got[1][0, 2:].tolist() == [1, 1]


@pytest.mark.parametrize("offset,ld", [(0, 5003), (1, 5003), (3, 5008), (2, 6001)])
def test_choice_from_rows_off_their_boundaries(K, offset, ld):
    rows, vocab = 6, 5001
    flat = torch.randn(rows * ld + 8, device="cuda")
    logits = flat[offset: offset + rows * ld].view(rows, ld)[:, :vocab]
    scores = -torch.rand(rows, device="cuda")
    _agree(_select(K, logits, scores, 3, 9), _best(logits.cpu().numpy(), scores.cpu().numpy(), 3, 9), vocab)


def test_choice_from_rows_that_lie_beyond_32_bits(K):
    """Rows more than 2^31 elements apart."""
    rows, vocab, ld = 2, 9001, (1 << 31) + 6
    flat = torch.empty(ld + vocab, device="cuda")
    logits = flat.as_strided((rows, vocab), (ld, 1))
    logits.copy_(torch.randn((rows, vocab), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda"))
    scores = torch.tensor([-1.0, -1.5], device="cuda")
    _agree(_select(K, logits, scores, 2, 20), _best(logits.cpu().numpy(), scores.cpu().numpy(), 2, 20), vocab)


def test_choice_refuses(K):
    x, s = torch.randn((4, 50), device="cuda"), torch.zeros(4, device="cuda")

    def out(g, p):
        return torch.empty((g, p), device="cuda"), torch.empty((g, p), dtype=torch.int32, device="cuda"), torch.empty((g, p), dtype=torch.int32, device="cuda")
    _refused(lambda: K.beam_select(x.bfloat16(), s, 2, *out(2, 4)))
    _refused(lambda: K.beam_select(x, s, 3, *out(1, 4)))
    _refused(lambda: K.beam_select(x, s, 0, *out(1, 4)))
    _refused(lambda: K.beam_select(x, s[:3], 2, *out(2, 4)))
    _refused(lambda: K.beam_select(x, s, 2, *out(2, 101)))
    _refused(lambda: K.beam_select(x, s, 4, *out(1, 129)))
    _refused(lambda: K.beam_select(x, s, 2, *out(1, 4)))
    _refused(lambda: K.beam_select(x.t(), torch.zeros(50, device="cuda"), 2, *out(25, 2)))
    _refused(lambda: K.beam_select(x.cpu(), s.cpu(), 2, *(t.cpu() for t in out(2, 4))))
    o = out(2, 4)
    _refused(lambda: K.beam_select(x, s, 2, o[0], o[1].long(), o[2]))
    K.beam_select(x[:0], s[:0], 2, *out(0, 4))            # no rows: nothing to do


# -------------------------------------------------------------------------------------- rows that move
def _filled(shape, dtype, g):
    if dtype in (torch.int32, torch.uint8):
        return torch.randint(0, 250, shape, generator=g, device="cuda").to(dtype)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _moved(store, rows, parents, used=None):
    want = store.clone()
    for r, p in enumerate(parents):
        a, b = rows[p], rows[r]
        if used is None:
            want[:, b] = store[:, a]
        else:
            want[:, b, :, :, : used[r]] = store[:, a, :, :, : used[r]]
    return want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.int32, torch.uint8])
@pytest.mark.parametrize("layers,total,tail,groups,beams", [
    (1, 1, (1,), 1, 1), (1, 9, (1,), 2, 4), (3, 20, (5,), 4, 5), (2, 70, (3, 2048), 1, 64), (5, 40, (16, 33, 8), 6, 6), (2, 130, (257,), 2, 64)])
@pytest.mark.parametrize("how", ["stay", "survivors", "any", "rotate", "one parent"])
def test_rows_take_over(K, layers, total, tail, groups, beams, dtype, how):
    g = torch.Generator(device="cuda").manual_seed(total + beams)
    store = _filled((layers, total) + tail, dtype, g)
    rows = torch.randperm(total, generator=g, device="cuda")[: groups * beams].to(torch.int32)
    rng = np.random.default_rng(beams)
    parents = np.arange(beams)
    if how == "survivors" and beams > 1:
        stays = rng.permutation(beams)[: beams // 2 + 1]
        parents = np.where(np.isin(parents, stays), parents, rng.choice(stays, beams))
    elif how == "any":
        parents = rng.integers(0, beams, beams)
    elif how == "rotate":                                  # one cycle through all, or several
        parents = np.roll(parents, 1) if beams < 6 else np.concatenate([np.roll(c, 1) for c in np.array_split(parents, 3)])
    elif how == "one parent":
        parents = np.full(beams, beams - 1)
    every = np.concatenate([parents + i * beams for i in range(groups)])
    want = _moved(store, rows.tolist(), every.tolist())
    K.reorder_rows(store, rows, torch.tensor(every, dtype=torch.int32, device="cuda"), beams)
    assert torch.equal(store, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kv_heads,page,dim", [(1, 8, 8), (2, 16, 64), (3, 5, 9), (8, 64, 128)])
@pytest.mark.parametrize("how", ["survivors", "any"])
def test_pages_take_over_the_tokens_in_use(K, kv_heads, page, dim, dtype, how):
    groups, beams, total = 3, 7, 40
    g = torch.Generator(device="cuda").manual_seed(page)
    store = _filled((4, total, 2, kv_heads, page, dim), dtype, g)
    rows = torch.randperm(total, generator=g, device="cuda")[: groups * beams].to(torch.int32)
    rng = np.random.default_rng(page)
    every = []
    for i in range(groups):
        stays = rng.permutation(beams)[:3]
        p = np.where(np.isin(np.arange(beams), stays), np.arange(beams), rng.choice(stays, beams)) if how == "survivors" else rng.integers(0, beams, beams)
        every += (p + i * beams).tolist()
    used = rng.integers(0, page + 1, groups * beams).tolist()
    if how == "any":                                       # rows that are read and taken over: as far as every row is in use
        used = [int(used[r // beams * beams]) for r in range(groups * beams)]
    want = _moved(store, rows.tolist(), every, used)
    K.reorder_rows(store, rows, torch.tensor(every, dtype=torch.int32, device="cuda"), beams, torch.tensor(used, dtype=torch.int32, device="cuda"))
    assert torch.equal(store, want)


def test_rows_that_do_not_exist_leave_everything_as_it_was(K):
    store = torch.randn((2, 6, 10), device="cuda")
    was = store.clone()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    K.reorder_rows(store, i32([0, 1, 2, 3]), i32([0, 5, -1, 99]), 4)        # parents outside the group
    K.reorder_rows(store, i32([0, 1, 2, 3]), i32([2, 1, 2, 3]), 2)          # row 0's is of the other group
    K.reorder_rows(store, i32([0, 6, -3, 70]), i32([2, 0, 0, 0]), 4)        # rows outside the storage
    K.copy_pages(store, i32([0, 6, -1, 3]), i32([6, 1, 2, 3]))
    K.copy_pages(store, i32([]), i32([]))
    K.reorder_rows(store, i32([]), i32([]), 4)
    assert torch.equal(store, was)


def test_storage_beyond_32_bits(K):
    """Rows that start past 2^32 bytes and 2^31 elements."""
    store = torch.zeros((3, 5, 300 << 20), dtype=torch.uint8, device="cuda")
    store[2, 4, -1000:] = 3
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    K.reorder_rows(store, i32([0, 4]), i32([1, 1]), 2)
    K.copy_pages(store, i32([4]), i32([3]))
    for r in (0, 3, 4):
        assert int(store[2, r, -1000:].sum()) == 3000
    assert int(store[2, 1].max()) == 0 and int(store[1].max()) == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.uint8])
@pytest.mark.parametrize("tail,used", [((1,), None), ((7, 3), None), ((2, 2, 16, 64), None), ((2, 2, 16, 64), "some"), ((2, 3, 5, 9), "some"),
                                       ((2, 8, 64, 128), "some")])
def test_pages_are_copied(K, tail, used, dtype):
    g = torch.Generator(device="cuda").manual_seed(len(tail))
    store = _filled((3, 50) + tail, dtype, g)
    order = torch.randperm(50, generator=g, device="cuda").to(torch.int32)
    src, dst = torch.cat([order[:10], order[:1].repeat(8)]), order[20: 38].contiguous()
    page = tail[2] if used else 0
    n_used = torch.randint(0, page + 1, (18,), generator=g, device="cuda", dtype=torch.int32) if used else None
    want = store.clone()
    for i, (a, b) in enumerate(zip(src.tolist(), dst.tolist())):
        if used:
            want[:, b, :, :, : int(n_used[i])] = store[:, a, :, :, : int(n_used[i])]
        else:
            want[:, b] = store[:, a]
    K.copy_pages(store, src, dst, n_used)
    assert torch.equal(store, want)


def test_moves_refuse(K):
    store = torch.randn((2, 6, 2, 1, 4, 8), device="cuda")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    _refused(lambda: K.reorder_rows(store, i32([0, 1, 2]), i32([0, 1, 2]), 2))
    _refused(lambda: K.reorder_rows(store, i32([0, 1]), i32([0, 1, 2]), 2))
    _refused(lambda: K.reorder_rows(store, i32([0] * 65), i32([0] * 65), 65))
    _refused(lambda: K.reorder_rows(store, i32([0, 1]).long(), i32([0, 1]), 2))
    _refused(lambda: K.reorder_rows(store[:, :3], i32([0, 1]), i32([0, 1]), 2))
    _refused(lambda: K.reorder_rows(store, i32([0, 1]), i32([0, 1]), 2, i32([1])))
    _refused(lambda: K.reorder_rows(store[..., 0].contiguous(), i32([0, 1]), i32([0, 1]), 2, i32([1, 1])))
    _refused(lambda: K.reorder_rows(store, i32([0, 1]).cpu(), i32([0, 1]), 2))
    _refused(lambda: K.copy_pages(store, i32([0, 1]), i32([2])))
    _refused(lambda: K.copy_pages(store, i32([0]), i32([2]).long()))
    _refused(lambda: K.copy_pages(store[0, 0, 0, 0, 0], i32([0]), i32([1])))
    _refused(lambda: K.copy_pages(store, i32([0]), i32([1]), i32([1, 2])))


# ------------------------------------------------------------------------------------- attention of beams
def _beams(groups, beams, heads, kv_heads, dim, page, shared, mine, seed=0, spread=0):
    """q, cache, block table, lengths and shared lengths; pages in no order, the shared part in pages of its own per beam where it ends inside one."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    count = sum(a // page + beams * (-(-(a + max(b)) // page) - a // page + 1) for a, b in zip(shared, mine))
    order = rng.permutation(count + 3)[:count].tolist()
    cache = torch.randn((count + 3, 2, kv_heads, page, dim), generator=g, device="cuda").to(torch.bfloat16)
    table, kv_len, at = [], [], 0
    blocks = max(-(-(a + max(b)) // page) for a, b in zip(shared, mine)) + spread
    for a, bs in zip(shared, mine):
        common = order[at: at + a // page]
        at += a // page
        first = None
        for b in bs:
            need = -(-(a + b) // page) - a // page
            private = order[at: at + need]
            at += need
            if a % page and need:
                if first is None:
                    first = private[0]
                else:
                    cache[private[0], :, :, : a % page] = cache[first, :, :, : a % page]
            row = common + private
            table.append(row + [-1] * (blocks - len(row)))
            kv_len.append(a + b)
    q = torch.randn((groups * beams, heads * dim), generator=g, device="cuda").to(torch.bfloat16)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return q, cache, i32(table), i32(kv_len), i32(shared)


def _attention(q, cache, table, kv_len, heads, kv_heads, dim, scale, window):
    page, rows = cache.shape[3], []
    bound = []
    for r, n in enumerate(kv_len.tolist()):
        first = max(0, n - window) if window else 0
        if n <= 0:
            rows.append(torch.zeros(heads * dim, dtype=torch.float64, device="cuda"))
            bound.append(torch.zeros(heads * dim, dtype=torch.float64, device="cuda"))
            continue
        at = torch.arange(first, n, device="cuda")
        kv = cache[table[r].long()[at // page], :, :, at % page].double()
        qq = q[r].double().view(kv_heads, heads // kv_heads, dim)
        p = torch.softmax(torch.einsum("kgd,tkd->kgt", qq, kv[:, 0]) * scale, -1)
        rows.append(torch.einsum("kgt,tkd->kgd", p, kv[:, 1]).reshape(-1))
        bound.append(torch.einsum("kgt,tkd->kgd", p, kv[:, 1].abs()).reshape(-1))
    return torch.stack(rows), torch.stack(bound)


def _near(got, want, weighted, dim, keys):
    """The stored output is rounded once (2^-8 of itself).  In front of that: a weight is off by its two pieces' 2^-16 and by its
    score's: a sum of `dim` products in 32 bits, |scale q . k| <= 40 here, off by dim * 2^-23 * 40 at the very worst; sums of
    `keys` terms add keys * 2^-23.  All of these act on the sum of |weight value|."""
    off = (got.double() - want).abs()
    assert torch.all(off <= 2.0 ** -8 * want.abs() + weighted * (2.0 ** -16 + (40 * dim + keys) * 2.0 ** -23))


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 8, 64), (32, 8, 64), (32, 8, 128), (5, 1, 64), (16, 1, 48), (40, 2, 128), (6, 2, 96), (8, 4, 16),
                                                (4, 2, 256)])
@pytest.mark.parametrize("beams", [1, 3, 4, 16])
def test_attention_of_beams(K, heads, kv_heads, dim, beams):
    shared, mine = [300, 1, 129, 64], [[1 + (7 * i + j) % 40 for j in range(beams)] for i in range(4)]
    q, cache, table, kv_len, sh = _beams(4, beams, heads, kv_heads, dim, 16, shared, mine, seed=dim + beams)
    out = torch.full_like(q, 9.0)
    K.attention_decode_beams(q, out, cache, table.clamp(min=0), kv_len, sh, beams, heads, kv_heads, dim, dim ** -0.5, None, 300, 40)
    _near(out, *_attention(q, cache, table, kv_len, heads, kv_heads, dim, dim ** -0.5, None), dim, 400)


@pytest.mark.parametrize("page", [1, 5, 8, 16, 32, 64, 128])
@pytest.mark.parametrize("shared,own", [(0, 1), (1, 1), (15, 2), (16, 1), (17, 63), (64, 64), (2000, 1), (513, 200), (128, 500)])
def test_attention_of_beams_lengths(K, page, shared, own):
    beams, heads, kv_heads, dim = 4, 8, 2, 64
    q, cache, table, kv_len, sh = _beams(2, beams, heads, kv_heads, dim, page, [shared, max(0, shared - 3)], [[own] * beams, [own + 2] * beams], seed=page)
    out = torch.empty_like(q)
    K.attention_decode_beams(q, out, cache, table.clamp(min=0), kv_len, sh, beams, heads, kv_heads, dim, 0.2, None, shared, own)
    _near(out, *_attention(q, cache, table, kv_len, heads, kv_heads, dim, 0.2, None), dim, shared + own + 2)


@pytest.mark.parametrize("window", [1, 7, 16, 100, 300, 5000])
@pytest.mark.parametrize("even", [True, False])
def test_attention_of_beams_with_a_window(K, window, even):
    """Rows of equal lengths share what the window leaves; pages behind it are given back and hold anything, no numbers too."""
    beams, heads, kv_heads, dim, page = 5, 8, 4, 64, 16
    mine = [[20] * beams, [1] * beams] if even else [[1 + j for j in range(beams)], [40 - j for j in range(beams)]]
    q, cache, table, kv_len, sh = _beams(2, beams, heads, kv_heads, dim, page, [250, 131], mine, seed=window)
    want = _attention(q, cache, table, kv_len, heads, kv_heads, dim, 0.125, window)
    for r, n in enumerate(kv_len.tolist()):                # pages that no key of the row's window lies in, if nobody else sees them
        for b in range(table.shape[1]):
            seen = [max(0, m - window) < (b + 1) * page for m in kv_len.tolist()]
            if not any(s and int(table[i, b]) == int(table[r, b]) for i, s in enumerate(seen)) and int(table[r, b]) >= 0:
                cache[int(table[r, b])] = math.nan
    out = torch.empty_like(q)
    K.attention_decode_beams(q, out, cache, table.clamp(min=0), kv_len, sh, beams, heads, kv_heads, dim, 0.125, window, 250, 40)
    _near(out, *want, dim, 300)


def test_attention_of_beams_reads_nothing_behind_a_rows_end(K):
    """Keys and values behind the last one are no numbers; rows shorter than what their group is said to share; rows of no keys."""
    beams, heads, kv_heads, dim, page = 4, 4, 2, 64, 16
    shared = [100, 40, 20]
    mine = [[-30, 0, 5, 11], [1, 1, 1, 1], [-20, 0, -19, 3]]
    q, cache, table, kv_len, sh = _beams(3, beams, heads, kv_heads, dim, page, shared, [[max(0, b) for b in m] for m in mine], seed=3, spread=2)
    kv_len = torch.tensor([a + b for a, m in zip(shared, mine) for b in m], dtype=torch.int32, device="cuda")
    want = _attention(q, cache, table, kv_len, heads, kv_heads, dim, 0.125, None)
    longest = {}
    for r, n in enumerate(kv_len.tolist()):
        for b, p in enumerate(table[r].tolist()):
            if p >= 0:
                longest[p] = max(longest.get(p, 0), min(page, max(0, n - b * page)))
    for p, used in longest.items():
        cache[p, :, :, used:] = math.nan
    spare = [p for p in range(cache.shape[0]) if p not in longest]
    cache[spare] = math.nan
    table = torch.where(table < 0, spare[0], table)
    out = torch.full_like(q, 5.0)
    K.attention_decode_beams(q, out, cache, table, kv_len, sh, beams, heads, kv_heads, dim, 0.125, None, 100, 11)
    _near(out, *want, dim, 120)
    assert int(kv_len[8]) == 0 and torch.all(out[8] == 0)


@pytest.mark.parametrize("dim", [64, 48])
def test_attention_of_beams_over_a_cache_beyond_32_bits(K, dim):
    """Pages that start past 2^31 elements and 2^32 bytes."""
    heads, kv_heads, beams, page, count = 8, 8, 2, 16, (1 << 31) // (2 * 8 * 16 * dim) + 60
    q, small, table, kv_len, sh = _beams(1, beams, heads, kv_heads, dim, page, [200], [[9, 30]], seed=2)
    cache = torch.empty((count, 2, kv_heads, page, dim), dtype=torch.bfloat16, device="cuda")
    cache[count - small.shape[0]:] = small
    table = torch.where(table < 0, table, table + count - small.shape[0])
    out = torch.empty_like(q)
    K.attention_decode_beams(q, out, cache, table.clamp(min=0), kv_len, sh, beams, heads, kv_heads, dim, 0.125, None, 200, 30)
    _near(out, *_attention(q, cache, table, kv_len, heads, kv_heads, dim, 0.125, None), dim, 230)


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 8), (64, 5), (48, 16)])
def test_attention_of_beams_with_pages_that_do_not_exist(K, dim, page):
    """Numbers outside the cache, in the shared part and in a row's own: pages of zeros."""
    heads, kv_heads, beams = 4, 2, 3
    q, cache, table, kv_len, sh = _beams(2, beams, heads, kv_heads, dim, page, [150, 70], [[40, 33, 21], [5, 1, 30]], seed=dim)
    zeros = int((set(range(cache.shape[0])) - set(table[table >= 0].tolist())).pop())
    cache[zeros] = 0
    for r, b, bad in ((0, 2, -1), (0, 3, 1 << 30), (1, 150 // page + 1, cache.shape[0]), (4, 1, -7), (5, 70 // page + 1, -(1 << 31))):
        if r in (0, 4):                                    # shared blocks: the whole group's
            rows = range(0, 3) if r == 0 else range(3, 6)
            for i in rows:
                table[i, b] = bad
        else:
            table[r, b] = bad
    used = torch.arange(table.shape[1], device="cuda")[None] * page < kv_len[:, None]
    want_table = torch.where((table < 0) | (table >= cache.shape[0]), zeros, table)
    out = torch.empty_like(q)
    K.attention_decode_beams(q, out, cache, torch.where(used, table, 0), kv_len, sh, beams, heads, kv_heads, dim, 0.125, None, 150, 40)
    _near(out, *_attention(q, cache, want_table, kv_len, heads, kv_heads, dim, 0.125, None), dim, 200)


def test_attention_of_beams_passes_on_what_is_no_number(K):
    q, cache, table, kv_len, sh = _beams(2, 2, 4, 2, 64, 16, [90, 90], [[9, 9], [9, 9]], seed=1)
    cache[int(table[0, 2]), 1, 0, 3, 5] = math.nan         # a shared value of the first group, key head 0
    out = torch.empty_like(q)
    K.attention_decode_beams(q, out, cache, table.clamp(min=0), kv_len, sh, 2, 4, 2, 64, 0.125, None, 90, 9)
    o = out.view(4, 4, 64)
    assert torch.all(o[:2, :2, 5].isnan()) and not o[:2, 2:].isnan().any() and not o[2:].isnan().any()
    cache[int(table[3, 5]), 0, 1, 12, 0] = math.nan        # a key of the last row's own, key head 1
    K.attention_decode_beams(q, out, cache, table.clamp(min=0), kv_len, sh, 2, 4, 2, 64, 0.125, None, 90, 9)
    assert out.view(4, 4, 64)[3, 2:].isnan().all() and not out.view(4, 4, 64)[2].isnan().any()


def test_attention_of_beams_strides_scratch_and_hints(K):
    """Rows of q and out inside wider ones, a table with more rows and columns, scratch of the caller's; the hints change how, not what."""
    heads, kv_heads, dim, beams = 8, 2, 64, 3
    q, cache, table, kv_len, sh = _beams(2, beams, heads, kv_heads, dim, 16, [700, 333], [[30] * 3, [2] * 3], seed=5)
    wide = torch.zeros((6, heads * dim + 24), dtype=torch.bfloat16, device="cuda")
    wide[:, 8: 8 + heads * dim] = q
    out = torch.full((6, heads * dim + 10), 3.0, dtype=torch.bfloat16, device="cuda")
    table = torch.nn.functional.pad(table.clamp(min=0), (0, 5, 0, 2))
    want = _attention(q, cache, table, kv_len, heads, kv_heads, dim, 0.125, None)
    for hints in ((700, 30), (0, 1), (100000, 100000)):
        splits = K.attention_beams_splits(*hints)
        a, b = K.decode_scratch_floats(6, heads, dim, sum(splits) + 1)
        K.attention_decode_beams(wide[:, 8: 8 + heads * dim], out[:, 1: 1 + heads * dim], cache, table, kv_len, sh, beams, heads, kv_heads, dim, 0.125,
                                 None, *hints, torch.empty(a, device="cuda"), torch.empty(b, device="cuda"))
        _near(out[:, 1: 1 + heads * dim], *want, dim, 730)
        assert torch.all(out[:, 0] == 3) and torch.all(out[:, 1 + heads * dim:] == 3)


def test_attention_of_beams_refuses(K):
    q, cache, table, kv_len, sh = _beams(2, 2, 4, 2, 64, 16, [20, 20], [[3, 3], [3, 3]])
    table = table.clamp(min=0)

    def call(**kw):
        a = dict(q=q, out=torch.empty_like(q), cache=cache, block_table=table, kv_len=kv_len, shared_len=sh, beams=2, num_heads=4, num_kv_heads=2,
                 head_dim=64, scale=0.1, window=None, most_shared=20, most_own=3)
        a.update(kw)
        return lambda: K.attention_decode_beams(**a)
    call()()
    for kw in (dict(q=q.float()), dict(beams=3), dict(beams=65), dict(beams=0), dict(num_heads=3), dict(head_dim=24), dict(head_dim=272), dict(window=0), dict(scale=0.0), dict(scale=math.nan),
               dict(cache=cache.float()), dict(cache=cache[:, :, :1]), dict(kv_len=kv_len.long()), dict(kv_len=kv_len[:3]), dict(shared_len=sh[:1]),
               dict(block_table=table[:3]), dict(block_table=table.long()), dict(out=torch.empty((4, 255), dtype=torch.bfloat16, device="cuda")),
               dict(q=torch.zeros((4, 264), dtype=torch.bfloat16, device="cuda")[:, 1: 257]), dict(q=q.cpu()),
               dict(part_o=torch.empty(3, device="cuda"), part_lse=torch.empty(3, device="cuda"))):
        _refused(call(**kw))
    K.attention_decode_beams(q[:0], q[:0].clone(), cache, table[:0], kv_len[:0], sh[:0], 2, 4, 2, 64, 0.1, None, 1, 1)


def test_tensors_of_another_device_are_refused(K, monkeypatch):
    """As if the current device were another one than the tensors'."""
    from rustinfer_b200.ops import library
    q, cache, table, kv_len, sh = _beams(1, 2, 4, 2, 64, 16, [20], [[3, 3]])
    i32 = torch.zeros(2, dtype=torch.int32, device="cuda")
    x = torch.randn((2, 40), device="cuda")
    monkeypatch.setattr(library, "_current_device", lambda: 1)
    _refused(lambda: K.beam_select(x, x[:, 0].contiguous(), 2, x[:1, :2].contiguous(), i32[None], i32[None]))
    _refused(lambda: K.reorder_rows(x[None], i32, i32, 2))
    _refused(lambda: K.copy_pages(x[None], i32, i32))
    _refused(lambda: K.attention_decode_beams(q, q.clone(), cache, table.clamp(min=0), kv_len, sh, 2, 4, 2, 64, 0.1, None, 20, 3))


# ------------------------------------------------------------------------------------- together, and elsewhere than on the default stream
def test_a_step_of_beams_captured_and_on_two_streams(K):
    """Choice, reorder and attention in one graph beside the same on another stream: each has its own scratch."""
    beams, groups, heads, kv_heads, dim, vocab = 4, 2, 8, 2, 64, 9001
    q, cache, table, kv_len, sh = _beams(groups, beams, heads, kv_heads, dim, 16, [200, 77], [[10] * 4, [3] * 4], seed=8)
    table = table.clamp(min=0)
    logits, scores = torch.randn((8, vocab), device="cuda"), -torch.rand(8, device="cuda")
    state = torch.randn((3, 10, 40), device="cuda")
    rows = torch.tensor([1, 3, 5, 7, 0, 2, 4, 6], dtype=torch.int32, device="cuda")
    best = [torch.empty((groups, beams), device="cuda")] + [torch.empty((groups, beams), dtype=torch.int32, device="cuda") for _ in range(2)]

    def step(best, state, out):
        K.beam_select(logits, scores, beams, *best)
        K.reorder_rows(state, rows, best[1].view(-1), beams)
        K.attention_decode_beams(q, out, cache, table, kv_len, sh, beams, heads, kv_heads, dim, 0.125, None, 200, 10)

    was, out = state.clone(), torch.empty_like(q)
    step(best, state, out)
    want = [t.clone() for t in (*best, state, out)]
    picked = best[1].cpu().numpy().reshape(-1).tolist()
    assert torch.equal(state, _moved(was, rows.tolist(), picked))
    graphs = []
    for _ in range(2):
        mine = [[t.clone() for t in best], was.clone(), torch.empty_like(q)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(*mine)
        graphs.append((graph, mine))
    side, eager = torch.cuda.Stream(), [[t.clone() for t in best], was.clone(), torch.empty_like(q)]
    side.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    for graph, _ in graphs:
        graph.replay()
    with torch.cuda.stream(side):
        step(*eager)
    torch.cuda.synchronize()
    for mine in [m for _, m in graphs] + [eager]:
        for a, b in zip((*mine[0], mine[1], mine[2]), want):
            assert torch.equal(a, b)
    logits.copy_(torch.randn((8, vocab), device="cuda"))   # a replay reads what the buffers hold by then
    graphs[0][1][1].copy_(was)
    graphs[0][0].replay()
    got = [t.cpu().numpy() for t in graphs[0][1][0]]
    _agree(got, _best(logits.cpu().numpy(), scores.cpu().numpy(), beams, beams), vocab)
