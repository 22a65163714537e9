"""The operators of beam search, as a program that keeps several continuations of a prompt calls them.

A case names an `op` and its sizes:

    select      the best continuations of every request over its beams and the vocabulary: running scores plus log-softmax
    reorder     every beam takes over what its parent's row holds, in place: state slots, or the pages that are partly filled
    pages       pages copied to others in every layer of a cache: a request that is forked, a pool that is compacted
    attention   a step of single tokens whose beams share the keys of their prompt and have some of their own

`run` computes a case from elementary torch operations, or with `own` through the framework's kernels.  Sizes are those of
the configurations that `bench.py` runs (heads of 64 and 128, 8 key heads, pages of 16, a vocabulary of 128,256) or generic.
"""
from __future__ import annotations

import math

import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "int32": torch.int32}


def listed():
    return [
        # one request of four beams, a step: latency decides
        dict(name="select one request", op="select", groups=1, beams=4, vocab=128256, picks=8, masked=0.0, dead=0),
        # a batch of requests with eight beams each; an odd vocabulary, rows off their 16-byte boundaries, words forbidden
        dict(name="select odd vocabulary", op="select", groups=16, beams=8, vocab=50021, picks=16, masked=0.1, dead=1),
        # many requests with wide beams and several stop words: the logits' stream decides
        dict(name="select wide beams", op="select", groups=32, beams=16, vocab=128256, picks=48, masked=0.0, dead=0),
        # convolution inputs of a small model: a few rows of a few kilobytes
        dict(name="states one request", op="reorder", what="states", dtype="bfloat16", layers=8, slots=33, elems=3 * 2048, groups=1,
             beams=4, moved=2),
        # recurrent states of a batch: 16 heads of 64 x 128 in 32-bit, 12 layers
        dict(name="states eight requests", op="reorder", what="states", dtype="float32", layers=12, slots=65, elems=16 * 64 * 128,
             groups=8, beams=8, moved=3),
        # the last pages of 64 beams, 16 layers of the 1B sizes, eleven tokens of sixteen in use
        dict(name="last pages eight requests", op="reorder", what="pages", dtype="bfloat16", layers=16, pages=700, kv_heads=8, page=16,
             dim=64, tokens=11, groups=8, beams=8, moved=4),
        # a prompt that continues in sixteen ways: its last page, fifteen copies
        dict(name="pages of a fork", op="pages", dtype="bfloat16", layers=16, pages=300, kv_heads=8, page=16, dim=64, copies=15, tokens=5),
        # a pool that is compacted: a thousand whole pages of the 8B sizes, 8 layers
        dict(name="pages compacted", op="pages", dtype="bfloat16", layers=8, pages=3000, kv_heads=8, page=16, dim=128, copies=1000, tokens=16),
        # one request of four beams behind a short prompt
        dict(name="attention one request", op="attention", groups=1, beams=4, heads=32, kv_heads=8, dim=64, page=16, shared=500, own=21,
             window=0, ragged=False),
        # the headline's context with eight beams a request, 1B sizes
        dict(name="attention eight requests", op="attention", groups=8, beams=8, heads=32, kv_heads=8, dim=64, page=16, shared=4096, own=60,
             window=0, ragged=False),
        # long prompts of different lengths, sixteen beams, 8B sizes
        dict(name="attention long prompts", op="attention", groups=4, beams=16, heads=32, kv_heads=8, dim=128, page=16, shared=9001, own=300,
             window=0, ragged=True),
        # a layer with a window, three beams, odd lengths
        dict(name="attention window", op="attention", groups=5, beams=3, heads=40, kv_heads=8, dim=128, page=16, shared=2777, own=45,
             window=1024, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["select", "select", "reorder", "reorder", "pages", "attention", "attention", "attention"])
    beams = rng.choice([1, 2, 3, 4, 5, 6, 8, 10, 12, 16])
    if op == "select":
        vocab = rng.choice([128256, _log(rng, 1000, 128256), _log(rng, 1000, 128256)])
        groups = _log(rng, 1, max(1, min(128, 512 * 128256 // (vocab * beams))))
        return dict(op=op, groups=groups, beams=beams, vocab=vocab, picks=beams * rng.choice([1, 2, 2, 3]),
                    masked=rng.choice([0.0, 0.0, rng.random()]), dead=rng.choice([0, 0, rng.randrange(beams)]))
    if op == "reorder":
        groups = _log(rng, 1, 64 // beams) if beams < 64 else 1
        moved = rng.randrange(beams)
        if rng.random() < 0.5:
            layers, dtype = _log(rng, 1, 24), rng.choice(["float32", "float32", "bfloat16", "int32"])
            elems = _log(rng, 1, min(1 << 18, (400 << 18) // (layers * (groups * beams + 1))))
            return dict(op=op, what="states", dtype=dtype, layers=layers, slots=groups * beams + rng.randint(1, 9), elems=elems, groups=groups,
                        beams=beams, moved=moved)
        page = rng.choice([8, 16, 16, 32, 64])
        return dict(op=op, what="pages", dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), layers=rng.randint(1, 16),
                    pages=groups * beams + _log(rng, 1, 300), kv_heads=rng.choice([1, 2, 4, 8]), page=page, dim=rng.choice([24, 64, 64, 128]),
                    tokens=rng.randint(1, page), groups=groups, beams=beams, moved=moved)
    if op == "pages":
        page, layers = rng.choice([8, 16, 16, 32, 64]), rng.randint(1, 16)
        kv_heads, dim = rng.choice([1, 2, 4, 8]), rng.choice([24, 64, 64, 128])
        copies = _log(rng, 1, max(1, min(1000, (250 << 20) // (layers * 4 * kv_heads * page * dim))))
        return dict(op=op, dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), layers=layers, pages=2 * copies + rng.randint(0, 50),
                    kv_heads=kv_heads, page=page, dim=dim, copies=copies, tokens=rng.choice([page, rng.randint(1, page)]))
    heads, kv_heads, dim = rng.choice([(32, 8, 64), (32, 8, 128), (40, 8, 128), (8, 8, 64), (16, 2, 64), (8, 2, 48), (6, 2, 96), (32, 4, 128)])
    groups = _log(rng, 1, max(1, 64 // beams))
    most = 4 * 16 * 9301 * 8 * 128 // (groups * max(beams, 5) * kv_heads * dim)
    shared = _log(rng, 1, min(16000, max(1, most - 300)))
    return dict(op=op, groups=groups, beams=beams, heads=heads, kv_heads=kv_heads, dim=dim, page=rng.choice([8, 16, 16, 32, 64]), shared=shared,
                own=_log(rng, 1, 300), window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]), ragged=rng.random() < 0.5)


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _lengths(case):
    """Keys that a request's beams share, and keys of their own, a request."""
    n = case["groups"]
    if not case["ragged"]:
        return [case["shared"]] * n, [case["own"]] * n
    return ([max(1, case["shared"] * (n - i) // n) for i in range(n)], [max(1, case["own"] * (2 * i + 1) // (2 * n)) for i in range(n)])


def _parents(case, g):
    """A step's outcome: `moved` rows of every request have no continuation and take over rows that have one."""
    n, k, moved = case["groups"], case["beams"], case["moved"]
    order = torch.rand((n, k), generator=g, device="cuda").argsort(1)
    stays, goes = order[:, moved:], order[:, :moved]
    parents = torch.arange(k, device="cuda").repeat(n, 1)
    pick = torch.randint(0, k - moved, (n, moved), generator=g, device="cuda")
    parents.scatter_(1, goes, stays.gather(1, pick))
    return (parents + torch.arange(n, device="cuda")[:, None] * k).reshape(-1).to(torch.int32)


def _values(shape, dtype, g):
    if dtype == torch.int32:
        return torch.randint(0, 1 << 17, shape, generator=g, device="cuda", dtype=torch.int32)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _prepare_select(case, g):
    n, k, v, p = case["groups"], case["beams"], case["vocab"], case["picks"]
    logits = 2.5 * torch.randn((n * k, v), generator=g, device="cuda")
    if case["masked"]:
        logits.masked_fill_(torch.rand((n * k, v), generator=g, device="cuda") < case["masked"], -math.inf)
    scores = -20 * torch.rand((n, k), generator=g, device="cuda")
    if case["dead"]:
        scores[:, k - case["dead"]:] = -math.inf
    return dict(logits=logits, scores=scores.reshape(-1), out_scores=torch.empty((n, p), device="cuda"),
                out_rows=torch.empty((n, p), dtype=torch.int32, device="cuda"), out_tokens=torch.empty((n, p), dtype=torch.int32, device="cuda"))


def _prepare_reorder(case, g):
    rows = case["groups"] * case["beams"]
    total = case["slots"] if case["what"] == "states" else case["pages"]
    tail = (case["elems"],) if case["what"] == "states" else (2, case["kv_heads"], case["page"], case["dim"])
    s = dict(store=_values((case["layers"], total) + tail, _TYPES[case["dtype"]], g),
             rows=torch.randperm(total, generator=g, device="cuda")[:rows].to(torch.int32), parents=_parents(case, g), tokens=None)
    if case["what"] == "pages":
        s["tokens"] = torch.full((rows,), case["tokens"], dtype=torch.int32, device="cuda")
    return s


def _prepare_pages(case, g):
    n = case["copies"]
    order = torch.randperm(case["pages"], generator=g, device="cuda").to(torch.int32)
    fork = 2 * n > case["pages"] or case["tokens"] < case["page"]
    return dict(store=_values((case["layers"], case["pages"], 2, case["kv_heads"], case["page"], case["dim"]), _TYPES[case["dtype"]], g),
                dst=order[:n].contiguous(), src=order[n: n + 1].repeat(n) if fork else order[n: 2 * n].contiguous(),
                tokens=torch.full((n,), case["tokens"], dtype=torch.int32, device="cuda"))


def _prepare_attention(case, g):
    k, ps, hkv, d = case["beams"], case["page"], case["kv_heads"], case["dim"]
    shared, mine = _lengths(case)
    rows = len(shared) * k
    blocks = max(-(-(a + b) // ps) for a, b in zip(shared, mine))
    count = sum(a // ps + k * (-(-(a + b) // ps) - a // ps) for a, b in zip(shared, mine))
    order = torch.randperm(count, generator=g, device="cuda").tolist()
    table, halves, at = [], [], 0
    for a, b in zip(shared, mine):
        common = order[at: at + a // ps]
        at += a // ps
        need = -(-(a + b) // ps) - a // ps
        for i in range(k):
            private = order[at: at + need]
            at += need
            if a % ps and i:                              # the shared keys of a page that is filled on by every beam lie in each one's copy
                halves.append((table[-i][a // ps], private[0], a % ps))
            table.append(common + private + [0] * (blocks - a // ps - need))
    cache = _values((count, 2, hkv, ps, d), torch.bfloat16, g)
    for src, dst, used in halves:
        cache[dst, :, :, :used] = cache[src, :, :, :used]
    return dict(q=_values((rows, case["heads"] * d), torch.bfloat16, g), out=torch.empty((rows, case["heads"] * d), dtype=torch.bfloat16, device="cuda"),
                cache=cache, table=torch.tensor(table, dtype=torch.int32, device="cuda"),
                kv_len=torch.tensor([a + b for a, b in zip(shared, mine) for _ in range(k)], dtype=torch.int32, device="cuda"),
                shared=torch.tensor(shared, dtype=torch.int32, device="cuda"), most_shared=max(shared), most_own=max(mine))


def prepare(case, seed):
    make = dict(select=_prepare_select, reorder=_prepare_reorder, pages=_prepare_pages, attention=_prepare_attention)[case["op"]]
    return dict(make(case, _generator(seed)), case=case)


# ------------------------------------------------------------------------------------------------ the plain forms
def _plain_select(case, s):
    # 64 bits: what is chosen hangs on differences of scores, however small
    n, k, v = case["groups"], case["beams"], case["vocab"]
    x = s["logits"].double()
    top = x.amax(1, keepdim=True)
    score = s["scores"].double()[:, None] + (x - (top + (x - top).exp().sum(1, keepdim=True).log()))
    best, at = score.view(n, k * v).sort(dim=1, descending=True, stable=True)
    at = at[:, : case["picks"]]
    rows = at // v + torch.arange(n, device=at.device)[:, None] * k
    return best[:, : case["picks"]].float(), rows.to(torch.int32), (at % v).to(torch.int32)


def _plain_reorder(case, s):
    store, to, source = s["store"], s["rows"].long(), s["rows"][s["parents"].long()].long()
    taken = store[:, source]
    if s["tokens"] is not None:
        used = torch.arange(case["page"], device=to.device) < s["tokens"][:, None]
        taken = torch.where(used[None, :, None, None, :, None], taken, store[:, to])
    store[:, to] = taken
    return store


def _plain_pages(case, s):
    store, src, dst = s["store"], s["src"].long(), s["dst"].long()
    used = torch.arange(case["page"], device=src.device) < s["tokens"][:, None]
    store[:, dst] = torch.where(used[None, :, None, None, :, None], store[:, src], store[:, dst])
    return store


def _plain_attention(case, s):
    rows, h, hkv, d = s["q"].shape[0], case["heads"], case["kv_heads"], case["dim"]
    keys, values = s["cache"][s["table"].long()].float().permute(2, 0, 3, 1, 4, 5).reshape(2, rows, hkv, -1, d).unbind(0)
    q = s["q"].float().view(rows, hkv, h // hkv, d)
    at = torch.arange(keys.shape[2], device=q.device)
    seen = at < s["kv_len"][:, None]
    if case["window"]:
        seen &= at >= s["kv_len"][:, None] - case["window"]
    weights = (q @ keys.transpose(2, 3) * d ** -0.5).masked_fill(~seen[:, None, None], -math.inf)
    weights = (weights - weights.amax(-1, keepdim=True)).exp()
    weights = weights / weights.sum(-1, keepdim=True)
    return (weights @ values).reshape(rows, h * d).to(torch.bfloat16)


def _own(case, s):
    from rustinfer_b200.ops import kernels as K
    op = case["op"]
    if op == "select":
        K.beam_select(s["logits"], s["scores"], case["beams"], s["out_scores"], s["out_rows"], s["out_tokens"])
        return s["out_scores"], s["out_rows"], s["out_tokens"]
    if op == "reorder":
        K.reorder_rows(s["store"], s["rows"], s["parents"], case["beams"], s["tokens"])
        return s["store"]
    if op == "pages":
        K.copy_pages(s["store"], s["src"], s["dst"], s["tokens"])
        return s["store"]
    K.attention_decode_beams(s["q"], s["out"], s["cache"], s["table"], s["kv_len"], s["shared"], case["beams"], case["heads"], case["kv_heads"],
                             case["dim"], case["dim"] ** -0.5, case["window"] or None, s["most_shared"], s["most_own"])
    return s["out"]


def run(state):
    case = state["case"]
    if own:
        return _own(case, state)
    return dict(select=_plain_select, reorder=_plain_reorder, pages=_plain_pages, attention=_plain_attention)[case["op"]](case, state)


def work(case):
    if case["op"] == "select":
        logits = case["groups"] * case["beams"] * case["vocab"]
        return dict(bytes=4 * logits + 4 * case["groups"] * case["beams"] + 12 * case["groups"] * case["picks"], flops=4 * logits)
    size = 2 if case.get("dtype") == "bfloat16" else 4
    if case["op"] == "reorder":
        row = case["elems"] if case["what"] == "states" else 2 * case["kv_heads"] * case["tokens"] * case["dim"]
        rows = case["groups"] * case["beams"]
        return dict(bytes=2 * case["layers"] * case["groups"] * case["moved"] * row * size + 8 * rows, flops=0)
    if case["op"] == "pages":
        row = case["layers"] * 2 * case["kv_heads"] * case["tokens"] * case["dim"] * size
        sources = 1 if 2 * case["copies"] > case["pages"] or case["tokens"] < case["page"] else case["copies"]
        return dict(bytes=(case["copies"] + sources) * row + 8 * case["copies"], flops=0)
    shared, mine = _lengths(case)
    keys = seen = 0
    for a, b in zip(shared, mine):
        first = max(0, a + b - case["window"]) if case["window"] else 0
        keys += max(0, a - first) + case["beams"] * (a + b - max(a, first))
        seen += case["beams"] * (a + b - first)
    rows = case["groups"] * case["beams"]
    return dict(bytes=4 * keys * case["kv_heads"] * case["dim"] + 4 * rows * case["heads"] * case["dim"],
                flops=4 * seen * case["heads"] * case["dim"])


# ------------------------------------------------------------------------------------------------ from the definitions, in 64 bits
def _exact_select(case, s):
    picked, k = [], case["beams"]
    for g in range(case["groups"]):
        part = slice(g * k, (g + 1) * k)
        total = (torch.log_softmax(s["logits"][part].double(), -1) + s["scores"][part].double()[:, None]).flatten()
        order = torch.sort(total, descending=True, stable=True)[1][: case["picks"]]
        picked.append((total[order], (g * k + order // case["vocab"]).int(), (order % case["vocab"]).int()))
    return tuple(torch.stack(p) for p in zip(*picked))


def _exact_attention(case, s):
    h, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    lengths, rows = s["kv_len"].tolist(), []
    for r, n in enumerate(lengths):
        first = max(0, n - case["window"]) if case["window"] else 0
        at = torch.arange(first, n, device="cuda")
        kv = s["cache"][s["table"][r].long()[at // case["page"]], :, :, at % case["page"]].double()       # [keys, 2, heads, dim]
        q = s["q"][r].double().view(hkv, h // hkv, d)
        p = torch.softmax(torch.einsum("kgd,tkd->kgt", q, kv[:, 0]) / math.sqrt(d), -1)
        rows.append(torch.einsum("kgt,tkd->kgd", p, kv[:, 1]).reshape(h * d))
    return torch.stack(rows)


def _exact_copies(case, s):
    store = s["store"].clone()
    src = s["rows"][s["parents"].long()] if case["op"] == "reorder" else s["src"]
    dst = s["rows"] if case["op"] == "reorder" else s["dst"]
    used = None if s["tokens"] is None else s["tokens"].tolist()
    for i, (a, b) in enumerate(zip(src.tolist(), dst.tolist())):
        if used is None:
            store[:, b] = s["store"][:, a]
        else:
            store[:, b, :, :, : used[i]] = s["store"][:, a, :, :, : used[i]]
    return store


def exact(case, seed):
    make = dict(select=_exact_select, reorder=_exact_copies, pages=_exact_copies, attention=_exact_attention)[case["op"]]
    return make(case, prepare(case, seed))
