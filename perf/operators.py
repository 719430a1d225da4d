"""Operators over the pages of a cache that the caller holds, as cases that can be timed and compared.

A cache is K and V apart, ``[layer][page][kv head][16][head_dim]`` in float16 or bfloat16, and a table of page numbers per sequence.

``tree``    attention of drafted tokens: every token sees its sequence's context and those drafted tokens that its bits name
``sparse``  a decode step that reads few pages: a score per page from 8-bit bounds of its keys, the best pages, attention over them
``bounds``  the 8-bit bounds of the pages that a step or a prompt has filled
``fork``    sequences branch: a child shares its parent's full pages and gets a copy of the last one
``copy``    whole pages in all layers
``keep``    the accepted drafted tokens move together behind the context, in all layers

Widths are those of ``synth.CONFIGS`` (1B: 32 heads, 8 of keys and values, 64 wide; 8B: 32, 8, 128; 70B: 64, 8, 128).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

PAGE = 16
DRAFTS = 64  # most drafted tokens of a sequence
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one user of a small model, a short chain of drafts in the middle of a chat: the smallest call, latency
        dict(name="tree, 1 x 4 at 512", op="tree", type="f16", seqs=1, drafts=4, context=512, kv=8, group=4, dim=64, ragged=False),
        # eight users with trees of different sizes and contexts of different lengths
        dict(name="tree, 8 x 16 at 8k, ragged", op="tree", type="bf16", seqs=8, drafts=16, context=8192, kv=8, group=4, dim=128, ragged=True),
        # large trees over long contexts at the widest model: as many products as bytes
        dict(name="tree, 4 x 64 at 32k", op="tree", type="f16", seqs=4, drafts=64, context=32000, kv=8, group=8, dim=128, ragged=False),
        # one user of a small model with a moderate context
        dict(name="sparse, 1 at 4k, 32 pages", op="sparse", type="f16", rows=1, context=4096, pages=32, kv=8, group=4, dim=64, ragged=False),
        # one user with a very long document
        dict(name="sparse, 1 at 128k, 128 pages", op="sparse", type="bf16", rows=1, context=131000, pages=128, kv=8, group=4, dim=128, ragged=False),
        # a full batch of users with long contexts of all lengths
        dict(name="sparse, 64 at 24k, 64 pages, ragged", op="sparse", type="bf16", rows=64, context=24576, pages=64, kv=8, group=4, dim=128, ragged=True),
        # every decode step: the last page of each of 64 sequences has a new key
        dict(name="bounds, a step of 64", op="bounds", type="bf16", seqs=64, context=300, new=1, kv=8, dim=128),
        # after a long prompt: all of its pages
        dict(name="bounds, a prompt of 64k", op="bounds", type="f16", seqs=1, context=65500, new=65500, kv=8, dim=128),
        # one sequence of the 1B shape goes on in eight branches
        dict(name="fork, 8 at 1000", op="fork", type="f16", layers=16, seqs=8, context=1000, kv=8, dim=64),
        # pages moved together to make room at one end of the pool, 8B shape
        dict(name="copy, 512 pages", op="copy", type="bf16", layers=32, pages=512, kv=8, dim=128),
        # one user's accepted path of a tree
        dict(name="keep, 1 x 5", op="keep", type="f16", layers=16, seqs=1, kept=5, context=512, kv=8, dim=64, ragged=False),
        # 64 users' accepted paths, 8B shape
        dict(name="keep, 64 x 8, ragged", op="keep", type="bf16", layers=32, seqs=64, kept=8, context=100, kv=8, dim=128, ragged=True),
    ]


def _log_uniform(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "sparse", "sparse", "bounds", "fork", "copy", "keep"])
    case = dict(op=op, type=rng.choice(sorted(TYPES)), kv=rng.choice([1, 2, 4, 8, 8]), dim=rng.choice([64, 128, 128]))
    if op == "tree":
        seqs, drafts = _log_uniform(rng, 1, 32), _log_uniform(rng, 1, DRAFTS)
        group = rng.choice([1, 2, 3, 4, 4, 7, 8, 16])
        most = min(32000, 2 ** 35 // (seqs * drafts * case["kv"] * group * case["dim"]), 2 ** 27 // (seqs * case["kv"] * case["dim"]))
        case.update(seqs=seqs, drafts=drafts, context=_log_uniform(rng, 1, max(1, most)), group=group, ragged=rng.random() < 0.7)
    elif op == "sparse":
        rows = _log_uniform(rng, 1, 64)
        case.update(rows=rows, context=_log_uniform(rng, 64, min(131000, 64 * 24576 // rows)), pages=_log_uniform(rng, 4, 128),
                    group=rng.choice([1, 2, 3, 4, 4, 7, 8, 16]), ragged=rng.random() < 0.7)
    elif op == "bounds":
        seqs = _log_uniform(rng, 1, 64)
        context = _log_uniform(rng, 1, min(65500, 65536 // seqs))
        case.update(seqs=seqs, context=context, new=rng.choice([1, _log_uniform(rng, 1, context), context]))
    elif op == "fork":
        case.update(layers=rng.choice([1, 2, 16, 32]), seqs=_log_uniform(rng, 1, 32), context=_log_uniform(rng, 1, 4000))
    elif op == "copy":
        case.update(layers=rng.choice([1, 2, 16, 32]), pages=_log_uniform(rng, 1, 512))
    else:
        case.update(layers=rng.choice([1, 2, 16, 32]), seqs=_log_uniform(rng, 1, 64), kept=_log_uniform(rng, 1, DRAFTS), context=_log_uniform(rng, 1, 500),
                    ragged=rng.random() < 0.7)
    return case


# ---------------------------------------------------------------------------------------------- inputs
def _lengths(case, seed):
    """Positions in the cache per sequence: all the same, or from a quarter of it up to it.  The same for every seed, as the work is."""
    n = case.get("seqs") or case.get("rows")
    if not case.get("ragged"):
        return np.full(n, case["context"], np.int64)
    r = np.random.default_rng(11)
    return np.maximum(1, (case["context"] * r.uniform(0.25, 1.0, n)).astype(np.int64))


def _sizes(case, key):
    """How many drafted or accepted tokens each sequence has."""
    n = np.full(case["seqs"], case[key], np.int64)
    return np.random.default_rng(12).integers(1, case[key] + 1, case["seqs"]) if case.get("ragged") else n


def _randn(shape, dtype, g, std=1.0):
    x = torch.empty(shape, dtype=dtype, device="cuda")
    flat = x.view(-1)
    for part in flat.split(1 << 28):  # in pieces: no fp32 copy of a whole cache
        part.normal_(0.0, std, generator=g)
    return x


def _cache(case, seed, held, layers=1, spare=0):
    """K, V and the table: `held` positions of every sequence, pages in a random order; channels of keys have offsets, as a model's have."""
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    pages = (held + PAGE - 1) // PAGE
    n = int(pages.sum()) + spare
    shape = (layers, n, case["kv"], PAGE, case["dim"])
    k, v = _randn(shape, TYPES[case["type"]], g), _randn(shape, TYPES[case["type"]], g)
    k += torch.randn(case["kv"], 1, case["dim"], generator=g, device="cuda").to(k.dtype)
    order = np.random.default_rng(seed).permutation(n).astype(np.int32)
    table = np.zeros((len(held), int(pages.max()) if len(held) else 1), np.int32)
    at = 0
    for s, p in enumerate(pages):
        table[s, :p] = order[at:at + p]
        at += p
    return g, k, v, torch.from_numpy(table).cuda(), order[at:]


def _visible(n, r):
    """Bits of a tree's n tokens: each grows from an earlier one or from the context and sees that one's tokens and itself."""
    bits = []
    for i in range(n):
        parent = int(r.integers(-1, i)) if i else -1
        bits.append((bits[parent] if parent >= 0 else 0) | 1 << i)
    return bits


def _ints(v):
    return torch.from_numpy(np.asarray(v, np.int32)).cuda()


def _queries(n, case, g):
    return _randn((n, case["kv"] * case["group"], case["dim"]), TYPES[case["type"]], g, 1.5)


def prepare(case, seed):
    s = dict(case, scale=case["dim"] ** -0.5)
    op, held = case["op"], None
    layers, spare = case.get("layers", 1), 0
    if op == "copy":
        held, spare = np.zeros(0, np.int64), 2 * case["pages"]
    else:
        held = _lengths(case, seed)
        if op == "fork":
            held, spare = held[:1], case["seqs"]
        sizes = _sizes(case, "drafts" if op == "tree" else "kept") if op in ("tree", "keep") else 0
    g, k, v, table, rest = _cache(case, seed, held + (sizes if op == "tree" else DRAFTS if op == "keep" else 0) if op != "copy" else held, layers, spare)
    r = np.random.default_rng(seed)
    s.update(k=k, v=v, table=table)
    if op == "tree":
        bits = [b for n in sizes for b in _visible(int(n), r)]
        first = np.concatenate([[0], np.cumsum(sizes)])
        s.update(q=_queries(int(first[-1]), case, g), first=_ints(first), context_lengths=_ints(held), max_context=int(held.max()),
                 visible=torch.from_numpy(np.array(bits, np.uint64).view(np.int64)).cuda())
    elif op == "sparse":
        codes, scales = _plain_bounds(k[0], torch.full((k.shape[1],), PAGE, device="cuda"))
        last = table.gather(1, _ints((held - 1) // PAGE).long()[:, None])[:, 0].long()
        codes[last], scales[last] = _plain_bounds(k[0][last], _ints((held - 1) % PAGE + 1))  # the last pages are filled in part
        s.update(q=_queries(case["rows"], case, g), n_pos=_ints(held), max_pos=int(held.max()), codes=codes, scales=scales)
    elif op == "bounds":
        shape = (k.shape[1], case["kv"], 2, case["dim"])
        s.update(codes=torch.zeros(shape, dtype=torch.int8, device="cuda"), scales=torch.zeros(shape[:2], device="cuda"),
                 first_pos=_ints(held - case["new"]), n_pos=_ints(held))
    elif op == "fork":
        n = case["seqs"]
        wide = torch.zeros((1 + n, table.shape[1]), dtype=torch.int32, device="cuda")
        wide[:1] = table
        s.update(table=wide, parent=_ints(np.zeros(n)), child=_ints(1 + np.arange(n)), n_pos=_ints(np.full(n, case["context"])), fresh=_ints(rest))
    elif op == "copy":
        s.update(table=_ints(np.zeros((1, 1))), src=_ints(rest[:case["pages"]]), dst=_ints(rest[case["pages"]:]))
    else:
        kept = np.full((case["seqs"], DRAFTS), -1, np.int32)
        for i, n in enumerate(sizes):
            kept[i, :n] = np.sort(r.permutation(DRAFTS)[:n])
        s.update(context_lengths=_ints(held), kept=_ints(kept), n_kept=_ints(sizes))
    if own:
        from orangu_b200 import CudaBackend, PagedCache

        global _backend
        _backend = _backend or CudaBackend.init(0)
        s["cache"] = PagedCache(_backend, s["k"], s["v"], s["table"])
    return s


_backend = None


# ---------------------------------------------------------------------------------------------- the plain forms
def _softmax_over(scores, seen):
    """softmax over the last axis of what is seen; rows that see nothing are zero."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    return e / e.sum(-1, keepdim=True).clamp_min(1e-30)


def _gathered(x, table):
    """[kv, S, P * 16, d] in fp32 of the pages [S, P] of one layer."""
    s, p = table.shape
    return x[table.long()].float().permute(2, 0, 1, 3, 4).reshape(x.shape[1], s, p * PAGE, x.shape[3])


def _plain_tree(s):
    first, ctx, q = s["first"].long(), s["context_lengths"].long(), s["q"]
    n, kv, group, dim = s["seqs"], s["kv"], s["group"], s["dim"]
    most = s["drafts"]
    k, v = _gathered(s["k"][0], s["table"]), _gathered(s["v"][0], s["table"])
    length = k.shape[2]
    # tokens padded to [S, most], and back at the end
    row = first[:-1, None] + torch.arange(most, device="cuda")
    real = row < first[1:, None]
    row = torch.where(real, row, torch.zeros_like(row))
    x = torch.arange(length, device="cuda")
    j = x - ctx[:, None]  # drafted token at a position [S, L]
    drafted = (j >= 0) & (j < (first[1:] - first[:-1])[:, None])
    bit = (s["visible"][row][:, :, None] >> j.clamp(0, 63)[:, None, :]) & 1
    seen = (x < ctx[:, None])[:, None, :] | (drafted[:, None, :] & (bit == 1))  # [S, T, L]
    qs = q[row].float().reshape(n, most, kv, group, dim).permute(2, 0, 3, 1, 4).reshape(kv, n, group * most, dim)
    w = torch.matmul(qs, k.transpose(2, 3)).mul_(s["scale"]).reshape(kv, n, group, most, length)
    w = _softmax_over(w, seen[None, :, None])
    o = torch.matmul(w.reshape(kv, n, group * most, length), v).reshape(kv, n, group, most, dim).permute(1, 3, 0, 2, 4)
    return o.reshape(n, most, kv * group, dim)[real].to(q.dtype)


def _plain_bounds(k, filled):
    """Codes [pages, kv, 2, dim] and scales [pages, kv] of pages [pages, kv, 16, dim] of which `filled` positions count."""
    there = (torch.arange(PAGE, device=k.device) < filled[:, None])[:, None, :, None]
    hi = k.masked_fill(~there, -math.inf).amax(2).float()
    lo = k.masked_fill(~there, math.inf).amin(2).float()
    top = torch.maximum(hi.abs(), lo.abs()).amax(-1)
    d = top / torch.full_like(top, 127.0)  # by a tensor: a division, not a product with a rounded inverse
    by = torch.where(d > 0, d, torch.ones_like(d))[..., None]
    codes = torch.stack([torch.ceil(hi / by), torch.floor(lo / by)], 2)
    return codes.clamp_(-127, 127).to(torch.int8), d


def _plain_select(s):
    q, table, n_pos = s["q"].float(), s["table"].long(), s["n_pos"].long()
    rows, kv, group, dim = q.shape[0], s["kv"], s["group"], s["dim"]
    top = q.abs().amax(-1)
    dq = top / torch.full_like(top, 127.0)
    c = torch.round(q / torch.where(dq > 0, dq, torch.ones_like(dq))[..., None]).reshape(rows, kv, group, dim)
    b = s["codes"][table].float().permute(0, 2, 3, 4, 1)  # [R, kv, 2, d, P]
    isum = torch.matmul(c.clamp_min(0), b[:, :, 0]) + torch.matmul(c.clamp_max(0), b[:, :, 1])  # whole numbers below 2^24: exact in any order
    score = ((dq.reshape(rows, kv, group, 1) * s["scales"][table].permute(0, 2, 1)[:, :, None]) * isum).amax(2)  # [R, kv, P]
    pages = (n_pos + PAGE - 1) // PAGE
    p = torch.arange(table.shape[1], device="cuda")
    n = s["pages"]
    score = torch.where((p < 1) | (p >= pages[:, None] - 2)[:, None], torch.full_like(score, math.inf), score)  # the first and the last two are kept
    score = torch.where((p < pages[:, None])[:, None], score, torch.full_like(score, -math.inf))
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :n]
    best = torch.sort(torch.where(best < pages[:, None, None], best, torch.full_like(best, 1 << 30)), dim=-1).values
    if best.shape[-1] < n:
        best = torch.nn.functional.pad(best, (0, n - best.shape[-1]), value=1 << 30)
    return torch.where(best < 1 << 30, best, torch.full_like(best, -1)).int()


def _plain_sparse(s):
    chosen = _plain_select(s)  # [R, kv, n]
    rows, kv, n = chosen.shape
    q, group, dim = s["q"], s["group"], s["dim"]
    page = s["table"].long()[:, None].expand(rows, kv, -1).gather(2, chosen.clamp_min(0).long())
    heads = torch.arange(kv, device="cuda")[None, :, None]
    k, v = (x[0][page, heads].float().reshape(rows, kv, n * PAGE, dim) for x in (s["k"], s["v"]))
    x = chosen[..., None] * PAGE + torch.arange(PAGE, device="cuda", dtype=torch.int32)
    seen = ((chosen >= 0)[..., None] & (x < s["n_pos"][:, None, None, None])).reshape(rows, kv, 1, n * PAGE)
    w = torch.matmul(q.float().reshape(rows, kv, group, dim), k.transpose(2, 3)) * s["scale"]
    o = torch.matmul(_softmax_over(w, seen), v.masked_fill(~seen.transpose(2, 3), 0.0))
    return chosen, o.reshape(rows, kv * group, dim).to(q.dtype)


def _plain_update(s):
    """Bounds of the pages that hold positions first_pos .. n_pos - 1."""
    p = torch.arange(s["table"].shape[1], device="cuda")
    touched = (p >= s["first_pos"][:, None] // PAGE) & (p * PAGE < s["n_pos"][:, None])
    filled = (s["n_pos"][:, None] - p * PAGE).clamp(max=PAGE)[touched]
    page = s["table"].long()[touched]
    s["codes"][page], s["scales"][page] = _plain_bounds(s["k"][0][page], filled)


def _plain_fork(s):
    table, parent, child, n_pos = s["table"], s["parent"].long(), s["child"].long(), s["n_pos"].long()
    p = torch.arange(table.shape[1], device="cuda")
    mine, old = table[child], table[parent]
    whole, part = p < (n_pos // PAGE)[:, None], (p == (n_pos // PAGE)[:, None]) & (n_pos % PAGE > 0)[:, None]
    table[child] = torch.where(whole, old, torch.where(part, s["fresh"][:, None], mine))
    src = old.gather(1, (n_pos // PAGE).clamp_max(table.shape[1] - 1)[:, None])[:, 0].long()
    ragged = (n_pos % PAGE > 0).nonzero()[:, 0]
    for x in (s["k"], s["v"]):
        x[:, s["fresh"].long()[ragged]] = x[:, src[ragged]]


def _plain_keep(s):
    n, ctx, kept = s["n_kept"].long(), s["context_lengths"].long(), s["kept"].long()
    j = torch.arange(DRAFTS, device="cuda")
    here = (j < n[:, None]).nonzero()
    seq, to = here[:, 0], here[:, 1]
    a, b = ctx[seq] + kept[seq, to], ctx[seq] + to
    table = s["table"].long()
    pa, pb = table[seq, a // PAGE], table[seq, b // PAGE]
    for x in (s["k"], s["v"]):
        x[:, pb, :, b % PAGE] = x[:, pa, :, a % PAGE]  # read whole before it is written


# ---------------------------------------------------------------------------------------------- one pass
def run(s):
    op = s["op"]
    if op == "tree":
        if not own:
            return _plain_tree(s)
        out = torch.empty_like(s["q"])
        s["cache"].attention_tree(s["q"], s["first"], s["context_lengths"], s["visible"], s["scale"], out, max_drafts=s["drafts"], max_context=s["max_context"],
                                  stream=torch.cuda.current_stream().cuda_stream)
        return out
    if op == "sparse":
        if not own:
            return _plain_sparse(s)
        out = torch.empty_like(s["q"])
        chosen = torch.empty((s["rows"], s["kv"], s["pages"]), dtype=torch.int32, device="cuda")
        st = torch.cuda.current_stream().cuda_stream
        s["cache"].select(s["q"], s["codes"], s["scales"], s["n_pos"], chosen, max_pos=s["max_pos"], keep_first=1, keep_last=2, stream=st)
        s["cache"].attention(s["q"], chosen, s["n_pos"], s["scale"], out, stream=st)
        return chosen, out
    st = torch.cuda.current_stream().cuda_stream if own else None
    if op == "bounds":
        if own:
            s["cache"].bounds(s["first_pos"], s["n_pos"], s["codes"], s["scales"], max_new=s["new"], stream=st)
        else:
            _plain_update(s)
        return s["codes"] * s["scales"][..., None, None], s["scales"]
    if op == "fork":
        if own:
            s["cache"].fork(s["parent"], s["child"], s["n_pos"], s["fresh"], stream=st)
        else:
            _plain_fork(s)
        return s["table"], s["k"], s["v"]
    if op == "copy":
        if own:
            s["cache"].copy(s["src"], s["dst"], stream=st)
        else:
            for x in (s["k"], s["v"]):
                x[:, s["dst"].long()] = x[:, s["src"].long()]
        return s["k"], s["v"]
    if own:
        s["cache"].keep(s["context_lengths"], s["kept"], s["n_kept"], stream=st)
    else:
        _plain_keep(s)
    return s["k"], s["v"]


def work(case):
    op, kv, dim = case["op"], case["kv"], case["dim"]
    vector = dim * 2  # bytes of one key or value
    if op == "tree":
        held, sizes = _lengths(case, 0), _sizes(case, "drafts")
        tokens = int(sizes.sum())
        seen = int((held * sizes).sum() + (sizes * (sizes + 1) // 2).sum())  # about: a tree's tokens see fewer of one another
        heads = kv * case["group"]
        return {"bytes": 2.0 * kv * vector * float((held + sizes).sum()) + 2.0 * tokens * heads * vector + 8.0 * tokens, "flops": 4.0 * dim * heads * seen}
    if op == "sparse":
        held = _lengths(case, 0)
        pages = (held + PAGE - 1) // PAGE
        read = np.minimum(pages, case["pages"])
        heads = kv * case["group"]
        return {"bytes": float(pages.sum()) * kv * (2 * dim + 4) + float(read.sum()) * kv * PAGE * 2 * vector + 2.0 * case["rows"] * heads * vector + 4.0 * kv * float(read.sum()),
                "flops": 4.0 * dim * heads * float(pages.sum()) + 4.0 * dim * heads * PAGE * float(read.sum())}
    if op == "bounds":
        held = _lengths(case, 0)
        first = (held - case["new"]) // PAGE
        pages = float(((held + PAGE - 1) // PAGE - first).sum())
        every = float(((held + PAGE - 1) // PAGE).sum())  # all bounds come back as values
        return {"bytes": float((held - first * PAGE).sum()) * kv * vector + pages * kv * (2 * dim + 4) + every * kv * (2 * dim * 5 + 4), "flops": 0.0}
    if op == "fork":
        part = case["context"] % PAGE
        return {"bytes": 2.0 * 2 * case["layers"] * case["seqs"] * (PAGE if part else 0) * kv * vector + 8.0 * case["seqs"] * -(-case["context"] // PAGE), "flops": 0.0}
    if op == "copy":
        return {"bytes": 2.0 * 2 * case["layers"] * case["pages"] * PAGE * kv * vector, "flops": 0.0}
    return {"bytes": 2.0 * 2 * case["layers"] * float(_sizes(case, "kept").sum()) * kv * vector, "flops": 0.0}


# ---------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """Attention and bounds from their definitions, a sequence (row) at a time in float64; moved values are those of another order of steps."""
    s = prepare(case, seed)
    table, op = s["table"].cpu().numpy(), case["op"]
    kv, dim = case["kv"], case["dim"]
    if op == "tree":
        first, ctx, bits = s["first"].tolist(), s["context_lengths"].tolist(), s["visible"].tolist()
        out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        for i in range(case["seqs"]):
            n, m = ctx[i], first[i + 1] - first[i]
            pages = torch.from_numpy(table[i, :(n + m + PAGE - 1) // PAGE].astype(np.int64)).cuda()
            mask = torch.ones(m, n + m, dtype=torch.bool, device="cuda")
            mask[:, n:] = torch.tensor([[bits[first[i] + t] >> j & 1 == 1 for j in range(m)] for t in range(m)], device="cuda")
            for h in range(kv):
                k, v = (x[0, pages, h].double().reshape(-1, dim)[:n + m] for x in (s["k"], s["v"]))
                q = s["q"][first[i]:first[i + 1], h * case["group"]:(h + 1) * case["group"]].double()
                e = torch.einsum("tgd,ld->tgl", q, k) / math.sqrt(dim)
                e = torch.where(mask[:, None], e, torch.full_like(e, -math.inf))
                out[first[i]:first[i + 1], h * case["group"]:(h + 1) * case["group"]] = torch.softmax(e, -1) @ v
        return out
    if op == "sparse":
        lengths, n = s["n_pos"].tolist(), case["pages"]
        q32 = s["q"].float().cpu().numpy().reshape(case["rows"], kv, case["group"], dim)
        out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        lists = np.full((case["rows"], kv, n), -1, np.int32)
        codes, scales = s["codes"].cpu().numpy(), s["scales"].cpu().numpy()
        for i, length in enumerate(lengths):
            count = (length + PAGE - 1) // PAGE
            pages = table[i, :count]
            for h in range(kv):
                best = np.full(count, -np.inf, np.float32)
                hi, lo = codes[pages, h, 0].astype(np.float64), codes[pages, h, 1].astype(np.float64)
                for g in range(case["group"]):
                    x = q32[i, h, g]
                    dq = np.float32(np.abs(x).max() / np.float32(127.0))
                    c = np.rint(x / (dq if dq > 0 else np.float32(1.0))).astype(np.float64)
                    whole = hi @ np.maximum(c, 0) + lo @ np.minimum(c, 0)
                    best = np.maximum(best, (dq * scales[pages, h]) * whole.astype(np.float32))
                kept = {p for p in range(count) if p < 1 or p >= count - 2}
                others = sorted((p for p in range(count) if p not in kept), key=lambda p: (-best[p], p))
                mine = sorted(list(kept) + others[:max(0, n - len(kept))])[:n]
                lists[i, h, :len(mine)] = mine
                at = torch.from_numpy(pages[mine].astype(np.int64)).cuda()
                where = torch.tensor([p * PAGE + t for p in mine for t in range(PAGE)], device="cuda")
                k, v = (x[0, at, h].double().reshape(-1, dim)[where < length] for x in (s["k"], s["v"]))
                q = s["q"][i, h * case["group"]:(h + 1) * case["group"]].double()
                out[i, h * case["group"]:(h + 1) * case["group"]] = torch.softmax(q @ k.T / math.sqrt(dim), -1) @ v
        return lists, out
    if op == "bounds":
        # a bound is a whole number of 127ths of the largest value that is no tighter than the keys
        value = torch.zeros(s["codes"].shape, dtype=torch.float64, device="cuda")
        unit = torch.zeros(s["scales"].shape, dtype=torch.float64, device="cuda")
        for i, (a, b) in enumerate(zip(s["first_pos"].tolist(), s["n_pos"].tolist())):
            p = np.arange(a // PAGE, (b + PAGE - 1) // PAGE)
            pages = torch.from_numpy(table[i, p].astype(np.int64)).cuda()
            k = s["k"][0, pages].double()
            late = torch.from_numpy((p[:, None] * PAGE + np.arange(PAGE)) >= b).cuda()[:, None, :, None]
            k = torch.where(late, k[:, :, :1], k)
            d = (k.abs().amax((2, 3)).float() / torch.tensor(127.0, device="cuda").expand(len(p), kv)).double()
            step = torch.where(d > 0, d, torch.ones_like(d))[..., None].float()
            up, down = torch.ceil(k.amax(2).float() / step), torch.floor(k.amin(2).float() / step)
            value[pages] = (torch.stack([up, down], 2).clamp(-127, 127) * d[..., None, None]).double()
            unit[pages] = d
        return value, unit
    k, v = s["k"], s["v"]
    if op == "copy":
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            k[:, b].copy_(k[:, a])
            v[:, b].copy_(v[:, a])
        return k, v
    if op == "fork":
        whole, part = divmod(case["context"], PAGE)
        for i, fresh in enumerate(s["fresh"].tolist()):
            s["table"][1 + i, :whole] = s["table"][0, :whole]
            if part:
                s["table"][1 + i, whole] = fresh
                for x in (k, v):
                    x[:, fresh] = x[:, int(table[0, whole])]
        return s["table"], k, v
    for i, (n, m) in enumerate(zip(s["context_lengths"].tolist(), s["n_kept"].tolist())):
        path = s["kept"][i, :m].tolist()
        for x in (k, v):
            moved = torch.stack([x[:, int(table[i, (n + a) // PAGE]), :, (n + a) % PAGE] for a in path])
            for j in range(m):
                x[:, int(table[i, (n + j) // PAGE]), :, (n + j) % PAGE] = moved[j]
    return k, v
