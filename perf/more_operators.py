"""Operators of a cache that is held in 4 bits and kept short, and of drafted tokens, as cases that can be timed and compared.

A cache is K and V apart in pages of 16 positions, and a table of page numbers per sequence.  Pages are float16, bfloat16, or 4 bits: a code from -8 to 7
an entry and a unit for each 32 entries of a position's key or value.

``store``   new keys and values become codes and units; read back as the values that they stand for
``attend``  attention of the newest tokens of each sequence: one, a part of a prompt (each sees what is before it) or a tree of drafts (each sees the context
            and those drafts that its bits name); ``weighed``: the weights that every position gets are added up, too
``evict``   a cache is cut to its first and last positions and those with the most weight, which move together, in all layers
``verify``  drafted tokens are accepted or not by the target's and the draft's probabilities and given random numbers

Widths are those of ``synth.CONFIGS`` (1B: 32 heads, 8 of keys and values, 64 wide; 8B: 32, 8, 128; 70B: 64, 8, 128; vocabulary 128256).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

PAGE = 16
GROUP = 32  # entries with one unit
DRAFTS = 64  # most nodes of a tree
LARGEST = 7168.0  # what larger entries count as
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # every decode step: one new key and value of each of 64 sequences
        dict(name="store, a step of 64", op="store", type="bf16", seqs=64, context=300, new=1, kv=8, dim=128, ragged=True),
        # after a long prompt: all of its keys and values
        dict(name="store, a prompt of 32k", op="store", type="f16", seqs=1, context=0, new=32000, kv=8, dim=128, ragged=False),
        # one user of a small model in the middle of a chat: the smallest call, latency
        dict(name="attend, 1 at 1000, 4 bits", op="attend", type="f16", pages="q4", seqs=1, context=1000, new=1, kv=8, group=4, dim=64, tree=False, weighed=False, ragged=False),
        # a full batch of users with contexts of all lengths: a decode step
        dict(name="attend, 64 at 16k, 4 bits, ragged", op="attend", type="bf16", pages="q4", seqs=64, context=16384, new=1, kv=8, group=4, dim=128, tree=False, weighed=False, ragged=True),
        # eight users with trees of drafts of different sizes
        dict(name="attend, 8 x 16 drafts at 8k, 4 bits, ragged", op="attend", type="f16", pages="q4", seqs=8, context=8192, new=16, kv=8, group=4, dim=128, tree=True, weighed=False, ragged=True),
        # the next part of a long prompt at the widest model
        dict(name="attend, 1000 more of a prompt at 8k, 4 bits", op="attend", type="bf16", pages="q4", seqs=1, context=8000, new=1000, kv=8, group=8, dim=128, tree=False, weighed=False, ragged=False),
        # a decode step that adds up the weights for a later cut
        dict(name="attend, 32 at 4k, weighed, ragged", op="attend", type="bf16", pages="bf16", seqs=32, context=4096, new=1, kv=8, group=4, dim=128, tree=False, weighed=True, ragged=True),
        # the last tokens of four prompts, whose weights say what the cut may drop
        dict(name="attend, 4 x 32 at 12k, weighed, 4 bits", op="attend", type="f16", pages="q4", seqs=4, context=12000, new=32, kv=8, group=4, dim=128, tree=False, weighed=True, ragged=False),
        # one user's cache of the 1B shape is cut to half
        dict(name="evict, 1 at 2k to 1k", op="evict", type="f16", pages="f16", layers=16, seqs=1, context=2050, keep=1000, kv=8, dim=64, ragged=False),
        # eight users' caches of the 8B shape are cut to a budget
        dict(name="evict, 8 at 4k to 2k, ragged", op="evict", type="bf16", pages="bf16", layers=32, seqs=8, context=4100, keep=2048, kv=8, dim=128, ragged=True),
        # one user's short chain of drafts
        dict(name="verify, 1 x 5", op="verify", type="f32", seqs=1, nodes=5, vocab=128256, chain=True, drafts=True, ragged=False),
        # 64 users' trees
        dict(name="verify, 64 x 16, trees, ragged", op="verify", type="f32", seqs=64, nodes=16, vocab=128256, chain=False, drafts=True, ragged=True),
    ]


def _log_uniform(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49))))))


def draw(rng):
    op = rng.choice(["store", "attend", "attend", "attend", "evict", "verify"])
    kind = rng.choice(["f16", "bf16"])
    shape = dict(kv=rng.choice([1, 2, 4, 8, 8]), dim=rng.choice([64, 128, 128]))
    if op == "store":
        seqs = _log_uniform(rng, 1, 64)
        return dict(op=op, type=kind, seqs=seqs, context=rng.choice([0, _log_uniform(rng, 1, 300)]), new=_log_uniform(rng, 1, 32000 // seqs), ragged=rng.random() < 0.7, **shape)
    if op == "attend":
        pages, tree, group = rng.choice(["q4", "q4", kind]), rng.random() < 0.4, rng.choice([1, 2, 3, 4, 4, 7, 8, 16])
        seqs = _log_uniform(rng, 1, 64)
        new = rng.choice([1, _log_uniform(rng, 1, DRAFTS), DRAFTS if tree else _log_uniform(rng, 1, 1000)])
        heads = shape["kv"] * group
        new = max(1, min(new, 2 ** 17 // (seqs * heads)))
        most = min(32000, 2 ** 34 // (seqs * new * heads * shape["dim"]), 2 ** (29 if pages == "q4" else 27) // (seqs * shape["kv"] * shape["dim"]))
        return dict(op=op, type=kind, pages=pages, seqs=seqs, context=_log_uniform(rng, 1, max(1, most)), new=new, group=group, tree=tree, weighed=rng.random() < 0.4,
                    ragged=rng.random() < 0.7, **shape)
    if op == "evict":
        seqs, layers, pages = _log_uniform(rng, 1, 16), rng.choice([1, 2, 16, 32]), rng.choice(["q4", kind, kind])
        layers = min(layers, 4) if pages == "q4" else layers
        context = _log_uniform(rng, 20, max(20, min(16000, 2 ** 29 // (seqs * layers * shape["kv"] * shape["dim"]))))
        return dict(op=op, type=kind, pages=pages, layers=layers, seqs=seqs, context=context, keep=_log_uniform(rng, 10, context + 5), ragged=rng.random() < 0.7, **shape)
    seqs = _log_uniform(rng, 1, 64)
    return dict(op=op, type=rng.choice(["f32", "f32", "f16", "bf16"]), seqs=seqs, nodes=_log_uniform(rng, 1, min(DRAFTS, 1024 // seqs)), vocab=rng.choice([2048, 32768, 128256, _log_uniform(rng, 500, 128256)]),
                chain=rng.random() < 0.5, drafts=rng.random() < 0.8, ragged=rng.random() < 0.7)


# ---------------------------------------------------------------------------------------------- inputs
def _lengths(case):
    """Positions in the cache per sequence: all the same, or from a quarter of it up to it.  The same for every seed, as the work is."""
    if not case["ragged"]:
        return np.full(case["seqs"], case["context"], np.int64)
    r = np.random.default_rng(11)
    return np.maximum(min(1, case["context"]), (case["context"] * r.uniform(0.25, 1.0, case["seqs"])).astype(np.int64))


def _sizes(case, key):
    """How many new tokens or nodes each sequence has."""
    n = case[key]
    return np.random.default_rng(12).integers(1, n + 1, case["seqs"]) if case["ragged"] else np.full(case["seqs"], n, np.int64)


def _randn(shape, dtype, g, std=1.0):
    x = torch.empty(shape, dtype=dtype, device="cuda")
    for part in x.view(-1).split(1 << 28):  # in pieces: no fp32 copy of a whole cache
        part.normal_(0.0, std, generator=g)
    return x


def _ints(v):
    return torch.from_numpy(np.asarray(v, np.int32)).cuda()


def _table(held, seed):
    """Pages in a random order, and how many there are."""
    pages = (held + PAGE - 1) // PAGE
    n = max(1, int(pages.sum()))
    order = np.random.default_rng(seed).permutation(n).astype(np.int32)
    table = np.zeros((len(held), max(1, int(pages.max()))), np.int32)
    at = 0
    for s, p in enumerate(pages):
        table[s, :p] = order[at:at + p]
        at += p
    return _ints(table), n


def _places(table, first, count):
    """Page and slot of positions first[s] .. first[s] + count[s] - 1 of all sequences, one after the other."""
    seq = torch.from_numpy(np.repeat(np.arange(len(count)), count)).cuda()
    x = torch.from_numpy(np.concatenate([np.arange(a, a + n) for a, n in zip(first, count)] + [np.zeros(0, np.int64)])).cuda()
    return table[seq, x // PAGE].long(), x % PAGE


def _packed(codes):
    """Codes [..., dim] as bytes [..., dim / 2]: entry 2 i in the low half of byte i."""
    c = (codes + 8).to(torch.uint8)
    return c[..., 0::2] | c[..., 1::2] << 4


def _cache_of_rows(s, case, held, g, layers=1):
    """Keys and values of `held` positions of every sequence, written to pages: those of the case's type, in 4 bits as codes and units, or by way of the cache."""
    kind, shape = case["pages"], (int(held.sum()), case["kv"], case["dim"])
    table, n = _table(held, s["seed"])
    s["table"] = table
    if kind != "q4":
        pool = (layers, n, case["kv"], PAGE, case["dim"])
        s["k"], s["v"] = _randn(pool, TYPES[kind], g), _randn(pool, TYPES[kind], g)
        s["k"] += torch.randn(case["kv"], 1, case["dim"], generator=g, device="cuda").to(s["k"].dtype)  # channels of keys have offsets, as a model's have
    elif own:
        s["k"], s["v"] = (torch.zeros((layers, n, case["kv"], 9 * case["dim"]), dtype=torch.uint8, device="cuda") for _ in range(2))
    else:
        s["codes"] = torch.zeros((layers, 2, n, case["kv"], PAGE, case["dim"] // 2), dtype=torch.uint8, device="cuda")
        s["units"] = torch.zeros((layers, 2, n, case["kv"], PAGE, case["dim"] // GROUP), dtype=torch.float16, device="cuda")
    if own:
        from orangu_b200 import CudaBackend, PagedCache

        global _backend
        _backend = _backend or CudaBackend.init(0)
        s["cache"] = PagedCache(_backend, s["k"], s["v"], table)
    if kind == "q4":
        page, slot = _places(table, np.zeros(len(held), np.int64), held)
        first, zero = _ints(np.concatenate([[0], np.cumsum(held)])), _ints(np.zeros(len(held)))
        for i in range(layers):
            k, v = _randn(shape, TYPES[case["type"]], g), _randn(shape, TYPES[case["type"]], g)
            k += torch.randn(case["kv"], case["dim"], generator=g, device="cuda").to(k.dtype)
            if own:
                s["cache"].store(k, v, first, zero, max_tokens=max(1, int(held.max())), layer=i, stream=torch.cuda.current_stream().cuda_stream)
                continue
            for j, x in enumerate((k, v)):
                for a in range(0, len(page), 1 << 17):
                    p, at = page[a:a + (1 << 17)], slot[a:a + (1 << 17)]
                    codes, units = _plain_codes(x[a:a + (1 << 17)])
                    s["codes"][i, j][p, :, at], s["units"][i, j][p, :, at] = _packed(codes), units.half()
    return s


_backend = None


def _visible(n, r):
    """Bits of a tree's n tokens: each grows from an earlier one or from the context and sees that one's tokens and itself."""
    bits = []
    for i in range(n):
        parent = int(r.integers(-1, i)) if i else -1
        bits.append((bits[parent] if parent >= 0 else 0) | 1 << i)
    return bits


def _probabilities(n, vocab, dtype, g):
    """Rows of a target and of a draft that is much like it."""
    target, draft = torch.empty((n, vocab), dtype=dtype, device="cuda"), torch.empty((n, vocab), dtype=dtype, device="cuda")
    for a in range(0, n, 64):
        x = torch.randn((min(64, n - a), vocab), generator=g, device="cuda") * 2.5
        y = x * 0.9 + torch.randn(x.shape, generator=g, device="cuda")
        target[a:a + 64], draft[a:a + 64] = torch.softmax(x, -1), torch.softmax(y, -1)
    return target, draft


def prepare(case, seed):
    g, r, op = torch.Generator("cuda"), np.random.default_rng(seed), case["op"]
    g.manual_seed(seed)
    s = dict(case, seed=seed)
    if op == "verify":
        sizes = _sizes(case, "nodes")
        first = np.concatenate([[0], np.cumsum(sizes)])
        n = int(first[-1])
        target, draft = _probabilities(n, case["vocab"], TYPES[case["type"]], g)
        parent = np.concatenate([[-1] + [i - 1 if case["chain"] else int(r.integers(0, i)) for i in range(1, m)] for m in sizes])
        above = torch.from_numpy(np.repeat(first[:-1], sizes) + np.maximum(parent, 0)).cuda()
        tokens = torch.cat([torch.multinomial(draft[above[a:a + 64]].float(), 1, generator=g)[:, 0] for a in range(0, n, 64)]).int()
        s.update(target=target, draft=draft if case["drafts"] else None, tokens=tokens, parent=_ints(parent), first=_ints(first), uniform=torch.rand(n, generator=g, device="cuda"), n=n)
        if own:
            from orangu_b200 import CudaBackend

            global _backend
            _backend = _backend or CudaBackend.init(0)
            s["backend"] = _backend
        return s
    held = _lengths(case)
    if op == "evict":
        _cache_of_rows(s, case, held, g, case["layers"])
        room = s["table"].shape[1] * PAGE
        s.update(n_pos=_ints(held), max_pos=int(held.max()), left=_ints(np.concatenate([[0], np.cumsum(np.minimum(held, case["keep"]))])),
                 zero=_ints(np.zeros(case["seqs"])), mass=torch.empty((case["layers"], case["seqs"], case["kv"], room), device="cuda").exponential_(1.0, generator=g) ** 2)
        return s
    sizes = _sizes(case, "new")
    first = np.concatenate([[0], np.cumsum(sizes)])
    s.update(first=_ints(first), context_lengths=_ints(held), max_context=int(held.max()), held=held, sizes=sizes)
    n = int(first[-1])
    if op == "store":
        s.update(k_new=_randn((n, case["kv"], case["dim"]), TYPES[case["type"]], g), v_new=_randn((n, case["kv"], case["dim"]), TYPES[case["type"]], g))
        s["k_new"] += torch.randn(case["kv"], case["dim"], generator=g, device="cuda").to(s["k_new"].dtype)
        table, pages = _table(held + sizes, seed)
        s["table"] = table
        s["page"], s["slot"] = _places(table, held, sizes)
        if own:
            from orangu_b200 import CudaBackend, PagedCache

            _backend = _backend or CudaBackend.init(0)
            s["cache"] = PagedCache(_backend, *(torch.zeros((1, pages, case["kv"], 9 * case["dim"]), dtype=torch.uint8, device="cuda") for _ in range(2)), table)
        else:
            s["codes"] = torch.zeros((2, pages, case["kv"], PAGE, case["dim"] // 2), dtype=torch.uint8, device="cuda")
            s["units"] = torch.zeros((2, pages, case["kv"], PAGE, case["dim"] // GROUP), dtype=torch.float16, device="cuda")
        return s
    _cache_of_rows(s, case, held + sizes, g)
    s.update(q=_randn((n, case["kv"] * case["group"], case["dim"]), TYPES[case["type"]], g, 1.5), scale=case["dim"] ** -0.5, visible=None, mass=None)
    if case["tree"]:
        bits = [b for m in sizes for b in _visible(int(m), r)]
        s["visible"] = torch.from_numpy(np.array(bits, np.uint64).view(np.int64)).cuda()
    if case["weighed"]:
        s["mass"] = torch.empty((case["seqs"], case["kv"], s["table"].shape[1] * PAGE), device="cuda").exponential_(1.0, generator=g)
    return s


# ---------------------------------------------------------------------------------------------- the plain forms
def _plain_codes(x):
    """Codes [..., dim] and units [..., dim / 32] of entries [..., dim], in fp32."""
    x = torch.nan_to_num(x.float(), nan=0.0).clamp(-LARGEST, LARGEST)
    x = x.reshape(*x.shape[:-1], -1, GROUP)
    hi, lo = x.amax(-1), x.amin(-1)
    m = torch.where(hi > -lo, hi, lo)
    a = m.abs() / 8
    # seven significant bits, and no finer than 2^-24, away from zero
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -30))) - 6)
    step = torch.where(a >= step * 128, step * 2, torch.where(a < step * 64, step / 2, step)).clamp_min(2.0 ** -24)  # (a logarithm may be off next to a power of two)
    d = torch.ceil(a / step) * step * -torch.sign(m)
    by = torch.where(d != 0, d, torch.ones_like(d))[..., None]
    c = torch.round(x / by).clamp(-8, 7)
    return c.reshape(*c.shape[:-2], -1), d


def _plain_values(codes, units):
    """Entries [..., dim] in fp32 of bytes [..., dim / 2] and units [..., dim / 32]."""
    c = torch.stack([codes & 15, codes >> 4], -1).float() - 8
    c = c.reshape(*codes.shape[:-1], units.shape[-1], GROUP)
    return (c * units.float()[..., None]).reshape(*codes.shape[:-1], -1)


def _softmax_over(scores, seen):
    """softmax over the last axis of what is seen; rows that see nothing are zero."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    return e / e.sum(-1, keepdim=True).clamp_min(1e-30)


def _pool(s, value, layer, pages):
    """fp32 keys or values [..., kv, 16, dim] of pages [...] of a layer."""
    if s["pages"] == "q4":
        return _plain_values(s["codes"][layer, value][pages], s["units"][layer, value][pages])
    return (s["v"] if value else s["k"])[layer][pages].float()


def _plain_store(s):
    for j, x in enumerate((s["k_new"], s["v_new"])):
        codes, units = _plain_codes(x)
        s["codes"][j][s["page"], :, s["slot"]], s["units"][j][s["page"], :, s["slot"]] = _packed(codes), units.half()
    return [_plain_values(s["codes"][j][s["page"], :, s["slot"]], s["units"][j][s["page"], :, s["slot"]]).half() for j in range(2)]


def _plain_attend(s):
    kv, group, dim, q = s["kv"], s["group"], s["dim"], s["q"]
    out = torch.empty_like(q)
    at = 0
    for i, (ctx, n) in enumerate(zip(s["held"].tolist(), s["sizes"].tolist())):  # a sequence at a time
        length = ctx + n
        pages = s["table"][i, :(length + PAGE - 1) // PAGE].long()
        k, v = (_pool(s, j, 0, pages).permute(1, 0, 2, 3).reshape(kv, -1, dim)[:, :length] for j in range(2))
        x, t = torch.arange(length, device="cuda"), torch.arange(n, device="cuda")
        if s["visible"] is None:
            seen = x < ctx + t[:, None] + 1
        else:
            bits = s["visible"][at:at + n]
            seen = (x < ctx) | ((bits[:, None] >> (x - ctx).clamp(0, 63) & 1) == 1)
        qs = q[at:at + n].float().reshape(n, kv, group, dim).permute(1, 2, 0, 3).reshape(kv, group * n, dim)
        w = torch.matmul(qs, k.transpose(1, 2)).mul_(s["scale"]).reshape(kv, group, n, length)
        w = _softmax_over(w, seen).reshape(kv, group * n, length)
        out[at:at + n] = torch.matmul(w, v).reshape(kv, group, n, dim).permute(2, 0, 1, 3).reshape(n, kv * group, dim).to(q.dtype)
        if s["mass"] is not None:
            got = w.sum(1)
            s["mass"][i, :, :ctx] += got[:, :ctx]
            s["mass"][i, :, ctx:length] = got[:, ctx:]
        at += n
    return out if s["mass"] is None else (out, s["mass"])


def _plain_evict(s):
    layers, seqs, kv, room = s["mass"].shape
    n, keep = s["n_pos"].long()[:, None], s["keep"]
    a, b = _ends(keep)
    x = torch.arange(room, device="cuda")
    key = torch.where((x < a) | (x >= n - b), torch.full_like(s["mass"][0, :, 0], math.inf), torch.zeros_like(s["mass"][0, :, 0]))[None, :, None] + s["mass"]
    key = torch.where((x < n)[None, :, None], key, torch.full_like(key, -math.inf))
    best = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep]
    best = torch.nn.functional.pad(best, (0, max(0, keep - room)), value=1 << 30)
    best = torch.where(best < n[None, :, None], best, torch.full_like(best, 1 << 30))
    kept = torch.sort(best, dim=-1).values
    there = kept < 1 << 30
    kept = torch.where(there, kept, torch.full_like(kept, -1))
    left = torch.minimum(s["n_pos"], torch.full_like(s["n_pos"], keep))
    table = s["table"].long()
    values = []
    for i in range(layers):
        seq, head, to = there[i].nonzero(as_tuple=True)
        src = kept[i][seq, head, to]
        pa, pb = table[seq, src // PAGE], table[seq, to // PAGE]
        s["mass"][i][seq, head, to] = s["mass"][i][seq, head, src]  # read whole before it is written
        for p in ((s["codes"][i, 0], s["codes"][i, 1], s["units"][i, 0], s["units"][i, 1]) if s["pages"] == "q4" else (s["k"][i], s["v"][i])):
            p[pb, head, to % PAGE] = p[pa, head, src % PAGE]
    if s["pages"] == "q4":  # what is left, as values
        seq = torch.repeat_interleave(torch.arange(seqs, device="cuda"), left.long(), output_size=sum(min(m, keep) for m in _lengths(s).tolist()))
        at = torch.arange(len(seq), device="cuda") - s["left"].long()[seq]
        page, slot = table[seq, at // PAGE], at % PAGE
        values = [_plain_values(s["codes"][i, j][page, :, slot], s["units"][i, j][page, :, slot]).half() for i in range(layers) for j in range(2)]
    return kept.int(), left, s["mass"], *(values if s["pages"] == "q4" else (s["k"], s["v"]))


def _ends(keep):
    """How many first and last positions a cut always keeps."""
    return min(4, keep // 4), min(64, keep // 2)


def _plain_verify(s):
    n, device = s["seqs"], "cuda"
    first, parent, tokens = s["first"].tolist(), s["parent"].tolist(), s["tokens"].tolist()
    u = s["uniform"].double()
    kept = torch.full((n, DRAFTS), -1, dtype=torch.int32, device=device)
    count, token = [], []
    for i in range(n):
        a = first[i]
        path, p, total = [0], s["target"][a].double(), torch.ones((), dtype=torch.float64, device=device)
        c = torch.zeros((), dtype=torch.float64, device=device)
        q = None if s["draft"] is None else s["draft"][a].double()
        w = p
        for j in range(1, first[i + 1] - a):
            if parent[a + j] != path[-1]:
                continue
            x = tokens[a + j]
            if (u[a + j] * total < w[x]) if q is None else (u[a + j] * total * q[x] < p[x] - c * q[x]):
                path.append(j)
                p, total, c = s["target"][a + j].double(), torch.ones_like(total), torch.zeros_like(c)
                q = None if s["draft"] is None else s["draft"][a + j].double()
                w = p
            elif q is None:
                total = (total - w[x]).clamp_min(0.0)
                w = w.clone()
                w[x] = 0.0
            else:
                c = c + total
                w = (p - c * q).clamp_min(0.0)
                total = w.sum()
        w = torch.where(w.sum() > 0, w, p)
        upto = torch.cumsum(w, 0)
        token.append((upto <= u[a] * upto[-1]).sum())
        kept[i, :len(path)] = torch.tensor(path, dtype=torch.int32, device=device)
        count.append(len(path))
    return kept, torch.tensor(count, dtype=torch.int32, device=device), torch.stack(token).int()


# ---------------------------------------------------------------------------------------------- one pass
def run(s):
    op = s["op"]
    if not own:
        return {"store": _plain_store, "attend": _plain_attend, "evict": _plain_evict, "verify": _plain_verify}[op](s)
    st = torch.cuda.current_stream().cuda_stream
    if op == "store":
        k, v = (torch.empty(s["k_new"].shape, dtype=torch.float16, device="cuda") for _ in range(2))
        s["cache"].store(s["k_new"], s["v_new"], s["first"], s["context_lengths"], max_tokens=s["new"], stream=st)
        s["cache"].load(k, v, s["first"], s["context_lengths"], max_tokens=s["new"], stream=st)
        return [k, v]
    if op == "attend":
        out = torch.empty_like(s["q"])
        s["cache"].attention_tokens(s["q"], s["first"], s["context_lengths"], s["scale"], out, max_tokens=s["new"], max_context=s["max_context"], visible=s["visible"], mass=s["mass"], stream=st)
        return out if s["mass"] is None else (out, s["mass"])
    if op == "evict":
        kept = torch.empty((s["layers"], s["seqs"], s["kv"], s["keep"]), dtype=torch.int32, device="cuda")
        left = torch.empty(s["seqs"], dtype=torch.int32, device="cuda")
        a, b = _ends(s["keep"])
        s["cache"].evict(s["n_pos"], s["mass"], kept, left, max_pos=s["max_pos"], keep_first=a, keep_last=b, stream=st)
        if s["pages"] != "q4":
            return kept, left, s["mass"], s["k"], s["v"]
        values = []
        for i in range(s["layers"]):
            k, v = (torch.empty((sum(min(m, s["keep"]) for m in _lengths(s).tolist()), s["kv"], s["dim"]), dtype=torch.float16, device="cuda") for _ in range(2))
            s["cache"].load(k, v, s["left"], s["zero"], max_tokens=s["keep"], layer=i, stream=st)
            values += [k, v]
        return kept, left, s["mass"], *values
    from orangu_b200 import verify_drafts

    kept = torch.empty((s["seqs"], DRAFTS), dtype=torch.int32, device="cuda")
    count, token = (torch.empty(s["seqs"], dtype=torch.int32, device="cuda") for _ in range(2))
    verify_drafts(s["backend"], s["target"], s["draft"], s["tokens"], s["parent"], s["first"], s["uniform"], kept, count, token, stream=st)
    return kept, count, token


def work(case):
    op = case["op"]
    if op == "verify":
        n = int(_sizes(case, "nodes").sum())
        size = 4 if case["type"] == "f32" else 2
        rows = 2 if case["drafts"] else 1  # of the last accepted node: what is left of its probabilities gives the next token
        return {"bytes": float(case["seqs"]) * (rows * case["vocab"] * size + 4 * DRAFTS + 8) + n * (rows * size + 12.0), "flops": 0.0}
    kv, dim, held = case["kv"], case["dim"], _lengths(case)
    entry = 9 / 16 if case.get("pages", "q4") == "q4" else 2.0  # bytes
    if op == "store":
        rows = float(_sizes(case, "new").sum()) * kv * dim * 2
        return {"bytes": rows * (2 + 2 * entry + 2), "flops": 0.0}  # read, written, read back, and the values
    if op == "evict":
        a, left = _ends(case["keep"])[0], np.minimum(held, case["keep"])
        moved = float(np.where(held > case["keep"], left - a, 0).sum()) * case["layers"] * kv
        back = float(left.sum()) * case["layers"] * kv * dim * 2 * (entry + 2) if case["pages"] == "q4" else 0.0
        return {"bytes": moved * (2 * 2 * dim * entry + 8) + 4.0 * case["layers"] * kv * (float(held.sum()) + case["seqs"] * case["keep"]) + back, "flops": 0.0}
    sizes, heads = _sizes(case, "new"), kv * case["group"]
    seen = float((held * sizes).sum() + (sizes * (sizes + 1) // 2).sum())  # about: a tree's tokens see fewer of one another
    masses = 8.0 * kv * float(held.sum()) + 4.0 * kv * float(sizes.sum()) if case["weighed"] else 0.0
    return {"bytes": 2.0 * kv * dim * entry * float((held + sizes).sum()) + 4.0 * float(sizes.sum()) * heads * dim + masses, "flops": 4.0 * dim * heads * seen}


# ---------------------------------------------------------------------------------------------- in 64 bits
def _exact_codes(x):
    """Entries that stand for x [..., dim] in 4 bits, in float64, a power of two and a ceiling at a time."""
    x = x.double().cpu().numpy()
    x = np.clip(np.where(np.isnan(x), 0.0, x), -LARGEST, LARGEST).reshape(*x.shape[:-1], -1, GROUP)
    most, least = x.max(-1), x.min(-1)
    a = np.maximum(most, -least) / 8
    _, e = np.frexp(a)  # a = f 2^e, f from 1/2 to 1
    step = np.ldexp(1.0, np.maximum(e - 7, -24))
    d = np.where(most > -least, -1.0, 1.0) * np.ceil(a / step) * step
    c = np.clip(np.rint(x / np.where(d != 0, d, 1.0)[..., None]), -8, 7)
    return torch.from_numpy((c * d[..., None]).reshape(*c.shape[:-2], -1)).cuda()


def exact(case, seed):
    """From the definitions in float64, a sequence at a time."""
    global own
    op, was = case["op"], own
    if op == "attend" and float(work(case)["flops"]) > 3e12:
        return None
    own = False  # inputs as arrays, whatever is measured
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if op == "store":
        return [_exact_codes(s["k_new"]), _exact_codes(s["v_new"])]
    if op == "verify":
        return _exact_verify(s)
    table = s["table"].cpu().numpy()
    if op == "evict":
        return _exact_evict(s, table)
    kv, group, dim = s["kv"], s["group"], s["dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    mass = None if s["mass"] is None else s["mass"].double()
    at = 0
    for i, (ctx, n) in enumerate(zip(s["held"].tolist(), s["sizes"].tolist())):
        pages = torch.from_numpy(table[i, :(ctx + n + PAGE - 1) // PAGE].astype(np.int64)).cuda()
        mask = torch.ones(n, ctx + n, dtype=torch.bool, device="cuda")
        if s["visible"] is None:
            mask[:, ctx:] = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
        else:
            bits = s["visible"][at:at + n].tolist()
            mask[:, ctx:] = torch.tensor([[b >> j & 1 == 1 for j in range(n)] for b in bits], device="cuda")
        for h in range(kv):
            k, v = (_exact_pages(s, j, pages, h).reshape(-1, dim)[:ctx + n] for j in range(2))
            got = torch.zeros(ctx + n, dtype=torch.float64, device="cuda")
            for gh in range(group):
                q = s["q"][at:at + n, h * group + gh].double()
                e = torch.where(mask, q @ k.T / math.sqrt(dim), torch.full((), -math.inf, dtype=torch.float64, device="cuda"))
                w = torch.nan_to_num(torch.softmax(e, -1), nan=0.0)
                out[at:at + n, h * group + gh] = w @ v
                got += w.sum(0)
            if mass is not None:
                mass[i, h, :ctx] += got[:ctx]
                mass[i, h, ctx:ctx + n] = got[ctx:]
        at += n
    return out if mass is None else (out, mass)


def _exact_pages(s, value, pages, head):
    if s["pages"] != "q4":
        return (s["v"] if value else s["k"])[0, pages, head].double()
    c, d = s["codes"][0, value][pages, head], s["units"][0, value][pages, head].double()
    c = torch.stack([c % 16, c // 16], -1).reshape(*c.shape[:-1], -1).double() - 8.0
    return c * torch.repeat_interleave(d, GROUP, dim=-1)


def _exact_evict(s, table):
    keep, held, mass = s["keep"], s["n_pos"].tolist(), s["mass"].cpu().numpy()
    layers, seqs, kv, _ = mass.shape
    a, b = _ends(keep)
    kept = np.full((layers, seqs, kv, keep), -1, np.int32)
    for i in range(seqs):
        n = held[i]
        for li in range(layers):
            for h in range(kv):
                if n <= keep:
                    mine = np.arange(n)
                else:
                    middle = np.arange(a, n - b)
                    order = middle[np.argsort(-mass[li, i, h, middle], kind="stable")][:keep - a - b]
                    mine = np.sort(np.concatenate([np.arange(a), order, np.arange(n - b, n)]))
                kept[li, i, h, :len(mine)] = mine
    new = mass.copy()
    left = np.minimum(held, keep).astype(np.int32)
    pools = []
    if s["pages"] != "q4":
        pools = [s["k"], s["v"]]
    values = []
    for li in range(layers):
        halves = [[], []]
        for i in range(seqs):
            m = int(left[i])
            at = torch.from_numpy(kept[li, i, :, :m].astype(np.int64)).cuda()
            tab = torch.from_numpy(table[i].astype(np.int64)).cuda()
            head = torch.arange(kv, device="cuda")[:, None]
            to = torch.arange(m, device="cuda")[None]
            for h in range(kv):
                new[li, i, h, :m] = mass[li, i, h, kept[li, i, h, :m]]
            for pool in pools:
                moved = pool[li][tab[at // PAGE], head, at % PAGE].clone()
                pool[li][tab[to // PAGE].expand(kv, m), head, (to % PAGE).expand(kv, m)] = moved
            if not pools:
                for j in range(2):
                    c, d = s["codes"][li, j][tab[at // PAGE], head, at % PAGE], s["units"][li, j][tab[at // PAGE], head, at % PAGE].double()
                    c = torch.stack([c % 16, c // 16], -1).reshape(kv, m, -1).double() - 8.0
                    halves[j].append((c * torch.repeat_interleave(d, GROUP, dim=-1)).permute(1, 0, 2))
        if not pools:
            values += [torch.cat(halves[0]), torch.cat(halves[1])]
    return kept, left, new, *(pools or values)


def _exact_verify(s):
    """The residual after each rejection is normalised, as the rule is stated."""
    first, parent, tokens, u = (s[k].cpu().numpy() for k in ("first", "parent", "tokens", "uniform"))
    n = s["seqs"]
    kept, count, token = np.full((n, DRAFTS), -1, np.int32), np.zeros(n, np.int32), np.zeros(n, np.int32)
    for i in range(n):
        a, nodes = int(first[i]), int(first[i + 1] - first[i])
        at, path = 0, [0]
        while True:
            r = s["target"][a + at].double().cpu().numpy()
            q = None if s["draft"] is None else s["draft"][a + at].double().cpu().numpy()
            total, went = 1.0, False
            for j in range(at + 1, nodes):
                if parent[a + j] != at:
                    continue
                x = tokens[a + j]
                if float(u[a + j]) * (total if q is None else q[x]) < r[x]:
                    at, went = j, True
                    path.append(j)
                    break
                if q is None:
                    total -= r[x]
                    r[x] = 0.0
                else:
                    r = np.maximum(r - q, 0.0)
                    r /= r.sum()
            if not went:
                break
        upto = np.cumsum(r)
        token[i] = np.searchsorted(upto, float(u[a]) * upto[-1], side="right")
        kept[i, :len(path)], count[i] = path, len(path)
    return kept, count, token
