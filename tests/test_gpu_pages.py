"""Operators over the pages of a caller's cache, through the public entry points, against the plain statements of pages_plain.py."""
import ctypes as C

import numpy as np
import pytest

import pages_plain as plain
from gpu_common import backend  # noqa: F401

pytestmark = pytest.mark.gpu
PAGE = 16
U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step of the outputs, relative


def tolerance(kind, dim):
    """Bound of an output's error but for its own rounding.  The weights: f16 ones are rounded (2^-11, in the sum and in the products alike, which
    adds up to twice that), bf16 ones go in with their remainder (2^-16); f16 weights below 2^-14 are off by 2^-25 at most.  A score's
    error, absolute, is that of a sum of dim products in fp32 with a factor in front (dim + 4 roundings of 2^-24, truncating adders: twice that),
    and a weight's relative error is as large, twice again in numerator and denominator; 2^-20 covers 2^x, the online sums and their merges."""
    weight = 2.0 ** -11 if kind == "f16" else 2.0 ** -16
    tiny = 2.0 ** -25 if kind == "f16" else 0.0
    return lambda v, qk, n: v * (2 * weight + n * tiny + 4 * (dim + 4) * 2.0 ** -24 * qk + 2.0 ** -20)


def device16(bits, kind):
    import torch

    return torch.from_numpy(np.ascontiguousarray(bits).view(np.int16)).cuda().view(torch.float16 if kind == "f16" else torch.bfloat16)


def ints(v):
    import torch

    return torch.from_numpy(np.ascontiguousarray(v, np.int32)).cuda()


def words(v):
    import torch

    return torch.from_numpy(np.array(v, np.uint64).view(np.int64)).cuda()


def float64(t):
    return t.float().cpu().numpy().astype(np.float64)


def check(got, want, tol, kind, what=""):
    assert np.isfinite(got).all(), what
    off = np.abs(got - want) - (tol[..., None] + U[kind] * (np.abs(want) + tol[..., None]) + 2.0 ** -25)
    assert off.max() <= 0, f"{what}: {off.max()} over the bound at {np.unravel_index(off.argmax(), off.shape)}"


class Made:
    """A cache of one or more layers with tables in a random order; positions that no sequence has are not numbers."""

    def __init__(self, be, kind, kv, dim, held, seed=0, layers=1, layer=0, spare=0, stride=None, seqs=None):
        from orangu_b200 import PagedCache

        r = np.random.default_rng(seed)
        pages = [-(-int(n) // PAGE) for n in held]
        n_pages = sum(pages) + spare + 1
        shape = (layers, n_pages, kv, PAGE, dim)
        k, kb = plain.bits16(shape, r, kind)
        v, vb = plain.bits16(shape, r, kind)
        order = r.permutation(n_pages)
        self.tables = np.full((seqs or len(held), stride or max(pages + [1])), -1, np.int64)
        filled = np.zeros((n_pages, PAGE), bool)
        at = 0
        for s, p in enumerate(pages):
            self.tables[s, :p] = order[at:at + p]
            at += p
            for x in range(int(held[s])):
                filled[self.tables[s, x // PAGE], x % PAGE] = True
        self.free = order[at:]
        junk = np.uint16(0x7e00 if kind == "f16" else 0x7fc0)
        for bits in (kb, vb):
            bits[:] = np.where(filled[None, :, None, :, None], bits, junk)
        self.k, self.v = k[layer], v[layer]
        self.kd, self.vd, self.td = device16(kb, kind), device16(vb, kind), ints(self.tables)
        self.cache = PagedCache(be, self.kd, self.vd, self.td)
        self.r, self.kind, self.layer = r, kind, layer


def random_tree(r, n):
    bits = []
    for i in range(n):
        parent = int(r.integers(-1, i)) if i else -1
        bits.append((bits[parent] if parent >= 0 else 0) | 1 << i)
    return bits


def run_tree(made, group, ctx, drafts, scale=None, extra=0, bits=None, max_ctx=None, strides=(0, 0), stream=None, layer=0):
    """Calls attention_tree; queries and outputs have `extra` rows behind the last token and `strides` entries between rows' ends and starts."""
    import torch

    kv, dim = made.k.shape[1], made.k.shape[3]
    first = np.concatenate([[0], np.cumsum(drafts)])
    n = int(first[-1]) + extra
    heads = kv * group
    q, qb = plain.bits16((n, heads, dim), made.r, made.kind, 1.5)
    wide = np.full((n, heads * dim + strides[0]), 0x7e00 if made.kind == "f16" else 0x7fc0, np.uint16)
    wide[:, :heads * dim] = qb.reshape(n, -1)
    qd = device16(wide, made.kind)[:, :heads * dim].view(n, heads, dim)
    outw = torch.full((n, heads * dim + strides[1]), 7.0, dtype=qd.dtype, device="cuda")
    out = outw[:, :heads * dim].view(n, heads, dim)
    if bits is None:
        bits = [b for m in drafts for b in random_tree(made.r, m)]
    bits = bits + [~0 & (1 << 64) - 1] * extra
    scale = dim ** -0.5 if scale is None else scale
    made.cache.attention_tree(qd, ints(first), ints(ctx), words(bits), scale, out, max_drafts=max(list(drafts) + [1]),
                              max_context=max(list(ctx) + [0]) if max_ctx is None else max_ctx, layer=layer, stream=stream or torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    want = np.full((n, heads, dim), 7.0)
    tol = plain.tree(q, made.k, made.v, made.tables, first, ctx, bits, scale, want, tolerance(made.kind, dim))
    assert (outw[:, heads * dim:] == 7.0).all()
    check(float64(out), want, tol, made.kind)
    return out


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kv,group,ctx,drafts", [
    (1, 1, [0], [1]), (2, 4, [5], [3]), (1, 16, [16], [1]), (2, 3, [15, 16, 17], [1, 2, 3]), (8, 4, [100, 0, 33], [4, 5, 1]), (2, 8, [40, 700, 1, 0], [7, 0, 4, 2]),
    (1, 4, [250], [16]), (2, 5, [130, 64], [13, 6]), (1, 7, [300], [33]), (1, 2, [77, 78], [64, 63]), (2, 8, [50, 333], [64, 20]), (1, 16, [90], [64])])
def test_tree(backend, kind, dim, kv, group, ctx, drafts):
    made = Made(backend, kind, kv, dim, [a + b for a, b in zip(ctx, drafts)], seed=len(ctx) + dim + group)
    run_tree(made, group, ctx, drafts, extra=2)


@pytest.mark.parametrize("kind,dim,group,drafts", [("f16", 128, 4, 4), ("bf16", 64, 4, 16), ("bf16", 128, 8, 64), ("f16", 64, 2, 21)])
def test_tree_of_long_contexts_is_cut_and_added_up(backend, kind, dim, group, drafts):
    ctx = [5000, 17, 2049]
    made = Made(backend, kind, 1, dim, [c + drafts for c in ctx], seed=drafts)
    a = run_tree(made, group, ctx, [drafts] * 3)
    made.r = np.random.default_rng(4)
    one = run_tree(made, group, ctx, [drafts] * 3)
    made.r = np.random.default_rng(4)
    for bound in (0, 1, 100, 1 << 31):  # the bound shares out the work and no more
        made.r = np.random.default_rng(4)
        run_tree(made, group, ctx, [drafts] * 3, max_ctx=bound)
    made.r = np.random.default_rng(4)
    again = run_tree(made, group, ctx, [drafts] * 3)
    assert (one.view(dtype=__import__("torch").int16) == again.view(dtype=__import__("torch").int16)).all()
    assert a.shape == again.shape


def test_tree_strides_layers_and_scales(backend):
    made = Made(backend, "bf16", 2, 128, [40, 70], seed=3, layers=3, layer=2)
    run_tree(made, 4, [30, 60], [10, 5], strides=(64, 8), layer=2, extra=1)
    run_tree(made, 4, [30, 60], [10, 5], strides=(8, 128), layer=2, scale=1.0)
    run_tree(made, 4, [30, 60], [10, 5], layer=2, scale=1e-6)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group,drafts,order", [(4, 2, 1), (4, 16, 1), (4, 64, 1), (8, 40, -1), (2, 20, -1)])
def test_tree_scores_that_grow_and_shrink_by_powers_of_two(backend, kind, dim, group, drafts, order):
    """Keys twice (or half) as large every 64 positions: every step has a new maximum, far above the last one, for half of the rows at least."""
    ctx = [64 * 12 + 5, 64 * 9]
    made = Made(backend, kind, 2, dim, [c + drafts for c in ctx], seed=drafts + dim)
    for s, c in enumerate(ctx):
        for x in range(c + drafts):
            page, slot, f = made.tables[s, x // PAGE], x % PAGE, 2.0 ** (min(order * (x // 64), 12) - (6 if order > 0 else -5))
            made.kd[0, page, :, slot] *= f
    made.k = float64(made.kd[0])  # (the smallest f16 keys have lost bits)
    run_tree(made, group, ctx, [drafts] * 2)


def test_tree_tokens_that_see_nothing_are_zero_and_others_do_not_notice(backend):
    made = Made(backend, "f16", 2, 64, [3, 20 + 4], seed=5)
    run_tree(made, 2, [0, 20], [3, 4], bits=[0, 0b111, 0b100, 0, 0b1111, 0b1, 0b1000])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("drafts", [3, 20, 64])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_tree_drafted_tokens_that_are_no_numbers_stay_with_those_who_see_them(backend, kind, drafts, bad):
    """Keys and values of one drafted token are no numbers: only tokens that see it may notice."""
    import torch

    ctx, victim = 21, drafts // 2
    made = Made(backend, kind, 1, 64, [ctx + drafts], seed=drafts)
    x = ctx + victim
    page, slot = int(made.tables[0, x // PAGE]), x % PAGE
    bits = [((1 << drafts) - 1) & ~(1 << victim)] * drafts  # nobody sees it
    for what in (made.vd, made.kd):
        what[0, page, :, slot, ::3] = bad
        clean = made.k.copy(), made.v.copy()
        made.k[page, :, slot], made.v[page, :, slot] = 0.0, 0.0
        run_tree(made, 4, [ctx], [drafts], bits=bits)
        made.k, made.v = clean
    # one that sees a value that is no number has none in those entries, and only there
    made = Made(backend, kind, 1, 64, [ctx + drafts], seed=drafts)
    page = int(made.tables[0, x // PAGE])
    made.vd[0, page, :, slot, ::3] = bad
    bits[0] = (1 << drafts) - 1
    q = torch.randn(drafts, 4, 64, device="cuda").to(made.kd.dtype)
    out = torch.empty_like(q)
    made.cache.attention_tree(q, ints([0, drafts]), ints([ctx]), words(bits), 0.125, out, max_drafts=drafts, max_context=ctx, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert not torch.isfinite(out[0, :, ::3]).any() and torch.isfinite(out[0, :, 1::3]).all() and torch.isfinite(out[1:]).all()


def test_tree_pages_that_are_not_there(backend):
    """Numbers outside the pool, and positions past the table's end, hold nothing."""
    made = Made(backend, "f16", 2, 128, [200, 90], seed=9)
    for entry, number in ((0, -1), (3, 1 << 30), (11, -(1 << 31)), (5, made.kd.shape[1])):
        made.tables[0, entry] = number
    made.td.copy_(ints(made.tables))
    run_tree(made, 4, [180, 80], [20, 10])
    made.tables[1, :] = -1
    made.td.copy_(ints(made.tables))
    run_tree(made, 4, [180, 80], [20, 10])
    import torch

    big = ints(np.array([2 ** 31 - 1, 2 ** 31 - 1]))  # contexts far past the table: what it names counts, drafted tokens behind it do not
    q = torch.randn(5, 8, 128, device="cuda").half()
    a, b = torch.empty_like(q), torch.empty_like(q)
    whole = made.td.shape[1] * PAGE
    st = torch.cuda.current_stream().cuda_stream
    made.kd.nan_to_num_(0.0), made.vd.nan_to_num_(0.0)
    for ctx, out in ((big, a), (ints([whole, whole]), b)):
        made.cache.attention_tree(q, ints([0, 3, 5]), ctx, words([0, 1, 2, 3, 1]), 0.1, out, max_drafts=3, max_context=whole, stream=st)
    torch.cuda.synchronize()
    assert torch.equal(a, b) and (a[3:] == 0).all() and torch.isfinite(a).all()


@pytest.mark.parametrize("group,dim", [(2, 64), (8, 64), (3, 128), (16, 128)])
def test_tree_of_many_sequences(backend, group, dim):
    """More sequences than a warp has lanes, some of them without drafted tokens, some without context."""
    r = np.random.default_rng(group)
    drafts = [int(v) for v in r.integers(0, 6, 75)]
    ctx = [0 if v < 20 else int(v) for v in r.integers(0, 400, 75)]
    made = Made(backend, "bf16", 2, dim, [a + b for a, b in zip(ctx, drafts)], seed=dim + group)
    run_tree(made, group, ctx, drafts)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_tree_short_pieces_with_and_without_rows_for_the_second_stream(backend, kind, dim):
    """Up to 512 rows a head in the call, but many sequences with 128 or fewer and contexts of a few tiles, several of them after one another in a CTA."""
    drafts = [64, 1, 16, 17, 2, 33, 48, 49, 0, 8] * 5
    ctx = [(37 * i) % 190 for i in range(len(drafts))]
    made = Made(backend, kind, 8, dim, [c + d for c, d in zip(ctx, drafts)], seed=dim)
    for _ in range(3):
        run_tree(made, 8, ctx, drafts)


def test_handles_come_and_go(backend):
    """A handle's workspace is used again by later ones: in the state that a new one has."""
    import torch

    from orangu_b200 import PagedCache

    made = Made(backend, "f16", 2, 64, [2500, 900], seed=3)
    first = {}
    for turn in range(3):
        for group, drafts in ((2, 4), (8, 20)):
            made.r = np.random.default_rng(group)
            out = run_tree(made, group, [2500 - drafts, 900 - drafts], [drafts, drafts])
            if turn:
                assert torch.equal(out, first[group])
            first[group] = out
        made.cache.close()
        made.cache = PagedCache(backend, made.kd, made.vd, made.td)


@pytest.mark.parametrize("group", [2, 8])
def test_tree_tokens_past_the_bound_and_odd_offsets_are_left_out(backend, group):
    import torch

    made = Made(backend, "f16", 1, 64, [30, 30, 30, 30], seed=2)
    q = torch.randn(12, group, 64, device="cuda").half()
    st = torch.cuda.current_stream().cuda_stream

    def run(first, max_drafts):
        out = torch.full_like(q, 5.0)
        made.cache.attention_tree(q, ints(first), ints([9] * (len(first) - 1)), words([7] * 12), 0.125, out, max_drafts=max_drafts, max_context=9, stream=st)
        torch.cuda.synchronize()
        return out

    out = run([0, 6, 8], 3)  # six tokens where three are allowed
    assert (out[3:6] == 5).all() and (out[8:] == 5).all() and not (out[:3] == 5).any() and not (out[6:8] == 5).any()
    out = run([0, 2, 1, 40, 3], 8)  # falling, and past the tokens
    assert (out[2:] == 5).all() and not (out[:2] == 5).any()
    assert (run([-3, 2, 2, 2], 8) == 5).all()


def test_positions_past_four_gigabytes(backend):
    """Pages at the far end of a pool of more than 2^32 bytes."""
    import torch

    from orangu_b200 import PagedCache

    n_pages, kv, dim = 150_000, 8, 128  # 32 KB a page
    k = torch.empty((1, n_pages, kv, PAGE, dim), dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    ids = [n_pages - 1, 5, 131_073, n_pages - 7]
    for p in ids:
        k[0, p].normal_(), v[0, p].normal_()
    cache = PagedCache(backend, k, v, ints([ids]))
    small = PagedCache(backend, k[:, ids].contiguous(), v[:, ids].contiguous(), ints([[0, 1, 2, 3]]))
    q = torch.randn(4, 32, dim, device="cuda").bfloat16()
    st = torch.cuda.current_stream().cuda_stream
    outs = []
    for c, pages in ((cache, n_pages), (small, 4)):
        out = torch.empty_like(q)
        c.attention_tree(q, ints([0, 4]), ints([58]), words([1, 3, 7, 9]), 0.1, out, max_drafts=4, max_context=58, stream=st)
        codes, scales = torch.zeros((pages, kv, 2, dim), dtype=torch.int8, device="cuda"), torch.zeros((pages, kv), device="cuda")
        c.bounds(ints([0]), ints([62]), codes, scales, max_new=62, stream=st)
        chosen = torch.empty((1, kv, 2), dtype=torch.int32, device="cuda")
        c.select(q[:1], codes, scales, ints([62]), chosen, max_pos=62, stream=st)
        row = torch.empty_like(q[:1])
        c.attention(q[:1], chosen, ints([62]), 0.1, row, stream=st)
        outs.append((out, codes[ids] if pages > 4 else codes, scales[ids] if pages > 4 else scales, chosen, row))
    cache.keep(ints([40]), ints([[5, 9]]), ints([2]), stream=st)
    small.keep(ints([40]), ints([[5, 9]]), ints([2]), stream=st)
    cache.copy(ints([n_pages - 1]), ints([140_000]), stream=st)
    torch.cuda.synchronize()
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    assert torch.equal(k[0, ids], small._arrays[0][0]) and torch.equal(v[0, ids], small._arrays[1][0])
    assert torch.equal(k[0, 140_000], k[0, n_pages - 1])


# ------------------------------------------------------------------------------------------- bounds and the choice of pages
def bounded(made, held, first=None, max_new=None):
    """codes and units by the library, checked against the plain ones."""
    import torch

    n, kv, dim = made.kd.shape[1], made.kd.shape[2], made.kd.shape[4]
    codes, scales = torch.full((n, kv, 2, dim), 99, dtype=torch.int8, device="cuda"), torch.full((n, kv), -1.0, device="cuda")
    first = [0] * len(held) if first is None else first
    made.cache.bounds(ints(first), ints(held), codes, scales, max_new=max(max(held, default=1), 1) if max_new is None else max_new, layer=made.layer,
                      stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    wc, ws = np.full((n, kv, 2, dim), 99, np.int8), np.full((n, kv), -1.0, np.float32)
    plain.bounds(made.k, made.tables, first, held, wc, ws)
    assert (codes.cpu().numpy() == wc).all() and (scales.cpu().numpy().view(np.uint32) == ws.view(np.uint32)).all()
    return codes, scales, wc, ws


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kv,held", [(1, [1]), (2, [16, 17, 15]), (8, [100, 1, 33, 0]), (3, [250])])
def test_bounds(backend, kind, dim, kv, held):
    made = Made(backend, kind, kv, dim, held, seed=kv + dim, layers=2, layer=1)
    bounded(made, held)
    for back in (1, 3, 20):  # the last positions only: whole pages are made again, others stay
        bounded(made, held, [max(0, n - back) for n in held], max_new=back)


def test_bounds_hold_and_odd_keys(backend):
    """code * unit is on the outer side of every key (to the rounding of a product and a division); keys that are no numbers, of no size or huge."""
    import torch

    made = Made(backend, "bf16", 2, 64, [64], seed=1)
    codes, scales, _, _ = bounded(made, [64])
    at = torch.from_numpy(made.tables[0]).cuda()
    k = made.kd[0, at].double()
    value = codes[at].double() * scales[at].double()[..., None, None]
    slack = scales[at].double()[..., None] * 127 * 2.0 ** -22
    assert (k.amax(2) <= value[:, :, 0] + slack).all() and (k.amin(2) >= value[:, :, 1] - slack).all()
    page = int(made.tables[0, 1])
    odd = made.k[page]
    odd[0, 3, 5], odd[0, :, 7], odd[1, 2, 9], odd[1, 4, 10], odd[1, 5, 11] = np.nan, np.nan, np.inf, -np.inf, 3e38
    odd[0, :, 20] = 0.0
    other = int(made.tables[0, 2])
    made.k[other] = 0.0
    for p in (page, other):
        made.kd[0, p] = device16(plain.to16(made.k[p], "bf16")[1], "bf16")
    made.k[page] = float64(made.kd[0, page])
    bounded(made, [64])


def choose(made, q, codes, scales, host, n_pos, n, keep_first=0, keep_last=0, row_seq=None, max_pos=None):
    import torch

    qv, qd = q
    rows, kv = qv.shape[0], made.k.shape[1]
    chosen = torch.full((rows, kv, n), -7, dtype=torch.int32, device="cuda")
    made.cache.select(qd, codes, scales, ints(n_pos), chosen, max_pos=max(n_pos) if max_pos is None else max_pos, keep_first=keep_first, keep_last=keep_last,
                      row_seq=None if row_seq is None else ints(row_seq), stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    seq = list(range(rows)) if row_seq is None else row_seq
    want = plain.select(qv, host[0], host[1], made.tables, n_pos, n, keep_first, keep_last, seq, kv)
    got = chosen.cpu().numpy()
    assert (got == want).all(), np.argwhere(got != want)[:5]
    return chosen, want


def queries(made, rows, group, std=1.5):
    v, b = plain.bits16((rows, made.k.shape[1] * group, made.k.shape[3]), made.r, made.kind, std)
    return v, device16(b, made.kind)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kv,group,held,n,keep", [
    (1, 1, [1], 1, (0, 0)), (2, 4, [400, 33, 160], 5, (1, 2)), (8, 4, [700], 12, (0, 1)), (1, 16, [333, 300, 16, 17], 4, (2, 2)), (2, 7, [1000, 20], 30, (3, 0)), (1, 3, [2000], 1, (0, 0)),
    (2, 8, [500] * 9, 8, (1, 1)), (2, 4, [64, 3], 128, (1, 2)), (1, 12, [1500, 1400], 70, (5, 9))])
def test_chosen_pages_and_their_attention(backend, kind, dim, kv, group, held, n, keep):
    import torch

    made = Made(backend, kind, kv, dim, held, seed=n + dim)
    codes, scales, wc, ws = bounded(made, held)
    q = queries(made, len(held), group)
    chosen, want = choose(made, q, codes, scales, (wc, ws), held, n, *keep)
    out = torch.full_like(q[1], 3.0)
    made.cache.attention(q[1], chosen, ints(held), 0.11, out, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    o, tol = plain.listed(q[0], made.k, made.v, made.tables, held, want, 0.11, range(len(held)), tolerance(kind, dim))
    check(float64(out), o, tol, kind)


def test_rows_of_a_portion_and_rows_of_no_sequence(backend):
    """Several rows of one sequence, each with the positions before it, as the tokens of a prompt's portion have them."""
    import torch

    held = [300, 90]
    made = Made(backend, "bf16", 2, 128, held, seed=8)
    codes, scales, wc, ws = bounded(made, held)
    row_seq, n_pos = [0, 0, 0, 1, -1, 1, 2, 0], [300, 299, 17, 90, 50, 1, 40, 0]
    q = queries(made, len(row_seq), 4)
    chosen, want = choose(made, q, codes, scales, (wc, ws), n_pos, 6, 1, 1, row_seq)
    out = torch.full_like(q[1], 3.0)
    made.cache.attention(q[1], chosen, ints(n_pos), 0.09, out, row_seq=ints(row_seq), stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    o, tol = plain.listed(q[0], made.k, made.v, made.tables, n_pos, want, 0.09, row_seq, tolerance("bf16", 128))
    check(float64(out), o, tol, "bf16")
    assert (out[4] == 0).all() and (out[6] == 0).all() and (out[7] == 0).all()


def test_equal_scores_go_to_the_first_pages(backend):
    import torch

    held = [80 * PAGE]
    made = Made(backend, "f16", 1, 64, held, seed=1)
    for group in ([3, 9, 10, 41], [5, 6, 7, 70], list(range(20, 36))):  # the same keys on several pages
        for p in group[1:]:
            made.kd[0, made.tables[0, p]] = made.kd[0, made.tables[0, group[0]]]
            made.k[made.tables[0, p]] = made.k[made.tables[0, group[0]]]
    codes, scales, wc, ws = bounded(made, held)
    for n in (1, 2, 7, 20, 33, 64, 79):
        for seed in range(3):
            choose(made, queries(made, 1, 2), codes, scales, (wc, ws), held, n)
    # every score the same
    q = np.zeros((1, 2, 64)), torch.zeros((1, 2, 64), dtype=torch.float16, device="cuda")
    for n in (1, 31, 32, 33, 79):
        _, want = choose(made, q, codes, scales, (wc, ws), held, n, 0, 1 if n > 1 else 0)
        assert want[0, 0, 0] == 0


@pytest.mark.parametrize("rows,pages,n", [(1, 5000, 128), (1, 9001, 1), (3, 700, 600), (40, 300, 20), (1, 129, 128), (2, 40000, 2000)])
def test_choice_among_many_pages(backend, rows, pages, n):
    """Clusters of one to eight CTAs; the bounds are random, as no keys have to be there for the choice."""
    import torch

    from orangu_b200 import PagedCache

    r = np.random.default_rng(pages)
    kv, group, dim = 2, 4, 64
    x = torch.zeros((1, pages, kv, PAGE, dim), dtype=torch.float16, device="cuda")
    tables = np.stack([r.permutation(pages) for _ in range(rows)])
    made = type("M", (), {})()
    made.cache, made.tables, made.k, made.r, made.kind = PagedCache(backend, x, x.clone(), ints(tables)), tables, np.zeros((1, kv, PAGE, dim)), r, "f16"
    hi = r.integers(-127, 128, (pages, kv, 1, dim))
    wc = np.concatenate([hi, np.minimum(hi, r.integers(-127, 128, hi.shape))], 2).astype(np.int8)
    ws = (r.random((pages, kv)) * 0.01 + 0.01).astype(np.float32)
    ws[::7] = 0.0
    n_pos = [pages * PAGE - int(v) for v in r.integers(0, 40, rows)]
    for std in (1.5, 1e-7, 60000.0):
        choose(made, queries(made, rows, group, std), torch.from_numpy(wc).cuda(), torch.from_numpy(ws).cuda(), (wc, ws), n_pos, n, 1 if n > 1 else 0, 0)


def test_more_rows_than_the_workspace_holds_scores_for(backend):
    """3000 rows of 8 heads and 700 pages are scored in two batches: the lists of the same rows in calls of their own."""
    import torch

    from orangu_b200 import PagedCache

    r = np.random.default_rng(5)
    rows, pages, kv, dim, n = 3000, 700, 8, 64, 24
    x = torch.randn((1, pages, kv, PAGE, dim), device="cuda").half()
    cache = PagedCache(backend, x, x.clone(), ints([r.permutation(pages)]))
    st = torch.cuda.current_stream().cuda_stream
    codes, scales = torch.zeros((pages, kv, 2, dim), dtype=torch.int8, device="cuda"), torch.zeros((pages, kv), device="cuda")
    cache.bounds(ints([0]), ints([pages * PAGE]), codes, scales, max_new=pages * PAGE, stream=st)
    q = torch.randn(rows, kv * 2, dim, device="cuda").half()
    seq, n_pos = ints([0] * rows), ints(r.integers(1, pages * PAGE + 1, rows))
    whole = torch.full((rows, kv, n), -9, dtype=torch.int32, device="cuda")
    parts = torch.full_like(whole, -8)
    cache.select(q, codes, scales, n_pos, whole, max_pos=pages * PAGE, keep_last=2, row_seq=seq, stream=st)
    for a in range(0, rows, 700):
        cache.select(q[a:a + 700], codes, scales, n_pos[a:a + 700], parts[a:a + 700], max_pos=pages * PAGE, keep_last=2, row_seq=seq[a:a + 700], stream=st)
    out = torch.empty_like(q)
    cache.attention(q, whole, n_pos, 0.125, out, row_seq=seq, stream=st)
    torch.cuda.synchronize()
    assert torch.equal(whole, parts)
    k, v, table = float64(x[0]), float64(x[0]), cache._arrays[2].cpu().numpy()
    some = [0, 1, 1333, 2998, 2999]
    lists, lens = whole.cpu().numpy(), n_pos.cpu().numpy()
    o, tol = plain.listed(float64(q)[some], k, v, table, lens[some], lists[some], 0.125, [0] * len(some), tolerance("f16", dim))
    check(float64(out)[some], o, tol, "f16")


def test_odd_queries_and_pages_that_are_not_there(backend):
    held = [600]
    made = Made(backend, "bf16", 1, 64, held, seed=12)
    codes, scales, wc, ws = bounded(made, held)
    for entry, number in ((4, -1), (5, 10 ** 9), (37, -5)):
        made.tables[0, entry] = number
    made.td.copy_(ints(made.tables))
    for value in (np.nan, np.inf, -np.inf, 3e38, 0.0):
        q = plain.bits16((1, 4, 64), made.r, "bf16")[0]
        q[0, 1, 5], q[0, 2] = value, value
        qv, qb = plain.to16(q, "bf16")
        choose(made, (qv, device16(qb, "bf16")), codes, scales, (wc, ws), held, 9, 1, 2)
        choose(made, (qv, device16(qb, "bf16")), codes, scales, (wc, ws), held, 37, 0, 0)  # one of the three has to be taken: the first


def test_lists_of_any_kind(backend):
    """Pages in any order, twice, outside the sequence, past its end; long lists of few rows are cut into stretches."""
    import torch

    held = [1000, 333]
    made = Made(backend, "f16", 2, 128, held, seed=4, stride=200)
    q = queries(made, 2, 4)
    lists = np.full((2, 2, 180), -1, np.int64)
    lists[0, 0, :9] = [5, 0, 62, 61, 5, 500, -3, 199, 2]
    lists[0, 1] = np.arange(180) % 63
    lists[1, 0, 170:] = 20  # the last, partly filled page ten times
    out = torch.full_like(q[1], 3.0)
    made.cache.attention(q[1], ints(lists), ints(held), 0.1, out, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    o, tol = plain.listed(q[0], made.k, made.v, made.tables, held, lists, 0.1, [0, 1], tolerance("f16", 128))
    check(float64(out), o, tol, "f16")
    assert (out[1, 4:] == 0).all()


def test_all_pages_are_the_whole_attention(backend):
    """With room for every page the result is the operator of the dense kind, ob_attention_decode."""
    import torch

    held = [777]
    made = Made(backend, "f16", 2, 64, held, seed=6)
    codes, scales, wc, ws = bounded(made, held)
    q = queries(made, 1, 4)
    chosen, want = choose(made, q, codes, scales, (wc, ws), held, 49)
    out = torch.empty_like(q[1])
    made.cache.attention(q[1], chosen, ints(held), 0.125, out, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    k, _ = plain.positions(made.k, made.tables[0], 777, made.kd.shape[1])
    v, _ = plain.positions(made.v, made.tables[0], 777, made.kd.shape[1])
    dense = backend.attention_decode(q[0].astype(np.float32), k.reshape(777, -1), v.reshape(777, -1), 8, 2, 64, 0.125, exact_order=False).reshape(1, 8, 64)
    assert np.abs(float64(out) - dense).max() < 2.0 ** -11 * 4 * (1 + np.abs(dense).max())  # this side's output and weights are rounded to f16


# ------------------------------------------------------------------------------------------- moves
def whole(t):
    return t.view(dtype=__import__("torch").int16).cpu().numpy()


@pytest.mark.parametrize("layers,kv,dim,n", [(1, 1, 64, 1), (3, 2, 128, 5), (2, 8, 128, 40), (2, 3, 64, 17)])
def test_copies_of_pages(backend, layers, kv, dim, n):
    import torch

    made = Made(backend, "bf16", kv, dim, [n * PAGE], seed=n, layers=layers, spare=n + 3)
    src, dst = made.tables[0, :n].copy(), made.free[:n].copy()
    want = [whole(x).copy() for x in (made.kd, made.vd)]
    if n > 4:
        src[1], dst[2], src[3], dst[4] = -1, 1 << 30, made.kd.shape[1], src[4]
    for a, b in zip(src, dst):
        if 0 <= a < made.kd.shape[1] and 0 <= b < made.kd.shape[1]:
            for w in want:
                w[:, b] = w[:, a]
    made.cache.copy(ints(src), ints(dst), stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert (whole(made.kd) == want[0]).all() and (whole(made.vd) == want[1]).all()


@pytest.mark.parametrize("layers,kv,dim,n_pos", [(1, 1, 64, [5]), (2, 2, 128, [16, 33, 0, 47]), (3, 8, 64, [100, 99])])
def test_forks(backend, layers, kv, dim, n_pos):
    import torch

    children = len(n_pos)
    made = Made(backend, "f16", kv, dim, [100, 60], seed=children, layers=layers, spare=children, seqs=2 + children)
    parent = [i % 2 if n <= 60 else 0 for i, n in enumerate(n_pos)]
    child = list(range(2, 2 + children))
    want = [whole(x).copy() for x in (made.kd, made.vd)]
    tables = made.tables.copy()
    for p, c, n, f in zip(parent, child, n_pos, made.free):
        tables[c, :n // PAGE] = tables[p, :n // PAGE]
        if n % PAGE:
            tables[c, n // PAGE] = f
            for w in want:
                w[:, f] = w[:, tables[p, n // PAGE]]
    made.cache.fork(ints(parent + [0, 9, 1]), ints(child + [0, 1, 77]), ints(n_pos + [50, 50, 50]), ints(list(made.free[:children]) + [0, 0, 0]), stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()  # (the three at the end name no child or no parent)
    assert (made.td.cpu().numpy() == tables).all()
    assert (whole(made.kd) == want[0]).all() and (whole(made.vd) == want[1]).all()


@pytest.mark.parametrize("layers,kv,dim", [(1, 1, 64), (2, 8, 128), (33, 3, 64)])
@pytest.mark.parametrize("kept", [[[0]], [[1, 3, 4], [], [63]], [list(range(64)), list(range(63, -1, -1))], [[5, 5, 2, 0, 1, 5], [2, 70, -1, 3]]])
def test_kept_positions(backend, layers, kv, dim, kept):
    import torch

    ctx = [20 + 13 * i for i in range(len(kept))]
    made = Made(backend, "bf16", kv, dim, [c + 64 for c in ctx], seed=layers, layers=layers)
    width = max(map(len, kept)) or 1
    lists = np.full((len(kept), width), 7, np.int64)
    want = [whole(x).copy() for x in (made.kd, made.vd)]
    for s, path in enumerate(kept):
        lists[s, :len(path)] = path
        for w in want:
            old = w.copy()
            for j, i in enumerate(path):
                if 0 <= i < 64:
                    a, b = ctx[s] + i, ctx[s] + j
                    w[:, made.tables[s, b // PAGE], :, b % PAGE] = old[:, made.tables[s, a // PAGE], :, a % PAGE]
    made.cache.keep(ints(ctx), ints(lists), ints([len(p) for p in kept]), stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert (whole(made.kd) == want[0]).all() and (whole(made.vd) == want[1]).all()


def test_kept_positions_that_are_not_there(backend):
    import torch

    made = Made(backend, "f16", 2, 64, [64, 40], seed=1)
    made.tables[0, 2], made.tables[1, 0] = -1, 1 << 29
    made.td.copy_(ints(made.tables))
    want = [whole(x).copy() for x in (made.kd, made.vd)]
    for w in want:
        w[:, made.tables[0, 3], :, 0] = w[:, made.tables[0, 3], :, 9]  # position 48 <- 57; 32 .. 47 are not there; 64 on are past the table
    made.cache.keep(ints([30, 2 ** 31 - 1]), ints([[5, 40, 3] + [4] * 15 + [27], [0] * 19]), ints([19, 500]), stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for w, x in zip(want, (made.kd, made.vd)):
        got = whole(x)
        # positions 30 and 31: from 35 (not there) and 70 (past the table); 32 .. 47 have no place
        assert (got == w).all()


# ------------------------------------------------------------------------------------------- as they are used together
def test_a_round_of_drafting(backend):
    """A sequence forks, a tree of drafts is attended, the accepted path moves together, and the next tokens, dense and over chosen pages, see what a cache
    that was filled token by token holds."""
    import torch

    dim, kv, group, ctx, drafts = 64, 2, 4, 200, 12
    path = [1, 4, 7, 11]
    made = Made(backend, "f16", kv, dim, [ctx + drafts], seed=77, spare=8, seqs=2, stride=20)
    st = torch.cuda.current_stream().cuda_stream
    n_pos = ctx + drafts
    made.cache.fork(ints([0]), ints([1]), ints([n_pos]), ints(made.free[:1]), stream=st)
    bits = [0] * drafts
    seen = 0
    for i in range(drafts):
        bits[i] = 1 << i
    for i in path:
        seen |= 1 << i
        bits[i] = seen
    q = queries(made, drafts, group)
    out = torch.empty_like(q[1])
    first, tables = [0, 0, drafts], None
    made.cache.attention_tree(q[1], ints(first), ints([ctx, ctx]), words(bits), 0.125, out, max_drafts=drafts, max_context=ctx, stream=st)
    # pages of the child that the move writes have to be its own: those from the context's last page on
    own = made.free[1:4]
    made.cache.copy(made.td[1, ctx // PAGE:ctx // PAGE + 1].clone(), ints(own[:1]), stream=st)
    torch.cuda.synchronize()
    made.td[1, ctx // PAGE] = int(own[0])
    made.cache.keep(ints([ctx, ctx]), ints([[0] * 4, path]), ints([0, 4]), stream=st)
    torch.cuda.synchronize()
    made.tables = made.td.cpu().numpy().astype(np.int64)
    want = np.zeros(q[0].shape)
    base = made.tables[0]
    tol = plain.tree(q[0], made.k, made.v, np.stack([base, base]), first, [ctx, ctx], bits, 0.125, want, tolerance("f16", dim))
    check(float64(out), want, tol, "f16")
    # the cache token by token: context, then the path
    pool = [np.concatenate([x, np.zeros_like(x[:16])]) for x in (made.k, made.v)]
    n = made.k.shape[0]
    table = list(range(n, n + 14))
    for x in pool:
        for p in range(ctx + 4):
            src = p if p < ctx else ctx + path[p - ctx]
            x[table[p // PAGE], :, p % PAGE] = x[base[src // PAGE], :, src % PAGE]
    held = ctx + 4
    codes = torch.zeros((made.kd.shape[1], kv, 2, dim), dtype=torch.int8, device="cuda")
    scales = torch.zeros((made.kd.shape[1], kv), device="cuda")
    made.cache.bounds(ints([0, 0]), ints([0, held]), codes, scales, max_new=held, stream=st)
    q1 = queries(made, 1, group)
    for pages in (13, 5):
        chosen = torch.empty((1, kv, pages), dtype=torch.int32, device="cuda")
        row = torch.empty_like(q1[1])
        made.cache.select(q1[1], codes, scales, ints([held]), chosen, max_pos=held, keep_last=1, row_seq=ints([1]), stream=st)
        made.cache.attention(q1[1], chosen, ints([held]), 0.125, row, row_seq=ints([1]), stream=st)
        torch.cuda.synchronize()
        lists = chosen.cpu().numpy()
        assert (lists >= 0).all() and (lists[..., -1] == 12).all()
        o, tol = plain.listed(q1[0], pool[0], pool[1], [table], [held], lists, 0.125, [0], tolerance("f16", dim))
        check(float64(row), o, tol, "f16")


def test_streams_captures_and_handles_side_by_side(backend):
    """Two handles of the same pages on two streams at a time; a captured round replayed with other inputs in the same memory."""
    import torch

    from orangu_b200 import PagedCache

    held = [3000, 1200]
    made = Made(backend, "bf16", 2, 128, held, seed=31)
    codes, scales, wc, ws = bounded(made, held)
    handles = [made.cache, PagedCache(backend, made.kd, made.vd, made.td)]
    streams = [torch.cuda.Stream() for _ in handles]
    lens, first, bits = ints(held), ints([0, 6, 10]), words([(1 << i % 6 + 1) - 1 for i in range(10)])
    ctx = ints([n - 8 for n in held])

    def once(cache, q, chosen, row, out, st):
        cache.select(q[:2], codes, scales, lens, chosen, max_pos=3000, keep_first=1, keep_last=1, stream=st)
        cache.attention(q[:2], chosen, lens, 0.1, row, stream=st)
        cache.attention_tree(q, first, ctx, bits, 0.1, out, max_drafts=6, max_context=2992, stream=st)

    def buffers():
        q = torch.randn(10, 8, 128, device="cuda").bfloat16()
        return q, torch.empty((2, 2, 40), dtype=torch.int32, device="cuda"), torch.empty_like(q[:2]), torch.empty_like(q)

    sets = [buffers() for _ in handles]
    alone = []
    for b in sets:
        once(made.cache, *b, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        alone.append([x.clone() for x in b[1:]])
        for x in b[1:]:
            x.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for h, s, b in zip(handles, streams, sets):
            once(h, *b, s.cuda_stream)
    torch.cuda.synchronize()
    for b, a in zip(sets, alone):
        assert all(torch.equal(x, y) for x, y in zip(b[1:], a))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        once(made.cache, *sets[0], torch.cuda.current_stream().cuda_stream)
    for k in (1, 0, 1):
        sets[0][0].copy_(sets[k][0] if k else sets[0][0])
        for x in sets[0][1:]:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(sets[0][1:], alone[1]))


# ------------------------------------------------------------------------------------------- refusals
def test_refusals(backend):
    import torch

    from orangu_b200 import OranguError, PagedCache, capi

    L, st = backend._lib, None
    x = torch.zeros((2, 4, 2, PAGE, 64), dtype=torch.float16, device="cuda")
    t = ints([[0, 1], [2, 3]])

    def made(**change):
        d = dict(k=x.data_ptr(), v=x.data_ptr(), layer_stride=x[0].numel(), type=1, n_layer=2, n_pages=4, n_head_kv=2, head_dim=64, n_seq=2, table_stride=2, tables=t.data_ptr())
        d.update(change)
        desc, h = capi.PagesDesc(**d), C.c_void_p()
        rc = L.ob_pages_create(backend._h, C.byref(desc), C.byref(h))
        if rc == 0:
            L.ob_pages_destroy(h)
        else:
            assert not h.value
        return rc

    assert made() == 0 and made(type=30) == 0
    host = torch.zeros(1 << 16, dtype=torch.float16)
    for change, rc in ((dict(type=0), -2), (dict(type=12), -2), (dict(head_dim=96), -2), (dict(head_dim=0), -2), (dict(n_pages=0), -1), (dict(n_layer=0), -1), (dict(n_head_kv=0), -1),
                       (dict(n_seq=0), -1), (dict(table_stride=0), -1), (dict(table_stride=1 << 28), -2), (dict(n_layer=20000), -2), (dict(n_head_kv=5000), -2), (dict(n_pages=1 << 31), -2),
                       (dict(layer_stride=8), -1), (dict(layer_stride=x[0].numel() + 4), -1), (dict(k=None), -1), (dict(tables=None), -1), (dict(v=x.data_ptr() + 2), -1),
                       (dict(k=host.data_ptr()), -1), (dict(tables=host.data_ptr()), -1)):
        assert made(**change) == rc, change
    assert L.ob_pages_create(None, None, None) == -1 and L.ob_pages_copy(None, 0, None, None, None) == -1
    L.ob_pages_destroy(None)

    cache = PagedCache(backend, x, x.clone(), t)
    q = torch.zeros((6, 4, 64), dtype=torch.float16, device="cuda")
    out = torch.full_like(q, 9.0)
    first, ctx, bits, lens = ints([0, 2, 6]), ints([3, 4]), words([1] * 6), ints([5] * 6)
    h, p = cache._h, lambda a: a.data_ptr()

    def tree(**change):
        a = dict(layer=0, n_seq=2, q=p(q), qs=256, n=6, first=p(first), ctx=p(ctx), bits=p(bits), heads=4, most=4, max_ctx=4, scale=0.1, out=p(out), os=256, st=st)
        a.update(change)
        return L.ob_pages_attention_tree(h, *a.values())

    assert tree() == 0 and tree(n_seq=0) == 0 and tree(n=0) == 0 and tree(most=0) == 0
    for change, rc in ((dict(layer=2), -1), (dict(n_seq=3), -1), (dict(heads=3), -1), (dict(heads=0), -1), (dict(heads=34, qs=34 * 64, os=34 * 64), -2), (dict(most=65), -2), (dict(scale=0.0), -1),
                       (dict(scale=-1.0), -1), (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1), (dict(qs=248), -1), (dict(os=260), -1), (dict(q=None), -1), (dict(q=p(q) + 2), -1),
                       (dict(out=p(out) + 8), -1), (dict(first=None), -1), (dict(bits=p(bits) + 4), -1), (dict(ctx=host.data_ptr()), -1), (dict(q=host.data_ptr()), -1), (dict(n=1 << 31), -1)):
        assert tree(**change) == rc, change
    codes, scales, chosen = torch.zeros((4, 2, 2, 64), dtype=torch.int8, device="cuda"), torch.zeros((4, 2), device="cuda"), torch.zeros((2, 2, 2), dtype=torch.int32, device="cuda")

    def select(**change):
        a = dict(codes=p(codes), scales=p(scales), n=2, q=p(q), qs=256, seq=None, n_pos=p(lens), heads=4, max_pos=32, n_select=2, first=1, last=1, chosen=p(chosen), st=st)
        a.update(change)
        return L.ob_pages_select(h, *a.values())

    assert select() == 0 and select(n=0) == 0 and select(max_pos=0) == 0
    for change, rc in ((dict(n=3), -1), (dict(heads=5), -1), (dict(n_select=0), -1), (dict(n_select=131073), -1), (dict(first=2), -1), (dict(first=0xffffffff, last=1), -1), (dict(codes=p(codes) + 1), -1),
                       (dict(scales=None), -1), (dict(seq=host.data_ptr()), -1), (dict(chosen=None), -1), (dict(qs=4), -1)):
        assert select(**change) == rc, change

    def attention(**change):
        a = dict(layer=1, n=2, q=p(q), qs=256, seq=None, n_pos=p(lens), heads=4, chosen=p(chosen), n_select=2, scale=0.1, out=p(out), os=256, st=st)
        a.update(change)
        return L.ob_pages_attention(h, *a.values())

    assert attention() == 0 and attention(n=0) == 0
    for change, rc in ((dict(layer=2), -1), (dict(n=3), -1), (dict(heads=0), -1), (dict(n_select=0), -1), (dict(n_select=131073), -1), (dict(scale=0.0), -1), (dict(chosen=None), -1), (dict(os=100), -1)):
        assert attention(**change) == rc, change
    i = p(lens)
    assert L.ob_pages_bounds(h, 0, 2, i, i, 4, p(codes), p(scales), st) == 0 and L.ob_pages_bounds(h, 0, 2, i, i, 0, p(codes), p(scales), st) == 0
    assert L.ob_pages_bounds(h, 2, 2, i, i, 4, p(codes), p(scales), st) == -1 and L.ob_pages_bounds(h, 0, 3, i, i, 4, p(codes), p(scales), st) == -1
    assert L.ob_pages_bounds(h, 0, 2, None, i, 4, p(codes), p(scales), st) == -1 and L.ob_pages_bounds(h, 0, 2, i, i, 4, p(codes) + 1, p(scales), st) == -1
    assert L.ob_pages_copy(h, 1, None, i, st) == -1 and L.ob_pages_copy(h, 0, None, None, st) == 0 and L.ob_pages_copy(h, 1 << 31, i, i, st) == -1
    assert L.ob_pages_fork(h, 1, i, i, i, None, st) == -1 and L.ob_pages_fork(h, 0, None, None, None, None, st) == 0
    assert L.ob_pages_keep(h, 3, i, i, 2, i, st) == -1 and L.ob_pages_keep(h, 2, i, i, 65, i, st) == -1 and L.ob_pages_keep(h, 2, i, i, 0, i, st) == -1 and L.ob_pages_keep(h, 2, i, None, 2, i, st) == -1
    backend.synchronize()
    # shapes and types in Python
    with pytest.raises(ValueError):
        PagedCache(backend, x.float(), x.float(), t)
    with pytest.raises(ValueError):
        PagedCache(backend, x, x[:1], t)
    with pytest.raises(ValueError):
        PagedCache(backend, x, x, t.long())
    with pytest.raises(ValueError):
        cache.attention_tree(q, first, ctx, bits[:5], 0.1, out, 4, 4)
    with pytest.raises(ValueError):
        cache.attention_tree(q, first, ctx, bits, 0.1, out[:5], 4, 4)
    with pytest.raises(ValueError):
        cache.attention_tree(q.bfloat16(), first, ctx, bits, 0.1, out, 4, 4)
    with pytest.raises(ValueError):
        cache.attention(q[:2], chosen[:, :1], lens[:2], 0.1, out[:2])
    with pytest.raises(OranguError):
        cache.attention(q, torch.zeros((6, 2, 2), dtype=torch.int32, device="cuda"), lens, 0.1, out)  # six rows, two tables
    with pytest.raises(OranguError):
        cache.copy(torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))  # host memory


def test_a_walk_of_more_than_31_bits_is_refused(backend):
    """Every (rows, sequence, head) piece counts as its tiles and six more: 2^22 sequences of one tile of 64 heads, in four tiles of 128 rows, are 7 2^30."""
    import torch

    from orangu_b200 import OranguError, PagedCache

    n_seq, heads = 1 << 22, 64
    k = torch.zeros((1, 1, heads, PAGE, 64), dtype=torch.float16, device="cuda")
    cache = PagedCache(backend, k, k.clone(), torch.zeros((n_seq, 1), dtype=torch.int32, device="cuda"))
    q = torch.zeros((1, heads * 16, 64), dtype=torch.float16, device="cuda")
    first, ctx = torch.zeros(n_seq + 1, dtype=torch.int32, device="cuda"), torch.zeros(n_seq, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 9.0)
    with pytest.raises(OranguError, match="too many positions"):
        cache.attention_tree(q, first, ctx, words([1]), 0.1, out, 32, 16)
    cache.attention_tree(q, first[:1025], ctx[:1024], words([1]), 0.1, out, 32, 16)  # (no tokens: nothing is written)
    torch.cuda.synchronize()
    assert bool((out == 9.0).all())
