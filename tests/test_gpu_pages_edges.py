"""Operators over the pages of a caller's cache at the edges of what they allow: equal scores, numbers that are none, long contexts, large tables, calls that
are captured first and replayed with other lengths, handles that outlive their context."""
import numpy as np
import pytest

import pages_plain as plain
from gpu_common import backend  # noqa: F401
from test_gpu_pages import PAGE, Made, check, device16, float64, ints, random_tree, run_tree, tolerance, words

pytestmark = pytest.mark.gpu


def current():
    import torch

    return torch.cuda.current_stream().cuda_stream


# ------------------------------------------------------------------------------------------- equal scores
class Bounds:
    """Bounds of `pages` pages for a choice alone; no keys have to be there for it."""

    def __init__(self, be, rows, pages, kv, dim, seed, kind="f16"):
        import torch

        from orangu_b200 import PagedCache

        self.r, self.kind, self.kv, self.dim = np.random.default_rng(seed), kind, kv, dim
        x = torch.zeros((1, pages, kv, PAGE, dim), dtype=torch.float16 if kind == "f16" else torch.bfloat16, device="cuda")
        self.tables = np.stack([self.r.permutation(pages) for _ in range(rows)])
        self.cache = PagedCache(be, x, x.clone(), ints(self.tables))
        hi = self.r.integers(-127, 128, (pages, kv, 1, dim))
        self.codes = np.concatenate([hi, np.minimum(hi, self.r.integers(-127, 128, hi.shape))], 2).astype(np.int8)
        self.scales = (self.r.random((pages, kv)) * 0.01 + 0.01).astype(np.float32)

    def choose(self, group, n_pos, n, keep_first, keep_last, zero=(), rounds=1):
        """Lists of random queries, those of the rows in `zero` all zero: equal scores."""
        import torch

        rows = len(n_pos)
        qv, qb = plain.bits16((rows, self.kv * group, self.dim), self.r, self.kind, 1.5)
        for row in zero:
            qv[row], qb[row] = 0.0, 0
        q = torch.from_numpy(qb.view(np.int16)).cuda().view(torch.float16 if self.kind == "f16" else torch.bfloat16)
        codes, scales, lens = torch.from_numpy(self.codes).cuda(), torch.from_numpy(self.scales).cuda(), ints(n_pos)
        want = plain.select(qv, self.codes, self.scales, self.tables, n_pos, n, keep_first, keep_last, list(range(rows)), self.kv)
        for _ in range(rounds):
            chosen = torch.full((rows, self.kv, n), -7, dtype=torch.int32, device="cuda")
            self.cache.select(q, codes, scales, lens, chosen, max_pos=max(n_pos), keep_first=keep_first, keep_last=keep_last, stream=current())
            torch.cuda.synchronize()
            assert (chosen.cpu().numpy() == want).all()


# (one kernel; two, 256 threads; two, 1024 threads)
@pytest.mark.parametrize("rows,pages,n", [(3, 3, 1), (2, 40, 7), (4, 500, 64), (160, 12, 5), (2, 700, 100), (1, 4500, 128)])
@pytest.mark.parametrize("keep", [(0, 0), (1, 2)])
def test_rows_of_zeros_among_others(backend, rows, pages, n, keep):
    """Padded rows of a batch: all of their scores are equal, their lists the first pages."""
    b = Bounds(backend, rows, pages, 2, 64, seed=rows + pages)
    n = max(n, sum(keep))
    n_pos = [pages * PAGE - int(v) for v in b.r.integers(0, 16, rows)]
    for zero in (range(rows), range(0, rows, 2)):
        b.choose(4, n_pos, n, *keep, zero=zero, rounds=20)
    b.scales[:] = 0.0  # bounds of a cache of zeros
    b.choose(4, n_pos, n, *keep)


@pytest.mark.parametrize("kind,dim", [("f16", 64), ("bf16", 128)])
@pytest.mark.parametrize("group", [9, 16])
def test_many_heads_scored_by_a_kernel_of_their_own(backend, kind, dim, group):
    """More than eight query heads a key/value head, rows of more pages than one CTA scores for itself."""
    b = Bounds(backend, 3, 900, 2, dim, seed=group + dim, kind=kind)
    b.choose(group, [900 * PAGE, 600 * PAGE - 3, 40], 30, 1, 2, zero=[1])


# ------------------------------------------------------------------------------------------- rows that are no numbers
FORMS = [(4, 3), (4, 20), (8, 40)]  # group, drafted tokens: up to 16 rows a key/value head, up to 128, more


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("group,drafts", FORMS)
@pytest.mark.parametrize("ctx", [[9, 21], [100] * 40, [0, 3000]])  # pieces of one tile, whole ones of several, cut ones
def test_a_query_that_is_no_number_has_no_result_and_no_neighbours(backend, kind, group, drafts, ctx):
    import torch

    made = Made(backend, kind, 2, 64, [c + drafts for c in ctx], seed=drafts)
    n = drafts * len(ctx)
    q = torch.randn(n, 2 * group, 64, device="cuda").to(made.kd.dtype)
    bits = words([b for _ in ctx for b in random_tree(made.r, drafts)])
    first, lens = ints([drafts * i for i in range(len(ctx) + 1)]), ints(ctx)

    def run():
        out = torch.full_like(q, 5.0)
        made.cache.attention_tree(q, first, lens, bits, 0.125, out, max_drafts=drafts, max_context=max(ctx), stream=current())
        torch.cuda.synchronize()
        return out

    clean = run()
    odd = [0, drafts // 2, n - 1]
    others = [t for t in range(n) if t not in odd]
    q[odd, :, 5] = float("nan")
    out = run()
    assert torch.isnan(out[odd]).all() and torch.isfinite(clean).all()
    assert torch.equal(out[others], clean[others])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("group,drafts", FORMS)
def test_a_token_that_sees_only_a_key_that_is_no_number_has_no_result(backend, kind, group, drafts):
    import torch

    made = Made(backend, kind, 2, 64, [drafts], seed=drafts)
    made.kd[0, int(made.tables[0, 0]), :, 1, 7] = float("nan")  # drafted token 1
    bits = [1 << i if i != 1 else 1 for i in range(drafts)]     # every token sees itself, and
    bits[2] = 0b10                                              # one sees token 1 alone
    q = torch.randn(drafts, 2 * group, 64, device="cuda").to(made.kd.dtype)
    out = torch.full_like(q, 5.0)
    made.cache.attention_tree(q, ints([0, drafts]), ints([0]), words(bits), 0.125, out, max_drafts=drafts, max_context=0, stream=current())
    torch.cuda.synchronize()
    assert torch.isnan(out[2]).all()
    assert torch.isfinite(out[[t for t in range(drafts) if t != 2]]).all()


# ------------------------------------------------------------------------------------------- weights
def fine(kind, v, n, score):
    """Bound of an output's error but for its own rounding, where the products of queries and keys are exact: weights go in as value and remainder (f16 2^-22,
    bf16 2^-16), f16 ones of less than 2^-21 of the largest are off by 2^-32 of it at most; both in numerator and denominator.  A score's product with
    the scale's power of two has three roundings; 2^-20 covers 2^x and the online sums."""
    weight, tiny = (2.0 ** -22, 2.0 ** -32) if kind == "f16" else (2.0 ** -16, 0.0)
    return v * (2 * weight + 2 * n * tiny + 4 * 2.0 ** -24 * 1.5 * score + 2.0 ** -20)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("group,drafts", FORMS)
@pytest.mark.parametrize("ctx", [300, 2000])
def test_weights_have_more_bits_than_the_cache(backend, kind, group, drafts, ctx):
    """Keys and queries of -1, 0 and 1: scores are exact, and what is left is the weights'."""
    import torch

    made = Made(backend, kind, 1, 64, [ctx + drafts], seed=ctx)
    signs = lambda *s: made.r.integers(-1, 2, s).astype(np.float64)  # noqa: E731
    made.k[:] = signs(*made.k.shape)
    made.kd.copy_(torch.from_numpy(made.k)[None])
    q = signs(drafts, group, 64)
    qd = torch.from_numpy(q).cuda().to(made.kd.dtype)
    out = torch.empty_like(qd)
    bits = [(2 << i) - 1 for i in range(drafts)]
    made.cache.attention_tree(qd, ints([0, drafts]), ints([ctx]), words(bits), 0.125, out, max_drafts=drafts, max_context=ctx, stream=current())
    torch.cuda.synchronize()
    want = np.zeros(q.shape)
    tol = plain.tree(q, made.k, made.v, made.tables, [0, drafts], [ctx], bits, 0.125, want, lambda v, qk, n: fine(kind, v, n, qk))
    check(float64(out), want, tol, kind)
    # the same positions as a list of pages
    pages = -(-ctx // PAGE)
    lists = ints(np.arange(pages)[None, None])
    row = torch.empty_like(qd[:1])
    made.cache.attention(qd[:1], lists, ints([ctx]), 0.125, row, stream=current())
    torch.cuda.synchronize()
    o, tol = plain.listed(q[:1], made.k, made.v, made.tables, [ctx], lists.cpu().numpy(), 0.125, [0], lambda v, qk, n: fine(kind, v, n, qk))
    check(float64(row), o, tol, kind)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("group,drafts", FORMS)
@pytest.mark.parametrize("power,first_value", [(25.2, -1.0), (21.09, 0.0)])
def test_many_small_weights_behind_a_large_one(backend, kind, group, drafts, power, first_value):
    """131,000 positions whose weights are 2^-25.2 (2^-21.09) of the first one's: together a third (six) percent.  As many sequences as leave the pieces (nearly)
    whole, all of them of the same pages."""
    import torch

    from orangu_b200 import PagedCache

    kv, dim, n, rows = 8, 64, 131_000, group * drafts
    seqs = 64 if rows <= 16 else 24
    pages = -(-(n + drafts) // PAGE)
    dtype = torch.float16 if kind == "f16" else torch.bfloat16
    k = torch.zeros((1, pages, kv, PAGE, dim), dtype=dtype, device="cuda")
    v = torch.ones_like(k)
    k[0, 0, :, 0], v[0, 0, :, 0] = power * np.log(2.0) / 8, first_value  # (the score is 64 times that, and the scale)
    score = float(k[0, 0, 0, 0, 0]) * 64 * 0.125
    cache = PagedCache(backend, k, v, ints(np.tile(np.arange(pages), (seqs, 1))))
    q = torch.ones((seqs * drafts, kv * group, dim), dtype=dtype, device="cuda")
    out = torch.empty_like(q)
    first = ints([drafts * i for i in range(seqs + 1)])
    cache.attention_tree(q, first, ints([n] * seqs), words([1] * (seqs * drafts)), 0.125, out, max_drafts=drafts, max_context=n, stream=current())
    torch.cuda.synchronize()
    rest = n * np.exp(-score)  # the other n - 1 positions and drafted token 0
    want = (rest + first_value) / (rest + 1)
    # What sums in fp32 may lose in an accumulator that takes 16 products a step, values and remainders apart: the tensor cores align the 17 terms of a
    # step to the largest with two more bits than fp32 has and cut off the rest, then cut the sum off to fp32: 17/4 + 1 last places, relative to what
    # has been added up so far.  An accumulator has a quarter of the positions (four warps), half (two streams) or all of them.
    chain = n / (4 if rows <= 16 else 2 if rows <= 128 else 1) / 16 * 2 * (17 / 4 + 1) * 2.0 ** -23
    lost = chain * ((rest + abs(first_value)) / (rest + 1) + abs(want))  # in the numerator and in the denominator
    check(float64(out), np.full(out.shape, want), np.full(out.shape[:2], fine(kind, 1.0, n, score) + lost), kind)


# ------------------------------------------------------------------------------------------- large tables
def test_a_table_whose_pages_times_heads_pass_32_bits(backend):
    """2^26 places of a table, most of them empty, and 72 heads: 4.8 10^9 pages in a walk."""
    import torch

    from orangu_b200 import PagedCache

    stride, kv, dim = 1 << 26, 72, 64
    r = np.random.default_rng(1)
    k, kb = plain.bits16((5, kv, PAGE, dim), r, "f16")
    v, vb = plain.bits16((5, kv, PAGE, dim), r, "f16")
    places = {0: 2, 7: 4, (1 << 25) + 3: 0, (1 << 26) - 2: 3, (1 << 26) - 1: 1}
    table = torch.full((1, stride), -1, dtype=torch.int32, device="cuda")
    for at, page in places.items():
        table[0, at] = page
    cache = PagedCache(backend, device16(kb[None], "f16"), device16(vb[None], "f16"), table)
    q, qb = plain.bits16((2, kv, dim), r, "f16", 1.5)
    out = torch.full((2, kv, dim), 9.0, dtype=torch.float16, device="cuda")
    ctx = stride * PAGE - 2  # the last two positions are the drafted ones
    for _ in range(2):       # (the counters are zero again)
        out.fill_(9.0)
        cache.attention_tree(device16(qb, "f16"), ints([0, 2]), ints([ctx]), words([1, 3]), 0.125, out, max_drafts=2, max_context=ctx, stream=current())
        torch.cuda.synchronize()
        flat = lambda x: np.concatenate([x[p].transpose(1, 0, 2) for p in places.values()])  # noqa: E731  [positions, kv, dim]
        want, tol = np.zeros(q.shape), np.zeros(q.shape[:2])
        for t in range(2):
            seen = np.ones(len(places) * PAGE, bool)
            seen[len(seen) - 2:] = [True, t == 1]
            o, big, qk, n = plain.attend(q[t], flat(k), flat(v), seen, 0.125)
            want[t], tol[t] = o, tolerance("f16", dim)(big, qk, n)
        check(float64(out), want, tol, "f16")


# ------------------------------------------------------------------------------------------- handles and their context
def free_bytes():
    import torch

    torch.cuda.synchronize()
    return torch.cuda.mem_get_info()[0]


def tiny_cache(be):
    import torch

    from orangu_b200 import PagedCache

    k = torch.zeros((1, 2, 1, PAGE, 64), dtype=torch.float16, device="cuda")
    return PagedCache(be, k, k.clone(), ints([[0, 1]]))


def test_a_handle_outlives_its_context():
    import torch

    from orangu_b200 import CudaBackend, OranguError

    be = CudaBackend.init(0)
    cache, lib = tiny_cache(be), be._lib
    q, out = torch.zeros((1, 1, 64), dtype=torch.float16, device="cuda"), torch.full((1, 1, 64), 9.0, dtype=torch.float16, device="cuda")
    lens, i = ints([5]), ints([0])
    calls = [lambda: cache.attention_tree(q, ints([0, 1]), lens, words([1]), 0.1, out, 1, 5), lambda: cache.attention(q, ints([[[0]]]), lens, 0.1, out), lambda: cache.copy(i, ints([1])),
             lambda: cache.keep(lens, ints([[0]]), i), lambda: cache.fork(i, i, lens, i)]
    before = free_bytes()
    be.close()
    assert free_bytes() - before >= 64 << 20  # the workspace of a handle that is open goes with the context
    for call in calls:
        with pytest.raises(OranguError):
            call()
    torch.cuda.synchronize()
    assert (out == 9.0).all()
    cache.close()
    cache.close()
    lib.ob_pages_destroy(None)


def test_a_workspace_that_may_be_in_use_is_not_given_away():
    """While a stream is captured the device cannot be waited for: the destroyed handle's workspace stays out of use, and later ones are reused as ever."""
    import ctypes as C

    import torch

    from orangu_b200 import CudaBackend

    be = CudaBackend.init(0)
    one, two = tiny_cache(be), tiny_cache(be)
    rt = C.CDLL([line.split()[-1] for line in open("/proc/self/maps") if "libcudart" in line][0])
    stream = torch.cuda.Stream()
    graph = C.c_void_p()
    torch.cuda.synchronize()
    assert rt.cudaStreamBeginCapture(C.c_void_p(stream.cuda_stream), 2) == 0
    one.close()
    rt.cudaStreamEndCapture(C.c_void_p(stream.cuda_stream), C.byref(graph))
    rt.cudaGetLastError()
    two.close()
    was = free_bytes()
    three = tiny_cache(be)  # takes what `two` left
    assert was - free_bytes() < 32 << 20
    four = tiny_cache(be)
    assert was - free_bytes() >= 64 << 20
    three.close(), four.close()
    was = free_bytes()
    be.close()
    assert free_bytes() - was >= 3 * 64 << 20  # the first one's, too


def test_a_wait_that_ran_out_is_reported_by_its_handle(backend):
    """The word that a kernel leaves when it gives up a wait is the handle's own: seen on the caller's stream, once, whoever else synchronizes."""
    import torch

    from orangu_b200 import CudaBackend, OranguError, capi

    other = CudaBackend.init(0)
    a, b, elsewhere = tiny_cache(backend), tiny_cache(backend), tiny_cache(other)
    stream = torch.cuda.Stream()
    st = stream.cuda_stream
    for used in (st, 0):
        capi.check(backend._h, backend._lib.ob_pages_wait_selftest(a._h, used or 1))
        torch.cuda.synchronize()
        for c in (b, elsewhere):
            c.synchronize(used)
        other.synchronize()
        with pytest.raises(OranguError, match="gave up a bounded wait"):
            a.synchronize(used)
        a.synchronize(used)  # said once,
        with pytest.raises(OranguError, match="gave up a bounded wait"):
            backend.synchronize()  # and once for all handles of the context
        backend.synchronize()
    # replays leave no trace on the host but that word
    q, out = torch.ones((20, 4, 64), dtype=torch.float16, device="cuda"), torch.empty((20, 4, 64), dtype=torch.float16, device="cuda")
    first, ctx, bits = ints([0, 20]), ints([5]), words([1] * 20)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        a.attention_tree(q, first, ctx, bits, 0.1, out, 20, 5, stream=st)
        capi.check(backend._h, backend._lib.ob_pages_wait_selftest(a._h, st))
        with pytest.raises(OranguError, match="captured"):
            a.synchronize(st)  # and the capture goes on
    a.synchronize(st)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        with pytest.raises(OranguError, match="gave up a bounded wait"):
            a.synchronize(st)
    assert (out[0] == 0).all()  # (a cache of zeros)
    a.close()
    c = tiny_cache(backend)  # the workspace that `a` left: the word is clear
    c.synchronize(st)
    backend.synchronize()
    other.close()


# ------------------------------------------------------------------------------------------- captures
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("group,drafts", [(4, 4), (4, 30), (8, 40)])
def test_a_replay_goes_by_the_lengths_tables_and_masks_of_its_time(backend, kind, group, drafts):
    """One captured round (bounds, choice in one kernel and in two, attention over lists and of trees, kept positions) replayed with everything on the device
    rewritten: contexts beyond the captured bound, sequences without drafted tokens or without context, tables in another order."""
    import torch

    from orangu_b200 import PagedCache

    kv, dim, seqs, stride = 2, 64, 4, 700
    r = np.random.default_rng(drafts)
    dtype = torch.float16 if kind == "f16" else torch.bfloat16
    k = torch.randn((2, seqs * stride, kv, PAGE, dim), device="cuda").to(dtype)
    v = torch.randn_like(k)
    n = seqs * drafts

    def inputs(lens, counts, seed):
        g = np.random.default_rng(seed)
        first = np.concatenate([[0], np.cumsum(counts)])
        bits = [int(g.integers(0, 1 << 62)) for _ in range(n)]
        return dict(tables=ints(g.permutation(seqs * stride).reshape(seqs, stride)), first=ints(first), lens=ints(lens), bits=words(bits), held=ints([a + b for a, b in zip(lens, counts)]),
                    zeros=ints([0] * seqs), kept=ints(np.sort(g.integers(0, max(counts), (seqs, 3)), -1)), n_kept=ints([min(3, c) for c in counts]),
                    q=torch.randn((n, kv * group, dim), device="cuda").to(dtype))

    sets = [inputs([100, 60, 30, 17], [drafts] * seqs, 1), inputs([9000, 0, 5000, 16], [drafts, 1, 0, drafts // 2], 2), inputs([0, 11000, 1, 10000], [0, drafts, drafts, 2], 3),
            inputs([100, 60, 30, 17], [drafts] * seqs, 1)]
    live = {a: b.clone() for a, b in sets[0].items()}
    pool = [k.clone(), v.clone()]
    cache = PagedCache(backend, pool[0], pool[1], live["tables"])

    def outputs():
        return dict(tree=torch.zeros((n, kv * group, dim), dtype=dtype, device="cuda"), row=torch.zeros((seqs, kv * group, dim), dtype=dtype, device="cuda"),
                    few=torch.zeros((seqs, kv, 20), dtype=torch.int32, device="cuda"), many=torch.zeros((seqs, kv, 30), dtype=torch.int32, device="cuda"),
                    codes=torch.zeros((k.shape[1], kv, 2, dim), dtype=torch.int8, device="cuda"), scales=torch.zeros((k.shape[1], kv), device="cuda"))

    def once(c, s, o, bound):
        st = current()
        for layer in range(2):
            c.bounds(s["zeros"], s["lens"], o["codes"], o["scales"], max_new=stride * PAGE, layer=layer, stream=st)
            c.select(s["q"][:seqs], o["codes"], o["scales"], s["lens"], o["few"], max_pos=512 * PAGE, keep_last=1, stream=st)
            c.select(s["q"][:seqs], o["codes"], o["scales"], s["lens"], o["many"], max_pos=stride * PAGE, keep_first=1, stream=st)
            c.attention(s["q"][:seqs], o["many"], s["lens"], 0.125, o["row"], layer=layer, stream=st)
            c.attention_tree(s["q"], s["first"], s["lens"], s["bits"], 0.125, o["tree"], max_drafts=drafts, max_context=bound, layer=layer, stream=st)
        c.keep(s["lens"], s["kept"], s["n_kept"], stream=st)

    got = outputs()
    once(cache, live, got, 100)  # (a first one that is not captured)
    pool[0].copy_(k), pool[1].copy_(v)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        once(cache, live, got, 100)
    for s in sets:
        for name, x in s.items():
            live[name].copy_(x)
        for x in got.values():
            x.zero_()
        pool[0].copy_(k), pool[1].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        fresh = [k.clone(), v.clone()]
        direct, want = PagedCache(backend, fresh[0], fresh[1], s["tables"]), outputs()
        once(direct, s, want, 100)  # (the bound shares out the work: the same one for the same sums)
        torch.cuda.synchronize()
        for name in got:
            assert torch.equal(got[name], want[name]), name
        assert torch.equal(pool[0], fresh[0]) and torch.equal(pool[1], fresh[1])
        cache.synchronize()
        direct.close()


def test_the_first_calls_of_a_process_are_captured():
    """Kernels that were never launched before, in a capture that allows nothing unsafe."""
    import os
    import subprocess
    import sys

    here = os.path.dirname(os.path.abspath(__file__))
    code = """
import torch
from orangu_b200 import CudaBackend, PagedCache
be = CudaBackend.init(0)
ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
k = torch.randn((1, 6, 1, 16, 64), device="cuda").half()
cache = PagedCache(be, k, k.clone(), ints([[0, 1, 2], [3, 4, 5]]))
q = torch.randn((8, 4, 64), device="cuda").half()
out, row, codes, scales = torch.zeros_like(q), torch.zeros_like(q[:2]), torch.zeros((6, 1, 2, 64), dtype=torch.int8, device="cuda"), torch.zeros((6, 1), device="cuda")
few, lens, first, bits = ints([[[0, 0]]] * 2), ints([33, 20]), ints([0, 4, 8]), torch.ones(8, dtype=torch.int64, device="cuda")
zeros, kept, src, dst = ints([0, 0]), ints([[1], [0]]), ints([0]), ints([5])
wide, wide_out = torch.randn((20, 16, 64), device="cuda").half(), torch.zeros((20, 16, 64), dtype=torch.float16, device="cuda")
wide_first, wide_bits = ints([0, 10, 20]), torch.ones(20, dtype=torch.int64, device="cuda")

def once():
    st = torch.cuda.current_stream().cuda_stream
    cache.bounds(zeros, lens, codes, scales, max_new=48, stream=st)
    cache.select(q[:2], codes, scales, lens, few, max_pos=48, stream=st)
    cache.attention(q[:2], few, lens, 0.1, row, stream=st)
    cache.attention_tree(q, first, lens, bits, 0.1, out, 4, 33, stream=st)
    cache.attention_tree(wide, wide_first, lens, wide_bits, 0.1, wide_out, 10, 33, stream=st)
    cache.keep(lens, kept, ints_one, stream=st)
    cache.fork(zeros[:1], src_one, lens[:1], dst, stream=st)
    cache.copy(src, dst, stream=st)

ints_one, src_one = ints([1, 1]), ints([1])
state = [x.clone() for x in cache._arrays]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    once()
g.replay()
torch.cuda.synchronize()
a = [x.clone() for x in (out, wide_out, row, few, codes, scales) + cache._arrays]
for x, y in zip(cache._arrays, state):
    x.copy_(y)
for x in (out, wide_out, row, few, codes, scales):
    x.zero_()
once()
torch.cuda.synchronize()
assert all(torch.equal(x, y) for x, y in zip(a, (out, wide_out, row, few, codes, scales) + cache._arrays)) and bool(out.any()) and bool(wide_out.any())
print("same")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=os.path.dirname(here), timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


# ------------------------------------------------------------------------------------------- long contexts
@pytest.mark.parametrize("kind,dim,group,drafts", [("f16", 128, 4, 4), ("bf16", 64, 2, 7), ("f16", 64, 4, 17), ("bf16", 128, 4, 16), ("f16", 128, 8, 17), ("bf16", 64, 16, 9)])
def test_trees_over_seventy_thousand_positions(backend, kind, dim, group, drafts):
    ctx = [70_001, 3, 20_000]
    counts = [drafts, 1, 2]
    made = Made(backend, kind, 1, dim, [a + b for a, b in zip(ctx, counts)], seed=dim + drafts)
    run_tree(made, group, ctx, counts)
