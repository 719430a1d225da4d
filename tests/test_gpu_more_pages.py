"""4-bit pages, attention of new tokens with the weights added up, caches that are cut down, and verified drafts, through the public entry points, against the plain
statements of more_pages_plain.py."""
import ctypes as C

import numpy as np
import pytest

import more_pages_plain as more
import pages_plain as plain
from gpu_common import backend  # noqa: F401
from test_gpu_pages import PAGE, device16, float64, ints, random_tree, words

pytestmark = pytest.mark.gpu
U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step of a type, relative


def current():
    import torch

    return torch.cuda.current_stream().cuda_stream


def weight_error(dim):
    """A weight's relative error.  A score's error, absolute, is that of a sum of dim products in fp32 with a factor in front (dim + 4 roundings of 2^-24, of
    truncating adders twice that); a weight's is as large, once more for the sum it is divided by (natural or binary exponents: below 1); the sums over n positions
    go page by page in fp32, 2^-23 each time; 2^-20 covers 2^x, the weight's remainder (2^-22) and the parts' factors."""
    return lambda qk, n: 4 * (dim + 4) * 2.0 ** -24 * qk + (n / PAGE + PAGE) * 2.0 ** -23 + 2.0 ** -20


class Held:
    """Sequences of `held` positions in pages of any type ("q4", or the type of the rows); unfilled places hold bytes that are no numbers."""

    def __init__(self, be, pages, kind, kv, dim, held, seed=0, layers=1, spare=0, std=1.0, gone=()):
        import torch

        from orangu_b200 import PagedCache

        r = self.r = np.random.default_rng(seed)
        count = [-(-int(n) // PAGE) for n in held]
        n_pages = sum(count) + spare + 1
        self.kind, self.pages, self.kv, self.dim, self.layers, self.n_pages, self.held = kind, pages, kv, dim, layers, n_pages, [int(n) for n in held]
        order = r.permutation(n_pages)
        self.tables = np.full((len(held), max(count + [1])), -1, np.int64)
        at = 0
        for s, p in enumerate(count):
            self.tables[s, :p] = order[at:at + p]
            at += p
        self.free = order[at:]
        rows = int(sum(self.held))
        first = np.concatenate([[0], np.cumsum(self.held)])
        self.k, self.v = [], []  # [layer][sequence]: [positions, kv, dim], as the pages hold them
        shape = (layers, n_pages, kv, 9 * dim) if pages == "q4" else (layers, n_pages, kv, PAGE, dim)
        if pages == "q4":
            pools = [torch.full(shape, 255, dtype=torch.uint8, device="cuda") for _ in range(2)]
        else:
            pools = [device16(np.full(shape, 0x7e00 if kind == "f16" else 0x7fc0, np.uint16), kind) for _ in range(2)]
        self.kd, self.vd, self.td = *pools, ints(self.tables)
        self.cache = PagedCache(be, self.kd, self.vd, self.td)
        for li in range(layers):
            made = []
            for pool in pools:
                x, b = plain.bits16((rows, kv, dim), r, kind, std)
                made.append((x, device16(b, kind)))
                if pages != "q4" and rows:
                    seq = np.repeat(np.arange(len(held)), self.held)
                    pos = np.concatenate([np.arange(n) for n in self.held])
                    pool[li, torch.from_numpy(self.tables[seq, pos // PAGE]).cuda(), :, torch.from_numpy(pos % PAGE).cuda()] = made[-1][1]
            if pages == "q4" and rows:
                self.cache.store(made[0][1], made[1][1], ints(first), ints([0] * len(held)), max_tokens=max(self.held), layer=li, stream=current())
            values = [more.in_four_bits(x) if pages == "q4" else x for x, _ in made]
            self.k.append([values[0][first[s]:first[s + 1]] for s in range(len(held))])
            self.v.append([values[1][first[s]:first[s + 1]] for s in range(len(held))])
        self.there = [np.ones(n, bool) for n in self.held]
        for s, p, number in gone:  # a page that is not there after all
            self.tables[s, p] = number
            self.there[s][p * PAGE:(p + 1) * PAGE] = False
        self.td.copy_(ints(self.tables))

    def values(self, layer=0):
        """What the cache holds now: [2][sequence][positions, kv, dim], by load or by the pages."""
        import torch

        rows, first = int(sum(self.held)), np.concatenate([[0], np.cumsum(self.held)])
        if self.pages == "q4":
            out = [torch.zeros((rows, self.kv, self.dim), dtype=torch.float16, device="cuda") for _ in range(2)]
            if rows:
                self.cache.load(*out, ints(first), ints([0] * len(self.held)), max_tokens=max(self.held), layer=layer, stream=current())
            return [[float64(x)[first[s]:first[s + 1]] for s in range(len(self.held))] for x in out]
        tables = self.td.cpu().numpy()
        return [[np.stack([float64(p[layer, int(tables[s, x // PAGE]), :, x % PAGE]) for x in range(n)]) if n else np.zeros((0, self.kv, self.dim)) for s, n in enumerate(self.held)]
                for p in (self.kd, self.vd)]


def run_tokens(made, group, ctx, counts, bits=None, weighed=False, extra=0, strides=(0, 0), max_tokens=None, max_context=None, layer=0, q_kind=None, q_std=1.5, scale=None, compare=True, heads_of_kv=None):
    """Calls attention_tokens and compares; `extra` rows behind the last token, `strides` entries between rows."""
    import torch

    kind = q_kind or made.kind
    first = np.concatenate([[0], np.cumsum(counts)])
    n, heads, dim = int(first[-1]) + extra, made.kv * group, made.dim
    q, qb = plain.bits16((n, heads, dim), made.r, kind, q_std)
    wide = np.full((n, heads * dim + strides[0]), 0x7e00 if kind == "f16" else 0x7fc0, np.uint16)
    wide[:, :heads * dim] = qb.reshape(n, -1)
    qd = device16(wide, kind)[:, :heads * dim].view(n, heads, dim)
    outw = torch.full((n, heads * dim + strides[1]), 7.0, dtype=qd.dtype, device="cuda")
    out = outw[:, :heads * dim].view(n, heads, dim)
    scale = dim ** -0.5 if scale is None else scale
    room = made.tables.shape[1] * PAGE + 3  # (rows of weights longer than they have to be)
    mass = made.r.exponential(1.0, (len(ctx), made.kv, room)).astype(np.float32) if weighed else None
    md = torch.from_numpy(mass).cuda() if weighed else None
    made.cache.attention_tokens(qd, ints(first), ints(ctx), scale, out, max_tokens=max(list(counts) + [1]) if max_tokens is None else max_tokens,
                                max_context=max(list(ctx) + [0]) if max_context is None else max_context, visible=words(bits + [0] * extra) if bits is not None else None, mass=md, layer=layer,
                                stream=current())
    made.cache.synchronize(current())  # (says so if a wait inside a kernel was given up)
    if not compare:
        return out, md
    want = np.full((n, heads, dim), 7.0)
    mass64 = mass.astype(np.float64) if weighed else None
    if heads_of_kv is not None:  # of heads apart only, by way of a cache that has those alone
        heads_of = np.concatenate([np.arange(h * group, (h + 1) * group) for h in heads_of_kv])
        pick = lambda x: [s[:, list(heads_of_kv)] for s in x]  # noqa: E731
        got, want, k, v, q = float64(out)[:, heads_of], want[:, heads_of], pick(made.k[layer]), pick(made.v[layer]), q[:, heads_of]
        mass64 = mass64[:, list(heads_of_kv)] if weighed else None
        md = md[:, list(heads_of_kv)] if weighed else None
    else:
        got, k, v = float64(out), made.k[layer], made.v[layer]
    # over 4-bit pages the weights of bfloat16 rows are f16 numbers, off by half a step of those
    rounded = U["f16"] if made.pages == "q4" and kind == "bf16" else 0.0
    tol, mass_tol = more.attend_tokens(q, k, v, made.there, first, ctx, bits, scale, want, mass64, weight_error(dim), rounded)
    assert np.isfinite(got).all()
    off = np.abs(got - want) - (tol[..., None] + U[kind] * (np.abs(want) + tol[..., None]) + 2.0 ** -25)
    assert off.max(initial=-1.0) <= 0, f"{off.max()} over the bound at {np.unravel_index(off.argmax(), off.shape)}"
    assert (outw[:, heads * dim:] == 7.0).all()
    if weighed:
        off = np.abs(md.cpu().numpy().astype(np.float64) - mass64) - mass_tol
        assert off.max() <= 0, f"masses: {off.max()} over the bound at {np.unravel_index(off.argmax(), off.shape)}"
    return out, md


# ------------------------------------------------------------------------------------------- rows into pages and back
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("dim,kv", [(64, 1), (128, 2), (64, 3), (128, 8)])
def test_store_and_load_are_the_definition(backend, kind, dim, kv):
    import torch

    made = Held(backend, "q4", kind, kv, dim, [40, 0, 1, 33], seed=dim + kv, layers=2)
    ctx, counts = [35, 0, 1, 16], [5, 0, 0, 17]
    first = np.concatenate([[0], np.cumsum(counts)])
    n = int(first[-1]) + 2  # two rows of no sequence
    x, b = plain.bits16((2, n, kv, dim), made.r, kind)
    b = b.copy()
    special = np.array([0, 0x8000, 0x7c00 if kind == "f16" else 0x7f80, 0xfc00 if kind == "f16" else 0xff80, 0x7e00 if kind == "f16" else 0x7fc0, 1, 0x8001, 0x03ff, 0x0400, 0x7bff if kind == "f16" else 0x7f7f], np.uint16)
    at = made.r.integers(0, b.size, b.size // 6)
    b.reshape(-1)[at] = special[made.r.integers(0, len(special), len(at))]
    b[0, 1] = 0  # zeros only
    b[0, 2, :, :32], b[1, 2, :, :32] = special[7], special[6]  # below the smallest steps
    b[1, 3] = plain.to16(np.tile([1.5, -1.5], dim // 2) * np.ones((kv, dim)), kind)[1]  # equal magnitudes: the negative one counts
    b[0, 4] = plain.to16(np.repeat(np.linspace(-8, 7.5, 32), dim // 32)[None] * np.ones((kv, 1)), kind)[1]  # halves: to the even code
    x = float64(device16(b, kind))
    wide = np.full((2, n, kv * dim + 8), 0x7e00 if kind == "f16" else 0x7fc0, np.uint16)
    wide[..., :kv * dim] = b.reshape(2, n, -1)
    k, v = (device16(w, kind)[:, :kv * dim].view(n, kv, dim) for w in wide)
    before = made.values(1), made.values(0)
    made.cache.store(k, v, ints(first), ints(ctx), max_tokens=17, layer=1, stream=current())
    out = [torch.full((n, kv * dim + 16), 7.0, dtype=torch.float16, device="cuda") for _ in range(2)]
    view = [o[:, :kv * dim].view(n, kv, dim) for o in out]
    made.cache.load(*view, ints(first), ints(ctx), max_tokens=17, layer=1, stream=current())
    torch.cuda.synchronize()
    want = more.in_four_bits(x)
    for j in range(2):
        got = float64(view[j])
        assert np.array_equal(got[:n - 2], want[j, :n - 2])
        assert (got[n - 2:] == 7.0).all() and (out[j][:, kv * dim:] == 7.0).all()
    after = made.values(1), made.values(0)
    for j in range(2):
        for s in range(4):
            assert np.array_equal(after[1][j][s], before[1][j][s])  # the other layer
            assert np.array_equal(after[0][j][s][:ctx[s]], before[0][j][s][:ctx[s]])
            assert np.array_equal(after[0][j][s][ctx[s]:], want[j, first[s]:first[s + 1]] if counts[s] else before[0][j][s][ctx[s]:])
    # bfloat16 rows: the same values, rounded
    half = [torch.zeros((n, kv, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    made.cache.load(*half, ints(first), ints(ctx), max_tokens=17, layer=1, stream=current())
    torch.cuda.synchronize()
    for j in range(2):
        assert torch.equal(half[j][:n - 2], view[j][:n - 2].bfloat16())


def test_four_bits_keep_what_sixteen_levels_can(backend):
    """An entry is off by half a step at most, but for those next to the far end of the sixteen codes: a step there."""
    made = Held(backend, "q4", "f16", 2, 128, [1], seed=3)
    x, b = plain.bits16((1, 2, 128), made.r, "f16")
    got = more.in_four_bits(x).reshape(1, 2, 4, 32)
    x = x.reshape(1, 2, 4, 32)
    step = np.abs(x).max(-1, keepdims=True) / 8 * (1 + 2.0 ** -6)
    assert (np.abs(got - x) <= np.where(np.abs(x) > 7 * step, step, step / 2) + 1e-12).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_store_leaves_out_what_is_not_there(backend, dim):
    import torch

    made = Held(backend, "q4", "f16", 2, dim, [32, 32, 32], seed=5, gone=[(1, 1, -1), (2, 0, 10_000)])
    before = made.kd.clone(), made.vd.clone()
    n = 60
    x = torch.randn((n, 2, dim), device="cuda").half()
    load = lambda first, ctx, most: made.cache.load(k, v, ints(first), ints(ctx), max_tokens=most, stream=current())  # noqa: E731
    for first, ctx, most in (([0, 20, 20, 20], [4_000_000_000 - (1 << 32), 0, 0], 60), ([0, -1, 20, 10], [0, 0, 0], 60), ([0, 0, 61, 61], [0, 0, 0], 60), ([5, 5, 5, 5], [0, 0, 0], 60), ([0, 0, 20, 40], [0, 16, -1], 60),
                             ([0, 0, 0, 10], [0, 0, 0], 60), ([0, 60, 60, 60], [32, 0, 0], 60), ([0, 60, 60, 60], [0, 0, 0], 0)):
        made.cache.store(x, x, ints(first), ints(ctx), max_tokens=most, stream=current())
        k, v = torch.full_like(x, 7.0), torch.full_like(x, 7.0)
        load(first, ctx, most)
        torch.cuda.synchronize()
        assert torch.equal(made.kd, before[0]) and torch.equal(made.vd, before[1]) and bool((k == 7.0).all()) and bool((v == 7.0).all()), (first, ctx)
    # 24 rows of which 16 have a place, and no more than max_tokens of a sequence
    k, v = torch.full_like(x, 7.0), torch.full_like(x, 7.0)
    made.cache.store(x, x, ints([0, 0, 24, 24]), ints([0, 0, 0]), max_tokens=24, stream=current())
    made.cache.load(k, v, ints([0, 0, 24, 24]), ints([0, 0, 0]), max_tokens=10, stream=current())
    torch.cuda.synchronize()
    want = more.in_four_bits(float64(x))
    assert np.array_equal(float64(k)[:10], want[:10]) and bool((k[10:] == 7.0).all())
    load([0, 0, 24, 24], [0, 0, 0], 24)
    torch.cuda.synchronize()
    assert np.array_equal(float64(v)[:16], want[:16]) and bool((v[16:] == 7.0).all())


# ------------------------------------------------------------------------------------------- attention of new tokens
SHAPES = [(1, 1, [0], [1]), (2, 4, [5], [1]), (1, 16, [16], [1]), (2, 3, [15, 16, 17], [1, 2, 3]), (8, 4, [100, 0, 33], [4, 5, 1]), (2, 8, [40, 700, 1, 0], [7, 0, 4, 2]), (1, 4, [250], [16]),
          (2, 5, [130, 64], [13, 6]), (1, 7, [300], [33]), (1, 2, [77, 78], [64, 63])]


@pytest.mark.parametrize("pages,kind", [("q4", "f16"), ("q4", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kv,group,ctx,counts", SHAPES)
def test_trees_and_chains_with_weights(backend, pages, kind, dim, kv, group, ctx, counts):
    made = Held(backend, pages, kind, kv, dim, [a + b for a, b in zip(ctx, counts)], seed=len(ctx) + dim + group)
    bits = [b for m in counts for b in random_tree(made.r, m)]
    run_tokens(made, group, ctx, counts, bits, weighed=True, extra=2)
    run_tokens(made, group, ctx, counts, None, weighed=True, strides=(8, 16))


@pytest.mark.parametrize("pages,kind", [("q4", "f16"), ("q4", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("dim,group,ctx,counts", [(128, 4, [0], [200]), (64, 3, [37, 0, 100], [129, 65, 1]), (128, 16, [70], [66]), (64, 1, [3, 500], [300, 64]), (128, 8, [1000], [130])])
def test_parts_of_prompts(backend, pages, kind, dim, group, ctx, counts):
    made = Held(backend, pages, kind, 2, dim, [a + b for a, b in zip(ctx, counts)], seed=dim + group)
    run_tokens(made, group, ctx, counts, None, weighed=True)
    run_tokens(made, group, ctx, counts, None, strides=(24, 8), extra=1)


@pytest.mark.parametrize("dim,group,counts", [(128, 8, [64, 40]), (64, 8, [64, 1]), (128, 4, [32, 20]), (64, 2, [60, 64]), (128, 16, [70, 9])])
def test_many_tiles_with_many_rows(backend, dim, group, counts):
    """More than twice as many tiles a CTA as its rings have places, in pieces of odd and even numbers of tiles."""
    ctx = [9000, 4100]
    made = Held(backend, "q4", "bf16", 8, dim, [a + b for a, b in zip(ctx, counts)], seed=dim + group)
    run_tokens(made, group, ctx, counts, None, weighed=group == 2, heads_of_kv=(0, 7))


@pytest.mark.parametrize("pages,kind,dim,group,counts", [("q4", "f16", 128, 4, [1, 1, 1]), ("q4", "bf16", 64, 4, [4, 1, 2]), ("bf16", "bf16", 128, 8, [1, 2, 1]), ("q4", "bf16", 128, 2, [20, 3, 40])])
def test_long_contexts_are_cut_and_added_up(backend, pages, kind, dim, group, counts):
    import torch

    ctx = [5000, 17, 2049]
    made = Held(backend, pages, kind, 1, dim, [a + b for a, b in zip(ctx, counts)], seed=dim + group)
    results = []
    for bound in (None, 0, 100, 1 << 31):  # the bound shares out the work and no more
        made.r = np.random.default_rng(4)
        results.append(run_tokens(made, group, ctx, counts, None, weighed=True, max_context=bound))
    for _ in range(3):
        made.r = np.random.default_rng(4)
        again = run_tokens(made, group, ctx, counts, None, weighed=True, compare=False)
        assert torch.equal(again[0], results[0][0]) and torch.equal(again[1], results[0][1])  # the same bits


@pytest.mark.parametrize("pages,kind", [("q4", "f16"), ("bf16", "bf16")])
def test_rows_that_see_nothing_and_pages_that_are_not_there(backend, pages, kind):
    made = Held(backend, pages, kind, 2, 128, [40, 20, 64], seed=9, gone=[(0, 0, -1), (2, 1, 1 << 20), (2, 3, -7)])
    run_tokens(made, 4, [36, 0, 60], [4, 3, 4], [1, 3, 0, 8, 0, 0, 0, 15, 0, 2, 1], weighed=True)
    made = Held(backend, pages, kind, 1, 64, [3, 7], seed=9, gone=[(0, 0, -1)])
    out, mass = run_tokens(made, 2, [0, 3], [3, 4], [0, 0, 0, 0, 1 << 63, 2, 4], weighed=True)
    assert bool((out[:3] == 0).all())


@pytest.mark.parametrize("pages,kind", [("q4", "f16"), ("q4", "bf16"), ("f16", "f16")])
def test_numbers_of_all_sizes(backend, pages, kind):
    """Queries from tiny to large: a power of two per row is taken out where they are bfloat16.  Scores up to about 30, whatever the sizes."""
    for q_std, scale in ((2.0 ** -12, 2.0 ** 8), (300.0, 2.0 ** -12)) + (((2.0 ** -60, 2.0 ** 56), (2.0 ** 70, 2.0 ** -74)) if kind == "bf16" else ()):
        made = Held(backend, pages, kind, 2, 128, [90], seed=11)
        run_tokens(made, 4, [80], [10], None, weighed=True, q_std=q_std, scale=scale)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_a_query_that_is_no_number_stays_in_its_row(backend, kind):
    import torch

    made = Held(backend, "q4", kind, 1, 128, [50], seed=2)
    q, qb = plain.bits16((4, 4, 128), made.r, kind)
    qb = qb.copy()
    clean = device16(qb, kind)
    qb[1, 2, 5] = 0x7e00 if kind == "f16" else 0x7fc0
    bad = device16(qb, kind)
    outs = [torch.zeros_like(clean) for _ in range(2)]
    for x, o in zip((clean, bad), outs):
        made.cache.attention_tokens(x, ints([0, 4]), ints([46]), 0.1, o, max_tokens=4, max_context=46, stream=current())
    torch.cuda.synchronize()
    same = torch.ones(4, 4, dtype=torch.bool, device="cuda")
    same[1, 2] = False
    assert torch.equal(outs[0][same], outs[1][same]) and bool(torch.isnan(outs[1][1, 2]).all())


def test_single_tokens_equal_the_tree_operator(backend):
    """Over f16 pages the new entry point is attention_tree: the same bits."""
    import torch

    made = Held(backend, "f16", "f16", 2, 64, [100, 40], seed=6)
    q, qb = plain.bits16((2, 8, 64), made.r, "f16")
    qd, a, b = device16(qb, "f16"), *(torch.zeros((2, 8, 64), dtype=torch.float16, device="cuda") for _ in range(2))
    made.cache.attention_tree(qd, ints([0, 1, 2]), ints([99, 39]), words([1, 1]), 0.125, a, 1, 99, stream=current())
    made.cache.attention_tokens(qd, ints([0, 1, 2]), ints([99, 39]), 0.125, b, 1, 99, stream=current())
    torch.cuda.synchronize()
    assert torch.equal(a, b)


@pytest.mark.parametrize("pages,kind", [("q4", "f16"), ("bf16", "bf16")])
def test_many_sequences_and_a_layer_of_several(backend, pages, kind):
    r = np.random.default_rng(1)
    counts = [int(v) for v in r.integers(0, 4, 70)]
    ctx = [int(v) for v in r.integers(0, 60, 70)]
    made = Held(backend, pages, kind, 2, 64, [a + b for a, b in zip(ctx, counts)], seed=8, layers=2)
    run_tokens(made, 4, ctx, counts, None, weighed=True, layer=1)


@pytest.mark.parametrize("pages,kind,group", [("q4", "f16", 4), ("q4", "bf16", 16), ("bf16", "bf16", 8)])
def test_prompts_that_reach_past_their_table_and_rows_before_the_first(backend, pages, kind, group):
    """Positions behind a table's last page are nobody's: the tokens there see what there is.  Rows of no sequence are left as they were, in front, too."""
    import torch

    made = Held(backend, pages, kind, 1, 64, [96, 40], seed=4)  # tables of six pages
    ctx, first = [20, 39], [3, 103, 104]
    q, qb = plain.bits16((110, group, 64), made.r, kind, 1.5)
    out = torch.full((110, group, 64), 7.0, dtype=torch.float16 if kind == "f16" else torch.bfloat16, device="cuda")
    mass = torch.zeros((2, 1, 96), device="cuda")
    made.cache.attention_tokens(device16(qb, kind), ints(first), ints(ctx), 0.125, out, max_tokens=100, max_context=39, mass=mass, stream=current())
    made.cache.synchronize(current())
    want, mass64 = np.full((110, group, 64), 7.0), np.zeros((2, 1, 96))
    tol, mass_tol = more.attend_tokens(q, made.k[0], made.v[0], made.there, first, ctx, None, 0.125, want, mass64, weight_error(64), U["f16"] if pages == "q4" and kind == "bf16" else 0.0)
    off = np.abs(float64(out) - want) - (tol[..., None] + U[kind] * (np.abs(want) + tol[..., None]) + 2.0 ** -25)
    assert off.max() <= 0 and (np.abs(mass.cpu().numpy() - mass64) <= mass_tol).all()


# ------------------------------------------------------------------------------------------- cutting caches down
def run_evict(made, n_pos, n_keep, first, last, mass, max_pos=None, width=None):
    import torch

    layers, kv, seqs = made.layers, made.kv, len(n_pos)
    room = made.tables.shape[1] * PAGE + (width or 0)
    m = np.zeros((layers, seqs, kv, room), np.float32)
    m[..., :mass.shape[-1]] = mass
    md = torch.from_numpy(m).cuda()
    kept, left = torch.full((layers, seqs, kv, n_keep), 7, dtype=torch.int32, device="cuda"), torch.full((seqs,), 7, dtype=torch.int32, device="cuda")
    before = [made.values(li) for li in range(layers)]
    made.cache.evict(ints(n_pos), md, kept, left, max_pos=max(n_pos) if max_pos is None else max_pos, keep_first=first, keep_last=last, stream=current())
    torch.cuda.synchronize()
    want, want_left = more.evict(m, n_pos, n_keep, first, last)
    assert np.array_equal(kept.cpu().numpy(), want) and np.array_equal(left.cpu().numpy(), want_left)
    after, got = [made.values(li) for li in range(layers)], md.cpu().numpy()
    for li in range(layers):
        for s in range(seqs):
            n = int(want_left[s])
            for h in range(kv):
                src = want[li, s, h, :n]
                ok = made.there[s][:n] & made.there[s][src]
                for j in range(2):
                    x = before[li][j][s][:, h].copy()
                    x[:n][ok] = x[src][ok]
                    here = np.concatenate([made.there[s]])
                    assert np.array_equal(after[li][j][s][here, h], x[here])  # what lies behind is as it was, too
                y = m[li, s, h].copy()
                y[:n] = y[src]
                assert np.array_equal(got[li, s, h], y, equal_nan=True)
    return kept


@pytest.mark.parametrize("pages,kind", [("q4", "f16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("dim,kv,layers,n_pos,n_keep,first,last", [
    (64, 1, 1, [17], 16, 0, 0), (128, 2, 2, [100, 5, 64, 0], 40, 4, 10), (64, 3, 1, [300, 299, 1], 299, 1, 298), (128, 2, 1, [700], 31, 0, 31), (64, 2, 3, [50, 60], 1, 0, 0), (128, 1, 1, [33], 100, 2, 2),
    (64, 2, 1, [1000, 999], 513, 500, 13)])
def test_evict(backend, pages, kind, dim, kv, layers, n_pos, n_keep, first, last):
    made = Held(backend, pages, kind, kv, dim, n_pos, seed=dim + n_keep, layers=layers)
    run_evict(made, n_pos, n_keep, first, last, made.r.exponential(1.0, (layers, len(n_pos), kv, made.tables.shape[1] * PAGE)).astype(np.float32), width=5)


@pytest.mark.parametrize("pages", ["q4", "f16"])
def test_evict_of_equal_weights_and_of_none(backend, pages):
    n_pos = [90, 90, 90]
    made = Held(backend, pages, "f16", 2, 64, n_pos, seed=1)
    mass = made.r.integers(0, 3, (1, 3, 2, 96)).astype(np.float32)  # equals: the first one stays
    mass[0, 1] = 0.5
    mass[0, 2, 0, ::3] = np.nan
    mass[0, 2, 1] = np.where(np.arange(96) % 2, np.inf, -0.0)
    run_evict(made, n_pos, 37, 2, 5, mass)
    made = Held(backend, pages, "f16", 1, 64, [64], seed=1, gone=[(0, 1, -1)])
    run_evict(made, [64], 20, 0, 0, np.tile(np.arange(64, dtype=np.float32), (1, 1, 1, 1)))


@pytest.mark.parametrize("n,n_keep,bound", [(5000, 1234, None), (40000, 300, None), (40000, 33000, 10), (9000, 4000, 1 << 31)])
def test_evict_of_long_caches(backend, n, n_keep, bound):
    made = Held(backend, "q4", "f16", 1, 64, [n, 100], seed=3)
    run_evict(made, [n, 100], n_keep, 4, 64, made.r.exponential(1.0, (1, 2, 1, made.tables.shape[1] * PAGE)).astype(np.float32), max_pos=bound)


@pytest.mark.parametrize("pages,kind", [("q4", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("dim", [64, 128])
def test_keep_moves_codes_units_and_weights(backend, pages, kind, dim):
    import torch

    made = Held(backend, pages, kind, 3, dim, [64, 80, 33, 20], seed=dim, layers=2)
    ctx = [5, 16, 0, 19]
    kept = np.full((4, 64), -1, np.int32)
    n_kept = [7, 64, 33, 5]
    kept[0, :7] = [0, 2, 3, 9, 15, 30, 58]
    kept[1] = made.r.permutation(64)
    kept[2, :33] = np.arange(33)[::-1]
    kept[3, :5] = [0, 64, -3, 70, 1]  # out of range; a place behind the table
    mass = made.r.exponential(1.0, (2, 4, 3, made.tables.shape[1] * PAGE)).astype(np.float32)
    md = torch.from_numpy(mass).cuda()
    before = [made.values(li) for li in range(2)]
    made.cache.keep(ints(ctx), ints(kept), ints(n_kept), stream=current(), mass=md)
    torch.cuda.synchronize()
    got = md.cpu().numpy()
    for li in range(2):
        after = made.values(li)
        for s in range(4):
            moves = [(ctx[s] + j, ctx[s] + int(kept[s, j])) for j in range(n_kept[s]) if 0 <= kept[s, j] < 64 and ctx[s] + max(j, int(kept[s, j])) < -(-made.held[s] // PAGE) * PAGE]
            for j in range(2):
                want = before[li][j][s].copy()
                for a, b in moves:
                    if a < made.held[s]:
                        want[a] = before[li][j][s][b]
                assert np.array_equal(after[j][s], want)
            want = mass[li, s].copy()
            for a, b in moves:
                want[:, a] = mass[li, s][:, b]
            assert np.array_equal(got[li, s], want)


@pytest.mark.parametrize("dim", [64, 128])
def test_four_bit_pages_are_copied_and_forked(backend, dim):
    import torch

    made = Held(backend, "q4", "f16", 3, dim, [40, 40], seed=1, layers=3, spare=4)
    src, dst = int(made.tables[0, 1]), int(made.free[0])
    k = made.kd.clone()
    made.cache.copy(ints([src]), ints([dst]), stream=current())
    torch.cuda.synchronize()
    k[:, dst] = k[:, src]
    assert torch.equal(made.kd, k)
    made.cache.fork(ints([0]), ints([1]), ints([37]), ints([int(made.free[1])]), stream=current())
    made.held = [37, 37]
    torch.cuda.synchronize()
    for li in range(3):
        for pool in made.values(li):
            assert np.array_equal(pool[0], pool[1])


# ------------------------------------------------------------------------------------------- verification
def distributions(r, n, vocab, kind, spread=2.0):
    x = r.standard_normal((n, vocab)) * spread
    y = x * 0.8 + r.standard_normal((n, vocab))
    p, q = (np.exp(z - z.max(1, keepdims=True)) for z in (x, y))
    p, q = (z / z.sum(1, keepdims=True) for z in (p, q))
    return [z.astype(np.float32).astype(np.float64) if kind == "f32" else plain.to16(z, kind)[0] for z in (p, q)]


def run_verify(be, kind, target, draft, tokens, parent, first, uniform, width=64, pad=0, seqs=None):
    import torch

    from orangu_b200 import verify_drafts

    def device(x):
        wide = np.full((x.shape[0], x.shape[1] + pad), np.nan)
        wide[:, :x.shape[1]] = x
        t = torch.from_numpy(wide.astype(np.float32)).cuda() if kind == "f32" else device16(plain.to16(wide, kind)[1], kind)
        return t[:, :x.shape[1]]

    n = len(first) - 1
    kept, count, token = torch.full((n, width), 7, dtype=torch.int32, device="cuda"), torch.full((n,), 7, dtype=torch.int32, device="cuda"), torch.full((n,), 7, dtype=torch.int32, device="cuda")
    verify_drafts(be, device(target), device(draft) if draft is not None else None, ints(tokens), ints(parent), ints(first), torch.from_numpy(np.asarray(uniform, np.float32)).cuda(), kept, count, token,
                  stream=current())
    torch.cuda.synchronize()
    got = [x.cpu().numpy() for x in (kept, count, token)]
    want = more.verify(target, draft, tokens, parent, first, np.asarray(uniform, np.float32), width)
    for g, w in zip(got, want):
        assert np.array_equal(g, w), (g, w)
    return got


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("drafted", [True, False])
@pytest.mark.parametrize("vocab,sizes,chain", [(1, [1, 3], True), (2, [5] * 20, False), (37, [1, 64, 0, 9, 70, 2], False), (1000, [8] * 40, True), (4099, [16, 3, 64], False), (128256, [6, 1], True)])
def test_verify(backend, kind, drafted, vocab, sizes, chain):
    r = np.random.default_rng(vocab + len(sizes))
    n = sum(sizes)
    first = np.concatenate([[0], np.cumsum(sizes)])
    target, draft = distributions(r, n, vocab, kind)
    parent = np.concatenate([np.array([-1] + [i - 1 if chain else int(r.integers(max(0, i - 4), i)) for i in range(1, m)], np.int64)[:m] for m in sizes])
    tokens = np.zeros(n, np.int64)
    for s in range(len(sizes)):
        for i in range(first[s] + 1, first[s + 1]):
            row = draft[first[s] + parent[i]]
            tokens[i] = r.choice(vocab, p=row / row.sum()) if row.sum() else 0
    run_verify(backend, kind, target, draft if drafted else None, tokens, parent, first, r.random(n), pad=3)


@pytest.mark.parametrize("vocab,sequences", [(700, 100), (700, 200), (20_000, 300)])
def test_verify_of_many_sequences(backend, vocab, sequences):
    """Fewer CTAs a sequence, and parts of more than 1024 tokens."""
    r = np.random.default_rng(sequences)
    sizes = r.integers(1, 4, sequences)
    first, n = np.concatenate([[0], np.cumsum(sizes)]), int(sizes.sum())
    target, draft = distributions(r, n, vocab, "f32")
    parent = np.concatenate([[-1, 0, 0][:m] for m in sizes])
    tokens = np.array([r.choice(vocab, p=row / row.sum()) for row in draft])
    run_verify(backend, "f32", target, draft, tokens, parent, first, r.random(n))


def test_verify_at_the_edges(backend):
    r = np.random.default_rng(5)
    vocab = 50
    target, draft = distributions(r, 6, vocab, "f32")
    same = target.copy()
    tokens, parent, first = np.array([0, 3, 4, 5, 6, 7]), np.array([-1, 0, 0, 1, 1, 2]), np.array([0, 6])
    for u in (0.0, 0.5, 1.0 - 2.0 ** -24, 1.0, np.nan, -1.0):  # 1, no number and less than 0 are out of range, and still answered
        run_verify(backend, "f32", target, draft, tokens, parent, first, np.full(6, u)) if u == u else None
        run_verify(backend, "f32", target, same, tokens, parent, first, np.full(6, u)) if u == u and u < 1 else None
        run_verify(backend, "f32", target, None, tokens, parent, first, np.full(6, u)) if u == u else None
    # parents and tokens out of range are never accepted
    for p, t in (([-1, 5, 0, 1, 1, 2], tokens), ([-1, 1, 0, 1, 1, 2], tokens), ([-1, -2, -1, 3, 9, 7], tokens), (parent, [0, -1, 50, 5, 6, 7]), (parent, [0, 3, 3, 3, 3, 3])):
        run_verify(backend, "f32", target, draft, np.array(t), np.array(p), first, np.zeros(6))
        run_verify(backend, "f32", target, None, np.array(t), np.array(p), first, np.full(6, 0.999))
    # rows that are zero, negative or no numbers
    odd = target.copy()
    odd[0] = 0.0
    odd[1, ::2], odd[2, 1::2], odd[2, 0] = np.nan, np.inf, -5.0
    run_verify(backend, "f32", odd, draft, tokens, parent, first, r.random(6))
    run_verify(backend, "f32", odd, None, tokens, parent, first, r.random(6))
    run_verify(backend, "f32", target, odd, tokens, parent, first, r.random(6))
    # a draft that is the target, rejected all the same (it cannot be but for u = 1): nothing is left, the target's own row counts
    run_verify(backend, "f32", same, same, tokens, parent, first, np.full(6, 1.0))
    # a path longer than the list
    run_verify(backend, "f32", target, draft, np.array([0, 1, 2, 3, 4, 5]), np.array([-1, 0, 1, 2, 3, 4]), first, np.zeros(6), width=3)
    # ranges that are none
    run_verify(backend, "f32", target, draft, tokens, parent, np.array([6, 6, 6]), np.zeros(6))


def test_verified_tokens_are_the_targets(backend):
    """40,000 sequences of one tree: the token after the root has the target's distribution, whatever the draft's."""
    import torch

    from orangu_b200 import verify_drafts

    r = np.random.default_rng(0)
    vocab, n, nodes = 8, 40_000, 4
    p, q = (x[0] for x in distributions(r, 1, vocab, "f32", 1.0))
    draws = r.choice(vocab, (n, nodes), p=q / q.sum())
    target = torch.from_numpy(np.tile(p.astype(np.float32), (n * nodes, 1))).cuda()
    draft = torch.from_numpy(np.tile(q.astype(np.float32), (n * nodes, 1))).cuda()
    kept, count, token = torch.zeros((n, 4), dtype=torch.int32, device="cuda"), *(torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(2))
    verify_drafts(backend, target, draft, ints(draws.reshape(-1)), ints(np.tile([-1, 0, 0, 0], n)), ints(np.arange(n + 1) * nodes), torch.from_numpy(r.random(n * nodes).astype(np.float32)).cuda(), kept, count,
                  token, stream=current())
    torch.cuda.synchronize()
    kept, count, token = kept.cpu().numpy(), count.cpu().numpy(), token.cpu().numpy()
    follows = np.where(count > 1, draws[np.arange(n), np.maximum(kept[:, 1], 0)], token)
    freq = np.bincount(follows, minlength=vocab) / n
    assert (np.abs(freq - p) < 5 * np.sqrt(p * (1 - p) / n)).all()  # five standard deviations
    assert (count > 1).mean() > 1 - 0.5 * np.abs(p - q).sum()       # more than one child: accepted more often than a single one would be


# ------------------------------------------------------------------------------------------- together
def test_rounds_of_serving_and_their_replay(backend):
    """Store, attention with weights, verification, keep, cut: two rounds in a stream, the same two as replays of one captured graph, and the plain statements."""
    import torch

    from orangu_b200 import verify_drafts

    kind, kv, group, dim, layers = "bf16", 2, 4, 64, 2
    held, counts, n_keep = [70, 40], [6, 4], 60
    rounds = 2

    def build():
        made = Held(backend, "q4", kind, kv, dim, [n + 26 for n in held], seed=21, layers=layers)
        return made

    first = np.concatenate([[0], np.cumsum(counts)])
    n, heads, vocab = int(first[-1]), kv * group, 33
    r = np.random.default_rng(3)
    rows = [[plain.bits16((2, layers, n, kv, dim), r, kind), plain.bits16((layers, n, heads, dim), r, kind, 1.5)] for _ in range(rounds)]
    probs = [distributions(r, n, vocab, "f32") for _ in range(rounds)]
    parent = np.array([-1, 0, 0, 1, 1, 2, -1, 0, 1, 2])
    tokens = [r.integers(0, vocab, n) for _ in range(rounds)]
    uniform = [r.random(n).astype(np.float32) for _ in range(rounds)]
    bits = []
    for s in range(2):
        mine = []
        for i in range(counts[s]):
            mine.append(1 << i | (mine[parent[first[s] + i]] if i else 0))
        bits += mine

    class State:
        pass

    def state():
        z = State()
        z.made = build()
        room = z.made.tables.shape[1] * PAGE
        z.kv_new, z.q = torch.zeros((2, layers, n, kv, dim), dtype=torch.bfloat16, device="cuda"), torch.zeros((layers, n, heads, dim), dtype=torch.bfloat16, device="cuda")
        z.target, z.draft, z.uniform, z.tokens = *(torch.zeros((n, vocab), device="cuda") for _ in range(2)), torch.zeros(n, device="cuda"), ints([0] * n)
        z.first, z.parent, z.bits, z.ctx = ints(first), ints(parent), words(bits), ints(held)
        z.mass, z.out = torch.zeros((layers, 2, kv, room), device="cuda"), torch.zeros((layers, n, heads, dim), dtype=torch.bfloat16, device="cuda")
        z.kept, z.count, z.token = torch.zeros((2, 64), dtype=torch.int32, device="cuda"), ints([0, 0]), ints([0, 0])
        z.chosen, z.left = torch.zeros((layers, 2, kv, n_keep), dtype=torch.int32, device="cuda"), ints([0, 0])
        return z

    def load(z, i):
        z.kv_new.copy_(device16(rows[i][0][1], kind)), z.q.copy_(device16(rows[i][1][1], kind))
        z.target.copy_(torch.from_numpy(probs[i][0].astype(np.float32))), z.draft.copy_(torch.from_numpy(probs[i][1].astype(np.float32)))
        z.uniform.copy_(torch.from_numpy(uniform[i])), z.tokens.copy_(ints(tokens[i]))

    def once(z):
        st = current()
        c = z.made.cache
        for li in range(layers):
            c.store(z.kv_new[0, li], z.kv_new[1, li], z.first, z.ctx, max_tokens=6, layer=li, stream=st)
            c.attention_tokens(z.q[li], z.first, z.ctx, dim ** -0.5, z.out[li], max_tokens=6, max_context=96, visible=z.bits, mass=z.mass[li], layer=li, stream=st)
        verify_drafts(backend, z.target, z.draft, z.tokens, z.parent, z.first, z.uniform, z.kept, z.count, z.token, stream=st)
        c.keep(z.ctx, z.kept, z.count, stream=st, mass=z.mass)
        z.ctx.add_(z.count)
        c.evict(z.ctx, z.mass, z.chosen, z.left, max_pos=96, keep_first=4, keep_last=16, stream=st)
        z.ctx.copy_(z.left)

    eager = state()
    for i in range(rounds):
        load(eager, i)
        once(eager)
    torch.cuda.synchronize()
    side, replayed = torch.cuda.Stream(), state()
    load(replayed, 0)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            once(replayed)
        for i in range(rounds):
            load(replayed, i)
            g.replay()
    torch.cuda.synchronize()
    for name in ("out", "mass", "kept", "count", "token", "chosen", "left", "ctx"):
        assert torch.equal(getattr(eager, name), getattr(replayed, name)), name
    assert torch.equal(eager.made.kd, replayed.made.kd) and torch.equal(eager.made.vd, replayed.made.vd)

    # the plain statements, by the masses and choices of the device where an order of nearly equal ones would depend on rounding
    made = build()
    ctx = list(held)
    k = [[x[:].copy() for x in made.k[li]] for li in range(layers)]
    v = [[x[:].copy() for x in made.v[li]] for li in range(layers)]
    mass = np.zeros((layers, 2, kv, made.tables.shape[1] * PAGE))
    for i in range(rounds):
        for li in range(layers):
            new = [more.in_four_bits(rows[i][0][0][j, li]) for j in range(2)]
            for s in range(2):
                k[li][s][ctx[s]:ctx[s] + counts[s]], v[li][s][ctx[s]:ctx[s] + counts[s]] = new[0][first[s]:first[s + 1]], new[1][first[s]:first[s + 1]]
            want = np.zeros((n, heads, dim))
            more.attend_tokens(rows[i][1][0][li], k[li], v[li], [np.ones(len(x), bool) for x in k[li]], first, ctx, bits, dim ** -0.5, want, mass[li], weight_error(dim))
        got = more.verify(probs[i][0], probs[i][1], tokens[i], parent, first, uniform[i])
        for s in range(2):
            path = got[0][s, :got[1][s]]
            for li in range(layers):
                for x in (k[li][s], v[li][s]):
                    x[ctx[s]:ctx[s] + len(path)] = x[ctx[s] + path]
                mass[li, s, :, ctx[s]:ctx[s] + len(path)] = mass[li, s][:, ctx[s] + path]
            ctx[s] += len(path)
        kept, left = more.evict(mass, ctx, n_keep, 4, 16)
        for s in range(2):
            for li in range(layers):
                for h in range(kv):
                    src = kept[li, s, h, :left[s]]
                    for x in (k[li][s], v[li][s]):
                        x[:left[s], h] = x[src, h]
                    mass[li, s, h, :left[s]] = mass[li, s, h, src]
            ctx[s] = int(left[s])
    assert np.array_equal(eager.count.cpu().numpy(), got[1]) and np.array_equal(eager.token.cpu().numpy(), got[2]) and np.array_equal(eager.chosen.cpu().numpy(), kept)
    assert eager.ctx.tolist() == ctx
    assert np.abs(float64(eager.out[layers - 1]) - want).max() < 2.0 ** -7 * np.abs(want).max()
    live = [np.arange(mass.shape[-1]) < c for c in ctx]
    assert max(np.abs(eager.mass.cpu().numpy()[:, s][..., live[s]] - mass[:, s][..., live[s]]).max() for s in range(2)) < 2.0 ** -15


def test_two_handles_side_by_side(backend):
    """Handles have workspaces of their own: two streams at once give what one after the other gives."""
    import torch

    both = [Held(backend, "q4", "f16", 2, 128, [3000, 500], seed=s) for s in (1, 2)]
    q = torch.randn((2, 8, 128), device="cuda").half()
    first, ctx = ints([0, 1, 2]), ints([2999, 499])
    mass = [torch.zeros((2, 2, made.tables.shape[1] * PAGE), device="cuda") for made in both]
    out = [torch.zeros_like(q) for _ in both]

    def call(i, st):
        both[i].cache.attention_tokens(q, first, ctx, 0.1, out[i], 1, 2999, mass=mass[i], stream=st)

    for i in range(2):
        call(i, current())
    torch.cuda.synchronize()
    want = [o.clone() for o in out], [m.clone() for m in mass]
    streams = [torch.cuda.Stream() for _ in both]
    for _ in range(10):
        for i in range(2):
            mass[i].zero_()
        torch.cuda.synchronize()
        for i in range(2):
            call(i, streams[i].cuda_stream)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out + mass, want[0] + want[1]))


# ------------------------------------------------------------------------------------------- refusals
def test_refusals(backend):
    import torch

    from orangu_b200 import OranguError, PagedCache, capi, verify_drafts

    L = backend._lib
    x = torch.zeros((2, 4, 2, 9 * 64), dtype=torch.uint8, device="cuda")
    half = torch.zeros((2, 4, 2, PAGE, 64), dtype=torch.float16, device="cuda")
    t, host = ints([[0, 1], [2, 3]]), torch.zeros(1 << 16, dtype=torch.float16)
    p = lambda a: a.data_ptr()  # noqa: E731

    def made(**change):
        d = dict(k=p(x), v=p(x), layer_stride=x[0].numel(), type=256, n_layer=2, n_pages=4, n_head_kv=2, head_dim=64, n_seq=2, table_stride=2, tables=p(t))
        d.update(change)
        desc, h = capi.PagesDesc(**d), C.c_void_p()
        rc = L.ob_pages_create(backend._h, C.byref(desc), C.byref(h))
        if rc == 0:
            L.ob_pages_destroy(h)
        return rc

    assert made() == 0
    for change, rc in ((dict(type=2), -2), (dict(type=255), -2), (dict(head_dim=96), -2), (dict(layer_stride=x[0].numel() + 8), -1), (dict(layer_stride=x[0].numel() - 16), -1), (dict(k=p(x) + 8), -1),
                       (dict(n_pages=1 << 27, n_layer=1), -2), (dict(v=host.data_ptr()), -1)):
        assert made(**change) == rc, change
    cache, wide = PagedCache(backend, x, x.clone(), t), PagedCache(backend, half, half.clone(), t)
    h, w = cache._h, wide._h
    q = torch.zeros((6, 4, 64), dtype=torch.float16, device="cuda")
    kv = torch.zeros((6, 2, 64), dtype=torch.float16, device="cuda")
    out, first, ctx, bits, i = torch.full_like(q, 9.0), ints([0, 2, 6]), ints([3, 4]), words([1] * 6), ints([5] * 64)
    mass, all_mass, fl = torch.zeros((2, 2, 32), device="cuda"), torch.zeros((2, 2, 2, 32), device="cuda"), torch.zeros(64, device="cuda")

    # operators of 16-bit pages over 4-bit ones, and the other way round
    assert L.ob_pages_attention_tree(h, 0, 2, p(q), 256, 6, p(first), p(ctx), p(bits), 4, 4, 4, 0.1, p(out), 256, None) == -2
    assert L.ob_pages_attention(h, 0, 2, p(q), 256, None, p(i), 4, p(i), 2, 0.1, p(out), 256, None) == -2
    assert L.ob_pages_select(h, p(x), p(fl), 2, p(q), 256, None, p(i), 4, 32, 2, 0, 0, p(i), None) == -2
    assert L.ob_pages_bounds(h, 0, 2, p(i), p(i), 4, p(x), p(fl), None) == -2

    def tokens(handle=h, **change):
        a = dict(layer=0, n_seq=2, q=p(q), type=1, qs=256, n=6, first=p(first), ctx=p(ctx), bits=None, heads=4, most=4, max_ctx=4, scale=0.1, out=p(out), os=256, mass=None, ms=0, st=None)
        a.update(change)
        return L.ob_pages_attention_tokens(handle, *a.values())

    assert tokens() == 0 and tokens(w) == 0 and tokens(n_seq=0) == 0 and tokens(n=0) == 0 and tokens(most=0) == 0 and tokens(mass=p(mass), ms=32) == 0 and tokens(type=30) == 0 and tokens(most=1 << 30) == 0
    for change, rc in ((dict(layer=2), -1), (dict(n_seq=3), -1), (dict(heads=3), -1), (dict(heads=0), -1), (dict(heads=34, qs=34 * 64, os=34 * 64), -2), (dict(bits=p(bits), most=65), -2), (dict(scale=0.0), -1),
                       (dict(scale=float("nan")), -1), (dict(qs=248), -1), (dict(os=260), -1), (dict(q=None), -1), (dict(q=p(q) + 2), -1), (dict(out=p(out) + 8), -1), (dict(first=None), -1),
                       (dict(bits=p(bits) + 4), -1), (dict(ctx=host.data_ptr()), -1), (dict(n=1 << 31), -1), (dict(type=0), -1), (dict(type=256), -1), (dict(mass=p(mass), ms=31), -1), (dict(mass=p(mass) + 2, ms=32), -1),
                       (dict(mass=host.data_ptr(), ms=32), -1), (dict(mass=p(mass), ms=32, n=1 << 20), -6)):
        assert tokens(**change) == rc, change
    assert tokens(w, type=30) == -1 and tokens(w, type=256) == -1

    def store(fn=L.ob_pages_store, handle=h, **change):
        a = dict(layer=0, n_seq=2, k=p(kv), v=p(kv), type=1, ks=128, vs=128, n=6, first=p(first), ctx=p(ctx), most=4, st=None)
        a.update(change)
        return fn(handle, *a.values())

    for fn in (L.ob_pages_store, L.ob_pages_load):
        assert store(fn) == 0 and store(fn, n_seq=0) == 0 and store(fn, most=0) == 0 and store(fn, n=0) == 0
        for change, rc in ((dict(handle=w), -2), (dict(layer=2), -1), (dict(n_seq=3), -1), (dict(type=0), -1), (dict(type=256), -1), (dict(ks=120), -1), (dict(vs=130), -1), (dict(k=None), -1), (dict(v=p(kv) + 2), -1),
                           (dict(first=None), -1), (dict(ctx=p(ctx) + 2), -1), (dict(k=host.data_ptr()), -1), (dict(n=1 << 31), -1)):
            assert store(fn, **change) == rc, change

    def evict(**change):
        a = dict(n_seq=2, n_pos=p(i), mass=p(all_mass), ms=32, max_pos=32, n_keep=4, first=1, last=1, kept=p(i) + 128, left=p(i) + 64, st=None)
        a.update(change)
        return L.ob_pages_evict(h, *a.values())

    assert evict(n_seq=0) == 0
    for change, rc in ((dict(n_seq=3), -1), (dict(n_keep=0), -1), (dict(first=4), -1), (dict(first=0xffffffff, last=2), -1), (dict(ms=31), -1), (dict(n_pos=None), -1), (dict(mass=None), -1), (dict(kept=host.data_ptr()), -1),
                       (dict(left=p(i)), -1), (dict(mass=p(all_mass) + 1), -1)):
        assert evict(**change) == rc, change
    assert L.ob_pages_keep_mass(h, 3, p(i), p(i), 2, p(i), p(all_mass), 32, None) == -1 and L.ob_pages_keep_mass(h, 2, p(i), p(i), 65, p(i), p(all_mass), 32, None) == -1
    assert L.ob_pages_keep_mass(h, 2, p(i), p(i), 2, p(i), p(all_mass), 31, None) == -1 and L.ob_pages_keep_mass(h, 2, p(i), p(i), 2, p(i), None, 32, None) == -1 and L.ob_pages_keep_mass(h, 0, None, None, 2, None, None, 32, None) == 0
    assert L.ob_pages_keep(h, 2, p(i), p(i), 65, p(i), None) == -1

    probs = torch.zeros((6, 10), device="cuda")

    def verify(ctx=backend._h, **change):
        a = dict(n_seq=2, n=6, vocab=10, type=0, target=p(probs), ts=10, draft=p(probs), ds=10, tokens=p(i), parent=p(i), first=p(first), uniform=p(fl), kept=p(i) + 128, ks=2, n_kept=p(i) + 64, next=p(i) + 80, st=None)
        a.update(change)
        return L.ob_drafts_verify(ctx, *a.values())

    assert verify(n_seq=0) == 0 and verify(None) == -1
    for change, rc in ((dict(type=8), -2), (dict(vocab=0), -1), (dict(vocab=1 << 31, ts=1 << 32, ds=1 << 32), -1), (dict(ts=9), -1), (dict(ds=9), -1), (dict(ks=0), -1), (dict(ks=65), -1), (dict(n=1 << 31), -1), (dict(target=None), -1),
                       (dict(draft=p(probs) + 2), -1), (dict(tokens=None), -1), (dict(parent=p(i) + 1), -1), (dict(first=host.data_ptr()), -1), (dict(uniform=None), -1), (dict(kept=None), -1), (dict(n_kept=None), -1),
                       (dict(next=None), -1), (dict(n_seq=(1 << 24) + 1), -1)):
        assert verify(**change) == rc, change
    backend.synchronize()
    torch.cuda.synchronize()
    # shapes and types in Python
    for call in (lambda: cache.attention_tree(q, first, ctx, bits, 0.1, out, 4, 4), lambda: cache.attention_tokens(q.float(), first, ctx, 0.1, out.float(), 4, 4), lambda: cache.attention_tokens(q, first, ctx, 0.1, out.bfloat16(), 4, 4),
                 lambda: cache.attention_tokens(q, first, ctx, 0.1, out, 4, 4, mass=mass[:1]), lambda: cache.attention_tokens(q, first, ctx, 0.1, out, 4, 4, visible=bits[:3]),
                 lambda: wide.attention_tokens(q.bfloat16(), first, ctx, 0.1, out.bfloat16(), 4, 4), lambda: cache.store(kv, kv[:3], first, ctx, 4), lambda: cache.store(kv, kv.bfloat16(), first, ctx, 4),
                 lambda: cache.load(kv.float(), kv.float(), first, ctx, 4), lambda: cache.store(q, q, first, ctx, 4), lambda: cache.evict(ctx, mass, ints([0]), ints([0, 0]), 4),
                 lambda: PagedCache(backend, x[..., :100].contiguous(), x[..., :100].contiguous(), t), lambda: PagedCache(backend, x, half, t)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(OranguError):
        wide.store(kv, kv, first, ctx, 4)
    n = ints([0, 0])
    for target, draft in ((probs.double(), None), (probs, probs.half()), (probs, probs[:3]), (probs.t(), None)):
        with pytest.raises(ValueError):
            verify_drafts(backend, target, draft, i[:6], i[:6], first, fl[:6], ints([[0], [0]]), n, n.clone())
