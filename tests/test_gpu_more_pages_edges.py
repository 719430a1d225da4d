"""4-bit pages, weights per position, cut caches and verified drafts where they went wrong once: values that cancel, keys that are no finite numbers, paths longer than
their list, numbers that are none."""
import numpy as np
import pytest

import more_pages_plain as more
import pages_plain as plain
from gpu_common import backend  # noqa: F401
from test_gpu_more_pages import U, Held, current, distributions, run_verify, weight_error
from test_gpu_pages import PAGE, device16, float64, ints, words

pytestmark = pytest.mark.gpu


def attend(made, q, kind, ctx, counts, bits, scale, mass=None):
    """Output of attention_tokens over `made`, as float64; `mass` (a device array) is added to."""
    import torch

    qd = device16(plain.to16(q, kind)[1], kind)
    out = torch.full_like(qd, 7.0)
    made.cache.attention_tokens(qd, ints(np.concatenate([[0], np.cumsum(counts)])), ints(ctx), scale, out, max_tokens=max(counts), max_context=max(ctx), visible=words(bits) if bits is not None else None, mass=mass,
                                stream=current())
    made.cache.synchronize(current())
    return float64(out)


# ------------------------------------------------------------------------------------------- weights and their remainders
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("dim,group,count", [(128, 4, 1), (64, 8, 1), (128, 2, 8), (64, 4, 8), (128, 4, 16), (64, 16, 7), (128, 8, 64), (64, 4, 64)])
def test_values_that_cancel(backend, kind, dim, group, count):
    """Two positions with nearly the same weight and opposite values: what is left of them is off by the weights' errors, which the output's rounding does not hide.  A
    weight that were one number of 11 bits would be off by up to 2^-11, a few times the bound (sum |q k| is about a half here)."""
    made = Held(backend, "q4", kind, 2, dim, [2 + count], seed=dim + group + count)
    x = made.r.standard_normal((2 + count, 2, dim))
    y = made.r.standard_normal((2 + count, 2, dim))
    y[1] = -y[0]
    rows = [plain.to16(z, kind) for z in (x, y)]
    made.cache.store(*(device16(b, kind) for _, b in rows), ints([0, 2 + count]), ints([0]), max_tokens=2 + count, stream=current())
    k, v = (more.in_four_bits(z) for z, _ in rows)
    q = plain.to16(made.r.standard_normal((count, 2 * group, dim)) * 0.1, kind)[0]
    scale, first, bits = 0.25 * 64 / dim / 4, [0, count], [0] * count  # drafts see the context alone
    want = np.zeros(q.shape)
    tol, _ = more.attend_tokens(q, [k], [v], made.there, first, [2], bits, scale, want, None, weight_error(dim))
    got = attend(made, q, kind, [2], [count], bits, scale)
    off = np.abs(got - want) - (tol[..., None] + U[kind] * (np.abs(want) + tol[..., None]) + 2.0 ** -25)
    assert off.max() <= 0, f"{off.max()} over the bound ({tol.max()}) at {np.unravel_index(off.argmax(), off.shape)}"


# ------------------------------------------------------------------------------------------- weights where keys are no finite numbers
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("dim,group,count", [(64, 1, 1), (128, 3, 1), (64, 4, 5), (128, 3, 40), (64, 7, 20)])
def test_a_key_that_every_row_puts_at_minus_infinity(backend, kind, dim, group, count):
    """Its weight is zero in every row, and in the columns that fill up a set there is none: what the position had gathered stays, whatever kernel the number of rows takes."""
    import torch

    ctx, at, entry = 50, 21, 5
    made = Held(backend, kind, kind, 2, dim, [ctx + count], seed=dim + group + count)
    page = int(made.tables[0, at // PAGE])
    made.kd[0, page, :, at % PAGE, entry] = float("inf")
    q = plain.to16(made.r.standard_normal((count, 2 * group, dim)), kind)[0]
    q[..., entry] = -np.abs(q[..., entry]) - 0.25
    q = plain.to16(q, kind)[0]  # as the device has them
    mass = made.r.exponential(1.0, (1, 2, made.tables.shape[1] * PAGE)).astype(np.float32)
    md, want, mass64 = torch.from_numpy(mass).cuda(), np.zeros(q.shape), mass.astype(np.float64)
    there = [made.there[0].copy()]
    there[0][at] = False  # a weight of zero
    tol, mass_tol = more.attend_tokens(q, made.k[0], made.v[0], there, [0, count], [ctx], None, dim ** -0.5, want, mass64, weight_error(dim))
    got = attend(made, q, kind, [ctx], [count], None, dim ** -0.5, md)
    off = np.abs(got - want) - (tol[..., None] + U[kind] * (np.abs(want) + tol[..., None]) + 2.0 ** -25)
    assert off.max() <= 0
    masses = md.cpu().numpy()
    assert np.isfinite(masses).all() and np.array_equal(masses[0, :, at], mass[0, :, at])
    assert (np.abs(masses - mass64) <= mass_tol).all()


# ------------------------------------------------------------------------------------------- cutting caches down
def test_a_list_of_almost_all_numbers(backend):
    """n_keep may be anything that 32 bits hold: what lies behind the last position is filled up to the end."""
    import torch

    n_keep = (1 << 32) - 1
    if torch.cuda.mem_get_info()[0] < 6 * n_keep:
        pytest.skip("not enough memory")
    made = Held(backend, "q4", "f16", 1, 64, [40], seed=1)
    kept, left, mass = torch.zeros((1, 1, 1, n_keep), dtype=torch.int32, device="cuda"), ints([0]), torch.ones((1, 1, 1, made.tables.shape[1] * PAGE), device="cuda")
    made.cache.evict(ints([40]), mass, kept, left, max_pos=40, stream=current())
    torch.cuda.synchronize()
    flat = kept.view(-1)
    assert left.item() == 40 and torch.equal(flat[:40].cpu(), torch.arange(40, dtype=torch.int32))
    assert all(bool((part == -1).all()) for part in flat[40:].split(1 << 28))
    del kept, flat
    torch.cuda.empty_cache()  # (17 GB)


# ------------------------------------------------------------------------------------------- verification
def in_list(parent, first, width):
    """The tree without the nodes whose paths are longer than the list: nobody's children."""
    out = np.array(parent).copy()
    for a, b in zip(first[:-1], first[1:]):
        depth = np.zeros(b - a, int)
        for i in range(1, b - a):
            depth[i] = depth[parent[a + i]] + 1
            if depth[i] >= width:
                out[a + i] = -1
    return out


def chain_with_siblings(m):
    """Every third node is the child of a node that has one already; the others go on from each other."""
    parent, last = [-1], 0
    for i in range(1, m):
        parent.append(last if i % 3 else max(0, parent[last]))
        last = i if i % 3 else last
    return parent


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("drafted", [True, False])
@pytest.mark.parametrize("width", [1, 2, 3, 5])
def test_a_path_ends_with_its_list(backend, kind, drafted, width):
    """No more nodes are accepted than the list holds, and the next token follows the last one in it."""
    import torch

    from orangu_b200 import verify_drafts

    r = np.random.default_rng(width)
    vocab, sizes = 300, [7, 1, 12, 64, 4] * 3
    first, n = np.concatenate([[0], np.cumsum(sizes)]), sum(sizes)
    target, draft = distributions(r, n, vocab, kind)
    draft = plain.to16(0.7 * target + 0.3 * draft, kind)[0] if kind != "f32" else (0.7 * target + 0.3 * draft).astype(np.float32).astype(np.float64)  # mostly accepted
    parent = np.concatenate([chain_with_siblings(m) for m in sizes])
    above = np.repeat(first[:-1], sizes) + np.maximum(parent, 0)
    tokens = np.array([r.choice(vocab, p=draft[a] / draft[a].sum()) if drafted else int(target[a].argmax()) for a in above])
    uniform = r.random(n).astype(np.float32) * (1.0 if drafted else 0.02)
    uniform[first[:-1]] = r.random(len(sizes))
    want = more.verify(target, draft if drafted else None, tokens, in_list(parent, first, width), first, uniform, width)
    assert (want[1] == width).sum() >= 5  # lists that are full
    device = lambda x: torch.from_numpy(x.astype(np.float32)).cuda() if kind == "f32" else device16(plain.to16(x, kind)[1], kind)  # noqa: E731
    kept, count, token = torch.full((len(sizes), width), 7, dtype=torch.int32, device="cuda"), ints([7] * len(sizes)), ints([7] * len(sizes))
    verify_drafts(backend, device(target), device(draft) if drafted else None, ints(tokens), ints(parent), ints(first), torch.from_numpy(uniform).cuda(), kept, count, token, stream=current())
    torch.cuda.synchronize()
    for got, w in zip((kept, count, token), want):
        assert np.array_equal(got.cpu().numpy(), w), (got, w)


@pytest.mark.parametrize("drafted", [True, False])
def test_no_nodes_at_all(backend, drafted):
    """A batch without drafts or certain tokens: empty arrays have no memory, and every sequence its answer."""
    import torch

    from orangu_b200 import verify_drafts

    rows, none = torch.zeros((0, 50), device="cuda"), ints([])
    kept, count, token = torch.full((3, 5), 7, dtype=torch.int32, device="cuda"), ints([7] * 3), ints([7] * 3)
    verify_drafts(backend, rows, rows if drafted else None, none, none, ints([0, 0, 0, 0]), torch.zeros(0, device="cuda"), kept, count, token, stream=current())
    torch.cuda.synchronize()
    assert bool((kept == -1).all()) and count.tolist() == [0, 0, 0] and token.tolist() == [-1, -1, -1]


@pytest.mark.parametrize("drafted", [True, False])
def test_random_numbers_that_are_none(backend, drafted):
    """They count as 0, as numbers below it do."""
    r = np.random.default_rng(8)
    target, draft = distributions(r, 6, 50, "f32")
    tokens, parent, first = np.array([0, 3, 4, 5, 6, 7]), np.array([-1, 0, 0, 1, 1, 2]), np.array([0, 6])
    for u in (np.full(6, np.nan), np.array([np.nan, 0.9, 0.9, 0.9, 0.9, 0.9]), np.array([0.7, 1.0, np.nan, 1.0, 1.0, np.nan]), np.array([-np.inf, np.inf, -1.0, 0.99, np.nan, 0.5])):
        run_verify(backend, "f32", target, draft if drafted else None, tokens, parent, first, u)
