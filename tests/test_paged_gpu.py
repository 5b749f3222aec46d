"""The paged KV cache's operators on the GPU against plain 64-bit implementations
(paged_testlib), at the sizes, layouts and masks where they can go wrong."""
import math

import numpy as np
import pytest

import paged_testlib as P

pytestmark = pytest.mark.gpu


def _up(x, cuda):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).to(cuda)


def _close(got, want, bound, what):
    err = np.abs(got.astype(np.float64) - want)
    assert np.isfinite(got).all(), what
    at = np.unravel_index(np.argmax(err - bound), err.shape)
    assert (err <= bound).all(), "%s: off by %.3g at %s, bound %.3g" % (what, err[at], at, bound[at])


# ------------------------------------------------------------ attention ------

def _attend(nne, cuda, seed, dtype, b, hq, hkv, d, page, lens, t, parents=None, counts=None,
            scale=None, tweak=None, q_layout="bthd"):
    """attend() on random pools against attention64; rows past counts stay."""
    import torch
    rng = np.random.default_rng(seed)
    pages = P.Pages(rng, b, hkv, d, page, lens, t, dtype=dtype)
    if tweak:
        tweak(pages)
    cache = pages.cache(nne, cuda)
    q = rng.standard_normal((b, hq, t, d), dtype=np.float32)
    if q_layout == "bthd":
        qd = _up(q.transpose(0, 2, 1, 3), cuda).transpose(1, 2)
    elif q_layout == "odd":         # no unit stride, not 16-byte aligned
        buf = torch.zeros(b, hq, d, 2 * t + 1, device=cuda)
        buf[..., 1::2] = _up(q, cuda).transpose(2, 3)
        qd = buf[..., 1::2].transpose(2, 3)
    else:
        qd = _up(q, cuda)
    draft = None
    if parents is not None:
        draft = nne.DraftTree(parents, counts, device=cuda)
    elif counts is not None:
        draft = nne.DraftTree.chain(b, t, counts, device=cuda)
    if q_layout == "odd":
        obuf = torch.full((b, hq, d, t + 3), 7.0, device=cuda)
        out = obuf[..., 2:2 + t].transpose(2, 3)
    else:
        out = torch.full((b, t, hq, d), 7.0, device=cuda).transpose(1, 2)
    got = cache.attend(0, qd, draft=draft, out=out, scale=scale)
    again = cache.attend(0, qd, draft=draft, out=out.clone(), scale=scale)
    torch.cuda.synchronize()
    assert got is out
    g = got.cpu().numpy()
    assert np.array_equal(g, again.cpu().numpy()), "two calls differ"
    if q_layout == "odd":
        rest = obuf.cpu().numpy()
        assert (rest[..., :2] == 7).all() and (rest[..., -1] == 7).all()
    for i in range(b):
        n = t if counts is None else int(counts[i])
        if n < t:
            assert (g[i, :, n:] == 7).all(), "row of a token that does not exist was written"
        if n == 0:
            continue
        mask = P.visible(int(lens[i]), n, None if parents is None else parents[i])
        want, bound = P.attention64(q[i, :, :n], pages.rows(pages.k, i, int(lens[i]) + n),
                                    pages.rows(pages.v, i, int(lens[i]) + n), mask,
                                    1 / math.sqrt(d) if scale is None else scale)
        _close(g[i, :, :n], want, bound, "sequence %d" % i)
    return g, pages


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("b,hq,hkv,d,page,lens", [
    (1, 1, 1, 64, 16, [0]),                    # nothing cached: the token sees itself
    (2, 4, 4, 64, 16, [1, 15]),
    (3, 8, 2, 128, 16, [16, 17, 300]),
    (1, 12, 12, 64, 1, [77]),                  # pages of one row
    (2, 6, 2, 128, 7, [33, 250]),              # pages that end inside every tile
    (2, 3, 1, 80, 24, [129, 64]),              # padded dims
    (1, 2, 2, 8, 5, [40]),
    (1, 8, 1, 96, 48, [1000]),
    (2, 4, 2, 256, 32, [31, 700]),
    (1, 5, 5, 136, 10, [90]),
    (1, 16, 1, 128, 64, [5000]),               # many parts, more than one stage of rows
    (1, 20, 1, 64, 100, [2049]),               # more than 16 rows of one head
    (1, 40, 1, 128, 64, [513]),                # more than 32
    (1, 70, 1, 64, 33, [200]),                 # more than 64: two row blocks
    (1, 40, 1, 256, 64, [300]),
])
def test_one_token(nne, cuda, dtype, b, hq, hkv, d, page, lens):
    _attend(nne, cuda, 11, dtype, b, hq, hkv, d, page, lens, 1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("b,hq,hkv,d,page,lens,t", [
    (2, 4, 2, 64, 16, [0, 3], 2),
    (3, 8, 2, 128, 16, [14, 31, 700], 5),
    (1, 4, 4, 128, 8, [63], 17),
    (2, 4, 1, 64, 24, [100, 1], 33),
    (1, 2, 1, 128, 64, [1000], 100),
    (1, 3, 3, 256, 16, [47], 65),
    (1, 8, 8, 72, 11, [20], 40),
    (1, 4, 1, 128, 32, [3000], 300),           # a prompt chunk: many row blocks
])
def test_chain(nne, cuda, dtype, b, hq, hkv, d, page, lens, t):
    _attend(nne, cuda, 12, dtype, b, hq, hkv, d, page, lens, t)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("b,hq,hkv,d,page,lens,t", [
    (1, 4, 2, 64, 16, [0], 7),
    (2, 8, 2, 128, 16, [30, 517], 13),
    (3, 4, 4, 64, 9, [5, 64, 31], 32),
    (2, 8, 2, 128, 64, [1000, 129], 64),
    (1, 4, 1, 128, 16, [77], 100),
    (1, 2, 2, 64, 32, [40], 256),
    (1, 6, 2, 80, 16, [333], 21),
    (1, 2, 1, 256, 16, [60], 40),
])
def test_tree(nne, cuda, dtype, b, hq, hkv, d, page, lens, t):
    rng = np.random.default_rng(5)
    _attend(nne, cuda, 13, dtype, b, hq, hkv, d, page, lens, t,
            parents=P.random_parents(rng, b, t))


@pytest.mark.parametrize("t", [1, 31, 33, 64, 255, 256])
def test_tree_shapes(nne, cuda, t):
    """A path (the deepest tree), a star (the widest), and many roots."""
    path = np.arange(t, dtype=np.int32) - 1
    star = np.where(np.arange(t) == 0, -1, 0).astype(np.int32)
    roots = np.full(t, -1, np.int32)
    parents = np.stack([path, star, roots])
    tree, pages = _attend(nne, cuda, 14, "bf16", 3, 2, 1, 64, 16, [10, 50, 0], t, parents=parents)
    chain, _ = _attend(nne, cuda, 14, "bf16", 3, 2, 1, 64, 16, [10, 50, 0], t)
    if 2 * t <= 64:     # a path is a chain, to the bit where one block holds all rows (a chain's
        assert np.array_equal(tree[0], chain[0])    # later blocks have more keys, cut elsewhere)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tree", [False, True])
def test_counts(nne, cuda, dtype, tree):
    rng = np.random.default_rng(6)
    parents = P.random_parents(rng, 5, 9) if tree else None
    _attend(nne, cuda, 15, dtype, 5, 4, 2, 64, 16, [0, 40, 3, 600, 17], 9, parents=parents,
            counts=[9, 0, 1, 5, 8])
    _attend(nne, cuda, 15, dtype, 2, 8, 1, 64, 16, [100, 3], 40,       # 320 rows: blocks without a token
            parents=P.random_parents(rng, 2, 40) if tree else None, counts=[3, 40])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_odd_strides_and_scale(nne, cuda, dtype):
    _attend(nne, cuda, 16, dtype, 2, 4, 2, 64, 16, [20, 90], 3, q_layout="odd", scale=0.3)
    _attend(nne, cuda, 16, dtype, 1, 4, 2, 128, 16, [90], 1, q_layout="bhtd", scale=-0.2)
    _attend(nne, cuda, 16, dtype, 1, 4, 2, 128, 16, [90], 1, q_layout="odd", scale=0.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_ragged_batch_of_more_sequences_than_a_launch(nne, cuda, dtype):
    rng = np.random.default_rng(7)
    lens = rng.integers(0, 200, 150)
    lens[77] = 3000
    _attend(nne, cuda, 17, dtype, 150, 2, 1, 64, 16, lens, 2)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_what_is_not_seen_has_no_part(nne, cuda, dtype, bad):
    """Rows behind a sequence's, tokens of other paths and tokens past counts hold
    values that are not finite; so do pages of no sequence."""
    import torch
    t, lens = 6, [21, 40]
    parents = np.array([[-1, 0, 0, 1, 2, -1], [-1, -1, 1, 1, 2, 0]], np.int32)
    counts = [6, 4]

    def tweak(pages):
        used = np.zeros(pages.n_pages, bool)
        for b in range(2):
            n = lens[b] + counts[b]
            used[pages.table[b, :-(-n // pages.page)]] = True
            for r in range(n, pages.page * (-(-n // pages.page))):
                for pool in (pages.k, pages.v):
                    pages.put(pool, b, r, np.full((2, 64), bad, np.float32))
        pages.k[:, ~used] = bad
        pages.v[:, ~used] = bad

    _attend(nne, cuda, 18, dtype, 2, 8, 2, 64, 16, lens, t, parents=parents, counts=counts,
            tweak=tweak)

    # One drafted token's row is not finite: the tokens below it see it, the
    # others' results are those of finite values.
    rng = np.random.default_rng(19)
    pages = P.Pages(rng, 1, 2, 64, 16, [21], t, dtype=dtype)
    q = rng.standard_normal((1, 8, t, 64), dtype=np.float32)
    tree = nne.DraftTree(parents[:1], device=cuda)
    clean = pages.cache(nne, cuda).attend(0, _up(q, cuda), draft=tree).cpu().numpy()
    below = P.visible(0, t, parents[0])[:, 1]          # sees token 1
    for pool in (pages.v, pages.k):
        keep = pool.copy()
        row = pages.rows(pool, 0, 23)[:, 22].copy()
        row[:, 5:9] = bad
        pages.put(pool, 0, 22, row)
        got = pages.cache(nne, cuda).attend(0, _up(q, cuda), draft=tree).cpu().numpy()
        torch.cuda.synchronize()
        assert np.array_equal(got[0][:, ~below], clean[0][:, ~below])
        if pool is pages.v:
            assert not np.isfinite(got[0][:, below, 5:9]).any()
            if np.isinf(bad):
                assert (got[0][:, below, 5:9] == bad).all()
        elif np.isnan(bad):
            assert not np.isfinite(got[0][:, below]).any()
        pool[...] = keep


def test_nan_in_a_counted_row_shows(nne, cuda):
    rng = np.random.default_rng(20)
    for dtype in ("f32", "bf16"):
        pages = P.Pages(rng, 1, 1, 64, 16, [50], 1, dtype=dtype)
        row = pages.rows(pages.k, 0, 20)[:, 19].copy()
        row[:, 0] = np.nan
        pages.put(pages.k, 0, 19, row)
        q = _up(rng.standard_normal((1, 2, 1, 64), dtype=np.float32), cuda)
        assert np.isnan(pages.cache(nne, cuda).attend(0, q).cpu().numpy()).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scores_of_any_size(nne, cuda, dtype):
    """Weights between 1 and 0, and all equal; queries and values far from 1."""
    rng = np.random.default_rng(21)
    for factor, vfactor in ((30.0, 1.0), (0.0, 1.0), (1e-20, 1e20), (1.0, 1e-30)):
        pages = P.Pages(rng, 1, 2, 128, 16, [400], 1, dtype=dtype)
        pages.v *= np.float32(vfactor)
        if dtype == "bf16":
            pages.v = P.bf16(pages.v)
        q = rng.standard_normal((1, 4, 1, 128), dtype=np.float32) * np.float32(factor)
        got = pages.cache(nne, cuda).attend(0, _up(q, cuda)).cpu().numpy()
        want, bound = P.attention64(q[0], pages.rows(pages.k, 0, 401), pages.rows(pages.v, 0, 401),
                                    np.ones((1, 401), bool), 1 / math.sqrt(128))
        _close(got[0], want, bound, "factor %g" % factor)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("t", [1, 24])
def test_float32_precision(nne, cuda, dtype, t):
    """Roundings to nearest are independent: of N(0, 1) inputs a score of d = 128
    products ends off by about sqrt(d) EPS times its partial sums' size of 1 at
    most, 7e-7, weights by that, and an output relative to the outputs' size too
    (both are sums over the same keys with signs at random).  An operand held to
    16 bits somewhere would give 2^-17 / sqrt(3), 4e-6."""
    rng = np.random.default_rng(22)
    pages = P.Pages(rng, 2, 2, 128, 16, [900, 333], t, dtype=dtype)
    q = rng.standard_normal((2, 8, t, 128), dtype=np.float32)
    got = pages.cache(nne, cuda).attend(0, _up(q, cuda)).cpu().numpy().astype(np.float64)
    for b, n in enumerate((900, 333)):
        want, _ = P.attention64(q[b], pages.rows(pages.k, b, n + t), pages.rows(pages.v, b, n + t),
                                P.visible(n, t, None), 1 / math.sqrt(128))
        assert np.linalg.norm(got[b] - want) <= 1e-6 * np.linalg.norm(want)


def test_a_contiguous_cache_is_one_page_a_sequence(nne, cuda):
    """The pools of a KVCache layer as a paged cache of one page per sequence:
    the same step as decode_step's, within both kernels' bounds."""
    import torch
    rng = np.random.default_rng(23)
    b, hq, hkv, d, cap = 3, 8, 2, 128, 333
    lens = np.array([0, 100, 332], np.int32)
    old = nne.KVCache(1, b, hkv, cap, d, device=cuda)
    old.k[0].copy_(_up(rng.standard_normal((b, hkv, cap, d), dtype=np.float32), cuda))
    old.v[0].copy_(_up(rng.standard_normal((b, hkv, cap, d), dtype=np.float32), cuda))
    old.set_lengths(0, lens)
    new = nne.PagedKVCache(1, b, hkv, cap, d, b, 1, device=cuda)
    new.k = old.k[0].clone()[None]
    new.v = old.v[0].clone()[None]
    new.set_table(np.arange(b)[:, None])
    new.set_lengths(lens)
    q, k, v = (_up(rng.standard_normal((b, h, 1, d), dtype=np.float32), cuda) for h in (hq, hkv, hkv))
    want = old.decode_step(0, q, k, v)
    new.append(0, k, v)
    got = new.attend(0, q)
    new.commit(1)
    torch.cuda.synchronize()
    assert torch.equal(new.k[0], old.k[0]) and torch.equal(new.v[0], old.v[0])
    assert np.array_equal(new.lens_host, old.lens_host[0])
    assert torch.equal(new.lens_dev, old.lens_dev[0])
    kk, vv = old.k[0].cpu().numpy(), old.v[0].cpu().numpy()
    for i in range(b):
        n = int(lens[i]) + 1
        _, bound = P.attention64(q[i].cpu().numpy(), kk[i, :, :n], vv[i, :, :n], np.ones((1, n), bool),
                                 1 / math.sqrt(d))
        _close(got[i].cpu().numpy(), want[i].cpu().numpy().astype(np.float64), 2 * bound, "sequence %d" % i)


def test_pool_beyond_32_bit_offsets(nne, cuda):
    """Rows whose byte and element offsets pass 2^32: the last pages of a pool of
    17 GiB."""
    import torch
    n_pages, hkv, page, d = 70000, 4, 128, 128       # 4.6e9 elements of K
    cache = nne.PagedKVCache(1, n_pages, hkv, page, d, 2, 4, dtype=torch.bfloat16, device=cuda)
    lens, t, hq = [300, 129], 3, 8
    table = np.array([[n_pages - 1, 5, n_pages - 2, -1], [n_pages - 70, n_pages - 69, -1, -1]])
    cache.set_table(table)
    rng = np.random.default_rng(24)
    k = P.bf16(rng.standard_normal((2, hkv, 303, d), dtype=np.float32))
    v = P.bf16(rng.standard_normal((2, hkv, 303, d), dtype=np.float32))
    for b in range(2):                               # rows in by append, 300 and 129
        counts = [0, 0]
        counts[b] = lens[b]
        ch = nne.DraftTree.chain(2, 303, counts, device=cuda)
        cache.append(0, _up(k, cuda), _up(v, cuda), draft=ch)
        cache.commit(ch.counts_dev, ch.counts_host)
    rows = [k[b][:, lens[b]:lens[b] + t] for b in range(2)], [v[b][:, lens[b]:lens[b] + t] for b in range(2)]
    cache.append(0, _up(np.stack(rows[0]), cuda), _up(np.stack(rows[1]), cuda))
    q = rng.standard_normal((2, hq, t, d), dtype=np.float32)
    got = cache.attend(0, _up(q, cuda)).cpu().numpy()
    for b in range(2):
        n = lens[b] + t
        assert np.array_equal(P.host(cache.k[0, table[b, 0], :, 7]), k[b][:, 7])
        want, bound = P.attention64(q[b], k[b][:, :n], v[b][:, :n], P.visible(lens[b], t, None),
                                    1 / math.sqrt(d))
        _close(got[b], want, bound, "sequence %d" % b)


def test_shared_prefix_pages(nne, cuda):
    rng = np.random.default_rng(25)
    pages = P.Pages(rng, 2, 2, 64, 16, [40, 40], 1)
    pages.table[1, :2] = pages.table[0, :2]
    cache = pages.cache(nne, cuda)
    q = rng.standard_normal((2, 4, 1, 64), dtype=np.float32)
    got = cache.attend(0, _up(q, cuda)).cpu().numpy()
    for b in range(2):
        want, bound = P.attention64(q[b], pages.rows(pages.k, b, 41), pages.rows(pages.v, b, 41),
                                    np.ones((1, 41), bool), 1 / 8)
        _close(got[b], want, bound, "sequence %d" % b)


# --------------------------------------------------------------- append ------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("b,hkv,d,page,lens,t", [
    (1, 1, 64, 16, [0], 1), (3, 2, 128, 16, [15, 16, 17], 1), (2, 4, 8, 3, [0, 5], 10),
    (2, 3, 80, 24, [23, 100], 33), (1, 2, 256, 1, [9], 7), (1, 8, 128, 64, [130], 500),
])
@pytest.mark.parametrize("rotate", ["no", "chain", "tree"])
def test_append(nne, cuda, dtype, b, hkv, d, page, lens, t, rotate):
    """The appended rows are RotaryEmbedding.apply's to the bit (then rounded to
    the pool's type), and nothing else in the pools changes."""
    import torch
    rng = np.random.default_rng(31)
    pages = P.Pages(rng, b, hkv, d, page, lens, t, layers=2, dtype=dtype)
    cache = pages.cache(nne, cuda)
    k = rng.standard_normal((b, t, hkv, d), dtype=np.float32)
    v = rng.standard_normal((b, hkv, d, t), dtype=np.float32)
    kd, vd = _up(k, cuda).transpose(1, 2), _up(v, cuda).transpose(2, 3)     # rows of V: no unit stride
    if rotate == "no":
        vd = vd.contiguous()
    rope = nne.RotaryEmbedding(d, max(lens) + t, device=cuda) if rotate != "no" else None
    draft, pos = None, np.asarray(lens)[:, None] + np.arange(t)
    if rotate == "tree":
        parents = P.random_parents(rng, b, t)
        draft = nne.DraftTree(parents, device=cuda)
        pos = np.asarray(lens)[:, None] + P.depths_of(parents)
    cache.append(1, kd, vd, rope=rope, draft=draft)
    torch.cuda.synchronize()
    turned = k.transpose(0, 2, 1, 3).copy()
    if rope is not None:
        for i in range(b):
            for j in range(t):
                turned[i, :, j] = rope.apply(kd[i:i + 1, :, j:j + 1], int(pos[i, j]))[0, :, 0].cpu().numpy()
    for i in range(b):
        for j in range(t):
            pages.put(pages.k, i, lens[i] + j, turned[i, :, j], layer=1)
            pages.put(pages.v, i, lens[i] + j, v[i, :, :, j], layer=1)
    assert np.array_equal(P.host(cache.k), pages.k)
    assert np.array_equal(P.host(cache.v), pages.v)
    assert np.array_equal(cache.lens_dev.cpu().numpy(), np.asarray(lens))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_counts_and_values(nne, cuda, dtype):
    """Rows past counts are not written; zeros, infinities and NaN arrive as they are."""
    rng = np.random.default_rng(32)
    pages = P.Pages(rng, 3, 1, 64, 16, [3, 14, 30], 4, dtype=dtype)
    cache = pages.cache(nne, cuda)
    k = rng.standard_normal((3, 1, 4, 64), dtype=np.float32)
    k[0, 0, 0, :6] = [0.0, -0.0, np.inf, -np.inf, np.nan, 1e-40]
    k[0, 0, 1, :2] = [3.3895e38, 1.00390625]         # rounds to inf in bf16; a tie
    counts = [2, 0, 4]
    cache.append(0, _up(k, cuda), _up(-k, cuda), draft=nne.DraftTree.chain(3, 4, counts, device=cuda))
    for i in range(3):
        for j in range(counts[i]):
            pages.put(pages.k, i, pages.lens[i] + j, k[i, :, j])
            pages.put(pages.v, i, pages.lens[i] + j, -k[i, :, j])
    for got, want in ((P.host(cache.k), pages.k), (P.host(cache.v), pages.v)):
        nan = np.isnan(want)
        assert np.array_equal(np.isnan(got), nan)
        assert np.array_equal(got[~nan].view(np.uint32), want[~nan].view(np.uint32))


# --------------------------------------------------------------- commit ------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layers,b,hkv,d,page,lens,t,j", [
    (1, 1, 1, 64, 16, [0], 1, 1), (3, 2, 2, 128, 16, [14, 100], 13, 5), (2, 3, 1, 8, 3, [0, 7, 31], 40, 40),
    (2, 2, 4, 80, 7, [5, 6], 64, 8), (5, 1, 3, 256, 32, [31], 30, 20),
])
def test_commit(nne, cuda, dtype, layers, b, hkv, d, page, lens, t, j):
    rng = np.random.default_rng(41)
    for trial in range(3):
        pages = P.Pages(rng, b, hkv, d, page, lens, t, layers=layers, dtype=dtype)
        cache = pages.cache(nne, cuda)
        paths = np.sort(np.argsort(rng.random((b, t)), 1)[:, :j], 1).astype(np.int32)
        if trial == 1 and j < t:
            paths = np.broadcast_to(np.arange(1, j + 1, dtype=np.int32), (b, j)).copy()   # shifted by one
        counts = rng.integers(0, j + 1, b).astype(np.int32)
        counts[-1] = j
        cache.commit(_up(counts, cuda), counts, _up(paths, cuda), paths)
        for layer in range(layers):
            for i in range(b):
                for n in range(counts[i]):
                    for pool in (pages.k, pages.v):
                        r = int(lens[i]) + int(paths[i, n])
                        row = pool[layer, pages.table[i, r // page], :, r % page].copy()
                        pages.put(pool, i, int(lens[i]) + n, row, layer=layer)
        assert np.array_equal(P.host(cache.k), pages.k)
        assert np.array_equal(P.host(cache.v), pages.v)
        assert np.array_equal(cache.lens_host, np.asarray(lens) + counts)
        assert np.array_equal(cache.lens_dev.cpu().numpy(), cache.lens_host)


def test_commit_first_tokens(nne, cuda):
    rng = np.random.default_rng(42)
    pages = P.Pages(rng, 3, 1, 64, 16, [0, 5, 30], 8)
    cache = pages.cache(nne, cuda)
    cache.commit(2)
    counts = np.array([0, 3, 6], np.int32)
    cache.commit(_up(counts, cuda), counts)
    assert list(cache.lens_host) == [2, 10, 38]
    assert list(cache.lens_dev.cpu().numpy()) == [2, 10, 38]
    assert np.array_equal(P.host(cache.k), pages.k)


# ----------------------------------------------------------------- norm ------

def _norm_bound(x, w, eps, cos, sin, pos):
    """A normalised value is off by (d + 12) EPS relative (the sum of squares d of
    them at most, halved by the root; the root, quotient and two products), the
    rotation adds two products and a sum of values no larger than both of the pair
    together."""
    n = np.abs(P.norm_rope64(x, w, eps, None, None, None))
    half = n.shape[-1] // 2
    pair = n + np.concatenate([n[..., half:], n[..., :half]], -1)
    return (x.shape[-1] / 2 + 12) * P.EPS * pair + 1e-38


@pytest.mark.parametrize("b,t,hq,hkv,d", [
    (1, 1, 1, 1, 64), (2, 3, 4, 2, 128), (3, 17, 5, 1, 80), (1, 9, 2, 2, 8), (2, 2, 3, 1, 2),
    (1, 5, 2, 1, 256), (1, 3, 2, 2, 512), (1, 2, 1, 1, 1024), (2, 7, 3, 3, 30), (1, 1, 12, 12, 136),
    (32, 1, 32, 8, 128),
])
@pytest.mark.parametrize("layout", ["bthd", "bhtd", "odd"])
def test_norm_rope(nne, cuda, b, t, hq, hkv, d, layout):
    import torch
    rng = np.random.default_rng(51)
    q = rng.standard_normal((b, hq, t, d), dtype=np.float32) * 3
    k = rng.standard_normal((b, hkv, t, d), dtype=np.float32) * 0.1
    wq, wk = (1 + 0.2 * rng.standard_normal(d, dtype=np.float32) for _ in range(2))
    start = rng.integers(0, 50, b).astype(np.int32)
    parents = P.random_parents(rng, b, t)
    rope = nne.RotaryEmbedding(d, 50 + t, device=cuda)

    def dev(x):
        if layout == "bthd":
            return _up(x.transpose(0, 2, 1, 3), cuda).transpose(1, 2)
        if layout == "odd":
            return _up(x.transpose(0, 1, 3, 2), cuda).transpose(2, 3)
        return _up(x, cuda)

    for tree in (False, True):
        draft = nne.DraftTree(parents, device=cuda) if tree else None
        pos = start[:, None] + (P.depths_of(parents) if tree else np.arange(t))
        qd, kd = dev(q), dev(k)
        qo, ko = nne.qk_norm_rope(qd, kd, _up(wq, cuda), _up(wk, cuda), rope, _up(start, cuda), start,
                                  eps=1e-5, draft=draft)
        for x, w, got in ((q, wq, qo), (k, wk, ko)):
            _close(got.cpu().numpy(), P.norm_rope64(x, w, 1e-5, rope.cos_host, rope.sin_host, pos),
                   _norm_bound(x, w, 1e-5, rope.cos_host, rope.sin_host, pos), "tree %s" % tree)
        # in place, the same bits
        a, c = nne.qk_norm_rope(qd, kd, _up(wq, cuda), _up(wk, cuda), rope, _up(start, cuda), start,
                                eps=1e-5, draft=draft, q_out=qd, k_out=kd)
        assert a is qd and c is kd
        assert torch.equal(qd, qo) and torch.equal(kd, ko)
    # the rotation alone is RotaryEmbedding.apply's, to the bit
    qd = dev(q)
    got, none = nne.qk_norm_rope(qd, None, None, None, rope, _up(start, cuda), start, eps=None)
    assert none is None and torch.equal(got, rope.apply(qd, start))
    # the norm alone, without weights
    got, _ = nne.qk_norm_rope(qd, None, None, None, None, None, None, eps=0.0)
    _close(got.cpu().numpy(), P.norm_rope64(q, None, 0.0, None, None, None),
           _norm_bound(q, None, 0.0, None, None, None), "norm alone")


def test_norm_of_zeros_and_one_sided_eps(nne, cuda):
    import torch
    x = torch.zeros(1, 2, 3, 64, device=cuda)
    got, _ = nne.qk_norm_rope(x, None, None, None, None, None, None, eps=1e-6)
    assert (got == 0).all()
    x[0, 0, 0, 3] = float("nan")
    got, _ = nne.qk_norm_rope(x, None, None, None, None, None, None, eps=1e-6)
    assert torch.isnan(got[0, 0, 0]).all() and (got[0, 1] == 0).all() and (got[0, 0, 1:] == 0).all()
