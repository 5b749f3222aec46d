"""The paged cache's operators as a serving loop uses them: together, over steps,
captured and replayed, on other streams and workspaces, and what they refuse."""
import ctypes
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


def _check_attend(got, q, k, v, table, page, lens, counts, parents, what, scale=None):
    """got [B, Hq, T, d] against attention64 over pools k, v [n_pages, Hkv, page, d]."""
    for b in range(len(lens)):
        n, ctx = int(counts[b]), int(lens[b])
        if n == 0:
            continue
        r = np.arange(ctx + n)
        kb, vb = (x[table[b, r // page], :, r % page].transpose(1, 0, 2) for x in (k, v))
        want, bound = P.attention64(q[b, :, :n], kb, vb, P.visible(ctx, n, None if parents is None else parents[b]),
                                    1 / math.sqrt(q.shape[-1]) if scale is None else scale)
        _close(got[b, :, :n], want, bound, "%s, sequence %d" % (what, b))


def _norm_bound(x, w, cos, sin, pos):
    """(d + 12) EPS of a normalised value (its sum of squares d of them at most, halved by
    the root; root, quotient, two products), and the rotation's two products and sum."""
    n = np.abs(P.norm_rope64(x, w, 1e-6, None, None, None))
    half = n.shape[-1] // 2
    c, s = np.abs(cos.astype(np.float64)[pos][:, None]), np.abs(sin.astype(np.float64)[pos][:, None])
    swapped = np.concatenate([n[..., half:], n[..., :half]], -1)
    return (x.shape[-1] + 16) * P.EPS * (n * c + swapped * s) + 1e-38


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hq,hkv,d,page", [(4, 2, 64, 16), (6, 2, 40, 5)])
def test_serving_loop(nne, cuda, dtype, hq, hkv, d, page):
    """Prompts, then steps of single tokens, chains and trees: norm and rotation, append,
    attention in two layers, commit; a sequence ends and another takes its place."""
    import torch
    rng = np.random.default_rng(61)
    b, layers, limit = 3, 2, 256
    cache = nne.PagedKVCache(layers, 60, hkv, page, d, b, -(-limit // page),
                             dtype=torch.bfloat16 if dtype == "bf16" else torch.float32, device=cuda)
    k_ref, v_ref = P.host(cache.k), P.host(cache.v)
    rope = nne.RotaryEmbedding(d, limit, device=cuda)
    cos, sin = rope.cos.cpu().numpy(), rope.sin.cpu().numpy()
    wq, wk = (1 + rng.standard_normal(d, dtype=np.float32) / 8 for _ in range(2))
    lens = np.zeros(b, np.int32)
    steps = [("prompt", 37)] + [("token", 1), ("chain", 4), ("tree", 13), ("token", 1), ("tree", 40), ("end", 0),
                                ("tree", 6), ("chain", 9)]
    for at, (kind, t) in enumerate(steps):
        if kind == "end":
            cache.release(1)
            lens[1] = 0
            continue
        counts = parents = None
        if kind == "prompt":
            counts = np.array([t, 0, 20], np.int32)
        elif kind == "chain":
            counts = rng.integers(1, t + 1, b).astype(np.int32)
        elif kind == "tree":
            parents = P.random_parents(rng, b, t)
        cache.allocate(lens + t)
        if parents is not None:
            draft = nne.DraftTree(parents, counts, device=cuda)
        else:
            draft = None if counts is None else nne.DraftTree.chain(b, t, counts, device=cuda)
        have = np.full(b, t) if counts is None else counts
        depths = P.depths_of(parents) if parents is not None else np.tile(np.arange(t), (b, 1))
        pos = lens[:, None] + depths
        for layer in range(layers):
            what = "step %d layer %d" % (at, layer)
            x = [rng.standard_normal((b, h, t, d), dtype=np.float32) for h in (hq, hkv, hkv)]
            q, k = nne.qk_norm_rope(_up(x[0], cuda), _up(x[1], cuda), _up(wq, cuda), _up(wk, cuda), rope,
                                    cache.lens_dev, cache.lens_host, draft=draft)
            qh, kh = q.cpu().numpy(), k.cpu().numpy()
            for got, src, w in ((qh, x[0], wq), (kh, x[1], wk)):
                _close(got, P.norm_rope64(src, w, 1e-6, cos, sin, pos), _norm_bound(src, w, cos, sin, pos), what)
            cache.append(layer, k, _up(x[2], cuda), draft=draft)
            table = cache.table_host
            for i in range(b):
                for n in range(int(have[i])):
                    r = int(lens[i]) + n
                    for pool, src in ((k_ref, kh), (v_ref, x[2])):
                        row = src[i, :, n]
                        pool[layer, table[i, r // page], :, r % page] = P.bf16(row) if dtype == "bf16" else row
            assert np.array_equal(P.host(cache.k), k_ref) and np.array_equal(P.host(cache.v), v_ref), what
            got = cache.attend(layer, q, draft=draft).cpu().numpy()
            _check_attend(got, qh, k_ref[layer], v_ref[layer], table, page, lens, have, parents, what)
        if parents is None:
            accepted = have if kind == "prompt" else np.array([rng.integers(0, n + 1) for n in have])
            accepted = accepted.astype(np.int32)
            cache.commit(_up(accepted, cuda), accepted)
        else:
            # the path to some node of each tree
            paths, accepted = np.zeros((b, t), np.int32), np.zeros(b, np.int32)
            for i in range(b):
                node, path = int(rng.integers(0, t)), []
                while node >= 0:
                    path.insert(0, node)
                    node = int(parents[i, node])
                accepted[i] = len(path)
                paths[i, :len(path)] = path
            cache.commit(_up(accepted, cuda), accepted, _up(paths, cuda), paths)
            for layer in range(layers):
                for i in range(b):
                    for n in range(accepted[i]):
                        src, dst = int(lens[i]) + int(paths[i, n]), int(lens[i]) + n
                        for pool in (k_ref, v_ref):
                            pool[layer, cache.table_host[i, dst // page], :, dst % page] = \
                                pool[layer, cache.table_host[i, src // page], :, src % page]
            assert np.array_equal(P.host(cache.k), k_ref) and np.array_equal(P.host(cache.v), v_ref)
        lens += accepted
        assert np.array_equal(cache.lens_host, lens)
        assert np.array_equal(cache.lens_dev.cpu().numpy(), lens)


@pytest.mark.parametrize("d,t", [(128, 701), (64, 1999)])
def test_norm_rope_of_long_inputs(nne, cuda, d, t):
    """Outputs of more than the L2s hold."""
    rng = np.random.default_rng(70)
    b, hq, hkv = 3, 32, 1
    assert b * t * (hq + hkv) * d * 4 > 1 << 25
    x = [rng.standard_normal((b, t, h, d), dtype=np.float32) for h in (hq, hkv)]
    w = [1 + rng.standard_normal(d, dtype=np.float32) / 8 for _ in range(2)]
    rope = nne.RotaryEmbedding(d, 4096, device=cuda)
    start = np.array([0, 2000, 7], np.int32)
    got = nne.qk_norm_rope(*(_up(a, cuda).transpose(1, 2) for a in x), *(_up(a, cuda) for a in w), rope,
                           _up(start, cuda), start)
    cos, sin = rope.cos.cpu().numpy(), rope.sin.cpu().numpy()
    pos = start[:, None] + np.arange(t)
    for g, src, weight in zip(got, x, w):
        src = src.transpose(0, 2, 1, 3)
        _close(g.cpu().numpy(), P.norm_rope64(src, weight, 1e-6, cos, sin, pos),
               _norm_bound(src, weight, cos, sin, pos), "long")


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("kind", ["token", "chain", "tree"])
def test_layer_step(nne, cuda, norm, kind):
    """forward_gqa_paged is its parts, called one after the other, to the bit."""
    import torch
    rng = np.random.default_rng(62)
    b, hq, hkv, d = 2, 4, 2, 32
    t = 1 if kind == "token" else 7
    layer = nne.GroupedQueryAttention(hq * d, hq, hkv, 64, device=cuda)
    if norm:
        w = [_up(1 + rng.standard_normal(d, dtype=np.float32) / 8, cuda) for _ in range(2)]
        layer.set_qk_norm(*w, eps=1e-5)
    draft = nne.DraftTree(P.random_parents(rng, b, t), device=cuda) if kind == "tree" else \
        nne.DraftTree.chain(b, t, [t, 3], device=cuda) if kind == "chain" else None
    caches = []
    for _ in range(2):
        c = nne.PagedKVCache(2, 8, hkv, 16, d, b, 4, device=cuda)
        c.allocate([20, 12])
        c.set_lengths([11, 4])
        c.k.copy_(_up(np.random.default_rng(5).standard_normal(tuple(c.k.shape), dtype=np.float32), cuda))
        c.v.copy_(_up(np.random.default_rng(6).standard_normal(tuple(c.v.shape), dtype=np.float32), cuda))
        caches.append(c)
    x = _up(rng.standard_normal((b, t, hq * d), dtype=np.float32), cuda)
    got = layer.forward_gqa_paged(x, caches[0], 1, draft=draft)
    c = caches[1]
    lin = torch.nn.functional.linear
    q, k, v = (lin(x, m).view(b, t, h, d).transpose(1, 2) for m, h in
               ((layer.wq, hq), (layer.wk, hkv), (layer.wv, hkv)))
    if norm:
        q, k = nne.qk_norm_rope(q, k, *w, layer.rope, c.lens_dev, c.lens_host, eps=1e-5, draft=draft)
        c.append(1, k, v, draft=draft)
    else:
        q, _ = nne.qk_norm_rope(q, None, None, None, layer.rope, c.lens_dev, c.lens_host, eps=None, draft=draft)
        c.append(1, k, v, rope=layer.rope, draft=draft)
    out = torch.zeros(b, t, hq, d, device=cuda)
    c.attend(1, q, draft=draft, out=out.transpose(1, 2))
    want = lin(out.view(b, t, hq * d), layer.wo)
    assert torch.equal(got, want)
    assert torch.equal(caches[0].k, c.k) and torch.equal(caches[0].v, c.v)
    assert list(caches[0].lens_host) == [11, 4]
    with pytest.raises(nne.EngineError):
        layer.forward_gqa_paged(x[0], c)


def test_replayed_steps(nne, cuda):
    """A captured step (append, attention, commit in two layers) replays at the lengths
    that the device holds, with eager steps between, and after the lengths were set anew."""
    import torch
    rng = np.random.default_rng(63)
    b, hq, hkv, d, page, t, layers = 3, 4, 2, 64, 16, 6, 2
    cap = 3200
    pages = P.Pages(rng, b, hkv, d, page, [3000, 40, 0], cap - 3000, layers=layers)
    for i in range(b):
        assert (pages.table[i] >= 0).sum() >= 200 // page
    cache = pages.cache(nne, cuda)
    spare = np.setdiff1d(np.arange(pages.n_pages), pages.table)
    assert len(spare) == 2
    parents = P.random_parents(rng, b, t)
    draft = nne.DraftTree(parents, device=cuda)
    q, k, v = (torch.zeros(layers, b, h, t, d, device=cuda) for h in (hq, hkv, hkv))
    out = torch.zeros(layers, b, hq, t, d, device=cuda)
    paths = np.array([[0, 2], [1, 3], [4, 5]], np.int32)
    counts = np.array([2, 1, 2], np.int32)
    dev = [_up(a, cuda) for a in (counts, paths)]

    def step():
        for layer in range(layers):
            cache.append(layer, k[layer], v[layer], draft=draft)
            cache.attend(layer, q[layer], draft=draft, out=out[layer])
        cache.commit(dev[0], counts, dev[1], paths)

    def fill():
        x = [rng.standard_normal(tuple(a.shape), dtype=np.float32) for a in (q, k, v)]
        for a, h in zip((q, k, v), x):
            a.copy_(_up(h, cuda))
        out.fill_(7.0)
        torch.cuda.synchronize()
        return x

    def check(x, lens, what):
        """The state after a step over ``lens``, and its results."""
        for layer in range(layers):
            for i in range(b):
                for n in range(t):
                    pages.put(pages.k, i, lens[i] + n, x[1][layer, i, :, n], layer=layer)
                    pages.put(pages.v, i, lens[i] + n, x[2][layer, i, :, n], layer=layer)
            _check_attend(out[layer].cpu().numpy(), x[0][layer], pages.k[layer], pages.v[layer], pages.table, page,
                          lens, [t] * b, parents, what)
            for i in range(b):
                for n in range(counts[i]):
                    for pool in (pages.k, pages.v):
                        r = lens[i] + int(paths[i, n])
                        pages.put(pool, i, lens[i] + n, pool[layer, pages.table[i, r // page], :, r % page].copy(),
                                  layer=layer)
        assert np.array_equal(P.host(cache.k), pages.k) and np.array_equal(P.host(cache.v), pages.v), what
        assert np.array_equal(cache.lens_dev.cpu().numpy(), lens + counts), what

    lens = pages.lens.astype(np.int64)
    x = fill()
    step()                                             # eager, and the warm-up
    check(x, lens, "eager")
    lens = lens + counts
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    assert np.array_equal(cache.lens_dev.cpu().numpy(), lens)          # capturing ran nothing
    for turn in range(7):
        x = fill()
        graph.replay()
        torch.cuda.synchronize()
        check(x, lens, "replay %d" % turn)
        lens = lens + counts
        cache.set_lengths(lens)                        # (the host's copy: replays leave it)
        if turn in (1, 4):                             # an eager step on the same workspace
            x = fill()
            step()
            torch.cuda.synchronize()
            check(x, lens, "eager after replay %d" % turn)
            lens = lens + counts
        if turn == 2:                                  # shorter than any part of the captured split
            lens = np.array([5, 0, 1], np.int64)
            cache.set_lengths(lens)
        if turn == 5:
            lens = np.array([2900, 130, 77], np.int64)
            cache.set_lengths(lens)


def test_graphs_on_one_workspace(nne, cuda):
    """Two captured steps of one cache, replayed in turn: they share its workspace."""
    import torch
    rng = np.random.default_rng(64)
    pages = P.Pages(rng, 2, 2, 128, 16, [2500, 1200], 40, dtype="bf16")
    cache = pages.cache(nne, cuda)
    work = []
    for t in (1, 33):
        q = rng.standard_normal((2, 8, t, 128), dtype=np.float32)
        parents = P.random_parents(rng, 2, t)
        work.append((q, _up(q, cuda), parents, nne.DraftTree(parents, device=cuda),
                     torch.zeros(2, 8, t, 128, device=cuda), torch.cuda.CUDAGraph()))
        cache.reserve_workspace(8, t)
    for q, qd, parents, draft, out, graph in work:
        cache.attend(0, qd, draft=draft, out=out)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            cache.attend(0, qd, draft=draft, out=out)
    for turn in range(4):
        for _, _, _, _, out, graph in work:
            out.fill_(7.0)
            graph.replay()
        torch.cuda.synchronize()
        for q, _, parents, _, out, _ in work:
            _check_attend(out.cpu().numpy(), q, pages.k[0], pages.v[0], pages.table, 16, pages.lens,
                          [q.shape[2]] * 2, parents, "turn %d" % turn)


def test_workspace_does_not_grow_under_capture(nne, cuda):
    import torch
    cache = nne.PagedKVCache(1, 4, 2, 1024, 64, 2, 2, device=cuda)
    cache.allocate(2048)
    cache.set_lengths(1900 * np.ones(2, np.int32))
    q, mark = torch.zeros(2, 4, 1, 64, device=cuda), torch.zeros(4, device=cuda)
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mark.add_(1)
        with pytest.raises(nne.InvalidArgument, match="under capture"):
            cache.attend(0, q, out=out)
    cache.reserve_workspace(4, 1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mark.add_(1)
        cache.attend(0, q, out=out)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert mark.cpu().tolist() == [3.0] * 4


@pytest.mark.parametrize("t", [1, 20])
def test_another_stream(nne, cuda, t):
    import torch
    rng = np.random.default_rng(65)
    pages = P.Pages(rng, 2, 2, 64, 16, [700, 90], t)
    cache = pages.cache(nne, cuda)
    x = [_up(rng.standard_normal((2, h, t, 64), dtype=np.float32), cuda) for h in (4, 2, 2)]
    rope = nne.RotaryEmbedding(64, 1024, device=cuda)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    cache.reserve_workspace(4, t, stream=side)
    q, k = nne.qk_norm_rope(x[0], x[1], None, None, rope, cache.lens_dev, cache.lens_host, stream=side)
    cache.append(0, k, x[2], stream=side)
    out = cache.attend(0, q, stream=side)
    cache.commit(t, stream=side)
    side.synchronize()
    lens = pages.lens.copy()
    kh = k.cpu().numpy()
    for i in range(2):
        for n in range(t):
            pages.put(pages.k, i, lens[i] + n, kh[i, :, n])
            pages.put(pages.v, i, lens[i] + n, x[2][i, :, n].cpu().numpy())
    _check_attend(out.cpu().numpy(), q.cpu().numpy(), pages.k[0], pages.v[0], pages.table, 16, lens, [t] * 2,
                  None, "side stream")
    assert np.array_equal(P.host(cache.k), pages.k)
    assert np.array_equal(cache.lens_dev.cpu().numpy(), lens + t)


@pytest.mark.parametrize("own", [False, True])
def test_workspaces_of_the_c_interface(nne, cuda, own):
    """ws NULL: the stream's own, and released with it; else the caller's, whose counters
    are zero again afterwards."""
    import torch
    lib = nne.lib()
    rng = np.random.default_rng(66)
    pages = P.Pages(rng, 2, 2, 64, 16, [3000, 1100], 5)
    cache = pages.cache(nne, cuda)
    q = rng.standard_normal((2, 8, 5, 64), dtype=np.float32)
    qd, out = _up(q, cuda), torch.zeros(2, 8, 5, 64, device=cuda)
    size = nne.NneWorkspaceSize()
    nne.check(lib.nne_paged_workspace_size(cache._addr[0][0], 8, 5, ctypes.byref(size)))
    records = torch.full((size.records_bytes,), 255, dtype=torch.uint8, device=cuda)    # (NaN)
    counters = torch.zeros(size.n_counters, dtype=torch.int32, device=cuda)
    ws = nne.NneWorkspace(records=records.data_ptr(), records_bytes=size.records_bytes,
                          counters=counters.data_ptr(), n_counters=size.n_counters)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        nne.check(lib.nne_paged_attention(cache._addr[0][0], qd.data_ptr(), None, out.data_ptr(), None, 8, 5,
                                          None, None, None, None, 0, 0.0, ctypes.byref(ws) if own else None,
                                          stream.cuda_stream))
    stream.synchronize()
    _check_attend(out.cpu().numpy(), q, pages.k[0], pages.v[0], pages.table, 16, pages.lens, [5, 5], None, "C call")
    assert not counters.any()
    assert (records != 255).any().item() == own
    lib.nne_stream_release(stream.cuda_stream)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("b,hq,hkv,d,page,lens,t,tree", [
    (1, 8, 4, 256, 64, [5278], 4, False),              # few rows, many wide parts: a merge of its own
    (1, 8, 2, 128, 16, [1733], 13, True),              # 16-row tiles of 52 rows
    (2, 4, 2, 256, 32, [484, 968], 29, True),
    (8, 8, 2, 128, 64, [2048, 900, 4096, 1500, 3000, 1024, 2600, 64], 64, True),   # 32-row tiles, parts
    (3, 2, 2, 64, 1, [2500, 700, 0], 3, False),        # pages of one row
    (2, 2, 1, 64, 3, [4099, 2], 9, True),
    (1, 4, 4, 64, 16, [30000], 1, False),
    (130, 2, 1, 64, 16, [64 + 37 * (i % 9) for i in range(130)], 18, False),       # two launches
    (1, 1, 1, 8, 8, [0], 1, False),
    (2, 40, 1, 16, 16, [100, 0], 1, False),            # 40 rows of one token
])
def test_splits(nne, cuda, dtype, b, hq, hkv, d, page, lens, t, tree):
    """Shapes that take each tile, split and merge, with tokens that do not exist."""
    import torch
    rng = np.random.default_rng(67)
    pages = P.Pages(rng, b, hkv, d, page, lens, t, dtype=dtype)
    cache = pages.cache(nne, cuda)
    q = rng.standard_normal((b, hq, t, d), dtype=np.float32)
    parents = P.random_parents(rng, b, t) if tree else None
    for counts in (np.full(b, t, np.int32), rng.integers(0, t + 1, b).astype(np.int32)):
        draft = nne.DraftTree(parents, counts, device=cuda) if tree else \
            nne.DraftTree.chain(b, t, counts, device=cuda)
        out = torch.full((b, hq, t, d), 7.0, device=cuda)
        for _ in range(2):
            cache.attend(0, _up(q, cuda), draft=draft, out=out)
        got = out.cpu().numpy()
        _check_attend(got, q, pages.k[0], pages.v[0], pages.table, page, lens, counts, parents, "counts")
        for i in range(b):
            assert (got[i, :, counts[i]:] == 7).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_siblings_that_are_not_finite(nne, cuda, dtype, bad):
    """Tokens of other branches hold infinities or NaN, over several row blocks and parts:
    who does not see them gets what it gets without them; who does, shows them."""
    rng = np.random.default_rng(68)
    b, hq, hkv, d, page, t = 2, 8, 2, 64, 16, 40
    lens = [1500, 9]
    pages = P.Pages(rng, b, hkv, d, page, lens, t, dtype=dtype)
    parents = P.random_parents(rng, b, t)
    counts = np.array([t, 31], np.int32)
    sick = [7, 20]                                     # one early, one late token of each sequence
    for i in range(b):
        for n in sick:
            r = lens[i] + n
            pages.k[0, pages.table[i, r // page], :, r % page] = bad
            pages.v[0, pages.table[i, r // page], :, r % page] = bad
        for n in range(counts[i], t):                  # and rows of tokens that do not exist
            r = lens[i] + n
            pages.v[0, pages.table[i, r // page], :, r % page] = bad
            pages.k[0, pages.table[i, r // page], :, r % page] = bad
    cache = pages.cache(nne, cuda)
    q = rng.standard_normal((b, hq, t, d), dtype=np.float32)
    got = cache.attend(0, _up(q, cuda), draft=nne.DraftTree(parents, counts, device=cuda)).cpu().numpy()
    for i in range(b):
        n = int(counts[i])
        mask = P.visible(lens[i], n, parents[i])
        seen = mask[:, [lens[i] + s for s in sick]].any(1)
        assert seen.any() and not seen.all()
        k, v = (pages.rows(x, i, lens[i] + n).copy() for x in (pages.k, pages.v))
        for x in (k, v):
            x[~np.isfinite(x)] = 0
        want, bound = P.attention64(q[i, :, :n], k, v, mask, 1 / math.sqrt(d))
        _close(got[i][:, :n][:, ~seen], want[:, ~seen], bound[:, ~seen], "sequence %d" % i)
        # (a row that sees them has an infinite or NaN score, whose softmax has no finite value
        # but where the score is -inf; its V then counts 0 times what is not finite)
        assert not np.isfinite(got[i][:, :n][:, seen]).all()


def test_empty_calls(nne, cuda):
    import torch
    cache = nne.PagedKVCache(1, 4, 2, 8, 16, 2, 2, device=cuda)
    cache.allocate(8)
    none = torch.zeros(2, 2, 0, 16, device=cuda)
    cache.append(0, none, none)
    assert cache.attend(0, torch.zeros(2, 4, 0, 16, device=cuda)).shape == (2, 4, 0, 16)
    cache.commit(0)
    q, k = nne.qk_norm_rope(none, none, None, None, None, None, None)
    assert q.shape == k.shape == (2, 2, 0, 16)
    no_seqs = nne.PagedKVCache(1, 4, 2, 8, 16, 0, 2, device=cuda)
    x = torch.zeros(0, 2, 3, 16, device=cuda)
    no_seqs.append(0, x, x)
    assert no_seqs.attend(0, x).shape == x.shape
    no_seqs.commit(0)
    # every token of every sequence absent: nothing is written
    out = torch.full((2, 4, 3, 16), 7.0, device=cuda)
    cache.attend(0, torch.zeros(2, 4, 3, 16, device=cuda), draft=nne.DraftTree.chain(2, 3, [0, 0], device=cuda),
                 out=out)
    assert (out == 7).all()
    # a sequence of no rows sees itself alone
    rng = np.random.default_rng(69)
    q, kv = (rng.standard_normal((2, h, 1, 16), dtype=np.float32) for h in (4, 2))
    cache.append(0, _up(kv, cuda), _up(kv, cuda))
    got = cache.attend(0, _up(q, cuda)).cpu().numpy()
    _check_attend(got, q, P.host(cache.k)[0], P.host(cache.v)[0], cache.table_host, 8, [0, 0], [1, 1], None, "alone")


def test_python_calls_refuse(nne, cuda):
    import torch
    cache = nne.PagedKVCache(2, 8, 2, 8, 16, 2, 4, device=cuda)
    cache.allocate(16)
    x, q = torch.zeros(2, 2, 3, 16, device=cuda), torch.zeros(2, 4, 3, 16, device=cuda)
    bad, shape = nne.InvalidArgument, nne.ShapeMismatch
    for error, call in [
            (bad, lambda: cache.append(2, x, x)), (bad, lambda: cache.append(-1, x, x)),
            (bad, lambda: cache.append(0, x.double(), x)), (bad, lambda: cache.append(0, x, x.cpu())),
            (bad, lambda: cache.append(0, x.bfloat16(), x)),
            (shape, lambda: cache.append(0, x, x[:, :, :2])), (shape, lambda: cache.append(0, x[:1], x[:1])),
            (shape, lambda: cache.append(0, q, q)),
            (nne.EngineError, lambda: cache.append(0, x[0], x[0])),
            (shape, lambda: cache.attend(0, q[:, :3])), (shape, lambda: cache.attend(0, q[..., :8])),
            (shape, lambda: cache.attend(0, q, out=q[:, :2])), (bad, lambda: cache.attend(0, q, out=q.double())),
            (bad, lambda: cache.attend(0, q.half())), (bad, lambda: cache.attend(2, q)),
            (shape, lambda: cache.attend(0, q, draft=nne.DraftTree.chain(2, 2, device=cuda))),
            (shape, lambda: cache.append(0, x, x, draft=nne.DraftTree.chain(1, 3, device=cuda))),
            (bad, lambda: cache.attend(0, q, draft=nne.DraftTree.chain(2, 3, device="cpu"))),
            (bad, lambda: cache.append(0, x, x, rope=nne.RotaryEmbedding(16, 8, device="cpu"))),
            (bad, lambda: cache.append(0, x, x, rope=nne.RotaryEmbedding(16, 2, device=cuda))),
            (shape, lambda: cache.append(0, x, x, rope=nne.RotaryEmbedding(8, 64, device=cuda))),
            (nne.CapacityError, lambda: cache.append(0, *[torch.zeros(2, 2, 33, 16, device=cuda)] * 2)),
            (bad, lambda: cache.append(0, *[torch.zeros(2, 2, 17, 16, device=cuda)] * 2)),       # no page
            (bad, lambda: cache.commit(-1)), (bad, lambda: cache.commit(33)),
            (bad, lambda: cache.commit(torch.zeros(2, device=cuda), np.zeros(2, np.int32))),
            (bad, lambda: cache.commit(torch.zeros(2, dtype=torch.int32), np.zeros(2, np.int32))),
            (shape, lambda: nne.qk_norm_rope(q, x, torch.ones(8, device=cuda), None, None, None, None)),
            (shape, lambda: nne.qk_norm_rope(q, x[:, :, :2], None, None, None, None, None)),
            (shape, lambda: nne.qk_norm_rope(q, x, None, None, None, None, None, q_out=x)),
            (bad, lambda: nne.qk_norm_rope(q, None, None, None, None, None, None, k_out=x)),
            (bad, lambda: nne.qk_norm_rope(q, x, torch.ones(16, device=cuda), None, None, None, None, eps=None)),
            (bad, lambda: nne.qk_norm_rope(q, x.cpu(), None, None, None, None, None)),
            (bad, lambda: nne.qk_norm_rope(q, x, None, None, nne.RotaryEmbedding(16, 64, device=cuda), None, None)),
            (bad, lambda: nne.qk_norm_rope(q, x, None, None, nne.RotaryEmbedding(16, 64, device=cuda), None, [0, 0])),
            (bad, lambda: cache.commit(torch.zeros(2, dtype=torch.int32, device=cuda))),
            (AttributeError, lambda: setattr(cache, "lens_host", np.zeros(2, np.int32))),
    ]:
        with pytest.raises(error):
            call()
    with pytest.raises(bad):                           # two sequences would write page 0
        cache.set_table([[0, 1], [0, 2]])
        cache.append(0, x, x)
    assert list(cache.lens_host) == [0, 0] and not cache.k.any() and not cache.v.any()


def test_replayed_tokens(nne, cuda):
    """A captured decode step -- norm and rotation, append, attention, commit of one -- is
    the eager one: the same rows in the pools, replay after replay."""
    import torch
    rng = np.random.default_rng(71)
    b, hq, hkv, d, page = 2, 6, 2, 64, 16
    pages = P.Pages(rng, b, hkv, d, page, [510, 33], 12)
    caches = [pages.cache(nne, cuda) for _ in range(2)]
    rope = nne.RotaryEmbedding(d, 1024, device=cuda)
    w = [_up(1 + rng.standard_normal(d, dtype=np.float32) / 8, cuda) for _ in range(2)]
    x = [torch.zeros(b, 1, h, d, device=cuda).transpose(1, 2) for h in (hq, hkv, hkv)]
    norms = [torch.zeros(b, h, 1, d, device=cuda) for h in (hq, hkv)]
    out = torch.zeros(b, hq, 1, d, device=cuda)

    def step(cache, q_out, k_out, o):
        q, k = nne.qk_norm_rope(x[0], x[1], *w, rope, cache.lens_dev, cache.lens_host, q_out=q_out, k_out=k_out)
        cache.append(0, k, x[2])
        cache.attend(0, q, out=o)
        cache.commit(1)
        return q

    def fill():
        for a in x:
            a.copy_(_up(rng.standard_normal(tuple(a.shape), dtype=np.float32), cuda))
        torch.cuda.synchronize()

    lens = pages.lens.copy()
    fill()
    step(caches[0], *norms, out)
    caches[0].set_lengths(lens)                        # the warm-up's token does not count
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(caches[0], *norms, out)
    for turn in range(6):
        fill()
        out.fill_(7.0)
        graph.replay()
        q = step(caches[1], None, None, None if turn % 2 else torch.zeros_like(out))
        torch.cuda.synchronize()
        assert torch.equal(norms[0], q), turn
        k, v = P.host(caches[1].k), P.host(caches[1].v)
        rows = [np.concatenate([pages.table[i, :(n + turn + page) // page] for i, n in enumerate(lens)])]
        for pool, want in ((caches[0].k, k), (caches[0].v, v)):
            assert np.array_equal(P.host(pool)[0][rows[0]], want[0][rows[0]]), turn
        _check_attend(out.cpu().numpy(), q.cpu().numpy(), k[0], v[0], pages.table, page, lens + turn, [1] * b, None,
                      "replay %d" % turn)
        assert caches[0].lens_dev.tolist() == caches[1].lens_dev.tolist() == (lens + turn + 1).tolist()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_pages_outside_the_pool(nne, cuda, dtype):
    """Without the host's table the device's own bounds hold: a row whose page lies outside
    is not written, and attention leaves it out."""
    import torch
    lib = nne.lib()
    rng = np.random.default_rng(72)
    b, hq, hkv, d, page, t = 2, 4, 2, 64, 8, 5
    pages = P.Pages(rng, b, hkv, d, page, [40, 21], t, dtype=dtype)
    cache = pages.cache(nne, cuda)
    bad = pages.table.copy()
    bad[0, 1], bad[0, 3], bad[1, 0] = -1, pages.n_pages, 2 ** 31 - 1     # of counted rows
    bad[1, 3] = -5                                                       # rows 24, 25 of the new ones
    cache.table_dev.copy_(_up(bad, cuda))
    q, k, v = (rng.standard_normal((b, h, t, d), dtype=np.float32) for h in (hq, hkv, hkv))
    dev = [_up(a, cuda) for a in (q, k, v)]
    out = torch.full((b, hq, t, d), 7.0, device=cuda)
    addr, stream = cache._addr[0][1], torch.cuda.current_stream().cuda_stream
    nne.check(lib.nne_paged_append(addr, dev[1].data_ptr(), None, dev[2].data_ptr(), None, t, None, None, None, None,
                                   None, None, 0, 0, stream))
    nne.check(lib.nne_paged_attention(addr, dev[0].data_ptr(), None, out.data_ptr(), None, hq, t, None, None, None,
                                      None, 0, 0.0, None, stream))
    torch.cuda.synchronize()
    for i in range(b):
        for n in range(t):
            r = int(pages.lens[i]) + n
            if 0 <= bad[i, r // page] < pages.n_pages:
                pages.put(pages.k, i, r, k[i, :, n])
                pages.put(pages.v, i, r, v[i, :, n])
    assert np.array_equal(P.host(cache.k), pages.k) and np.array_equal(P.host(cache.v), pages.v)
    for i in range(b):
        n = int(pages.lens[i]) + t
        there = np.array([0 <= bad[i, r // page] < pages.n_pages for r in range(n)])
        assert there.any() and not there.all()
        want, bound = P.attention64(q[i], pages.rows(pages.k, i, n), pages.rows(pages.v, i, n),
                                    P.visible(n - t, t, None) & there, 1 / math.sqrt(d))
        _close(out.cpu().numpy()[i], want, bound, "sequence %d" % i)


def test_replay_after_the_workspace_grew(nne, cuda):
    """A captured call keeps its records where they were when the workspace grows."""
    import torch
    rng = np.random.default_rng(73)
    pages = P.Pages(rng, 2, 2, 64, 16, [2500, 900], 64)
    cache = pages.cache(nne, cuda)
    q = [rng.standard_normal((2, 4, t, 64), dtype=np.float32) for t in (1, 64)]
    dev = [_up(a, cuda) for a in q]
    out = torch.zeros_like(dev[0])
    cache.attend(0, dev[0], out=out)
    torch.cuda.synchronize()
    before = cache._ws.records.data_ptr()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attend(0, dev[0], out=out)
    for turn in range(3):
        big = cache.attend(0, dev[1])
        assert cache._ws.records.data_ptr() != before
        filler = [torch.full((1 << 20,), float("nan"), device=cuda) for _ in range(8)]   # (what was freed)
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        _check_attend(out.cpu().numpy(), q[0], pages.k[0], pages.v[0], pages.table, 16, pages.lens, [1, 1], None, "replay")
        _check_attend(big.cpu().numpy(), q[1], pages.k[0], pages.v[0], pages.table, 16, pages.lens, [64, 64], None, "eager")
        assert all(torch.isnan(f).all() for f in filler)
