"""Plain 64-bit implementations of the paged-cache operators, and the bounds
that float32 results are held to."""
import numpy as np

EPS = 2.0 ** -24           # half a step of float32


def bf16(x):
    """x rounded to bfloat16 (to nearest, ties to even), as float32."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    u = (u + 0x7fff + ((u >> 16) & 1)) & 0xffff0000
    return u.astype(np.uint32).view(np.float32).reshape(np.shape(x))


def depths_of(parents):
    d = np.zeros_like(parents)
    for b in range(parents.shape[0]):
        for t in range(parents.shape[1]):
            if parents[b, t] >= 0:
                d[b, t] = d[b, parents[b, t]] + 1
    return d


def random_parents(rng, b, t):
    p = np.floor(rng.random((b, t)) * np.arange(1, t + 1)).astype(np.int32) - 1
    p[:, :1] = -1
    return p


def visible(n_ctx, t, parents):
    """[t, n_ctx + t] truth values of one sequence; parents [t] or None: a chain."""
    m = np.zeros((t, n_ctx + t), bool)
    m[:, :n_ctx] = True
    for i in range(t):
        at = i
        while at >= 0:
            m[i, n_ctx + at] = True
            at = int(parents[at]) if parents is not None else at - 1
    return m


def attention64(q, k, v, mask, scale):
    """q [Hq, T, d], k and v [Hkv, n, d], mask [T, n] -> (out, bound on a float32
    kernel's error), both [Hq, T, d].

    The bound: a score is a sum of d products of float32 values, each product and
    sum off by at most EPS of the sum of magnitudes A = scale * sum |q k|, so by
    (d + 4) EPS A (the scale and log2(e) folded into q and the subtraction of the
    maximum among the 4); a weight is then off by that and 4 EPS of exp2, relative
    to itself; numerator and denominator add up to n such weights in some order,
    n EPS more each, and rescale or merge at most 64 times.  Their quotient is
    off by twice that, relative to sum p |v|."""
    hq, hkv = q.shape[0], k.shape[0]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for h in range(hq):
        q1, k1, v1 = (x.astype(np.float64) for x in (q[h], k[h // (hq // hkv)], v[h // (hq // hkv)]))
        s = np.where(mask, q1 @ k1.T * scale, -np.inf)
        a = np.where(mask, np.abs(q1) @ np.abs(k1).T * abs(scale), 0.0).max(1)
        m = s.max(1, keepdims=True)
        p = np.exp(s - np.where(np.isfinite(m), m, 0))
        p = p / np.maximum(p.sum(1, keepdims=True), 1e-300)
        vz = np.where(mask.any(0)[:, None], v1, 0)
        out[h] = p @ vz
        rel = (q.shape[2] + 4) * EPS * a + (k.shape[1] + 68) * EPS
        bound[h] = 2 * rel[:, None] * (p @ np.abs(vz)) + 1e-38
    return out, bound


def norm_rope64(x, w, eps, cos, sin, pos):
    """x [B, H, T, d], pos [B, T]; w None: ones; eps None: no norm; cos None: no rotation."""
    x = x.astype(np.float64)
    if eps is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        if w is not None:
            x = x * w.astype(np.float64)
    if cos is None:
        return x
    half = x.shape[-1] // 2
    c, s = cos.astype(np.float64)[pos][:, None], sin.astype(np.float64)[pos][:, None]
    return x * c + np.concatenate([-x[..., half:], x[..., :half]], -1) * s


class Pages:
    """A host model of the pools: [n_pages][Hkv][page][d] float32 arrays."""

    def __init__(self, rng, b, hkv, d, page, lens, room, layers=1, dtype="f32", spare=2):
        need = -(-(np.asarray(lens, np.int64) + room) // page)
        self.n_pages = int(need.sum()) + spare
        self.max_pages = max(1, int(need.max()) if b else 1)
        ids = rng.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((b, self.max_pages), -1, np.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = ids[at:at + n]
            at += n
        self.page, self.lens = page, np.asarray(lens, np.int32)
        shape = (layers, self.n_pages, hkv, page, d)
        self.k = rng.standard_normal(shape, dtype=np.float32)
        self.v = rng.standard_normal(shape, dtype=np.float32)
        self.dtype = dtype
        if dtype == "bf16":
            self.k, self.v = bf16(self.k), bf16(self.v)

    def rows(self, pool, b, n, layer=0):
        """The first n rows of sequence b, [Hkv, n, d]."""
        r = np.arange(n)
        return pool[layer][self.table[b, r // self.page], :, r % self.page].transpose(1, 0, 2)

    def put(self, pool, b, row, values, layer=0):
        """values [Hkv, d] into row ``row`` of sequence b."""
        pool[layer, self.table[b, row // self.page], :, row % self.page] = \
            bf16(values) if self.dtype == "bf16" else values

    def cache(self, nne, cuda):
        import torch
        layers, n_pages, hkv, page, d = self.k.shape
        c = nne.PagedKVCache(layers, n_pages, hkv, page, d, len(self.lens), self.max_pages,
                             dtype=torch.bfloat16 if self.dtype == "bf16" else torch.float32,
                             device=cuda)
        c.k.copy_(torch.from_numpy(self.k))
        c.v.copy_(torch.from_numpy(self.v))
        c.set_table(self.table)
        c.set_lengths(self.lens)
        return c


def host(pool):
    return pool.float().cpu().numpy()
