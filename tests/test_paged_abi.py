"""Paged-cache checks that need no GPU: what the entry points refuse, on the host
and before any device access, with which error and with lengths left alone."""
import ctypes

import numpy as np
import pytest

FAKE = 4096                # never dereferenced: validation fails first
I32 = ctypes.POINTER(ctypes.c_int32)


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def ip(a):
    return None if a is None else a.ctypes.data_as(I32)


class Cache:
    """An nne_paged_cache_t of two sequences, 4 pages of 8 rows each."""

    def __init__(self, nne, lens=(5, 9), pages=((0, 1, 2, 3), (4, 5, 6, 7)), **other):
        self.lens = np.array(lens, np.int32)
        self.table = None if pages is None else np.array(pages, np.int32)
        f = dict(k=FAKE, v=FAKE, dtype=0, n_pages=8, Hkv=2, page_size=8, d=16, B=len(lens),
                 max_pages=4, table=FAKE, table_host=None if pages is None else self.table.ctypes.data,
                 lens_dev=FAKE, lens_host=self.lens.ctypes.data)
        f.update(other)
        self.c = nne.NnePagedCache(*[f[name] for name, _ in nne.NnePagedCache._fields_])
        self.p = ctypes.byref(self.c)


def append(nne, cache, t=3, counts=None, depths=None, rope=(None, None, 0, 0), k=FAKE, dev=FAKE):
    return nne.lib().nne_paged_append(
        cache.p, k, None, k, None, t, dev if counts is not None else None, ip(counts),
        dev if depths is not None else None, ip(depths), *rope, None)


def attend(nne, cache, hq=4, t=3, counts=None, parents=None, q=FAKE, ws=None, dev=FAKE):
    return nne.lib().nne_paged_attention(
        cache.p, q, None, q, None, hq, t, dev if counts is not None else None, ip(counts),
        dev if parents is not None else None, ip(parents), 0, 0.0, ws, None)


def commit(nne, cache, counts, paths=None, layers=2, stride=8 * 2 * 8 * 16, j=3, dev=FAKE):
    return nne.lib().nne_paged_commit(
        cache.p, layers, stride, dev, ip(counts), FAKE if paths is not None else None, ip(paths), j,
        None, None)


def refused(nne, rc, code, text):
    assert rc == code, nne.lib().nne_last_error()
    assert text in nne.lib().nne_last_error().decode()


BAD_GEOMETRY = [
    (dict(dtype=2), "dtype"),
    (dict(d=12), "multiple of 8"),
    (dict(d=264), "multiple of 8"),
    (dict(d=0), "multiple of 8"),
    (dict(n_pages=0), "geometry"),
    (dict(Hkv=0), "geometry"),
    (dict(page_size=0), "geometry"),
    (dict(max_pages=0), "geometry"),
    (dict(B=-1), "geometry"),
    (dict(n_pages=1 << 20, Hkv=1 << 10, page_size=2), "below 2^31"),
    (dict(n_pages=1 << 40), "geometry"),
    (dict(n_pages=1 << 20, Hkv=8, page_size=16, d=256), "64 GiB"),
    (dict(max_pages=1 << 28), "tokens behind"),
    (dict(lens_host=None), "lens_host"),
]


@pytest.mark.parametrize("fields,text", BAD_GEOMETRY)
def test_geometry(nne, fields, text):
    size = nne.NneWorkspaceSize()
    c = Cache(nne, **fields)
    counts = np.array([1, 1], np.int32)
    refused(nne, append(nne, c), nne.NNE_EINVAL, text)
    refused(nne, attend(nne, c), nne.NNE_EINVAL, text)
    refused(nne, commit(nne, c, counts), nne.NNE_EINVAL, text)
    refused(nne, nne.lib().nne_paged_workspace_size(c.p, 4, 3, ctypes.byref(size)), nne.NNE_EINVAL, text)


def test_null_cache(nne):
    refused(nne, nne.lib().nne_paged_append(None, FAKE, None, FAKE, None, 1, None, None, None, None, None,
                                            None, 0, 0, None), nne.NNE_EINVAL, "null paged cache")


@pytest.mark.parametrize("name", ["k", "v", "table", "lens_dev"])
def test_null_and_misaligned_device_arrays(nne, name):
    for call in (append, attend):
        refused(nne, call(nne, Cache(nne, **{name: None})), nne.NNE_EINVAL, "null tensor pointer")
    if name in "kv":
        for call in (append, attend):
            refused(nne, call(nne, Cache(nne, **{name: FAKE + 8})), nne.NNE_EINVAL, "16-byte aligned")
        refused(nne, commit(nne, Cache(nne, **{name: FAKE + 8}), np.array([1, 1], np.int32)),
                nne.NNE_EINVAL, "16-byte aligned")


def test_null_tensors(nne):
    refused(nne, append(nne, Cache(nne), k=None), nne.NNE_EINVAL, "null tensor pointer")
    refused(nne, attend(nne, Cache(nne), q=None), nne.NNE_EINVAL, "null tensor pointer")


def test_room(nne):
    c = Cache(nne, lens=(30, 0))                       # 32 rows each
    refused(nne, append(nne, c), nne.NNE_ECAPACITY, "3 new rows of sequence 0 of length 30 exceed")
    refused(nne, attend(nne, c), nne.NNE_EINVAL, "3 new rows")
    # counts that fit pass this check (and the next refuses: no tensor)
    refused(nne, append(nne, c, counts=np.array([2, 3], np.int32), k=None), nne.NNE_EINVAL, "null tensor")
    refused(nne, append(nne, Cache(nne, lens=(-1, 0))), nne.NNE_ECAPACITY, "sequence 0")
    assert list(c.lens) == [30, 0]


def test_counts(nne):
    for bad in ([4, 0], [0, -1]):
        counts = np.array(bad, np.int32)
        for call in (append, attend):
            refused(nne, call(nne, Cache(nne), counts=counts), nne.NNE_EINVAL, "outside [0, 3]")
    for call in (append, attend):
        refused(nne, call(nne, Cache(nne), counts=np.array([1, 1], np.int32), dev=None), nne.NNE_EINVAL,
                "on the device and on the host")


def test_pages(nne):
    missing = Cache(nne, pages=((0, -1, 2, 3), (4, 5, 6, 7)))
    # rows 5..7 lie in the first page, row 8 has none
    refused(nne, append(nne, missing, t=4), nne.NNE_EINVAL, "row 8 of sequence 0 has no page")
    refused(nne, attend(nne, missing, t=4), nne.NNE_EINVAL, "row 8 of sequence 0 has no page")
    refused(nne, append(nne, missing, k=None), nne.NNE_EINVAL, "null tensor")
    refused(nne, commit(nne, missing, np.array([4, 0], np.int32), j=4), nne.NNE_EINVAL, "row 8 of sequence 0")
    outside = Cache(nne, pages=((8, 1, 2, 3), (4, 5, 6, 7)))
    refused(nne, attend(nne, outside), nne.NNE_EINVAL, "has no page")
    assert list(missing.lens) == [5, 9]


def test_a_page_takes_new_rows_of_one_sequence(nne):
    two = Cache(nne, pages=((5, 1, 2, 3), (4, 5, 6, 7)))
    refused(nne, append(nne, two), nne.NNE_EINVAL, "page 5 would take new rows of two places")
    refused(nne, commit(nne, two, np.array([2, 2], np.int32), paths=np.array([[0, 1, 2]] * 2, np.int32)),
            nne.NNE_EINVAL, "page 5 would take new rows of two places")
    assert list(two.lens) == [5, 9]
    # a shared page of counted rows alone is fine: the next check refuses
    shared = Cache(nne, lens=(8, 9), pages=((4, 1, 2, 3), (4, 5, 6, 7)))
    refused(nne, append(nne, shared, k=None), nne.NNE_EINVAL, "null tensor")
    one = Cache(nne, lens=(5, 9), pages=((0, 0, 2, 3), (4, 5, 6, 7)))
    refused(nne, append(nne, one, t=4), nne.NNE_EINVAL, "page 0 would take new rows of two places")


def test_parents(nne):
    def parents(*row):
        return np.array([[-1, 0, 1], row], np.int32)

    for bad in ((-2, 0, 0), (0, 0, 0), (-1, 1, 0), (-1, 0, 2)):
        refused(nne, attend(nne, Cache(nne), parents=parents(*bad)), nne.NNE_EINVAL, "a parent comes before")
    # a token that does not exist may have any
    refused(nne, attend(nne, Cache(nne), parents=parents(-1, 0, 7), counts=np.array([3, 2], np.int32), q=None),
            nne.NNE_EINVAL, "null tensor")
    refused(nne, attend(nne, Cache(nne), parents=parents(-1, 0, 0), dev=None), nne.NNE_EINVAL,
            "on the device and on the host")
    big = Cache(nne, lens=(0, 0), page_size=128, pages=None)
    refused(nne, attend(nne, big, t=257, parents=np.full((2, 257), -1, np.int32)), nne.NNE_EINVAL,
            "at most 256 tokens")


def test_heads(nne):
    size = nne.NneWorkspaceSize()
    for hq in (0, -2, 3):
        refused(nne, attend(nne, Cache(nne), hq=hq), nne.NNE_EINVAL, "divisible")
        refused(nne, nne.lib().nne_paged_workspace_size(Cache(nne).p, hq, 3, ctypes.byref(size)),
                nne.NNE_EINVAL, "divisible")
    refused(nne, attend(nne, Cache(nne), hq=1 << 30), nne.NNE_EINVAL, "query rows")
    refused(nne, attend(nne, Cache(nne), hq=1 << 40), nne.NNE_EINVAL, "divisible")


def test_rotation(nne):
    c = Cache(nne)
    refused(nne, append(nne, c, rope=(FAKE, None, 64, 16)), nne.NNE_EINVAL, "both its tables")
    refused(nne, append(nne, c, rope=(FAKE, FAKE, 64, 32)), nne.NNE_ESHAPE, "expected shape [32], got [16]")
    refused(nne, append(nne, c, rope=(FAKE, FAKE, 0, 16)), nne.NNE_EINVAL, "max_seq_len 0")
    refused(nne, append(nne, c, rope=(FAKE, FAKE, 11, 16)), nne.NNE_EINVAL, "[9, 12) exceeds RoPE max_seq_len 11")
    depths = np.array([[0, 1, 2], [0, 1, 1]], np.int32)
    refused(nne, append(nne, c, rope=(FAKE, FAKE, 10, 16), depths=depths), nne.NNE_EINVAL, "exceeds RoPE")
    refused(nne, append(nne, c, rope=(FAKE, FAKE, 11, 16), depths=depths, k=None), nne.NNE_EINVAL, "null tensor")
    depths[0, 0] = -6
    refused(nne, append(nne, c, rope=(FAKE, FAKE, 64, 16), depths=depths), nne.NNE_EINVAL, "[-1, 8) exceeds")
    refused(nne, append(nne, c, rope=(FAKE, FAKE, 64, 16), depths=depths, dev=None), nne.NNE_EINVAL,
            "depths are needed")
    refused(nne, append(nne, c, rope=(FAKE + 4, FAKE, 64, 16)), nne.NNE_EINVAL, "16-byte aligned")


def test_commit(nne):
    c = Cache(nne)
    ok = np.array([2, 1], np.int32)
    path = np.array([[0, 2, 5], [1, 9, 9]], np.int32)
    refused(nne, commit(nne, c, None), nne.NNE_EINVAL, "counts_host")
    refused(nne, commit(nne, c, np.array([4, 0], np.int32), path), nne.NNE_EINVAL, "outside [0, 3]")
    refused(nne, commit(nne, c, np.array([0, -1], np.int32), path), nne.NNE_EINVAL, "outside [0, 3]")
    refused(nne, commit(nne, c, np.array([1, 3], np.int32), path), nne.NNE_EINVAL, "9 after 9")
    refused(nne, commit(nne, c, ok, np.array([[-1, 2, 5], [1, 2, 3]], np.int32)), nne.NNE_EINVAL, "-1 after -1")
    refused(nne, commit(nne, c, ok, np.array([[0, 27, 5], [1, 2, 3]], np.int32)), nne.NNE_EINVAL,
            "row 32 of sequence 0 is past its 4 pages")
    refused(nne, commit(nne, c, ok, path, layers=-1), nne.NNE_EINVAL, "layers")
    refused(nne, commit(nne, c, ok, path, stride=-4), nne.NNE_EINVAL, "layers")
    refused(nne, commit(nne, c, ok, path, stride=6), nne.NNE_EINVAL, "16-byte multiples")
    refused(nne, commit(nne, Cache(nne, dtype=1), ok, path, stride=12), nne.NNE_EINVAL, "16-byte multiples")
    # one count for all: counts_host[0]
    refused(nne, commit(nne, c, np.array([24], np.int32), j=24, dev=None), nne.NNE_EINVAL,
            "row 32 of sequence 1")
    assert list(c.lens) == [5, 9]


def test_workspaces(nne):
    lib = nne.lib()
    c = Cache(nne, lens=(4000, 9), page_size=4096, n_pages=2, max_pages=1, pages=((0,), (1,)))
    size = nne.NneWorkspaceSize()
    assert lib.nne_paged_workspace_size(c.p, 4, 3, ctypes.byref(size)) == nne.NNE_OK
    assert size.records_bytes > 0 and size.n_counters >= 4
    more = nne.NneWorkspaceSize()
    for t in (4, 16, 40, 1000, 4000):
        assert lib.nne_paged_workspace_size(c.p, 4, t, ctypes.byref(more)) == nne.NNE_OK
        assert more.records_bytes >= size.records_bytes and more.n_counters >= size.n_counters
        size = nne.NneWorkspaceSize(more.records_bytes, more.n_counters)
    assert size.records_bytes <= 1 << 28
    small = nne.NneWorkspace(records=FAKE, records_bytes=64, counters=FAKE, n_counters=16)
    refused(nne, attend(nne, c, ws=ctypes.byref(small)), nne.NNE_EINVAL, "record bytes")
    few = nne.NneWorkspace(records=FAKE, records_bytes=1 << 30, counters=FAKE, n_counters=1)
    refused(nne, attend(nne, c, ws=ctypes.byref(few)), nne.NNE_EINVAL, "counters")
    odd = nne.NneWorkspace(records=FAKE + 8, records_bytes=1 << 30, counters=FAKE, n_counters=16)
    refused(nne, attend(nne, c, ws=ctypes.byref(odd)), nne.NNE_EINVAL, "aligned")
    assert lib.nne_paged_workspace_size(c.p, 4, 3, None) == nne.NNE_EINVAL


def test_nothing_to_do(nne):
    """No sequences or no tokens: success without any device array."""
    none = dict(k=None, v=None, table=None, lens_dev=None)
    for c, t in ((Cache(nne, lens=(), pages=None, **none), 3), (Cache(nne, **none), 0)):
        assert append(nne, c, t=t, k=None) == nne.NNE_OK
        assert attend(nne, c, t=t, q=None) == nne.NNE_OK
        assert commit(nne, c, np.zeros(2, np.int32), j=0) == nne.NNE_OK


def norm(nne, q_shape=(2, 4, 3, 16), k_shape=(2, 2, 3, 16), weights=(FAKE, FAKE), has_norm=1, eps=1e-6,
         rope=(FAKE, FAKE, 64, 16), start=(0, 7), depths=None, q=FAKE, k=FAKE, k_out=FAKE, dev=FAKE):
    start = None if start is None else np.array(start, np.int32)
    return nne.lib().nne_qk_norm_rope(
        q, i64(*q_shape), None, q, None, k, i64(*k_shape), None, k_out, None, *weights, has_norm, eps,
        *rope, dev, ip(start), dev if depths is not None else None, ip(depths), None)


def test_norm_rope(nne):
    einval, eshape = nne.NNE_EINVAL, nne.NNE_ESHAPE
    refused(nne, norm(nne, k_shape=(2, 2, 4, 16)), eshape, "expected shape [2, 2, 3, 16], got [2, 2, 4, 16]")
    refused(nne, norm(nne, k_shape=(2, 2, 3, 8)), eshape, "got [2, 2, 3, 8]")
    refused(nne, norm(nne, q_shape=(2, -4, 3, 16)), einval, "out of range")
    refused(nne, norm(nne, q_shape=(1 << 20, 4, 1 << 20, 16), k_shape=(1 << 20, 4, 1 << 20, 16)), einval,
            "out of range")
    refused(nne, norm(nne, q_shape=(2, 4, 3, 15), k_shape=(2, 2, 3, 15)), einval, "must be even")
    refused(nne, norm(nne, eps=-1e-6), einval, "eps")
    refused(nne, norm(nne, eps=float("nan")), einval, "eps")
    refused(nne, norm(nne, has_norm=0), einval, "weights without a norm")
    refused(nne, norm(nne, rope=(None, FAKE, 64, 16)), einval, "both its tables")
    refused(nne, norm(nne, rope=(FAKE, FAKE, 64, 32)), eshape, "expected shape [32], got [16]")
    refused(nne, norm(nne, rope=(FAKE, FAKE, 9, 16)), einval, "[7, 10) exceeds RoPE max_seq_len 9")
    refused(nne, norm(nne, start=(-1, 0)), einval, "[-1, 2) exceeds")
    refused(nne, norm(nne, start=None), einval, "start positions")
    refused(nne, norm(nne, dev=None), einval, "null tensor pointer")
    refused(nne, norm(nne, q=None), einval, "null tensor pointer")
    refused(nne, norm(nne, k_out=None), einval, "null tensor pointer")
    depths = np.array([[0, 1, 2], [0, 1, 60]], np.int32)
    refused(nne, norm(nne, depths=depths), einval, "exceeds RoPE")
    assert norm(nne, q_shape=(0, 4, 3, 16), k_shape=(0, 2, 3, 16), start=()) == nne.NNE_OK
    assert norm(nne, q_shape=(2, 4, 0, 16), k_shape=(2, 2, 0, 16)) == nne.NNE_OK


def test_python_objects_refuse(nne):
    """What needs no device array: the classes' own checks, on the CPU."""
    bad = nne.InvalidArgument
    for geometry in ((1, 0, 2, 8, 16, 2, 4), (1, 4, 2, 8, 16, -1, 4), (-1, 4, 2, 8, 16, 2, 4)):
        with pytest.raises(bad):
            nne.PagedKVCache(*geometry, device="cpu")
    import torch
    with pytest.raises(bad):
        nne.PagedKVCache(1, 4, 2, 8, 16, 2, 4, dtype=torch.float16, device="cpu")
    c = nne.PagedKVCache(2, 6, 2, 8, 16, 2, 4, device="cpu")
    assert c.num_layers() == 2 and c.capacity() == 32
    for table in ([[0, 1]], [[0] * 5] * 2, [0, 1]):
        with pytest.raises(nne.ShapeMismatch):
            c.set_table(table)
    for table in ([[6], [0]], [[-2], [0]]):
        with pytest.raises(bad):
            c.set_table(table)
    for lens in ([1], [-1, 0], [33, 0], [1, 0]):
        with pytest.raises(bad):
            c.set_lengths(lens)
    with pytest.raises(nne.CapacityError):
        c.allocate(33)
    with pytest.raises(nne.CapacityError):
        c.allocate([32, 24])                           # 4 and 3 pages of 6
    assert (c.table_host == -1).all()
    c.allocate([17, 8])
    assert (c.table_host >= 0).sum(1).tolist() == [3, 1]
    before = c.table_host.copy()
    c.allocate([17, 16])                               # pages it has stay
    assert (c.table_host[before >= 0] == before[before >= 0]).all()
    assert len(set(c.table_host[c.table_host >= 0])) == 5
    c.set_lengths([17, 16])
    with pytest.raises(bad):
        c.set_table([[0, 1], [2, 3]])                  # 17 rows need three
    for seq in (-1, 2):
        with pytest.raises(bad):
            c.release(seq)
    c.release(0)
    assert c.lens_host.tolist() == [0, 16] and (c.table_host[0] == -1).all()
    assert c.lens_dev.tolist() == [0, 16] and (c.table_dev.numpy() == c.table_host).all()
    for pool in (torch.zeros(2, 6, 2, 8, 8), torch.zeros(2, 6, 2, 16, 8)):
        with pytest.raises(nne.ShapeMismatch):
            c.k = pool
    with pytest.raises(bad):
        c.v = torch.zeros(2, 6, 2, 8, 16, dtype=torch.bfloat16)
    with pytest.raises(bad):
        c.v = torch.zeros(2, 6, 2, 16, 8).transpose(3, 4)
    x = torch.zeros(2, 2, 1, 16)
    for call in (lambda: c.append(0, x, x), lambda: c.attend(0, x), lambda: c.commit(1),
                 lambda: nne.qk_norm_rope(x, x, None, None, None, None, None)):
        with pytest.raises(bad):
            call()                                     # not on a GPU
    with pytest.raises(bad):
        c.append(2, x, x)


def test_draft_trees_refuse(nne):
    for parents in ([[-1, 1]], [[-2, 0]], [[0, 0]]):
        with pytest.raises(nne.InvalidArgument):
            nne.DraftTree(parents, device="cpu")
    with pytest.raises(nne.InvalidArgument):
        nne.DraftTree([-1, 0], device="cpu")
    for counts in ([3], [-1]):
        with pytest.raises(nne.InvalidArgument):
            nne.DraftTree([[-1, 0]], counts=counts, device="cpu")
        with pytest.raises(nne.InvalidArgument):
            nne.DraftTree.chain(1, 2, counts=counts, device="cpu")
    tree = nne.DraftTree([[-1, 0, 0, 2, -1], [-1, 0, 9, 9, 9]], counts=[5, 2], device="cpu")
    assert tree.depths_host.tolist() == [[0, 1, 1, 2, 0], [0, 1, 0, 0, 0]]
    with pytest.raises(nne.ShapeMismatch):
        tree._check(2, 4, -1)


@pytest.mark.parametrize("name", ["qk_norm_rope", "paged_append", "paged_attention", "paged_commit",
                                  "qk_norm_rope_t", "paged_append_t"])
def test_malformed_native_calls_raise(nne, name):
    call = getattr(nne._native(), name)
    with pytest.raises(TypeError):
        call()
    with pytest.raises((TypeError, AttributeError)):
        call(*[object()] * 3)
    with pytest.raises(TypeError):
        call(*[None] * 40)


def test_native_calls_on_tensors(nne):
    """The calls that read tensors themselves: None for a tensor that does not fit, else
    the ABI's answer (index -1: CPU tensors, which the ABI's checks refuse or do not reach)."""
    import torch
    f32, i32 = torch.float32, torch.int32
    native = nne._native()
    cache = Cache(nne)
    addr = ctypes.addressof(cache.c)
    k, q = torch.zeros(2, 2, 30, 16), torch.zeros(2, 4, 30, 16)

    def append(k, v, addr=addr, index=-1):
        return native.paged_append_t(f32, index, addr, k, v, None, None, None, None, None, None, 0, 0, 0)

    assert append(k, k) == nne.NNE_ECAPACITY                  # 30 rows behind 5 and 9 of 32
    for bad in (k.double(), k[0], k[:1], k[:, :1], k[..., :8], k.numpy(), torch.zeros(1, 2, 2, 30, 16)):
        assert append(bad, k) is None and append(k, bad) is None
    assert append(k, k, index=0) is None and append(k, k, addr=0) is None
    cos = torch.zeros(8, 16)
    start, host = torch.zeros(2, dtype=i32), np.array([0, 7], np.int32)

    def norm(q=q, qo=q, k=k, ko=k, qw=None, kw=None, cos=cos, start=start, host=host, d=16):
        return native.qk_norm_rope_t(f32, -1, i32, q, qo, k, ko, qw, kw, True, 1e-6, cos, cos, 8, d, start, host,
                                     None, None, 0)

    assert norm() == nne.NNE_EINVAL                           # rows 7..36 of 8
    assert b"exceeds RoPE max_seq_len" in nne.lib().nne_last_error()
    assert norm(d=8) == nne.NNE_ESHAPE
    assert norm(k=None, ko=None) == nne.NNE_EINVAL
    w = torch.ones(16)
    assert norm(qw=w, kw=w) == nne.NNE_EINVAL
    for bad in (dict(q=q.double()), dict(q=q[0]), dict(qo=q[:1]), dict(k=None), dict(ko=None), dict(ko=q),
                dict(qw=torch.ones(8)), dict(kw=torch.ones(32)[::2]), dict(qw=w.double()), dict(kw=w[None]),
                dict(cos=cos.double()), dict(start=start.long()), dict(start=start[:1]), dict(start=None),
                dict(start=torch.zeros(4, dtype=i32)[::2]), dict(host=None), dict(host=host[:1]),
                dict(host=host.astype(np.int64)), dict(host=[0, 7]), dict(host=np.zeros(4, np.int32)[::2])):
        assert norm(**bad) is None, bad
