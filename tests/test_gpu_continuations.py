"""GPU parity of the operators for several continuations of a prompt.

Attention, against a 64-bit evaluation of the formula on the same fp16 cache
rows. What the kernel may be off by, from its arithmetic:
  - q and the weights are carried as fp16 part + fp16 remainder: each part is
    off by half a step (2^-11 relative), so a value by 2^-22;
  - a score is a sum of hd products over hd/16 steps of two instructions, each
    of which may lose 2^-23 of the largest partial sum, A = sum |q_d k_d| /
    sqrt(hd) at most: |ds| <= (2^-22 + (hd / 8) 2^-23 + 2^-22) A, the last
    term for the scaling and the subtraction of the maximum;
  - e^s is off by 2 |ds| in the weights' ratio to their sum, plus 2^-21 for
    exp2f and the split;
  - the weighted sum over n keys takes n/16 steps of two instructions and a
    rescaling, 2^-23 each of sum p |v| <= max |v|.
so |do| <= (2 |ds| + 2^-21 + (n / 8 + 4) 2^-23) max |v|, worst case. The
2-norm over a whole output, in which roundings of either sign average out, is
held to 2^-16 (a 64th of one fp16 step of every element) as well.
"""
import ctypes as C

import numpy as np
import pytest

from prosperoai_b200 import _native
from prosperoai_b200.api import KvView

pytestmark = pytest.mark.gpu

SENTINEL = np.float32(-12345.5)


def i32(v):
    return np.ascontiguousarray(v, np.int32)


class Cache:
    """A cache of random fp16 rows on the device, with the host's copy."""

    def __init__(self, dev, rng, lens, page, hk, hd, layers=1, spare=0, pad=0, table=None, n_pages=None, max_pages=None,
                 cap=None):
        self.dev, self.hk, self.hd, self.layers = dev, hk, hd, layers
        n_seq = len(lens)
        if page:
            need = [-(-max(int(n), 0) // page) for n in lens]
            self.max_pages = max_pages or max(max(need), 1)
            self.n_pages = n_pages or max(sum(need) + spare, 1)
            if table is None:
                table = np.full((n_seq, self.max_pages), -1, np.int32)
                perm, at = rng.permutation(self.n_pages), 0
                for s, k in enumerate(need):
                    table[s, :k] = perm[at:at + k]
                    at += k
            self.table = i32(table)
            self.page = page
        else:
            self.page, self.max_pages, self.n_pages, self.table = cap or max(max(lens), 1), 1, n_seq, None
        # head rows are padded by `pad` elements, so that strides differ from the sizes
        self.head = self.page * hd + pad
        shape = (layers, self.n_pages, hk, self.head)
        self.k = rng.standard_normal(shape).astype(np.float16)
        self.v = rng.standard_normal(shape).astype(np.float16)
        self.dk, self.dv = dev.put(self.k), dev.put(self.v)
        self.dt = dev.put(self.table) if self.table is not None else None
        self.view = KvView(self.dk.ptr, self.dv.ptr, self.dt.ptr if self.dt else None, layers, n_seq, hk, hd, self.page,
                           self.n_pages, self.max_pages, self.n_pages * hk * self.head, hk * self.head, self.head)

    def put(self):
        self.dk.upload(self.k)
        self.dv.upload(self.v)

    def where(self, s, pos):
        """(page, first element of the row) of a position, or None."""
        j = pos // self.page
        if j >= self.max_pages:
            return None
        page = s if self.table is None else int(self.table[s, j])
        return (page, pos % self.page * self.hd) if 0 <= page < self.n_pages else None

    def rows(self, plane, layer, s, n):
        """[kv head][n][hd] in 64 bits and which of the n positions exist."""
        out = np.zeros((self.hk, n, self.hd))
        there = np.zeros(n, bool)
        for p in range(n):
            at = self.where(s, p)
            if at:
                out[:, p] = plane[layer, at[0], :, at[1]:at[1] + self.hd].astype(np.float64)
                there[p] = True
        return out, there

    def download(self):
        self.k = self.dk.download(np.float16).reshape(self.k.shape)
        self.v = self.dv.download(np.float16).reshape(self.v.shape)
        return self.k, self.v


def random_tree(rng, n):
    """sees[i][j] of n nodes, parents among the 6 before."""
    sees = np.zeros((n, n), bool)
    for i in range(n):
        if i:
            sees[i] = sees[rng.integers(max(0, i - 6), i)]
        sees[i, i] = True
    return sees


def pack(sees_of, most):
    words = -(-most // 64)
    out = []
    for sees in sees_of:
        for row in sees:
            v = sum(1 << int(j) for j in np.flatnonzero(row))
            out.append([v >> 64 * w & (1 << 64) - 1 for w in range(words)])
    return np.array(out, np.uint64).reshape(-1, words)


def attend(cache, layer, lens, sees_of, q, h):
    """The formula in 64 bits, and each element's bound."""
    out, bound, row = np.zeros(q.shape), np.zeros(q.shape), 0
    g, hd = h // cache.hk, cache.hd
    for s, sees in enumerate(sees_of):
        n = int(lens[s]) + len(sees)
        with np.errstate(invalid="ignore"):
            k, there = cache.rows(cache.k, layer, s, n)
            v, _ = cache.rows(cache.v, layer, s, n)
        for i in range(len(sees)):
            ok = there.copy()
            ok[int(lens[s]):] &= sees[i]
            if ok.any():
                for hh in range(h):
                    kk, vv = k[hh // g][ok], v[hh // g][ok]
                    qq = q[row, hh].astype(np.float64)
                    with np.errstate(invalid="ignore", over="ignore"):
                        sc = kk @ qq / np.sqrt(hd)
                        p = np.exp(sc - sc.max())
                        out[row, hh] = p @ vv / p.sum()
                        a = (np.abs(kk) @ np.abs(qq)).max() / np.sqrt(hd)
                        ds = (2.0 ** -21 + hd / 8 * 2.0 ** -23) * a
                        bound[row, hh] = (2 * ds + 2.0 ** -21 + (ok.sum() / 8 + 4) * 2.0 ** -23) * np.abs(vv).max()
            row += 1
    return out, bound


def run_tree(dev, cache, layer, lens, counts, h, mask, q, graph=False):
    off = np.concatenate([[0], np.cumsum(counts)])
    rows, most = int(off[-1]), max(max(counts), 1)
    out = dev.put(np.full(q.size, SENTINEL, np.float32))
    keep = [dev.put(i32(lens)), dev.put(i32(off)), dev.put(mask) if mask is not None else None, dev.put(q)]
    dev.attn_tree(cache.view, layer, h, max(rows, 1), most, keep[0], keep[1], keep[2], keep[3], out)
    return out.download(np.float32).reshape(q.shape)


def close(got, want, bound):
    assert np.all(np.isfinite(got))
    assert np.all(np.abs(got - want) <= bound), np.max(np.abs(got - want) / np.maximum(bound, 1e-30))
    norm = np.linalg.norm(want)
    assert np.linalg.norm(got - want) <= 2.0 ** -16 * norm


SHAPES = [
    # lens, nodes, page, h, hk, hd
    ([0], [1], 16, 2, 1, 128), ([1], [1], 0, 2, 1, 64), ([63], [1], 16, 4, 4, 128), ([64], [1], 128, 8, 1, 64),
    ([65], [2], 16, 32, 8, 128), ([511, 0, 130], [1, 1, 1], 128, 32, 8, 128), ([200, 7], [16, 3], 48, 14, 2, 64),
    ([300], [33], 100, 6, 2, 128), ([70, 0, 1000, 5], [5, 0, 17, 9], 64, 16, 2, 128), ([129, 40], [65, 20], 16, 8, 8, 64),
    ([90], [130], 32, 4, 1, 128), ([37, 500], [1, 64], 0, 32, 8, 128), ([5000], [8], 128, 8, 2, 128),
    ([3000, 2, 777, 64, 0, 1500, 31, 900], [4, 1, 7, 16, 2, 1, 12, 3], 128, 10, 2, 128), ([17], [31], 1, 2, 1, 64),
    ([40], [20], 16, 64, 1, 128), ([333, 20], [40, 9], 24, 4, 2, 128), ([250], [5], 8, 8, 2, 64), ([1000], [6], 0, 6, 2, 128),
    ([260, 131], [70, 3], 20, 8, 2, 128), ([127, 128, 129, 255], [1, 1, 1, 1], 256, 8, 8, 128),
]


@pytest.mark.parametrize("lens,nodes,page,h,hk,hd", SHAPES)
@pytest.mark.parametrize("kind", ["tree", "chain"])
def test_attention(dev, lens, nodes, page, h, hk, hd, kind):
    rng = np.random.default_rng(sum(lens) * 31 + sum(nodes) + hd)
    total = [a + b for a, b in zip(lens, nodes)]
    cache = Cache(dev, rng, total, page, hk, hd, layers=2, spare=2, pad=8, cap=max(total) + 3)
    sees = [random_tree(rng, n) if kind == "tree" else np.tril(np.ones((n, n), bool)) for n in nodes]
    q = rng.standard_normal((sum(nodes), h, hd)).astype(np.float32)
    mask = pack(sees, max(nodes)) if kind == "tree" else None
    got = run_tree(dev, cache, 1, lens, nodes, h, mask, q)
    close(got, *attend(cache, 1, lens, sees, q, h))
    again = run_tree(dev, cache, 1, lens, nodes, h, mask, q)
    assert np.array_equal(got.view(np.uint32), again.view(np.uint32))


@pytest.mark.parametrize("scale", [1e-30, 1e-3, 30.0, 1e5])
def test_attention_of_small_and_large_queries(dev, scale):
    """Scores from all equal to one that takes all the weight; queries beyond fp16's range. (A score's
    bound grows with its size: past 1 the output may be any mean of the V rows, and only that is held.)"""
    rng = np.random.default_rng(4)
    cache = Cache(dev, rng, [700], 64, 2, 128)
    sees = [random_tree(rng, 12)]
    q = (rng.standard_normal((12, 8, 128)) * scale).astype(np.float32)
    got = run_tree(dev, cache, 0, [688], [12], 8, pack(sees, 12), q)
    want, bound = attend(cache, 0, [688], sees, q, 8)
    assert np.all(np.isfinite(got))
    assert np.all(np.abs(got - want) <= np.minimum(bound, 2 * np.abs(cache.v).max()))
    if scale == 1e5:  # the gap between the best score and the next is far above its error in nearly all rows
        assert np.mean(np.abs(got - want) <= 2.0 ** -20) > 0.9


def test_rows_that_see_nothing_and_masks_of_holes(dev):
    rng = np.random.default_rng(8)
    table = [[0, -1, 2, 9], [-1, -1, 5, 6], [3, 4, 77, -5]]
    cache = Cache(dev, rng, [64] * 3, 16, 2, 64, table=table, n_pages=8, max_pages=4)
    lens, nodes = [50, 0, 40], [6, 5, 3]  # the second's nodes lie in holes, the others' partly
    sees = [random_tree(rng, n) for n in nodes]
    sees[0][2] = False
    sees[2][:] = False
    q = rng.standard_normal((14, 4, 64)).astype(np.float32)
    got = run_tree(dev, cache, 0, lens, nodes, 4, pack(sees, 6), q)
    want, bound = attend(cache, 0, lens, sees, q, 4)
    close(got, want, bound)
    assert not got[6:11].any()
    empty = [np.zeros((4, 4), bool)]
    one = Cache(dev, rng, [16], 16, 2, 64)
    assert not run_tree(dev, one, 0, [0], [4], 4, pack(empty, 4), q[:4]).any()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("page", [0, 16])
def test_nonfinite_rows_reach_only_those_that_see_them(dev, bad, page):
    rng = np.random.default_rng(9)
    lens, n, h, hd = [70], 20, 4, 64
    cache = Cache(dev, rng, [128], page, 2, hd, cap=128)
    sees = [random_tree(rng, n)]
    sees[0][:, 7] = False
    sees[0][3, 7] = True
    q = rng.standard_normal((n, h, hd)).astype(np.float32)
    clean, bound = attend(cache, 0, lens, sees, q, h)
    for pos in [77] + list(range(90, 128)):  # node 7, and the stale rows behind the last node
        p, e = cache.where(0, pos)
        cache.k[0, p, :, e:e + hd] = bad
        cache.v[0, p, :, e:e + hd] = bad
    cache.put()
    got = run_tree(dev, cache, 0, lens, [n], h, pack(sees, n), q)
    others = np.arange(n) != 3
    close(got[others], clean[others], bound[others])
    assert not np.isfinite(got[3]).any()
    # a V row alone, one element of it: only that element of the row that sees it
    p, e = cache.where(0, 77)
    cache.k[0, p, :, e:e + hd] = 0
    cache.v[0, p, :, e:e + hd] = 0
    cache.v[0, p, :, e + 5] = bad
    cache.put()
    got = run_tree(dev, cache, 0, lens, [n], h, pack(sees, n), q)
    assert np.array_equal(np.isfinite(got[3]), np.tile(np.arange(hd) != 5, (h, 1)))
    close(got[others], clean[others], bound[others])


def test_rows_outside_the_sequences_stay(dev):
    rng = np.random.default_rng(10)
    cache = Cache(dev, rng, [40, 40], 16, 1, 64)
    q = rng.standard_normal((12, 2, 64)).astype(np.float32)
    out = dev.put(np.full(q.size, SENTINEL, np.float32))
    off = dev.put(i32([2, 5, 10]))  # rows 0, 1, 10, 11 belong to no sequence; max_nodes 4 leaves out node 4 of the second
    dev.attn_tree(cache.view, 0, 2, 12, 4, dev.put(i32([20, 30])), off, None, dev.put(q), out)
    got = out.download(np.float32).reshape(q.shape)
    assert np.all(got[[0, 1, 9, 10, 11]] == SENTINEL) and not np.any(got[2:9] == SENTINEL)
    # offsets that point outside the rows
    for off in ([-3, 4, 4], [9, 20, 30], [12, 14, 2], [5, 5, 2]):
        out.upload(np.full(q.size, SENTINEL, np.float32))
        dev.attn_tree(cache.view, 0, 2, 12, 4, dev.put(i32([20, 30])), dev.put(i32(off)), None, dev.put(q), out)
        got = out.download(np.float32).reshape(q.shape)
        touched = set()
        for s in range(2):
            if 0 <= off[s] < off[s + 1] and off[s] < 12:
                touched |= set(range(off[s], min(off[s + 1], 12, off[s] + 4)))
        assert {i for i in range(12) if not np.any(got[i] == SENTINEL)} == touched


def test_attention_replayed_with_other_lengths(dev):
    """A captured call follows the lengths and masks that lie on the device when it is replayed."""
    rng = np.random.default_rng(11)
    L = _native.load()
    cache = Cache(dev, rng, [600, 600], 64, 2, 128)
    q = rng.standard_normal((10, 4, 128)).astype(np.float32)
    lens, off = dev.put(i32([3, 4])), dev.put(i32([0, 5, 10]))
    sees = [random_tree(rng, 5), random_tree(rng, 5)]
    mask, dq, out = dev.put(pack(sees, 5)), dev.put(q), dev.alloc(q.nbytes)
    dev.attn_tree(cache.view, 0, 4, 10, 5, lens, off, mask, dq, out)
    g = C.c_void_p()
    _native.check(L.pai_b200_graph_begin(dev.ctx), "begin")
    dev.attn_tree(cache.view, 0, 4, 10, 5, lens, off, mask, dq, out)
    _native.check(L.pai_b200_graph_end(dev.ctx, C.byref(g)), "end")
    try:
        for now in ([3, 4], [595, 0], [64, 320]):
            lens.upload(i32(now))
            sees = [random_tree(rng, 5), random_tree(rng, 5)]
            mask.upload(pack(sees, 5))
            _native.check(L.pai_b200_graph_launch(dev.ctx, g), "launch")
            close(out.download(np.float32).reshape(q.shape), *attend(cache, 0, now, sees, q, 4))
    finally:
        dev.sync()
        L.pai_b200_graph_destroy(g)


def test_rows_past_32_bit_offsets(dev):
    """A page whose first element lies past 2^32."""
    rng = np.random.default_rng(12)
    small = Cache(dev, rng, [80], 16, 1, 64)
    stride = 1 << 30  # elements between pages: page 5 starts at 5 * 2^30
    n = 5 * stride + 16 * 64
    bk, bv = dev.alloc(n * 2), dev.alloc(n * 2)
    L = _native.load()
    for buf, plane in ((bk, small.k), (bv, small.v)):
        for page in range(small.n_pages):
            a = np.ascontiguousarray(plane[0, page])
            _native.check(L.pai_b200_memcpy_h2d(dev.ctx, buf.ptr + (page + 1) * stride * 2, a.ctypes.data, a.nbytes), "h2d")
    dev.sync()
    table = dev.put(small.table + 1)
    v = small.view
    view = KvView(bk.ptr, bv.ptr, table.ptr, 1, 1, 1, 64, 16, 6, v.max_pages, 0, stride, 16 * 64)
    q = rng.standard_normal((3, 2, 64)).astype(np.float32)
    out = dev.alloc(q.nbytes)
    dev.attn_tree(view, 0, 2, 3, 3, dev.put(i32([77])), dev.put(i32([0, 3])), None, dev.put(q), out)
    want = attend(small, 0, [77], [np.tril(np.ones((3, 3), bool))], q, 2)
    close(out.download(np.float32).reshape(q.shape), *want)


# ---- rotary append ------------------------------------------------------------------------------------


@pytest.mark.parametrize("hd,page,depths", [(128, 16, True), (64, 0, False), (96, 7, True), (8, 64, True), (256, 100, False)])
def test_rope_append(dev, hd, page, depths):
    rng = np.random.default_rng(hd + page)
    lens, nodes, h, hk, layers = [5, 0, 33], [4, 1, 9], 6, 2, 2
    cache = Cache(dev, rng, [a + b for a, b in zip(lens, nodes)], page, hk, hd, layers=layers, spare=1, pad=8, cap=60)
    if page:
        cache.table[2, 35 // page:36 // page + 1] = -1  # a hole: nodes there are not stored
        cache.dt.upload(cache.table)
    rows = sum(nodes)
    qkv = rng.standard_normal((rows, h + 2 * hk, hd)).astype(np.float32)
    depth = i32(rng.integers(-1, 12, rows)) if depths else None
    table_len = 40
    ang = rng.standard_normal((table_len, hd // 2)).astype(np.float32)
    cos, sin = np.cos(ang), np.sin(ang)
    q = dev.put(np.full((rows + 1) * h * hd, SENTINEL, np.float32))
    off = i32(np.concatenate([[0], np.cumsum(nodes)]))
    keep = [dev.put(x) for x in (i32(lens), off, qkv, cos, sin)] + [dev.put(depth) if depths else None]
    dev.rope_append(cache.view, 1, h, rows, max(nodes), keep[0], keep[1], keep[5], keep[2], keep[3], keep[4], table_len, q)
    got = q.download(np.float32).reshape(rows + 1, h, hd)
    assert np.all(got[rows] == SENTINEL)
    k0, v0, row, r2 = cache.k.copy(), cache.v.copy(), 0, hd // 2
    for s, n in enumerate(nodes):
        for i in range(n):
            p = lens[s] + (int(depth[row]) if depths else i)
            if not 0 <= p < table_len:
                assert np.all(np.isnan(got[row]))
            else:
                c, d = cos[p], sin[p]
                x0, x1 = qkv[row, :, :r2], qkv[row, :, r2:]
                rot = np.concatenate([x0 * c - x1 * d, x0 * d + x1 * c], -1)  # float32: one rounding an operation
                assert np.array_equal(got[row].view(np.uint32), rot[:h].view(np.uint32))
                at = cache.where(s, lens[s] + i)
                if at:
                    k0[1, at[0], :, at[1]:at[1] + hd] = rot[h:h + hk].astype(np.float16)
                    v0[1, at[0], :, at[1]:at[1] + hd] = qkv[row, h + hk:].astype(np.float16)
            row += 1
    k1, v1 = cache.download()
    assert np.array_equal(k0.view(np.uint16), k1.view(np.uint16)) and np.array_equal(v0.view(np.uint16), v1.view(np.uint16))


# ---- accepted rows ------------------------------------------------------------------------------------


@pytest.mark.parametrize("page,hd,layers,most,alias", [(16, 64, 2, 4, False), (0, 128, 1, 9, True), (5, 8, 3, 40, False),
                                                       (128, 128, 2, 64, True), (7, 256, 1, 1, False)])
def test_accept(dev, page, hd, layers, most, alias):
    rng = np.random.default_rng(page + most)
    lens = [0, 3, 50, 31, 20, 11, 9]
    nodes = 2 * most + 2
    cache = Cache(dev, rng, [n + nodes for n in lens], page, 3, hd, layers=layers, pad=8, cap=200)
    path = np.full((len(lens), most), -7, np.int32)
    n_path = []
    for s in range(len(lens)):
        n = int(rng.integers(0, most + 1)) if s else most
        path[s, :n] = np.sort(rng.choice(nodes, n, replace=False))
        n_path.append(n)
    path[1], n_path[1] = np.arange(most), most  # nothing moves
    path[2, -1], n_path[2] = nodes - 1, most
    if most > 2:
        path[2, :most] = np.arange(most) + 2
        path[2, most - 1] = path[2, most - 2]   # not ascending: the path ends there
        path[3, 0], n_path[3] = -1, most        # a negative node: nothing is kept
        n_path[4] = -5
        path[5], n_path[5] = np.arange(most), most + 9  # more than the row holds
        path[6], n_path[6] = np.arange(most) + 100000, most  # behind the last page
    if page and most > 2:
        cache.table[5, (lens[5] + most - 1) // page] = cache.n_pages  # a hole at its last target
        cache.dt.upload(cache.table)
    k0, v0, kept = cache.k.copy(), cache.v.copy(), []
    for s, ln in enumerate(lens):
        n, before = 0, -1
        for e in path[s][:max(n_path[s], 0)]:
            a, b = (cache.where(s, ln + int(e)), cache.where(s, ln + n)) if e > before else (None, None)
            if not a or not b:
                break
            for new, old in ((k0, cache.k), (v0, cache.v)):
                new[:, b[0], :, b[1]:b[1] + hd] = old[:, a[0], :, a[1]:a[1] + hd]
            n, before = n + 1, e
        kept.append(ln + n)
    dl = dev.put(i32(lens))
    out = dl if alias else dev.alloc(4 * len(lens))
    dev.kv_accept(cache.view, most, dl, dev.put(path), dev.put(i32(n_path)), out)
    assert out.download(np.int32).tolist() == kept
    k1, v1 = cache.download()
    assert np.array_equal(k0.view(np.uint16), k1.view(np.uint16)) and np.array_equal(v0.view(np.uint16), v1.view(np.uint16))


# ---- forks ----------------------------------------------------------------------------------------------


def fork_reference(cache, lens, parents, grow):
    """The header's rules, one sequence after the other: (table, lens, granted, copies)."""
    n, page, n_pages, width = len(lens), cache.page, cache.n_pages, cache.max_pages
    cap = width * page
    new, length, g = [], [], []
    for i in range(n):
        p = parents[i] if parents is not None else i
        live = 0 <= p < n
        ln = min(max(int(lens[p]), 0), cap) if live else 0
        row = [-1] * width
        for j in range(-(-ln // page)):
            e = int(cache.table[p, j])
            row[j] = e if 0 <= e < n_pages else -1
        new.append(row)
        length.append(ln)
        g.append(max(int(grow[i]), 0) if live and grow is not None else 0)
    uses = {}  # page -> rows in use by each holder
    for i in range(n):
        for j in range(-(-length[i] // page)):
            if new[i][j] >= 0:
                uses.setdefault(new[i][j], []).append(min(page, length[i] - j * page))
    keeper = {}
    for i in range(n):
        mine = length[i] % page
        if g[i] and mine:
            last = new[i][length[i] // page]
            if last >= 0 and mine == max(uses[last]) and last not in keeper:
                keeper[last] = i
    free = [e for e in range(n_pages) if e not in uses]
    granted, copies, at, dry = [0] * n, [], 0, False
    table = [row[:] for row in new]
    for i in range(n):
        if not g[i] or length[i] + g[i] > cap:
            continue
        have, mine = -(-length[i] // page), length[i] % page
        last = new[i][have - 1] if mine else None
        if mine and last < 0:
            continue
        copy = bool(mine) and keeper.get(last) != i
        upto = -(-(length[i] + g[i]) // page)
        want = upto - have + copy
        if want and (dry or at + want > len(free)):
            dry = True
            continue
        if copy:
            copies.append((last, free[at], mine))
            table[i][have - 1] = free[at]
        for j in range(have, upto):
            table[i][j] = free[at + copy + j - have]
        at += want
        granted[i] = g[i]
    return table, length, granted, copies


def check_fork(dev, cache, lens, parents, grow, alias=False):
    table, length, granted, copies = fork_reference(cache, lens, parents, grow)
    k0, v0 = cache.k.copy(), cache.v.copy()
    for src, dst, rows in copies:
        for new, old in ((k0, cache.k), (v0, cache.v)):
            new[:, dst, :, :rows * cache.hd] = old[:, src, :, :rows * cache.hd]
    n = len(lens)
    dl = dev.put(i32(lens))
    dt, dlo, dg = dev.alloc(4 * n * cache.max_pages), dl if alias else dev.alloc(4 * n), dev.alloc(4 * n)
    dev.kv_fork(cache.view, 0, dl, dev.put(i32(parents)) if parents is not None else None,
                dev.put(i32(grow)) if grow is not None else None, dt, dlo, dg)
    assert dt.download(np.int32).reshape(n, -1).tolist() == table
    assert dlo.download(np.int32).tolist() == length
    assert dg.download(np.int32).tolist() == granted
    k1, v1 = cache.download()
    assert np.array_equal(k0.view(np.uint16), k1.view(np.uint16)) and np.array_equal(v0.view(np.uint16), v1.view(np.uint16))
    return table, length, granted


@pytest.mark.parametrize("seed", range(24))
def test_fork_pages(dev, seed):
    """A chain of random forks of a small cache: shared pages, ended sequences, full pages, too few pages, holes."""
    rng = np.random.default_rng(seed)
    page, hd, n = int(rng.choice([1, 4, 16, 33])), int(rng.choice([8, 64])), int(rng.integers(1, 9))
    width, n_pages = int(rng.integers(2, 7)), int(rng.integers(3, 24))
    table = np.full((n, width), -1, np.int32)
    cache = Cache(dev, rng, [1] * n, page, 2, hd, layers=2, pad=8, table=table, n_pages=n_pages, max_pages=width)
    lens = [0] * n
    for step in range(6):
        parents = [int(rng.integers(-1, n + 1)) if rng.random() < 0.7 else i for i in range(n)] if step else None
        grow = [int(rng.choice([0, 1, 2, page, 2 * page + 1, -3, 1000])) for _ in range(n)] if rng.random() < 0.9 else None
        new, length, granted = check_fork(dev, cache, lens, parents, grow, alias=bool(step & 1))
        cache.table[:] = new
        if rng.random() < 0.3:
            cache.table[int(rng.integers(n)), int(rng.integers(width))] = int(rng.choice([-2, n_pages, n_pages + 100]))
        cache.dt.upload(cache.table)
        # a sequence takes some of the room that it got, or gives positions back
        lens = [max(0, ln + int(rng.integers(-1, g + 1)) if g else ln) for ln, g in zip(length, granted)]


def test_fork_of_many_sequences(dev):
    rng = np.random.default_rng(77)
    n, page, width = 300, 16, 5
    cache = Cache(dev, rng, [1] * n, page, 1, 8, table=np.full((n, width), -1, np.int32), n_pages=1500, max_pages=width)
    new, lens, granted = check_fork(dev, cache, [0] * n, None, [int(x) for x in rng.integers(0, 80, n)])
    cache.table[:] = new
    cache.dt.upload(cache.table)
    lens = [int(rng.integers(0, g + 1)) for g in granted]
    check_fork(dev, cache, lens, [int(x) for x in rng.integers(-1, n, n)], [1] * n)


@pytest.mark.parametrize("n,hd,first,alias", [(1, 64, 0, True), (4, 128, 0, False), (8, 8, 5, True), (9, 64, 0, False), (32, 16, 3, True)])
def test_fork_runs(dev, n, hd, first, alias):
    rng = np.random.default_rng(n)
    cap = 41
    cache = Cache(dev, rng, [cap] * n, 0, 2, hd, layers=2, pad=8, cap=cap)
    lens = [int(rng.integers(first, cap + 1)) for _ in range(n)]
    parents = rng.permutation(n)
    parents[:n // 3] = rng.integers(-2, n + 2, n // 3)
    grow = [int(x) for x in rng.integers(-1, 30, n)]
    k0, v0, length = cache.k.copy(), cache.v.copy(), []
    for i, p in enumerate(int(x) for x in parents):
        live = 0 <= p < n
        length.append(lens[p] if live else 0)
        if live and length[i] > first:
            for new, old in ((k0, cache.k), (v0, cache.v)):
                new[:, i, :, first * hd:length[i] * hd] = old[:, p, :, first * hd:length[i] * hd]
    granted = [g if 0 <= p < n and g > 0 and ln + g <= cap else 0 for g, p, ln in zip(grow, parents, length)]
    dl = dev.put(i32(lens))
    dlo, dg = dl if alias else dev.alloc(4 * n), dev.alloc(4 * n)
    dev.kv_fork(cache.view, first, dl, dev.put(i32(parents)), dev.put(i32(grow)), None, dlo, dg)
    assert dlo.download(np.int32).tolist() == length and dg.download(np.int32).tolist() == granted
    k1, v1 = cache.download()
    assert np.array_equal(k0.view(np.uint16), k1.view(np.uint16)) and np.array_equal(v0.view(np.uint16), v1.view(np.uint16))


# ---- beam selection -------------------------------------------------------------------------------------


def beam_reference(logits, scores, done, pad, n_out):
    """Every candidate's score in 64 bits, ranked by (score, flat index): per prompt (score, parent, token)."""
    prompts, beams, vocab = logits.shape
    x = np.where(np.isnan(logits), -np.inf, logits).astype(np.float64)
    with np.errstate(invalid="ignore", divide="ignore"):
        top = x.max(-1, keepdims=True)
        z = np.where(x == top, 0.0, x - top)
        logp = z - np.log(np.exp(z).sum(-1, keepdims=True))
        cand = scores.astype(np.float64)[..., None] + np.where(top == -np.inf, -np.inf, logp)
    if done is not None:
        for a, b in zip(*np.nonzero(done)):
            cand[a, b] = -np.inf
            cand[a, b, pad] = scores[a, b]
    cand = np.where(np.isnan(cand), -np.inf, cand).reshape(prompts, -1)
    order = np.argsort(-cand, axis=-1, kind="stable")[:, :n_out]
    return cand, order


# exp of a logit as 2^((x - c) log2 e), c a thread's value up to 2 from its maximum: x - c, the product and the constant
# are off by 2^-24, 2^-24 and 2^-25 of |x - c|, whose mean under the weights is at most log(vocab) + 4 < 16: 40 * 2^-24;
# 2^-22 for 2^x, twice; 6 additions in 32 bits; the slice's sum is rounded to 32 bits: 55 * 2^-24 in log Z, below 2^-18.
# The score is rounded once more.
def beam_tol(s):
    return 2.0 ** -18 + 2.0 ** -24 * np.abs(s)


def check_beams(dev, logits, scores, done, pad, n_out, stride=None):
    prompts, beams, vocab = logits.shape
    stride = stride or vocab
    host = np.full((prompts * beams, stride), np.float32(1e30))  # what lies between rows must not matter
    host[:, :vocab] = logits.reshape(-1, vocab)
    out = [dev.alloc(4 * prompts * n_out) for _ in range(3)]
    dev.beam_select(prompts, beams, vocab, dev.put(host), stride, dev.put(scores.astype(np.float32)),
                    dev.put(i32(done)) if done is not None else None, pad, n_out, *out)
    gs = out[0].download(np.float32).reshape(prompts, n_out)
    gp = out[1].download(np.int32).reshape(prompts, n_out)
    gt = out[2].download(np.int32).reshape(prompts, n_out)
    cand, order = beam_reference(logits, scores, done, pad, n_out)
    for i in range(prompts):
        ws = cand[i, order[i]]
        for k in range(n_out):
            if k >= order.shape[1] or ws[k] == -np.inf:
                assert (gs[i, k], gp[i, k], gt[i, k]) == (-np.inf, -1, pad)
                continue
            tol = beam_tol(ws[k]) if np.isfinite(ws[k]) else 0.0
            assert gs[i, k] == ws[k] or abs(gs[i, k] - ws[k]) <= tol
            flat = (gp[i, k] - i * beams) * vocab + gt[i, k]
            # equal to the reference's choice, or another candidate whose score cannot be told from it
            assert flat == order[i, k] or 0 < abs(cand[i, flat] - ws[k]) <= 2 * tol
        chosen = [(a, b) for a, b in zip(gp[i], gt[i]) if a >= 0]
        assert len(set(chosen)) == len(chosen)
    return gs, gp, gt


@pytest.mark.parametrize("prompts,beams,vocab,n_out,stride", [
    (1, 1, 1, 1, None), (1, 1, 5, 8, None), (1, 4, 300, 4, None), (2, 3, 2048, 6, 2050), (3, 5, 8192, 10, None),
    (1, 8, 8193, 16, 8196), (1, 2, 128256, 4, None), (5, 1, 4097, 1, 4099), (1, 64, 777, 64, None), (2, 7, 30000, 64, 30004),
    (1, 13, 128256, 26, None), (1, 64, 40000, 64, None), (1, 1, 128256, 64, None)])
@pytest.mark.parametrize("ended", [False, True])
def test_beams(dev, prompts, beams, vocab, n_out, stride, ended):
    rng = np.random.default_rng(vocab + beams)
    logits = (rng.standard_normal((prompts, beams, vocab)) * 3).astype(np.float32)
    scores = (-5 * rng.random((prompts, beams))).astype(np.float32)
    done = (rng.random((prompts, beams)) < 0.3) if ended else None
    check_beams(dev, logits, scores, done, vocab // 2, n_out, stride)


@pytest.mark.parametrize("vocab", [40, 2000, 20000])
def test_beams_of_equal_scores(dev, vocab):
    """All logits equal: the lowest beam and token first, through the path for many equal values."""
    logits = np.full((2, 3, vocab), np.float32(0.25))
    scores = np.zeros((2, 3), np.float32)
    gs, gp, gt = check_beams(dev, logits, scores, None, 0, 20)
    assert gp.tolist() == [[0] * 20, [3] * 20] and gt.tolist() == [list(range(20))] * 2
    logits[:, :, vocab // 3] = 4.0  # one better token in every beam, equal over the beams
    gs, gp, gt = check_beams(dev, logits, scores, None, 0, 5)
    assert gp[0].tolist() == [0, 1, 2, 0, 0] and gt[0].tolist() == [vocab // 3] * 3 + [0, 1]
    # the first step of a search: all beams the same, all but one dead
    scores[:, 1:] = -np.inf
    gs, gp, gt = check_beams(dev, logits, scores, None, 0, 5)
    assert gp[0].tolist() == [0] * 5


@pytest.mark.parametrize("pick", [1, 16, 64])
@pytest.mark.parametrize("kind", ["random", "rising", "falling", "equal", "masked", "steps", "lowest"])
def test_beams_of_many_rows(dev, kind, pick):
    """Rows enough that a CTA goes through a whole vocabulary: every way in which later logits meet the earlier best."""
    prompts, beams, vocab = 150, 4, 13001
    rng = np.random.default_rng(pick)
    x = np.arange(vocab)
    if kind == "random":
        logits = rng.standard_normal((prompts, beams, vocab))
    elif kind == "rising":
        logits = np.broadcast_to(x / 1024.0, (prompts, beams, vocab))
    elif kind == "falling":
        logits = np.broadcast_to(-x / 1024.0, (prompts, beams, vocab))
    elif kind == "equal":
        logits = np.full((prompts, beams, vocab), -2.5)
    elif kind == "masked":
        logits = np.where(rng.random((prompts, beams, vocab)) < 0.002, rng.standard_normal((prompts, beams, vocab)), -np.inf)
        logits[7] = -np.inf
        logits[8, :, :9000] = np.nan
        logits[9, 1, 12000:12003] = np.inf
    elif kind == "lowest":  # masks of the type's lowest value: candidates like any others
        lowest = np.finfo(np.float32).min
        logits = np.where(rng.random((prompts, beams, vocab)) < 0.0002, rng.standard_normal((prompts, beams, vocab)), lowest)
        logits[3, :, :8192] = -np.inf
        logits[4] = np.where(x > 9000, lowest, -np.inf)
    else:  # equal values within a tile, larger ones in the next
        logits = np.broadcast_to((x // 4096).astype(float), (prompts, beams, vocab))
    scores = (-rng.random((prompts, beams))).astype(np.float32)
    check_beams(dev, np.ascontiguousarray(logits, np.float32), scores, None, 1, pick)


def test_beams_with_masked_and_infinite_logits(dev):
    rng = np.random.default_rng(3)
    logits = rng.standard_normal((1, 6, 9000)).astype(np.float32)
    logits[0, 0] = -np.inf                      # nothing can follow
    logits[0, 1, 7:] = -np.inf                  # seven tokens can
    logits[0, 2] = np.nan
    logits[0, 3, ::2] = np.nan
    logits[0, 4, [5, 8999]] = np.inf            # they share the probability
    logits[0, 5] = np.finfo(np.float32).min
    scores = np.array([[-1, -2, -3, np.nan, -0.5, -40]], np.float32)
    check_beams(dev, logits, scores, None, 3, 12)
    check_beams(dev, logits, scores, np.array([[1, 0, 0, 1, 0, 0]], bool), 3, 12)
    # fewer candidates than asked for
    gs, gp, gt = check_beams(dev, logits[:, :3], scores[:, :3], None, 3, 12)
    assert gp[0].tolist() == [1] * 7 + [-1] * 5


# ---- a run of them ----------------------------------------------------------------------------------------


def test_drafts_and_beams_over_shared_pages(dev):
    """Beams over one paged cache: fork, append, attend, accept, select, fork again; the rows that the
    attention then reads are those a cache without pages holds after the same steps."""
    rng = np.random.default_rng(21)
    n, h, hk, hd, page, width, pages = 4, 4, 2, 64, 16, 8, 40
    cache = Cache(dev, rng, [1] * n, page, hk, hd, layers=2, table=np.full((n, width), -1, np.int32), n_pages=pages,
                  max_pages=width)
    plain = [[np.zeros((2, hk, 0, hd)) for _ in range(n)] for _ in range(2)]  # [k, v][sequence], committed rows
    ang = np.outer(np.arange(width * page), 10000.0 ** (-np.arange(hd // 2) / (hd // 2)))
    cos, sin = dev.put(np.cos(ang).astype(np.float32)), dev.put(np.sin(ang).astype(np.float32))
    lens, tables = dev.put(i32([0] * n)), [dev.alloc(4 * n * width), cache.dt]
    granted, host_lens, score = dev.alloc(4 * n), [0] * n, np.zeros((1, n), np.float32)
    for step in range(7):
        # beams continue their parents, with room for the drafted nodes
        vocab = 500
        logits = (rng.standard_normal((1, n, vocab)) * 3).astype(np.float32)
        sc, parents, tokens = (dev.alloc(4 * n) for _ in range(3))
        dev.beam_select(1, n, vocab, dev.put(logits), vocab, dev.put(score), None, 0, n, sc, parents, tokens)
        nodes = [int(x) for x in rng.integers(1, 9, n)]
        new = tables[step & 1]
        cache.view.table = tables[1 - (step & 1)].ptr
        dev.kv_fork(cache.view, 0, lens, parents, dev.put(i32(nodes)), new, lens, granted)
        cache.view.table = new.ptr
        par = parents.download(np.int32).tolist()
        score = sc.download(np.float32).reshape(1, n)
        assert granted.download(np.int32).tolist() == nodes
        host_lens = [host_lens[p] for p in par]
        assert lens.download(np.int32).tolist() == host_lens
        plain = [[x[p] for p in par] for x in plain]
        cache.table = new.download(np.int32).reshape(n, width)
        # drafts: append in both layers, attend in both
        off = i32(np.concatenate([[0], np.cumsum(nodes)]))
        rows = int(off[-1])
        sees = [random_tree(rng, k) for k in nodes]
        depth = i32(np.concatenate([s.sum(1) - 1 for s in sees]))
        keep = [dev.put(off), dev.put(depth), dev.put(pack(sees, max(nodes)))]
        for layer in range(2):
            qkv = dev.put(rng.standard_normal((rows, h + 2 * hk, hd)).astype(np.float32))
            q, out = dev.alloc(rows * h * hd * 4), dev.alloc(rows * h * hd * 4)
            dev.rope_append(cache.view, layer, h, rows, max(nodes), lens, keep[0], keep[1], qkv, cos, sin, width * page, q)
            dev.attn_tree(cache.view, layer, h, rows, max(nodes), lens, keep[0], keep[2], q, out)
            cache.download()
            for s in range(n):  # the committed rows, as the steps before left them
                for plane, own in ((cache.k, plain[0]), (cache.v, plain[1])):
                    assert np.array_equal(cache.rows(plane, layer, s, host_lens[s])[0], own[s][layer])
            qh = q.download(np.float32).reshape(rows, h, hd)
            close(out.download(np.float32).reshape(rows, h, hd), *attend(cache, layer, host_lens, sees, qh, h))
        # accept a path from the root to a random node
        paths = [np.flatnonzero(s[rng.integers(len(s))]) for s in sees]
        most = max(map(len, paths))
        path = np.zeros((n, most), np.int32)
        for s, p in enumerate(paths):
            path[s, :len(p)] = p
            for a, plane in ((0, cache.k), (1, cache.v)):
                took = np.stack([cache.rows(plane, la, s, host_lens[s] + nodes[s])[0][:, host_lens[s] + p] for la in range(2)])
                plain[a][s] = np.concatenate([plain[a][s], took], 2)
            host_lens[s] += len(p)
        dev.kv_accept(cache.view, most, lens, dev.put(path), dev.put(i32([len(p) for p in paths])), lens)
        assert lens.download(np.int32).tolist() == host_lens


def test_a_beam_step_captured_and_replayed(dev):
    """Selection, fork and attention as one graph: every replay works on what lies on the device then."""
    rng = np.random.default_rng(31)
    L = _native.load()
    beams, vocab, hd, page = 4, 5003, 64, 16
    lens = [20, 20, 20, 20]
    cache = Cache(dev, rng, lens, page, 1, hd, layers=2, spare=8, max_pages=3)
    start = dict(k=cache.k.copy(), v=cache.v.copy(), table=cache.table.copy())
    logits, scores = dev.alloc(4 * beams * vocab), dev.alloc(4 * beams)
    out = [dev.alloc(4 * beams) for _ in range(3)]
    dl, grow, table2 = dev.put(i32(lens)), dev.put(i32([3] * beams)), dev.alloc(4 * beams * cache.max_pages)
    lens2, granted = dev.alloc(4 * beams), dev.alloc(4 * beams)
    after = KvView.from_buffer_copy(cache.view)
    after.table = table2.ptr
    q = rng.standard_normal((beams, 2, hd)).astype(np.float32)
    off, dq, att = dev.put(i32(range(beams + 1))), dev.put(q), dev.alloc(q.nbytes)

    def step():
        dev.beam_select(1, beams, vocab, logits, vocab, scores, None, 0, beams, *out)
        dev.kv_fork(cache.view, 0, dl, out[1], grow, table2, lens2, granted)
        dev.attn_tree(after, 1, 2, beams, 1, lens2, off, None, dq, att)

    logits.upload(np.zeros((beams, vocab), np.float32))
    scores.upload(np.zeros(beams, np.float32))
    step()  # sizes the scratch
    dev.sync()
    g = C.c_void_p()
    _native.check(L.pai_b200_graph_begin(dev.ctx), "begin")
    step()
    _native.check(L.pai_b200_graph_end(dev.ctx, C.byref(g)), "end")
    try:
        for turn in range(3):
            cache.k, cache.v, cache.table = start["k"].copy(), start["v"].copy(), start["table"].copy()
            cache.put()
            x = rng.standard_normal((1, beams, vocab)).astype(np.float32)
            sc = (-rng.random((1, beams))).astype(np.float32)
            logits.upload(x[0])
            scores.upload(sc)
            _native.check(L.pai_b200_graph_launch(dev.ctx, g), "launch")
            got = out[1].download(np.int32)
            cand, order = beam_reference(x, sc, None, 0, beams)
            assert got.tolist() == (order[0] // vocab).tolist()
            table, length, room, copies = fork_reference(cache, lens, got.tolist(), [3] * beams)
            for src, dst, rows in copies:
                for plane in (cache.k, cache.v):
                    plane[:, dst, :, :rows * hd] = plane[:, src, :, :rows * hd]
            assert table2.download(np.int32).reshape(beams, -1).tolist() == table
            assert (lens2.download(np.int32).tolist(), granted.download(np.int32).tolist()) == (length, room)
            cache.table = i32(table)
            sees = [np.ones((1, 1), bool)] * beams
            close(att.download(np.float32).reshape(q.shape), *attend(cache, 1, length, sees, q, 2))
    finally:
        dev.sync()
        L.pai_b200_graph_destroy(g)


def test_contexts_at_once():
    """Two contexts, each on a thread of its own, give the bits that they give alone."""
    import threading

    from prosperoai_b200.api import Device

    rng = np.random.default_rng(8)
    shapes = [([700, 90], [1, 1]), ([260], [40])]
    jobs = []
    for lens, nodes in shapes:
        d = Device(0)
        cache = Cache(d, rng, [n + k for n, k in zip(lens, nodes)], 64, 2, 128)
        rows = sum(nodes)
        q = d.put(rng.standard_normal((rows, 8, 128)).astype(np.float32))
        x = d.put(rng.standard_normal((rows, 9001)).astype(np.float32))
        sc = d.put(np.zeros(rows, np.float32))
        outs = [d.alloc(rows * 8 * 128 * 4)] + [d.alloc(4 * 8) for _ in range(3)]
        off = d.put(i32(np.concatenate([[0], np.cumsum(nodes)])))
        jobs.append((d, cache, d.put(i32(lens)), off, max(nodes), rows, q, x, sc, outs))

    def work(job, times, results):
        d, cache, lens, off, most, rows, q, x, sc, outs = job
        for _ in range(times):
            d.attn_tree(cache.view, 0, 8, rows, most, lens, off, None, q, outs[0])
            d.beam_select(1, rows, 9001, x, 9001, sc, None, 0, 8, *outs[1:])
        results.append([o.download(np.uint32) for o in outs])

    alone, both = [], [[], []]
    for job in jobs:
        work(job, 1, alone)
    threads = [threading.Thread(target=work, args=(job, 60, both[i])) for i, job in enumerate(jobs)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(alone, both):
        for u, v in zip(a, b[0]):
            np.testing.assert_array_equal(u, v)
    for job in jobs:
        for item in (job[1].dk, job[1].dv, job[1].dt, job[2], job[3], *job[6:9], *job[9]):
            item.free()
        job[0].close()
