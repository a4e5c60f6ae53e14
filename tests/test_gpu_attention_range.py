"""Tree attention over the whole range of its inputs, in every form of its kernels.

The bounds are those of test_gpu_continuations.attend unless a test says otherwise.
"""
import numpy as np
import pytest

from prosperoai_b200 import _native
from prosperoai_b200.api import KvView
from test_gpu_continuations import Cache, attend, close, i32, pack, random_tree, run_tree

pytestmark = pytest.mark.gpu

# page, nodes, h, hk, hd: the rows of a kv head (nodes x h / hk), the page size and head_dim choose the kernel
FORMS = {
    "few 8": (16, 2, 8, 2, 128), "few 16": (0, 4, 4, 1, 128), "few 32": (64, 8, 8, 2, 128), "few 8 of 64": (16, 2, 8, 2, 64),
    "few 16 of 64": (0, 4, 8, 2, 64), "many": (16, 12, 8, 2, 128), "many of 64": (0, 40, 4, 2, 64),
    "any page": (20, 5, 8, 2, 128), "any page of 64": (7, 3, 4, 2, 64), "any page, rows": (100, 12, 8, 2, 128),
    "any page, rows of 64": (20, 40, 4, 2, 64),
}
forms = pytest.mark.parametrize("page,n,h,hk,hd", list(FORMS.values()), ids=list(FORMS))


def one_sequence(dev, rng, form, past, spare=16):
    page, n, h, hk, hd = form
    cache = Cache(dev, rng, [past + n + spare], page, hk, hd, cap=past + n + spare)
    return cache, rng.standard_normal((n, h, hd)).astype(np.float32)


# ---- what is not a number reaches the rows that attend it, and no others ------------------------------------


@forms
def test_nan_queries(dev, page, n, h, hk, hd):
    """As rotary append leaves them for a position behind its tables."""
    rng = np.random.default_rng(hd + n)
    cache, q = one_sequence(dev, rng, (page, n, h, hk, hd), 70)
    sees = [random_tree(rng, n)]
    want, bound = attend(cache, 0, [70], sees, q, h)
    q[1, h - 1, 3] = np.nan
    got = run_tree(dev, cache, 0, [70], [n], h, pack(sees, n), q)
    others = np.ones((n, h), bool)
    others[1, h - 1] = False
    assert np.isnan(got[1, h - 1]).all()
    close(got[others], want[others], bound[others])


@forms
@pytest.mark.parametrize("past", [0, 16, 48, 64, 130])
def test_one_nan_key(dev, page, n, h, hk, hd, past):
    """The first key behind 16 positions may be the only one that a warp's share of a tile shows a row."""
    rng = np.random.default_rng(past + n)
    cache, q = one_sequence(dev, rng, (page, n, h, hk, hd), past)
    sees = [random_tree(rng, n)]
    sees[0][:, 0] = False
    sees[0][0] = np.arange(n) == 0
    want, bound = attend(cache, 0, [past], sees, q, h)
    p, e = cache.where(0, past)
    cache.k[0, p, :, e + 1] = np.nan
    cache.put()
    got = run_tree(dev, cache, 0, [past], [n], h, pack(sees, n), q)
    assert np.isnan(got[0]).all()
    close(got[1:], want[1:], bound[1:])


@forms
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_nonfinite_nodes(dev, page, n, h, hk, hd, bad):
    rng = np.random.default_rng(n * hd)
    cache, q = one_sequence(dev, rng, (page, n, h, hk, hd), 70)
    sees = [random_tree(rng, n)]
    sees[0][:, 1] = np.arange(n) == 1
    want, bound = attend(cache, 0, [70], sees, q, h)
    others = np.arange(n) != 1
    for pos in [71] + list(range(70 + n, 70 + n + 16)):  # node 1, and the stale rows behind the last node
        p, e = cache.where(0, pos)
        cache.k[0, p, :, e:e + hd] = bad
        cache.v[0, p, :, e:e + hd] = bad
    cache.put()
    got = run_tree(dev, cache, 0, [70], [n], h, pack(sees, n), q)
    assert not np.isfinite(got[1]).any()
    close(got[others], want[others], bound[others])
    # one element of the node's V row: that element of the row that sees it
    p, e = cache.where(0, 71)
    cache.k[0, p, :, e:e + hd] = 0
    cache.v[0, p, :, e:e + hd] = 0
    cache.v[0, p, :, e + 5] = bad
    cache.put()
    got = run_tree(dev, cache, 0, [70], [n], h, pack(sees, n), q)
    assert np.array_equal(np.isfinite(got[1]), np.tile(np.arange(hd) != 5, (h, 1)))
    close(got[others], want[others], bound[others])


# ---- queries of unequal elements ------------------------------------------------------------------------------


@forms
@pytest.mark.parametrize("outlier", [64, 1024, 8192])
def test_outlier_query_dimensions(dev, page, n, h, hk, hd, outlier):
    """One large dimension of q against a K channel that is small by as much, as the channels of trained models are: the
    other dimensions count as much as that one. Half of fp16's smallest step is 2^-25, and a row's largest element lies
    at 2^14 or above: what is too small for both of its parts is off by 2^-39 of it, a score by 2^-39 max |q| sum |k| /
    sqrt(hd) more than with equal elements."""
    rng = np.random.default_rng(outlier + n)
    cache, q = one_sequence(dev, rng, (page, n, h, hk, hd), 300)
    row = cache.page * hd
    cache.k[..., 0:row:hd] = (cache.k[..., 0:row:hd].astype(np.float32) / outlier).astype(np.float16)
    cache.put()
    q[..., 0] = 3 * outlier * np.where(rng.random((n, h)) < 0.5, -1, 1)
    sees = [random_tree(rng, n)]
    want, bound = attend(cache, 0, [300], sees, q, h)
    most = np.abs(cache.k.astype(np.float64)[..., :row].reshape(-1, hd)).sum(-1).max()
    bound = bound + 2 * 2.0 ** -39 * np.abs(q).max() * most / np.sqrt(hd) * np.abs(cache.v.astype(np.float64)).max()
    close(run_tree(dev, cache, 0, [300], [n], h, pack(sees, n), q), want, bound)


# ---- scores of any size ---------------------------------------------------------------------------------------


@forms
@pytest.mark.parametrize("scale", [1e6, 1e7, 2e7, 4e7, 1e8, 1e9, 1e12, 1e20])
def test_large_scores(dev, page, n, h, hk, hd, scale):
    """Scores whose steps are larger than the exponents of the weights. The outputs are means of the V rows; where the best
    score is further from the next than both may be off (2^-20 + hd / 8 2^-23 of sum |q_d k_d| / sqrt(hd) each) and e^-40
    more, the output is the best key's V row."""
    rng = np.random.default_rng(n + hd)
    past = 500
    cache, q = one_sequence(dev, rng, (page, n, h, hk, hd), past)
    q = (q * np.float32(scale)).astype(np.float32)
    sees = [random_tree(rng, n)]
    got = run_tree(dev, cache, 0, [past], [n], h, pack(sees, n), q)
    assert np.isfinite(got).all()
    k, _ = cache.rows(cache.k, 0, 0, past + n)
    v, _ = cache.rows(cache.v, 0, 0, past + n)
    top, decided = np.abs(v).max(), 0
    assert np.abs(got).max() <= top * (1 + 2.0 ** -19)
    for i in range(n):
        ok = np.concatenate([np.ones(past, bool), sees[0][i]])
        for j in range(h):
            kk, qq = k[j // (h // hk)][ok], q[i, j].astype(np.float64)
            sc = kk @ qq / np.sqrt(hd)
            ds = (2.0 ** -20 + hd / 8 * 2.0 ** -23) * (np.abs(kk) @ np.abs(qq)).max() / np.sqrt(hd)
            best = sc.argmax()
            if np.partition(sc, -2)[-2] < sc[best] - 2 * ds - 40:
                decided += 1
                tol = (2.0 ** -21 + (len(kk) / 8 + 4) * 2.0 ** -23) * top
                assert np.abs(got[i, j] - v[j // (h // hk)][ok][best]).max() <= tol
    assert decided > n * h // 2


@forms
@pytest.mark.parametrize("query,key", [(1e33, 1.0), (1e29, 1.0), (1.7e38, 2.0 ** -10), (3e38, 2.0 ** -14), (1e-40, 60000.0), (0.0, 1.0)])
@pytest.mark.parametrize("sign", [1, -1])
def test_equal_scores_of_any_size(dev, page, n, h, hk, hd, query, key, sign):
    """All keys have the same score, whatever it is: the output is the mean of the V rows. The weights are equal, so
    only the sum's roundings are left: 2^-23 for each of n / 8 + 4 steps, 2^-21 for the weights' parts."""
    rng = np.random.default_rng(n)
    past = 300
    cache, q = one_sequence(dev, rng, (page, n, h, hk, hd), past)
    row = cache.page * hd
    cache.k[..., 0:row:hd] = key
    cache.put()
    q[:] = 0
    q[..., 0] = sign * query
    sees = [random_tree(rng, n)]
    got = run_tree(dev, cache, 0, [past], [n], h, pack(sees, n), q)
    v, _ = cache.rows(cache.v, 0, 0, past + n)
    for i in range(n):
        ok = np.concatenate([np.ones(past, bool), sees[0][i]])
        want = np.repeat(v[:, ok].mean(1), h // hk, 0)
        assert np.abs(got[i] - want).max() <= (2.0 ** -21 + (ok.sum() / 8 + 4) * 2.0 ** -23) * np.abs(v).max()


# ---- holes, empty rows, long trees ----------------------------------------------------------------------------


@pytest.mark.parametrize("page,n,h,hk,hd", [f for f in FORMS.values() if f[0]], ids=[k for k, f in FORMS.items() if f[0]])
def test_holes_and_rows_that_see_nothing(dev, page, n, h, hk, hd):
    rng = np.random.default_rng(page + n)
    lens, nodes = [230, 0, 90], [n, n, max(n - 1, 1)]
    width = -(-(230 + n) // page) + 1
    table = rng.permutation(3 * width).reshape(3, width)
    table[rng.random((3, width)) < 0.3] = -1
    table[0, 0], table[2, -1] = 3 * width, -(1 << 31)
    table[1, :-(-n // page)] = -1  # every node of a sequence without a past
    cache = Cache(dev, rng, [1] * 3, page, hk, hd, table=table, n_pages=3 * width, max_pages=width)
    sees = [random_tree(rng, k) for k in nodes]
    sees[0][0] = False
    sees[2][:] = False
    q = rng.standard_normal((sum(nodes), h, hd)).astype(np.float32)
    got = run_tree(dev, cache, 0, lens, nodes, h, pack(sees, n), q)
    close(got, *attend(cache, 0, lens, sees, q, h))
    assert not got[n:2 * n].any()
    # nothing committed, nothing seen
    alone = Cache(dev, rng, [n], page, hk, hd)
    assert not run_tree(dev, alone, 0, [0], [n], h, pack([np.zeros((n, n), bool)], n), q[:n]).any()


@pytest.mark.parametrize("lens,nodes,page,h,hk,hd", [
    ([50], [1024], 16, 2, 1, 64), ([10, 300], [200, 513], 20, 2, 2, 128), ([700], [257], 0, 2, 1, 128), ([0], [131], 100, 1, 1, 64),
    ([33, 1, 0], [1, 1024, 129], 64, 1, 1, 128)])
@pytest.mark.parametrize("kind", ["tree", "chain"])
def test_long_trees(dev, lens, nodes, page, h, hk, hd, kind):
    """Masks of up to 16 words, row tiles behind the first."""
    rng = np.random.default_rng(sum(nodes))
    total = [a + b for a, b in zip(lens, nodes)]
    cache = Cache(dev, rng, total, page, hk, hd, cap=max(total))
    sees = [random_tree(rng, n) if kind == "tree" else np.tril(np.ones((n, n), bool)) for n in nodes]
    q = rng.standard_normal((sum(nodes), h, hd)).astype(np.float32)
    got = run_tree(dev, cache, 0, lens, nodes, h, pack(sees, max(nodes)) if kind == "tree" else None, q)
    close(got, *attend(cache, 0, lens, sees, q, h))


# ---- dependent launches ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("page,n,h,hk,hd", [FORMS[k] for k in ("few 16", "many", "any page")], ids=["few", "many", "any page"])
def test_dependent_launches(dev, page, n, h, hk, hd):
    """Selection, fork, append, attention and acceptance, each launched while the one before runs (pai_b200_set_pdl), give
    the bits that they give one behind the other."""
    L, rng = _native.load(), np.random.default_rng(n)
    beams, vocab, past = 4, 3001, 61
    width = -(-(past + 3 * n) // page) if page else 1
    table = rng.permutation(2 * beams * width).reshape(2, beams, width)[0] if page else None
    cache = Cache(dev, rng, [past] * beams, page, hk, hd, layers=2, table=table, n_pages=2 * beams * width if page else None,
                  max_pages=width if page else None, cap=past + 3 * n)
    rows, lens = beams * n, i32([past - b for b in range(beams)])
    off, path = i32(np.arange(beams + 1) * n), i32([[0, n - 1]] * beams)
    sees = [random_tree(rng, n) for _ in range(beams)]
    ang = rng.standard_normal((past + 4 * n, hd // 2)).astype(np.float32)
    given = dict(logits=rng.standard_normal((beams, vocab)).astype(np.float32), scores=np.zeros(beams, np.float32),
                 qkv=rng.standard_normal((rows, h + 2 * hk, hd)).astype(np.float32), cos=np.cos(ang), sin=np.sin(ang), lens=lens,
                 off=off, path=path, n_path=i32([2] * beams), mask=pack(sees, n), grow=i32([n] * beams))
    d = {k: dev.put(v) for k, v in given.items()}
    out = {k: dev.alloc(4 * size) for k, size in dict(score=beams, parent=beams, token=beams, table=beams * width, lens=beams,
                                                      granted=beams, q=rows * h * hd, att=rows * h * hd, after=beams).items()}
    forked = KvView.from_buffer_copy(cache.view)
    if page:
        forked.table = out["table"].ptr

    def step():
        cache.put()
        for o in out.values():
            o.upload(np.zeros(o.nbytes // 4, np.int32))
        dev.beam_select(1, beams, vocab, d["logits"], vocab, d["scores"], None, 0, beams, out["score"], out["parent"], out["token"])
        dev.kv_fork(cache.view, 0, d["lens"], out["parent"], d["grow"], out["table"] if page else None, out["lens"], out["granted"])
        for layer in range(2):
            dev.rope_append(forked, layer, h, rows, n, out["lens"], d["off"], None, d["qkv"], d["cos"], d["sin"], len(ang), out["q"])
            dev.attn_tree(forked, layer, h, rows, n, out["lens"], d["off"], d["mask"], out["q"], out["att"])
        dev.kv_accept(forked, 2, out["lens"], d["path"], d["n_path"], out["after"])
        return [o.download(np.uint32) for o in out.values()] + [cache.dk.download(np.uint16), cache.dv.download(np.uint16)]

    want = step()
    assert (want[5] == n).all() and np.isfinite(want[7].view(np.float32)).all()  # room for all, attended
    _native.check(L.pai_b200_set_pdl(dev.ctx, 1), "set_pdl")
    try:
        for _ in range(20):
            for a, b in zip(step(), want):
                np.testing.assert_array_equal(a, b)
    finally:
        L.pai_b200_set_pdl(dev.ctx, 0)
