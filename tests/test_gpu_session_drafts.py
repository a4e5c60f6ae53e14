"""Drafted trees and beams on a decode session.

A verification computes what stepping the nodes one after the other computes,
in another order and (above 8 rows) with the prefill's GEMM on bf16 tiles. Its
logits are held to 2e-2 of the largest, the bound that the prefill's hidden
states are held to: the stepped logit of a greedy token is then at most twice
that below the stepped maximum. What runs the same kernels on the same bits is compared bit by bit.
"""
import numpy as np
import pytest

from oracle import py_oracle as po
from prosperoai_b200 import _native
from prosperoai_b200.api import Model, Session
from test_gpu_model import SMALL

pytestmark = pytest.mark.gpu

INVALID, NOMEM, UNSUPPORTED = -1, -2, -3
SHARED = dict(SMALL, n_head_kv=1)


@pytest.fixture(scope="module", params=[("q8_0", SMALL, po.Q8_0), ("q4_k", SHARED, po.Q4_K)], ids=lambda p: p[0])
def model(dev, request):
    _, cfg, wtype = request.param
    m = Model(dev, dict(cfg, wtype=wtype))
    m.synthesize(7300 + wtype)
    yield m
    m.close()


def stepped(model, batch, history, paths):
    """Logits [batch][len] after every token of paths [batch][len] behind history [batch][n], one step each."""
    s = Session(model, batch, 256)
    s.prefill(history)
    out = [s.step(np.array(paths)[:, i], True)[1].reshape(batch, -1) for i in range(np.array(paths).shape[1])]
    s.close()
    return np.stack(out, 1)


def told_apart(logits):
    """Where the greedy token is decided: the top two are further apart than both may be off."""
    top = np.sort(logits, -1)
    return top[..., -1] - top[..., -2] > 2 * 2e-2 * np.abs(logits).max(-1)


def same_greedy(got, logits):
    """The maximum of logits that are off by 2e-2 each at most: the stepped greedy token wherever it is told apart."""
    chosen = np.take_along_axis(logits, np.asarray(got, np.int64)[..., None], -1)[..., 0]
    assert (chosen >= logits.max(-1) - 2 * 2e-2 * np.abs(logits).max(-1)).all()


@pytest.mark.parametrize("batch,n", [(1, 1), (1, 7), (2, 4), (8, 1), (1, 9), (4, 13), (2, 70)])
def test_verified_chain_is_what_steps_give(model, batch, n):
    rng = np.random.default_rng(100 * batch + n)
    vocab = model.cfg["vocab"]
    history, draft = rng.integers(0, vocab, (batch, 21)), rng.integers(0, vocab, (batch, n))
    want = stepped(model, batch, history, draft)
    s = Session(model, batch, 256)
    first = s.prefill(history)
    got = s.verify(draft)
    same_greedy(got, want)
    # nothing was committed: the steps give the bits they give without it
    assert s.pos == 21
    np.testing.assert_array_equal(s.tokens(), first)
    again = np.stack([s.step(draft[:, i], True)[1].reshape(batch, -1) for i in range(n)], 1)
    np.testing.assert_array_equal(again, want)
    s.close()


TREE = [-1, 0, 0, -1, 1, 2, 2, 3, 5, 5, 8, -1, 9]


@pytest.mark.parametrize("batch,n", [(1, 8), (1, 13), (4, 13), (8, 13)])
def test_tree_then_accepted_path(model, batch, n):
    """Every branch as if it were stepped alone; the accepted nodes are the cache of the steps after."""
    rng = np.random.default_rng(batch)
    vocab = model.cfg["vocab"]
    history, draft = rng.integers(0, vocab, (batch, 130)), rng.integers(0, vocab, (batch, n))
    parents = TREE[:n]
    s = Session(model, batch, 256)
    s.prefill(history)
    got = s.verify(draft, parents)
    leaves = [i for i in range(n) if i not in parents]
    for leaf in leaves:
        path = []
        while leaf >= 0:
            path.insert(0, leaf)
            leaf = parents[leaf]
        same_greedy(got[:, path], stepped(model, batch, history, draft[:, path]))
    # each sequence keeps another path of the same length, then goes on alone
    choices = [p for p in ([0, 1, 4], [0, 2, 5], [0, 2, 6]) if p[-1] < n]
    path = np.array([choices[b % len(choices)] for b in range(batch)])
    tail = rng.integers(0, vocab, (batch, 4))
    kept = np.take_along_axis(draft, path, 1)
    s.accept(path, tail[:, 0])
    assert s.pos == 133
    logits = []
    s.run(1)  # the tokens given to accept
    logits.append(s.tokens())
    for i in range(1, 4):
        logits.append(s.step(tail[:, i], True)[1].reshape(batch, -1))
    s.close()
    want = stepped(model, batch, history, np.concatenate([kept, tail], 1))[:, 3:]
    same_greedy(logits[0][:, None], want[:, :1])
    for i in range(1, 4):
        assert np.abs(logits[i] - want[:, i]).max() <= 2e-2 * np.abs(want[:, i]).max()


def test_drafts_of_drafts(model):
    """Verify and accept in turn (as a drafting loop does) give the greedy decode's tokens."""
    rng = np.random.default_rng(3)
    vocab = model.cfg["vocab"]
    history = rng.integers(0, vocab, (1, 40))
    s = Session(model, 1, 256)
    plain = [int(s.prefill(history)[0])]
    sure = []
    for _ in range(40):
        nxt, logits = s.step(np.array(plain[-1:]), True)
        sure.append(bool(told_apart(logits)))
        plain.append(int(nxt[0]))
    s.reset()
    tok = int(s.prefill(history)[0])
    out, rounds = [tok], 0
    while len(out) <= 40:
        at = len(out) - 1
        draft = [out[-1], *plain[at + 1:at + 5]]
        if rounds % 3 == 1 and len(draft) > 3:
            draft[2] = (draft[2] + 1) % vocab  # a wrong guess: the nodes behind it are dropped
        nxt = s.verify([draft])[0]
        k = 1
        while k < len(draft) and draft[k] == nxt[k - 1]:
            k += 1
        s.accept([list(range(k))], [nxt[k - 1]])
        out += draft[1:k] + [int(nxt[k - 1])]
        rounds += 1
    for i, (a, b) in enumerate(zip(out, plain)):
        if a != b:
            assert not sure[i - 1]  # a near tie may fall the other way, and the texts part there
            assert i > 5
            break
    s.close()


@pytest.mark.parametrize("batch,n", [(1, 4), (2, 9)])
def test_verifications_of_one_size_follow_their_inputs(model, batch, n):
    """The second call of a size is captured and replayed from then on: tokens, trees and positions are those of each call."""
    rng = np.random.default_rng(n)
    vocab = model.cfg["vocab"]
    history = rng.integers(0, vocab, (batch, 30))
    s = Session(model, batch, 256)
    s.prefill(history)
    for turn in range(5):
        draft = rng.integers(0, vocab, (batch, n))
        parents = [-1] + [int(rng.integers(-1, i)) for i in range(1, n)] if turn else None
        fresh = Session(model, batch, 256)
        fresh.prefill(history[:, :30])
        for i in range(30, history.shape[1]):
            fresh.step(history[:, i])
        got, want = s.verify(draft, parents), fresh.verify(draft, parents)
        fresh.close()
        np.testing.assert_array_equal(got, want)
        if turn == 2:
            s.verify(draft[:, :1])  # another size in between
        if turn == 3:  # the kernels carry the limit on their waits
            _native.check(_native.load().pai_b200_set_wait_limit(model.dev.ctx, 3_000_000_000), "set_wait_limit")
            np.testing.assert_array_equal(s.verify(draft, parents), want)
            _native.check(_native.load().pai_b200_set_wait_limit(model.dev.ctx, 0), "set_wait_limit")
        s.step(draft[:, 0])
        history = np.concatenate([history, draft[:, :1]], 1)
    s.close()


def log_softmax(x):
    x = x.astype(np.float64)
    return x - x.max(-1, keepdims=True) - np.log(np.exp(x - x.max(-1, keepdims=True)).sum(-1, keepdims=True))


@pytest.mark.parametrize("batch", [2, 4, 8])
def test_beam_search(model, batch):
    """Selections against a 64-bit ranking, and caches that follow their beams."""
    rng = np.random.default_rng(40 + batch)
    vocab, P = model.cfg["vocab"], 19
    prompt = np.repeat(rng.integers(0, vocab, (1, P)), batch, 0)
    s = Session(model, batch, 256)
    s.prefill(prompt[:, :-1])
    logits = s.step(prompt[:, -1], True)[1].reshape(batch, vocab)
    scores = np.full(batch, -np.inf, np.float32)
    scores[0] = 0
    texts, past = [[] for _ in range(batch)], None
    for i in range(6):
        cand = scores[:, None].astype(np.float64) + log_softmax(logits)
        got, parents, tokens = s.beam(scores, first=P)
        assert len(set(zip(parents.tolist(), tokens.tolist()))) == batch
        chosen = cand[parents, tokens]
        tol = 2.0 ** -18 + 2.0 ** -24 * np.abs(chosen)  # the selection's own bound
        assert (np.abs(got - chosen) <= tol).all()
        assert (np.abs(np.sort(cand.ravel())[::-1][:batch] - chosen) <= 2 * tol).all()
        assert (np.diff(got) <= 0).all()
        texts = [texts[p] + [int(t)] for p, t in zip(parents, tokens)]
        scores = got
        s.run(1)  # on the chosen tokens
        alone = Session(model, batch, 256)
        alone.prefill(prompt[:, :-1])
        alone.step(prompt[:, -1])
        for j in range(i + 1):
            want = alone.step(np.array([t[j] for t in texts], np.int32), True)[1].reshape(batch, vocab)
        alone.close()
        logits = want
        np.testing.assert_array_equal(s.tokens(), want.argmax(-1))
    assert s.pos == P + 6
    s.close()


def test_beams_that_ended_or_died(model):
    batch, vocab = 4, model.cfg["vocab"]
    rng = np.random.default_rng(9)
    s = Session(model, batch, 128)
    s.prefill(rng.integers(0, vocab, (batch, 5)))
    # only ended beams: one candidate each, best first; the dead beam's place stays empty
    sc, parents, tokens = s.beam([-3.0, -1.0, -np.inf, -2.0], done=[1, 1, 1, 1], pad=7)
    np.testing.assert_array_equal(sc, np.array([-1, -2, -3, -np.inf], np.float32))
    np.testing.assert_array_equal(parents, [1, 3, 0, -1])
    np.testing.assert_array_equal(tokens, [7] * 4)
    s.run(1)
    assert s.pos == 6 and np.isfinite(s.step([1, 2, 3, 4], True)[1]).all()
    s.close()


def refused(code, f, *args):
    with pytest.raises(_native.PaiError) as e:
        f(*args)
    assert e.value.status == code


def test_refusals(model):
    vocab = model.cfg["vocab"]
    s = Session(model, 2, 128)
    refused(INVALID, s.beam, [0, 0])  # nothing to select from
    refused(INVALID, s.accept, [[0], [0]], [1, 1])
    s.prefill(np.ones((2, 10), np.int32))
    for bad in ([1], [-2], [0]):
        refused(INVALID, s.verify, [[1], [1]], bad)
    refused(INVALID, s.verify, [[1, vocab], [1, 1]])
    refused(INVALID, s.verify, [[1, 1], [-1, 1]])
    refused(NOMEM, s.verify, np.ones((2, 119), np.int32))
    refused(UNSUPPORTED, s.verify, np.ones((2, 1025), np.int32))
    s.verify(np.ones((2, 118), np.int32))
    s.verify(np.ones((2, 3), np.int32), [-1, -1, 0])
    for path in ([[1], [3]], [[0], [-1]], [[0, 2], [0, 1]], [[2], [0]], [[0, 0], [0, 2]], [[0, 2, 2], [0, 2, 2]]):
        refused(INVALID, s.accept, path, [1, 1])
    refused(INVALID, s.accept, [[0], [0]], [1, vocab])
    assert s.pos == 10
    s.accept([[1], [0]], [1, 1])
    assert s.pos == 11
    refused(INVALID, s.accept, [[1], [0]], [1, 1])  # once only
    refused(INVALID, s.beam, [0, 0])  # the logits are older than the position
    s.verify(np.ones((2, 3), np.int32))
    s.run(1)
    refused(INVALID, s.accept, [[0], [0]], [1, 1])  # a step came between
    s.verify(np.ones((2, 3), np.int32))
    refused(INVALID, lambda: s.beam([0, 0], first=13))
    refused(INVALID, lambda: s.beam([0, 0], pad=vocab))
    s.beam([0, 0], first=12)
    refused(INVALID, s.accept, [[0], [0]], [1, 1])
    refused(INVALID, s.beam, [0, 0])
    s.verify(np.ones((2, 3), np.int32))
    s.reset()
    refused(INVALID, s.accept, [[0], [0]], [1, 1])
    s.verify(np.ones((2, 3), np.int32))  # without a committed position
    s.accept([[0, 1], [0, 1]], [1, 1])
    assert s.pos == 2
    s.close()


def test_operators_on_the_session_view(model):
    """The view addresses the rows that pai_b200_session_write_kv fills."""
    cfg = model.cfg
    s = Session(model, 2, 128)
    kv = s.kv_view()
    assert (kv.n_layer, kv.n_seq, kv.kv_heads, kv.head_dim, kv.page_tokens) == (
        cfg["n_layer"], 2, cfg["n_head_kv"], cfg["head_dim"], 128)
    rng = np.random.default_rng(1)
    rows = rng.standard_normal((kv.kv_heads, 5, kv.head_dim)).astype(np.float16)
    s.write_kv(1, 1, rows, -rows)
    whole = kv.n_layer * kv.layer_stride
    host = np.empty(whole, np.float16)
    for ptr, want in ((kv.k, rows), (kv.v, -rows)):
        _native.check(_native.load().pai_b200_memcpy_d2h(model.dev.ctx, host.ctypes.data, ptr, host.nbytes), "d2h")
        model.dev.sync()
        for h in range(kv.kv_heads):
            at = kv.layer_stride + kv.page_stride + h * kv.head_stride
            got = host[at:at + 5 * kv.head_dim].reshape(5, -1)
            np.testing.assert_array_equal(got, want[h])
    s.close()
