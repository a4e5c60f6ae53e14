"""Contexts on a caller's stream: operators in order with the other work of that stream, without a wait on the host."""
import ctypes as C

import numpy as np
import pytest

from prosperoai_b200 import _native
from prosperoai_b200.api import Device, KvView, Model, PaiError, Session

INVALID, INIT = -1, -8
BEAMS, VOCAB, STEPS = 4, 30011, 12


def test_refusals_without_a_device():
    import torch
    L = _native.load()
    assert L.pai_b200_init_on_stream(0, None, None) == INVALID
    assert L.pai_b200_stream(None) is None
    if not torch.cuda.is_available():
        ctx = C.c_void_p()
        assert L.pai_b200_init_on_stream(0, None, C.byref(ctx)) == INIT and not ctx.value


class Loop:
    """Selection, fork and attention on tensors that torch fills just before and reads just behind."""

    def __init__(self, dev, torch):
        self.dev, self.torch = dev, torch
        g = torch.Generator(device="cuda").manual_seed(7)
        i32 = dict(dtype=torch.int32, device="cuda")
        self.logits = torch.zeros(BEAMS, VOCAB, device="cuda")
        self.scores = torch.zeros(BEAMS, device="cuda")
        self.out = [torch.zeros(BEAMS, device="cuda"), torch.zeros(BEAMS, **i32), torch.zeros(BEAMS, **i32)]
        self.k = torch.randn(1, BEAMS, 1, 64, 64, generator=g, device="cuda").half()
        self.v = torch.randn(1, BEAMS, 1, 64, 64, generator=g, device="cuda").half()
        self.lens, self.off = torch.full((BEAMS,), 40, **i32), torch.arange(BEAMS + 1, **i32)
        self.lens_out, self.granted = torch.zeros(BEAMS, **i32), torch.zeros(BEAMS, **i32)
        self.q, self.att = torch.zeros(BEAMS, 2, 64, device="cuda"), torch.zeros(BEAMS, 2, 64, device="cuda")
        self.view = KvView.of(self.k.data_ptr(), self.v.data_ptr(), n_layer=1, n_seq=BEAMS, kv_heads=1, head_dim=64, page_tokens=64,
                              n_pages=BEAMS)
        self.a = torch.randn(2048, 2048, generator=g, device="cuda")
        self.source = torch.randn(STEPS, BEAMS, VOCAB, generator=g, device="cuda")
        self.queries = torch.randn(STEPS, BEAMS, 2, 64, generator=g, device="cuda")

    def step(self, i, slow=True):
        if slow:  # keeps the stream busy, so that a kernel out of order would read what was there before
            for _ in range(3):
                self.a = (self.a @ self.a).clamp_(-1, 1)
        self.logits.copy_(self.source[i])
        self.q.copy_(self.queries[i])
        for x in (*self.out, self.lens_out, self.granted, self.att):
            x.fill_(-7)
        self.ops()
        return [x.clone() for x in (*self.out, self.lens_out, self.att, self.k, self.v)]

    def ops(self):
        at = [x.data_ptr() for x in self.out]
        self.dev.beam_select(1, BEAMS, VOCAB, self.logits.data_ptr(), VOCAB, self.scores.data_ptr(), None, 0, BEAMS, *at)
        self.dev.kv_fork(self.view, 0, self.lens.data_ptr(), at[1], None, None, self.lens_out.data_ptr(), self.granted.data_ptr())
        self.dev.attn_tree(self.view, 0, 2, BEAMS, 1, self.lens_out.data_ptr(), self.off.data_ptr(), None, self.q.data_ptr(),
                           self.att.data_ptr())


def same(a, b):
    for x, y in zip(a, b):
        np.testing.assert_array_equal(x.cpu().numpy(), y.cpu().numpy())


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["side", "default"])
def test_in_order_with_torch(which):
    import torch
    torch.cuda.synchronize()
    # each step waited for, by a context with a stream of its own
    dev = Device(0)
    loop, want = Loop(dev, torch), []
    for i in range(STEPS):
        torch.cuda.synchronize()
        loop.logits.copy_(loop.source[i])
        loop.q.copy_(loop.queries[i])
        torch.cuda.synchronize()
        loop.ops()
        dev.sync()
        want.append([x.clone() for x in (*loop.out, loop.lens_out, loop.att, loop.k, loop.v)])
    torch.cuda.synchronize()
    dev.close()
    # all steps enqueued, waited for once
    stream = torch.cuda.Stream() if which == "side" else torch.cuda.default_stream()
    with torch.cuda.stream(stream):
        dev = Device(0, stream=stream.cuda_stream)
        assert dev.stream == stream.cuda_stream
        loop = Loop(dev, torch)
        got = [loop.step(i) for i in range(STEPS)]
    stream.synchronize()
    for a, b in zip(got, want):
        same(a, b)
    dev.sync()
    dev.close()
    with torch.cuda.stream(stream):  # the stream is the caller's, and stays
        assert int(torch.ones(5, device="cuda").sum()) == 5


@pytest.mark.gpu
def test_captured_with_torch():
    import torch
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        dev = Device(0, stream=stream.cuda_stream)
        loop = Loop(dev, torch)
        start = [loop.k.clone(), loop.v.clone()]
        want = [loop.step(i, slow=False) for i in range(3)]  # the first sizes the scratch
        g = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(g, stream=stream):
            loop.ops()
        loop.k.copy_(start[0])
        loop.v.copy_(start[1])
        for i in range(3):
            loop.logits.copy_(loop.source[i])
            loop.q.copy_(loop.queries[i])
            g.replay()
            same([x.clone() for x in (*loop.out, loop.lens_out, loop.att, loop.k, loop.v)], want[i])
        # scratch that would have to grow while the stream is captured: refused, and the capture is still sound
        big = torch.zeros(64, 40000, device="cuda")
        more = [torch.zeros(64, device="cuda"), torch.zeros(64, dtype=torch.int32, device="cuda"),
                torch.zeros(64, dtype=torch.int32, device="cuda")]
        fresh = Device(0, stream=stream.cuda_stream)
        g2 = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(g2, stream=stream):
            loop.ops()
            with pytest.raises(PaiError):
                fresh.beam_select(1, 64, 40000, big.data_ptr(), 40000, big.data_ptr(), None, 0, 64, *(x.data_ptr() for x in more))
        g2.replay()
        stream.synchronize()
        del g, g2
    fresh.close()
    dev.close()


@pytest.mark.gpu
def test_a_session_needs_a_stream_that_can_be_captured():
    import torch
    from test_gpu_model import SMALL
    from oracle import py_oracle as po
    cfg = dict(SMALL, wtype=po.Q8_0)
    prompt = np.arange(12, dtype=np.int32).reshape(1, -1)
    tokens = []
    for stream in (None, torch.cuda.Stream()):
        dev = Device(0) if stream is None else Device(0, stream=stream.cuda_stream)
        m = Model(dev, cfg)
        m.synthesize(11)
        s = Session(m, 1, 128)
        tokens.append([int(s.prefill(prompt)[0])] + [int(s.step(np.array([t], np.int32))[0]) for t in range(3)])
        s.close()
        m.close()
        dev.close()
    assert tokens[0] == tokens[1]
    dev = Device(0, stream=0)
    m = Model(dev, cfg)
    m.synthesize(11)
    with pytest.raises(PaiError):
        Session(m, 1, 128)
    dev.sync()
    m.close()
    dev.close()
