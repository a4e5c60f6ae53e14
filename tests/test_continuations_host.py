"""Operators for several continuations of a prompt: what needs no GPU.

Every refusal happens before the context is touched, so the calls here get
a block of zeroed memory in its place. The page arithmetic that all the
kernels share (kv_view.cuh) is compiled for the host and compared with the
formula of the header, holes and absurd lengths among its inputs.
"""
import ctypes as C
import os
import random
import shutil
import subprocess

import pytest

from prosperoai_b200 import _native
from prosperoai_b200._native import KvView

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, UNSUPPORTED, MISMATCH = -1, -3, -6
CTX = C.create_string_buffer(4096)  # stands where a context would: refused calls do not read it
A = 0x10000                         # an aligned address that no refused call follows


def view(**changes):
    kv = KvView.of(A, A, n_layer=2, n_seq=4, kv_heads=2, head_dim=128, page_tokens=16, n_pages=8, table=A, max_pages=3)
    for name, value in changes.items():
        setattr(kv, name, value)
    return kv


VIEW_REFUSALS = [
    (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(k=A + 8), INVALID), (dict(v=A + 2), INVALID),
    (dict(n_layer=0), INVALID), (dict(n_seq=0), INVALID), (dict(kv_heads=0), INVALID), (dict(head_dim=0), INVALID),
    (dict(page_tokens=0), INVALID), (dict(n_pages=0), INVALID), (dict(max_pages=0), INVALID),
    (dict(layer_stride=7), INVALID), (dict(page_stride=12), INVALID), (dict(head_stride=16 * 128 + 4), INVALID),
    (dict(head_stride=15 * 128), MISMATCH), (dict(head_dim=100), UNSUPPORTED),
    (dict(head_dim=264, head_stride=16 * 264), UNSUPPORTED),
    (dict(table=None), INVALID), (dict(table=None, max_pages=1, n_pages=3), INVALID), (dict(n_seq=1025), UNSUPPORTED),
    (dict(max_pages=1 << 28), INVALID), (dict(max_pages=1 << 22, n_seq=1024), UNSUPPORTED),
]


def calls(kv):
    L = _native.load()
    r = C.byref(kv) if kv is not None else None
    return {
        "append": lambda ctx=CTX, layer=0, h=4, rows=5, most=3, lens=A, off=A, qkv=A, cos=A, sin=A, top=9, q=A:
            L.pai_b200_rope_append_f16kv(ctx, r, layer, h, rows, most, lens, off, None, qkv, cos, sin, top, q),
        "attn": lambda ctx=CTX, layer=0, h=4, rows=5, most=3, lens=A, off=A, mask=None, q=A, out=A:
            L.pai_b200_attn_tree_f16kv(ctx, r, layer, h, rows, most, lens, off, mask, q, out),
        "accept": lambda ctx=CTX, most=4, lens=A, path=A, n=A, out=A:
            L.pai_b200_kv_accept_f16(ctx, r, most, lens, path, n, out),
        "fork": lambda ctx=CTX, lens=A, table=2 * A, lens_out=A, granted=A:
            L.pai_b200_kv_fork_f16(ctx, r, 0, lens, None, None, table, lens_out, granted),
    }


@pytest.mark.parametrize("op", ["append", "attn", "accept", "fork"])
@pytest.mark.parametrize("changes,status", VIEW_REFUSALS)
def test_cache_view_refusals(op, changes, status):
    assert calls(view(**changes))[op]() == status
    assert _native.load().pai_b200_last_error()


@pytest.mark.parametrize("op", ["append", "attn", "accept", "fork"])
def test_null_context_and_view(op):
    assert calls(view())[op](ctx=None) == INVALID
    assert calls(None)[op]() == INVALID


@pytest.mark.parametrize("op", ["append", "attn"])
@pytest.mark.parametrize("args,status", [
    (dict(layer=2), INVALID), (dict(h=0), INVALID), (dict(h=5), INVALID), (dict(h=8192), INVALID), (dict(rows=0), INVALID),
    (dict(rows=1 << 31), INVALID), (dict(most=0), INVALID), (dict(most=1025), UNSUPPORTED), (dict(lens=None), INVALID),
    (dict(off=None), INVALID), (dict(q=None), INVALID), (dict(q=A + 4), INVALID)])
def test_node_refusals(op, args, status):
    assert calls(view())[op](**args) == status


@pytest.mark.parametrize("op,args,status", [
    ("append", dict(qkv=None), INVALID), ("append", dict(cos=None), INVALID), ("append", dict(sin=A + 8), INVALID),
    ("append", dict(qkv=A + 8), INVALID), ("append", dict(top=0), INVALID), ("attn", dict(out=None), INVALID),
    ("attn", dict(out=A + 8), INVALID), ("attn", dict(mask=A + 4), INVALID), ("accept", dict(most=0), INVALID),
    ("accept", dict(most=1025), UNSUPPORTED), ("accept", dict(path=None), INVALID), ("accept", dict(n=None), INVALID),
    ("accept", dict(lens=None), INVALID), ("accept", dict(out=None), INVALID), ("fork", dict(lens=None), INVALID),
    ("fork", dict(table=None), INVALID), ("fork", dict(lens_out=None), INVALID), ("fork", dict(granted=None), INVALID),
    ("fork", dict(table=A + 4 * 11), INVALID), ("fork", dict(table=A - 4 * 11), INVALID)])
def test_argument_refusals(op, args, status):
    assert calls(view())[op](**args) == status


def test_attention_takes_head_dim_64_and_128():
    assert calls(view(head_dim=96, head_stride=16 * 96))["attn"]() == UNSUPPORTED


def test_fork_without_table_takes_32_sequences():
    assert calls(view(table=None, max_pages=1, n_seq=33, n_pages=33))["fork"]() == UNSUPPORTED


@pytest.mark.parametrize("args,status", [
    (dict(ctx=None), INVALID), (dict(logits=None), INVALID), (dict(scores=None), INVALID), (dict(out=None), INVALID),
    (dict(prompts=0), INVALID), (dict(beams=0), INVALID), (dict(vocab=0), INVALID), (dict(n_out=0), INVALID),
    (dict(stride=99), MISMATCH), (dict(pad=-1), INVALID), (dict(pad=100), INVALID), (dict(beams=65), UNSUPPORTED),
    (dict(n_out=65), UNSUPPORTED), (dict(prompts=65536), UNSUPPORTED), (dict(vocab=1 << 26, stride=1 << 26), UNSUPPORTED),
    (dict(logits=A + 2), INVALID)])
def test_beam_refusals(args, status):
    a = dict(ctx=CTX, prompts=1, beams=4, vocab=100, logits=A, stride=100, scores=A, pad=0, n_out=4, out=A)
    a.update(args)
    assert _native.load().pai_b200_beam_select_f32(a["ctx"], a["prompts"], a["beams"], a["vocab"], a["logits"], a["stride"],
                                                   a["scores"], None, a["pad"], a["n_out"], a["out"], A, A) == status


PROGRAM = r"""
#include <cstdio>
#include <vector>
#include "kernels/kv_view.cuh"
extern "C" pai_status_t b200_fail(pai_status_t st, const char *, ...) { return st; }
extern "C" pai_status_t b200_cuda(int, const char *) { return 0; }
int main() {
  int n;
  while (std::scanf("%d", &n) == 1) {
    KvDev c{};
    int paged;
    unsigned long long page_stride;
    std::scanf("%d %u %u %u %u %u %llu", &paged, &c.n_seq, &c.hd, &c.page_tokens, &c.n_pages, &c.max_pages, &page_stride);
    c.page_stride = page_stride;
    std::vector<int32_t> table(c.n_seq * c.max_pages);
    for (auto &e : table) std::scanf("%d", &e);
    if (paged) c.table = table.data();
    for (int i = 0; i < n; i++) {
      unsigned s, pos;
      std::scanf("%u %u", &s, &pos);
      std::printf("%lld\n", (long long)kv_row(c, s, pos));
    }
    int32_t len, off[2];
    unsigned long long rows;
    unsigned most, first;
    std::scanf("%d %d %d %llu %u", &len, &off[0], &off[1], &rows, &most);
    std::printf("%u\n", kv_len(c, &len, 0));
    const unsigned k = kv_nodes(off, 0, rows, most, &first);
    std::printf("%u %u\n", first, k);
  }
}
"""


def test_page_arithmetic(tmp_path):
    nvcc = "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc) and not shutil.which("nvcc"):
        pytest.skip("no nvcc")
    src = tmp_path / "rows.cu"
    src.write_text(PROGRAM)
    subprocess.run([nvcc if os.path.exists(nvcc) else "nvcc", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a",
                    "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "prosperoai_b200", "csrc"), str(src), "-o",
                    str(tmp_path / "rows")], check=True)
    r = random.Random(5)
    given, want = [], []
    for _ in range(200):
        paged = r.random() < 0.8
        n_seq, hd, tokens = r.randint(1, 4), r.choice([8, 64, 128]), r.choice([1, 7, 16, 100, 1 << 20])
        max_pages = r.randint(1, 5) if paged else 1
        n_pages = r.randint(1, 6) if paged else n_seq
        stride = r.choice([tokens * hd, 1 << 34])
        table = [r.choice([r.randint(0, n_pages - 1)] * 4 + [-1, n_pages, -(1 << 31), (1 << 31) - 1]) for _ in range(n_seq * max_pages)]
        asks = [(r.randrange(n_seq), r.choice([0, tokens - 1, tokens, r.randrange(max_pages * tokens + 3), (1 << 32) - 1]))
                for _ in range(8)]
        given.append(f"{len(asks)} {int(paged)} {n_seq} {hd} {tokens} {n_pages} {max_pages} {stride}")
        given.append(" ".join(map(str, table)))
        given += [f"{s} {p}" for s, p in asks]
        for s, p in asks:
            page = -1 if p // tokens >= max_pages else table[s * max_pages + p // tokens] if paged else s
            want.append(str(page * stride + p % tokens * hd if 0 <= page < n_pages else -1))
        length, a, b = r.choice([-5, 0, 3, 1 << 30]), r.choice([-1, 0, 2, 50]), r.choice([-3, 0, 2, 9, 60, (1 << 31) - 1])
        rows, most = r.choice([1, 5, 55]), r.choice([1, 4, 64])
        given.append(f"{length} {a} {b} {rows} {most}")
        want.append(str(min(max(length, 0), max_pages * tokens)))
        none = a < 0 or b <= a or a >= rows
        want.append("0 0" if none else f"{a} {min(b - a, rows - a, most)}")
    got = subprocess.run([str(tmp_path / "rows")], input="\n".join(given), capture_output=True, text=True, check=True).stdout
    assert got.split("\n")[:-1] == want


def test_session_refusals_without_a_session():
    L = _native.load()
    words = (C.c_int32 * 8)()
    floats = (C.c_float * 8)()
    assert L.pai_b200_session_kv_view(None, C.byref(KvView())) == INVALID
    assert L.pai_b200_session_verify(None, words, None, 1, words) == INVALID
    assert L.pai_b200_session_accept(None, words, 1, words) == INVALID
    assert L.pai_b200_session_beam(None, floats, None, 0, 0, floats, words, words) == INVALID
