"""Memory of a session's prefill, drafts and beams, on the CPU.

b200_model.c is compiled as it is, with host memory in the place of device memory and kernels that do nothing, so that
any allocation can be made to fail.
"""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, INVALID, NOMEM = 0, -1, -2

# The entry points that the session's host code calls. Allocation number `fail_at` fails (0: none).
STUBS = r"""
#include <stdarg.h>
#include <stdint.h>
#include <stdlib.h>
#include <string.h>
uint64_t fail_at, calls, bytes_held;
int b200_fail(int st, const char *fmt, ...) { (void)fmt; return st; }
static int take(uint64_t bytes, void **out) {
  *out = NULL;
  if (++calls == fail_at) return -2;
  *out = calloc(1, bytes ? bytes : 1);
  bytes_held += bytes;
  return 0;
}
int pai_b200_alloc(void *c, uint64_t bytes, void **out) { (void)c; return take(bytes, out); }
int pai_b200_host_alloc(void *c, uint64_t bytes, void **out) { (void)c; return take(bytes, out); }
int pai_b200_free(void *c, void *p) { (void)c; free(p); return 0; }
int pai_b200_host_free(void *c, void *p) { (void)c; free(p); return 0; }
static int copy(void *d, const void *s, uint64_t n) { if (n) memcpy(d, s, n); return 0; }
int pai_b200_memcpy_h2d(void *c, void *d, const void *s, uint64_t n) { (void)c; return copy(d, s, n); }
int pai_b200_memcpy_d2h(void *c, void *d, const void *s, uint64_t n) { (void)c; return copy(d, s, n); }
int pai_b200_memcpy_d2d(void *c, void *d, const void *s, uint64_t n) { (void)c; return copy(d, s, n); }
int pai_b200_memset(void *c, void *d, int v, uint64_t n) { (void)c; memset(d, v, n); return 0; }
uint64_t b200_ctx_wait_ns(void *c) { (void)c; return 1; }
#define NOTHING(name) int name(void) { return 0; }
NOTHING(pai_b200_sync) NOTHING(b200_decode_launch) NOTHING(b200_launch_embed) NOTHING(b200_launch_rmsnorm_xq) NOTHING(b200_launch_gemv)
NOTHING(b200_launch_gemv_norm) NOTHING(b200_launch_argmax) NOTHING(b200_launch_xprep) NOTHING(pai_b200_gemm_f32)
NOTHING(pai_b200_kv_accept_f16) NOTHING(pai_b200_kv_fork_f16) NOTHING(pai_b200_beam_select_f32)
NOTHING(pai_b200_graph_begin) NOTHING(pai_b200_graph_launch) NOTHING(pai_b200_graph_destroy)
NOTHING(b200_graph_destroy) NOTHING(b200_decode_plan_destroy) NOTHING(b200_tp_mark_failed)
int pai_b200_graph_end(void *c, void **g) { (void)c; *g = NULL; return 0; }
"""

PROGRAM = r"""
#include <stdio.h>
#include "host/b200_model.c"
extern uint64_t fail_at, calls, bytes_held;
enum { B = 2, E = 64, V = 96 };
static pai_b200_session_t *session(pai_b200_model_t *m) {
  pai_b200_session_t *s = calloc(1, sizeof(*s));
  memset(m, 0, sizeof(*m));
  m->cfg.n_embd = E, m->cfg.vocab = V, m->cfg.head_dim = 64, m->cfg.wtype = m->cfg.etype = PAI_B200_Q8_0;
  m->tp = 1, m->hl = m->hkl = 1, m->k_o = 64, m->n_qkv = 192, m->ffl = 128, m->vl = V; /* no layers */
  s->m = m, s->batch = B, s->max_ctx = 256;
  s->x = calloc(B * E, 4), s->logits = calloc(B * V, 4), s->tok_in = calloc(64, 1), s->tok_out = calloc(64, 1);
  s->dpos = calloc(64, 1), s->htok = calloc(64, 1), s->kc = calloc(1, 64), s->vc = calloc(1, 64);
  s->xq_buf = calloc(1, b200_xq_bytes(B, E) + 64);
  s->xq_e = b200_xq_view(s->xq_buf, B, E);
  s->beam_ready = 1, s->pos = 3;
  return s;
}
static int call(pai_b200_session_t *s, const char *what) {
  int32_t tok[B * 4] = {1, 2, 3, 4, 5, 6, 7, 8}, next[B * 4], parents[B], tokens[B];
  float score[B] = {0, 0};
  s->beam_ready = 1;
  switch (what[0]) {
    case 'p': return pai_b200_session_prefill(s, tok, 4, next);
    case 'v': return pai_b200_session_verify(s, tok, NULL, 4, next);
    default: return pai_b200_session_beam(s, score, NULL, 0, 0, score, parents, tokens);
  }
}
int main(int argc, char **argv) {
  (void)argc;
  pai_b200_model_t m;
  pai_b200_session_t *s = session(&m);
  if (argv[1][0] == 'l') { /* the layers run between a verification and its acceptance */
    int32_t path[B] = {0, 0}, next[B] = {1, 1};
    s->plan = (void *)s;
    const int a = call(s, "verify"), b = pai_b200_session_accept(s, path, 1, next);
    const int c = call(s, "verify"), d = pai_b200_session_run_layers(s, atoi(argv[2]));
    const int e = pai_b200_session_accept(s, path, 1, next);
    printf("%d %d %d %d %d\n", a, b, c, d, e);
    return 0;
  }
  fail_at = strtoull(argv[2], NULL, 10);
  const int first = call(s, argv[1]);
  const int second = call(s, argv[1]);
  printf("%d %d %llu %llu\n", first, second, (unsigned long long)calls, (unsigned long long)bytes_held);
  return 0;
}
"""


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    if not shutil.which("gcc"):
        pytest.skip("no gcc")
    at = tmp_path_factory.mktemp("session")
    (at / "stubs.c").write_text(STUBS)
    (at / "program.c").write_text(PROGRAM)
    inc = ["-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "prosperoai_b200", "csrc")]
    subprocess.run(["gcc", "-std=c11", "-O1", "-g", "-w", *inc, "-c", str(at / "stubs.c"), "-o", str(at / "stubs.o")], check=True)
    subprocess.run(["gcc", "-std=c11", "-O1", "-g", "-w", *inc, str(at / "program.c"), str(at / "stubs.o"), "-lm",
                    "-Wl,--unresolved-symbols=ignore-all", "-o", str(at / "program")], check=True)

    def go(what, fail_at):
        p = subprocess.run([str(at / "program"), what, str(fail_at)], capture_output=True, text=True)
        assert p.returncode == 0, f"{what} with allocation {fail_at} failing ended with {p.returncode}"
        return [int(x) for x in p.stdout.split()]

    return go


@pytest.mark.parametrize("what", ["prefill", "verify", "beam"])
def test_a_call_after_a_failed_allocation(run, what):
    """Whichever allocation fails, the call says so and the next one has everything it works on."""
    first, second, allocations, _ = run(what, 0)
    assert (first, second) == (OK, OK) and allocations > 0
    for n in range(1, allocations + 1):
        first, second, made, _ = run(what, n)
        assert (first, second) == (NOMEM, OK)
        assert made == allocations + 1  # the failed one again, nothing twice


def test_beams_hold_their_staging_only(run):
    """A selection works on arrays of batch entries: none of the row arrays of a prefill or a verification."""
    assert run("beam", 0)[2] == 2
    assert run("beam", 0)[3] < 2 << 20 < run("verify", 0)[3]


def test_layers_that_run_alone_overwrite_verified_nodes(run):
    """pai_b200_session_run_layers appends the step's K/V where the first node's lie: the nodes cannot be accepted any more."""
    assert run("layers", 0) == [OK] * 5
    assert run("layers", 1) == [OK] * 4 + [INVALID]
