"""Parts of tree attention's units (attn_tree.cuh): what the joining kernel may read.

An entry that the cut of the work makes is taken as it is. One that no CTA wrote, because a wait had run out before,
holds whatever the scratch held: it may name no slot outside the scratch, and no more parts than there are CTAs.
"""
import os
import random
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include "kernels/attn_tree.cuh"
extern "C" pai_status_t b200_fail(pai_status_t st, const char *, ...) { return st; }
extern "C" pai_status_t b200_cuda(int, const char *) { return 0; }
extern "C" int b200_ctx_device(pai_b200_ctx_t *) { return 0; }
extern "C" int b200_ctx_pdl(pai_b200_ctx_t *) { return 0; }
extern "C" void *b200_ctx_stream(pai_b200_ctx_t *) { return nullptr; }
int main() {
  unsigned parts, first, slots;
  while (std::scanf("%u %u %u", &parts, &first, &slots) == 3) {
    const unsigned n = unit_parts(parts, first, slots);
    std::printf("%u", n);
    for (unsigned q = 0; q < n; q++) std::printf(" %u", part_slot(first, q));
    std::printf("\n");
  }
}
"""


@pytest.fixture(scope="module")
def parts(tmp_path_factory):
    nvcc = "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc) and not shutil.which("nvcc"):
        pytest.skip("no nvcc")
    at = tmp_path_factory.mktemp("parts")
    (at / "parts.cu").write_text(PROGRAM)
    subprocess.run([nvcc if os.path.exists(nvcc) else "nvcc", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a",
                    "--expt-relaxed-constexpr", "-I", os.path.join(ROOT, "include"), "-I",
                    os.path.join(ROOT, "prosperoai_b200", "csrc"), str(at / "parts.cu"), "-o", str(at / "parts")], check=True)

    def run(asks):
        text = "\n".join(" ".join(map(str, a)) for a in asks)
        out = subprocess.run([str(at / "parts")], input=text, capture_output=True, text=True, check=True).stdout
        return [[int(x) for x in line.split()] for line in out.splitlines()]

    return run


def test_entries_of_the_cut(parts):
    """Units that CTAs c0 .. c1 share: the first one's first or last part, the first parts of the others."""
    asks, want = [], []
    for grid in (2, 5, 147, 148):
        for c0 in range(0, grid, max(1, grid // 7)):
            for c1 in {c0, c0 + 1, (c0 + grid) // 2, grid - 1}:
                if not c0 <= c1 < grid:
                    continue
                for last in (0, 1):
                    asks.append((c1 - c0 + 1, 2 * c0 + last, 2 * grid))
                    want.append([c1 - c0 + 1, 2 * c0 + last] + [2 * c for c in range(c0 + 1, c1 + 1)])
    assert parts(asks) == want


def test_entries_that_nothing_wrote(parts):
    r = random.Random(3)
    odd = [0, 1, 2, 147, 148, 149, 295, 296, 297, 0x3F800000, 0x7FC00000, 0x7FFFFFFF, 0x80000000, 0xC2F60000, 0xFFFFFFFE,
           0xFFFFFFFF]
    asks = [(a, b, s) for a in odd for b in odd for s in (2, 10, 296)]
    asks += [(r.getrandbits(32) >> r.randrange(32), r.getrandbits(32) >> r.randrange(32), 2 * r.randint(1, 148)) for _ in range(3000)]
    for (a, b, slots), got in zip(asks, parts(asks)):
        n, named = got[0], got[1:]
        assert n in (0, a) and len(named) == n <= slots // 2
        assert all(x < slots for x in named) and len(set(named)) == n
