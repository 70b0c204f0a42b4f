"""The choice of kernel and shape for the experts' products
(cuda_inf_amd/csrc/moe_shape.h): the sizes that the GPU tests launch reach every one
that a call can."""
import os
import shutil
import subprocess

import numpy as np
import pytest

import ffn_sizes

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FEW, STREAM, TILE = range(3)

SOURCE = r"""
#include <cstdio>
#include <set>
#include <tuple>
#include "moe_shape.h"
using namespace cia;
int main(int argc, char**) {
  if (argc == 1) {  // sizes on stdin
    int up, E, K, N;
    long long P;
    while (std::scanf("%d %lld %d %d %d", &up, &P, &E, &K, &N) == 5) {
      const MoeShape s = moe_shape(up, P, E, K, N);
      std::printf("%d %d %d %d\n", s.kernel, s.a, s.b, s.splits);
    }
    return 0;
  }
  std::set<std::tuple<int, int, int, int, bool>> all;
  for (int up = 0; up < 2; up++)
    for (int E : {1, 2, 4, 7, 16, 32, 60, 128, 256})
      for (long long P : {1, 2, 5, 8, 9, 12, 16, 17, 24, 32, 40, 64, 65, 96, 128, 180, 256, 384, 385, 512, 513, 700,
                          1024, 1025, 1500, 4096, 16384, 16385, 1 << 20})
        for (int K = 128; K <= 32768; K = K < 8448 ? K + 128 : 2 * K)
          for (int N = 128; N <= 32768; N = N < 4096 ? N + 128 : N + 1024) {
            const MoeShape s = moe_shape(up, P, E, K, N);
            all.insert({up, s.kernel, s.a, s.b, s.splits > 1});
            // what the launches assume
            if (s.kernel == kMoeFew && (P > kFewPairs || K > 128 * s.a * s.b)) return 1;
            if (s.kernel == kMoeStream &&
                (P > kStreamPairs || (s.b > 1 && P > 64) || ((K >> 7) + s.splits - 1) / s.splits > kStreamWaves * s.a))
              return 2;
            if (s.splits * P > y_rows(P) || (up && s.splits > 1)) return 3;
            if (s.kernel == kMoeTile && s.splits > K / 128) return 4;
          }
  for (auto& [up, kernel, a, b, split] : all) std::printf("%d %d %d %d %d\n", up, kernel, a, b, split);
}
"""


@pytest.fixture(scope="module")
def shape(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    d = tmp_path_factory.mktemp("moe_shape")
    src, exe = str(d / "shape.cpp"), str(d / "shape")
    with open(src, "w") as f:
        f.write(SOURCE)
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", os.path.join(ROOT, "cuda_inf_amd", "csrc"), src, "-o", exe], check=True)

    def run(sizes=None):
        r = subprocess.run([exe] if sizes is not None else [exe, "all"], text=True, capture_output=True, timeout=60,
                           input="".join("%d %d %d %d %d\n" % s for s in sizes or ()))
        assert r.returncode == 0, f"assumption {r.returncode}"
        return [tuple(map(int, l.split())) for l in r.stdout.splitlines()]

    return run


def launched(up, P, k, E, K, N, rows, kernel, a, b, splits):
    """What a size launches: the kernel's shape, and the code inside it by how many
    rows an expert (a tile) has."""
    yield up, kernel, a, b, int(splits > 1)
    ids = ffn_sizes.pair_ids(P, k, E, rows)
    counts = [P] if ids is None else np.bincount(ids[ids >= 0], minlength=E).tolist()
    for n in filter(None, counts):
        if kernel == TILE:
            if n >= 128:
                yield "tile rows", up, a, 4
            if n % 128:
                yield "tile rows", up, a, (n % 128 + 31) // 32
        if kernel == STREAM:
            for left in range(n, 0, -16 * b):
                yield "stream rows", up, a, b, 4 if b >= 4 and left > 32 else 2 if b >= 2 and left > 16 else 1


def test_the_tests_launch_every_shape(shape):
    need = set(shape())
    need |= {("tile rows", up, nt, n) for up in (0, 1) for nt in (1, 2, 3) for n in (1, 2, 3, 4)}
    need |= {("stream rows", 1, a, b, n) for _, kernel, a, b, _ in shape() if kernel == STREAM
             for n in (1, 2, 4) if n <= b}
    have = set()
    for up, sizes in ((1, ffn_sizes.UP), (0, ffn_sizes.DOWN)):
        got = shape([(up, P, E, K, N) for P, _, E, K, N, _ in sizes])
        for size, s in zip(sizes, got):
            have |= set(launched(up, *size, *s))
    assert not need - have, sorted(map(str, need - have))


def test_what_the_launches_assume(shape):
    assert len(shape()) > 20  # (the assumptions are looked at on the way)
