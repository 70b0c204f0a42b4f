"""The sampler's chunks and the layout of its workspace (cuda_inf_amd/csrc/sample_shape.h):
parts lie where 16 bytes can be read at once, apart from each other, and within the stated
size for a batch and every smaller one."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r"""
#include <cstdio>
#include <initializer_list>
#include "sample_shape.h"
using namespace cia;
int main() {
  for (int V : {1, 60, 8192, 16384, 16385, 20000, 24576, 24577, 50001, 65536, 131072, 262143, 262144, 262145, 300000,
                1 << 20, 1 << 22}) {
    int64_t least = 0;
    for (int B = 0; B <= 2100; B++) {
      const SampleSpace s = sample_space(B, V);
      // (rows of one large chunk need none)
      const int64_t n = V > kMaxChunk ? (int64_t)B * s.chunks : 0;
      if (s.bins % 16 || s.tops % 16 || s.bins < n * (int64_t)sizeof(ChunkHead) || s.tops - s.bins < n * kBins * 8) {
        std::printf("B=%d V=%d: bins at %lld, tops at %lld\n", B, V, (long long)s.bins, (long long)s.tops);
        return 1;
      }
      if (s.end - s.tops < (s.chunk == kMinChunk ? n * kTop * 8 : 0)) return 2;
      // the chunks are a row, and none is empty
      if ((int64_t)s.chunk * s.chunks < V || (int64_t)s.chunk * (s.chunks - 1) >= V) return 3;
      least = s.end > least ? s.end : least;
      if (sample_space_bytes(B, V) < least) {
        std::printf("B=%d V=%d: %lld of %lld bytes\n", B, V, (long long)sample_space_bytes(B, V), (long long)least);
        return 4;
      }
      // no more than the larger of the layouts of B rows and fewer, and a few bytes
      if (sample_space_bytes(B, V) > least + 16) return 5;
    }
  }
  return 0;
}
"""


def test_workspace_layout(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    src, exe = str(tmp_path / "space.cpp"), str(tmp_path / "space")
    with open(src, "w") as f:
        f.write(SOURCE)
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", os.path.join(ROOT, "cuda_inf_amd", "csrc"), src, "-o", exe], check=True)
    r = subprocess.run([exe], text=True, capture_output=True, timeout=60)
    assert r.returncode == 0, f"assumption {r.returncode}: {r.stdout}"
