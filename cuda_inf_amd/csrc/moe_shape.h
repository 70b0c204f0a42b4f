// moe_shape.h -- which kernel, and which of its shapes, the experts' products of a
// call take (moe_int4.hip), by the number of pairs, the experts and the widths.
// Plain C++, so that the CPU tests see what a size launches.
#pragma once

#include <cstdint>

namespace cia {

constexpr int kTileRows = 128;  // rows of a row tile
constexpr int kUnits = 256;     // compute units

// Up to so many pairs a tile's workgroup finds its rows from the ids by itself (which
// saves the plan's launch, 4 us).
constexpr int kOwnPairs = 1024;

// Streams: waves of a workgroup, which split K; pairs, a thread each; the longest K of
// one part, 4 scale groups a wave.
constexpr int kStreamWaves = 8, kStreamPairs = 64 * kStreamWaves;
constexpr int kStreamMaxK = 4 * 8 * 128;
// groups a wave -> row tiles that x leaves registers for
constexpr int stream_mt(int kg) { return kg <= 2 ? 4 : 2; }

// Down of few pairs in one launch
constexpr int kFewPairs = 8;

// The most row tiles P pairs of E experts can make
constexpr int64_t max_tiles(int64_t P, int E) { return P / kTileRows + (P < E ? P : E); }

// Row tiles, about: an expert's last one is partly filled, and with few rows costs
// less.
constexpr double row_tiles(int64_t P, int E) {
  return E > 1 ? (double)P / kTileRows + 0.75 * (double)(P < E ? P : E) : (double)((P + kTileRows - 1) / kTileRows);
}

// Rows of y: P, and room for parts of K where few pairs leave the chip empty
constexpr int64_t y_rows(int64_t P) { return P >= 4096 ? P : (8 * P < 4096 ? 8 * P : 4096); }

// Parts of K of a down launch in tiles: as many as the chip's 512 places hold of
// workgroups of 128 columns, each part of 4 groups or more.
constexpr int k_splits(int64_t P, int E, int H, int F) {
  int64_t n = (int64_t)(512.0 / (row_tiles(P, E) * ((H + 127) / 128)));
  n = n < y_rows(P) / P ? n : y_rows(P) / P;
  n = n < F / 512 ? n : F / 512;
  return n < 1 ? 1 : (int)n;
}

// Whether the weights are streamed rather than multiplied in tiles: while experts
// have 2 (up), 1.5 (down) rows on average, or pairs are few.  Calls in us, streamed /
// in tiles: 4 of 32 experts of 1792, H = 2048, up 16 tokens 21.0 / 24.5, 20 26.9 /
// 25.0, 40 30.6 / 30.4, down 12 15.6 / 16.7, 20 23.7 / 18.1; 8 of 128 of 1536, H =
// 4096, up 8 66 / 76, 32 119 / 114, down 24 64 / 67, 64 90 / 87; 2 of 8 of 2048, H =
// 1024, up 32 9.7 / 10.5, 40 13.3 / 11.1, down 4 8.5 / 8.5, 12 13.7 / 11.0; the dense
// form of 7168, H = 2048, up 32 rows 11.5 / 12.3, 64 16.1 / 14.6, down 16 12.1 / 13.8,
// 24 14.4 / 13.9.  (Down takes a K of two parts as well.)
constexpr bool streams(bool up, int64_t P, int E, int K) {
  const int64_t most = up ? 2 * (int64_t)E : 3 * (int64_t)E / 2, few = up ? 64 : 16;
  return P <= (most > few ? most : few) && K <= (up ? 1 : 2) * kStreamMaxK;
}

// Column tiles a wave, of 1, 2 and 3: a workgroup's time goes with kNT + 3, and the
// call's with its rounds of the 512 workgroups that the chip holds, of which the
// first is never less than nine tenths.  (Of 125 sizes of 7 layers the choice is 0.6 %
// slower on average than the best of the three, always 2 would be 5 %, always 1 21 %;
// 4 of 32 experts of 1792, H = 2048, in us: 45 tokens down 25.7 / 21.3 / 24.7, 220 up
// 62.4 / 47.0 / 50.8.)
constexpr int tile_nt(int64_t P, int E, int nv, int splits) {
  int best = 1;
  double least = 0.0;
  for (int nt = 1; nt <= 3; nt++) {
    const double rounds = row_tiles(P, E) * ((nv + 64 * nt - 1) / (64 * nt)) * splits / 512.0;
    const double t = (rounds < 0.9 ? 0.9 : rounds) * (nt + 3);
    if (nt == 1 || t < least) {
      best = nt;
      least = t;
    }
  }
  return best;
}

enum MoeKernel { kMoeFew, kMoeStream, kMoeTile };
struct MoeShape {
  MoeKernel kernel;
  int splits;  // parts of K, each into rows of y of its own
  int a;       // few: waves; stream: scale groups a wave; tile: column tiles a wave
  int b;       // few: scale groups a wave; stream: row tiles; tile: 1 with a plan
};

// P pairs of E experts, K inputs, N outputs (up: of each of the two)
constexpr MoeShape moe_shape(bool up, int64_t P, int E, int K, int N) {
  if (!up && P <= kFewPairs && K <= kStreamMaxK)
    return {kMoeFew, 1, K <= 1024 ? 8 : 16, K <= 2048 ? 1 : 2};
  if (streams(up, P, E, K)) {
    const int splits = up ? 1 : (K + kStreamMaxK - 1) / kStreamMaxK;
    const int part = ((K >> 7) + splits - 1) / splits;  // groups
    const int kg = part <= 8 ? 1 : part <= 16 ? 2 : 4;
    // 16 rows at a time where experts hardly have more; up to 64 rows of up's few
    // pairs of few experts
    return {kMoeStream, splits, kg, up && P > 8 * (int64_t)E ? stream_mt(kg) : 1};
  }
  const int splits = up ? 1 : k_splits(P, E, N, K);
  return {kMoeTile, splits, tile_nt(P, E, up ? 2 * N : N, splits), P > kOwnPairs};
}

}  // namespace cia
