// sample_shape.h -- how the sampler cuts its rows into chunks, and what its workspace
// holds (sample.hip).  Plain C++, so that the CPU tests see what a size is given.
#pragma once

#include <cstdint>

namespace cia {

constexpr int kBins = 672;  // of a chunk: 42 octaves, 16 bins each
constexpr int kMinChunk = 8192;
constexpr int kMaxChunk = 2 * kMinChunk;
constexpr int kTop = 512;  // tokens of a smaller chunk that it puts out by themselves, at most

// of a chunk of a row
struct ChunkHead {
  double n;      // ceil of its largest x; -inf: no token, inf: logits of +inf
  float top;     // its largest logit
  uint32_t idx;  // the first token that has it
  int depth;     // bins whose tokens are in its top
  int listed;    // tokens of its top
};

// Chunks of 16384 logits where there are more than 1024 of them, or a row has more than 32 of
// the smaller ones; else of 8192, with their tops: of the largest tokens the choice
// mostly falls on, the row need not be read again.  us with 8192 / 16384, of rows of 131 072:
//   rows (chunks of 16384)         1 (8)   32 (256)     64 (512)   128 (1024)    256 (2048)
//   top-k and top-p          18.5 / 26.7  22.8 / 31.4  27.7 / 34.8  35.4 / 40.9   55.0 / 57.6
//   top-p, broad: read again 27.4 / 29.4  55.2 / 50.4  59.4 / 53.4  69.8 / 61.7   90.7 / 74.5
// (Which filters a row has is known on the device alone.  At 1024 chunks narrow rows gain 13 %
// by the smaller ones and broad rows lose as much; below it narrow rows gain more, above it
// broad rows lose more.)
constexpr int kMostTopped = 1024;
constexpr int row_chunks(int V, int chunk) { return (V + chunk - 1) / chunk; }
constexpr int sample_chunk(int B, int V) {
  return (int64_t)B * row_chunks(V, kMaxChunk) > kMostTopped || V > 32 * kMinChunk ? kMaxChunk : kMinChunk;
}

// Where a workspace of B rows has its parts, in bytes from its start: the heads of all chunks
// of all rows, [kBins] uint64 of each, and of smaller chunks [kTop] uint64 of each.  Rows of up
// to kMaxChunk are read by their own workgroups, which need none of it.
struct SampleSpace {
  int chunk, chunks;  // logits of a chunk, chunks of a row
  int64_t bins, tops, end;
};
constexpr SampleSpace sample_space(int B, int V) {
  const int chunk = sample_chunk(B, V), chunks = row_chunks(V, chunk);
  const int64_t n = V > kMaxChunk ? (int64_t)B * chunks : 0;
  // (bins are read 16 bytes at a time)
  const int64_t bins = (n * (int64_t)sizeof(ChunkHead) + 15) & ~(int64_t)15;
  const int64_t tops = bins + n * kBins * 8;
  return SampleSpace{chunk, chunks, bins, tops, tops + (chunk == kMinChunk ? n * kTop * 8 : 0)};
}

// Bytes for B rows of V or fewer: a smaller batch may have smaller chunks.
constexpr int64_t sample_space_bytes(int B, int V) {
  const int topped = kMostTopped / row_chunks(V, kMaxChunk);  // rows
  const int64_t all = sample_space(B, V).end, fewer = sample_space(B < topped ? B : topped, V).end;
  return 16 + (all > fewer ? all : fewer);
}

}  // namespace cia
