// sample.hip -- a token for each row of logits from a given random number, after
// temperature, top-k, top-p and min-p, on gfx950.
//
// In descending order of the logits (the lowest index first among equals) each filter
// keeps a prefix, and so does the draw: a prefix sum of w = exp((l - max) / T) that
// reaches a goal.  No row is sorted.  With x = 16 log2(e) l / T, a token's bin is
// ceil(x), a sixteenth of an octave of w, and the counts and masses of the 672 bins
// below the largest (42 octaves; what lies lower has no weight) say in which bin a
// prefix ends:
//   k_sample_bins  reads the logits once: the bins of each chunk of a row;
//   k_sample_pick  adds up a row's chunks, takes the few tokens that a filter or the
//                  draw can end at from the chunks that have them, and puts those in
//                  order;
//   k_sample_row   does both for a row of up to 16384 logits, which stays in registers.
// Bins lie at whole x, so that those of chunks with other maxima only need a shift.
// Masses are added as integers, 2^34 for a bin's upper edge, so that sums do not depend
// on the order of atomics; over the largest logit's own, so that rows of equals have
// whole sums.
//
// Bound by memory for large batches, which read a row once or, for a broad nucleus,
// twice (4 V bytes a pass in fp32): 256 rows of 131 072, top-p, take 79 us, 29-30 of them the
// bins (134 MB at 4.5-4.7 TB/s; their atomics are 3 % of it) and 48-50 the choice, of which its
// pass is 19 (7 TB/s, part of it from the last-level cache).  By chains of dependent steps
// for few: one row of 65 536 with all filters takes 16 us, 6 for the bins and 10 for the
// choice; one row of 4000 8.0 in its one launch, of 60 7.8 (a call alone takes the host
// about 6).  What such steps cost is not arithmetic: a step of a scan through LDS 140
// cycles (by DPP a few), an atomic on one word by all threads 4500 (by one lane a wave
// 200), a barrier with what waits at it 150.
#include <type_traits>

#include "common.h"
#include "cuda_inf_batch.h"
#include "sample_shape.h"

namespace cia {

constexpr int kSampleThreads = 512;  // of a row's workgroup
constexpr int kSampleWaves = kSampleThreads / 64;
constexpr int kSlots = 36;    // tokens that a thread takes from a row into LDS
constexpr int kCap = 7680;   // tokens that are tried to be taken: 15 a thread
constexpr int kSmall = 16;  // tokens put in order by one wave (256 broad rows 74.2 us for 76.8; up to 48 slower)
constexpr int kAll = 1024;   // tokens put in order at all
constexpr int kSub = kSampleThreads;  // parts of a bin's keys
constexpr int kStep = 4 * kSampleThreads;  // logits of a step of k_sample_pick
constexpr int kMaxChunks = CIA_SAMPLE_MAX_VOCAB / kMaxChunk;  // 256
constexpr int kCountShift = 49;  // of a chunk's bin: count << 49 | mass; 2^14 tokens of 2^34

struct SampleArgs {
  const void* logits;
  int64_t stride;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* u;
  int32_t* ids;
  float* p;
  int B, V;
  int chunk, chunks;  // logits of a chunk, chunks of a row
  ChunkHead* heads;   // [B][chunks]
  uint64_t* bins;     // [B][chunks][kBins]
  uint64_t* tops;     // [B][chunks][kTop], of smaller chunks
};

// order-preserving bits of a number; -0 as 0
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __builtin_bit_cast(float, k ^ ((uint32_t)((int32_t)~k >> 31) | 0x80000000u));
}

// Four neighbouring logits of a row from i on, in two steps, so that many loads can be out
// before any is looked at.  `_in`: those past the row's end V are -inf; the row's last four
// are read for them, and moved.
template <bool kHalf>
struct Logits {
  using T = typename std::conditional<kHalf, _Float16, float>::type;
  typename std::conditional<kHalf, f16x4, f32x4>::type x;
  __device__ __forceinline__ void load(const void* row, int i) { __builtin_memcpy(&x, (const T*)row + i, sizeof(x)); }
  __device__ __forceinline__ void load_in(const void* row, int i, int V) { load(row, min(i, V - 4)); }
  // (of a row of less than 4)
  __device__ __forceinline__ void load_few(const void* row, int V) {
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = ((const T*)row)[max(e + V - 4, 0)];
  }
  __device__ __forceinline__ f32x4 get_in(int i, int V) const {
    const int past = i - min(i, V - 4);
    f32x4 y = get();
    const float none = -__builtin_inff();
    if (past & 1) y = f32x4{y[1], y[2], y[3], none};
    if (past & 2) y = f32x4{y[2], y[3], none, none};
    return past > 3 ? f32x4{none, none, none, none} : y;
  }
  __device__ __forceinline__ f32x4 get() const {
    f32x4 y;
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = (float)x[e];
    return y;
  }
};

// 2^(f / 16) for f in (-1, 0]: the polynomial of degree 4 through the Chebyshev points of
// the interval, 2.5e-12 off.  Its coefficients are pinned to scalar registers: as literals
// each costs two moves a use (8 of the 26 vector instructions of a logit).
struct PowerOf2 {
  double c0 = 0.9999999999975604, c1 = 4.3321698663009583e-02, c2 = 9.383838162057435e-04,
         c3 = 1.3548068750879863e-05, c4 = 1.4361898916011284e-07, unit = 262144.0;
  __device__ __forceinline__ PowerOf2() {
    asm("" : "+s"(c0), "+s"(c1), "+s"(c2), "+s"(c3), "+s"(c4), "+s"(unit));
  }
  __device__ __forceinline__ double operator()(double f) const {
    return __builtin_fma(__builtin_fma(__builtin_fma(__builtin_fma(c4, f, c3), f, c2), f, c1), f, c0);
  }
  // the same in units of 2^-34, rounded by an addition of 2^18, whose low half is 0
  __device__ __forceinline__ uint64_t mass(double f) const {
    return __builtin_bit_cast(uint64_t, (*this)(f) + unit) - __builtin_bit_cast(uint64_t, 262144.0);
  }
};

// a bin's upper edge, bin 0's being 1: 2^(-bin / 16)
__device__ __forceinline__ double bin_edge(int bin) {
  const int i = bin & 3, j = bin >> 2 & 3;
  const double e = i == 0 ? 1.0 : i == 1 ? 0.9576032806985737 : i == 2 ? 0.9170040432046712 : 0.8781260801866497;
  const double q = j == 0 ? 1.0 : j == 1 ? 0.8408964152537145 : j == 2 ? 0.7071067811865476 : 0.5946035575013605;
  return e * q * __builtin_bit_cast(double, (uint64_t)(1023 - (bin >> 4)) << 52);
}

__device__ __forceinline__ double temperature_scale(float t) { return 16 * 1.44269504088896340736 / (double)t; }

// ---------------------------------------------------------------- the bins
// Of rows of more than kMaxChunk.  grid = rows * chunks, block = kThreads, 4 kVec logits of the chunk a thread, in registers:
// all loads of a chunk are out together, and its largest is known before its bins.  19 vector
// instructions a logit with all that is around them, vector units 47 % busy (256 rows of 131 072).
template <bool kHalf, int kThreads, int kVec>
__global__ __launch_bounds__(kThreads) void k_sample_bins(SampleArgs a) {
  constexpr int kWaves = kThreads / 64, kEach = 4 * kThreads;
  constexpr bool kTops = kVec * kEach == kMinChunk;
  __shared__ int wcount[kWaves], depth, listed;
  __shared__ unsigned long long bins[kBins];
  __shared__ float wtop[kWaves];
  __shared__ uint32_t widx[kWaves];
  const int b = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks, tid = threadIdx.x;
  const void* row = (const char*)a.logits + (int64_t)b * a.stride * (kHalf ? 2 : 4);
  const int i0 = chunk * (kVec * kEach) + 4 * tid;
  const bool whole = (chunk + 1) * (kVec * kEach) <= a.V;
  Logits<kHalf> in[kVec];
#pragma unroll
  for (int i = 0; i < kVec; i++) in[i].load_in(row, i0 + kEach * i, a.V);
  const float t = a.temperature ? a.temperature[b] : 1.0f;
  for (int i = tid; i < kBins; i += kThreads) bins[i] = 0;
  f32x4 x[kVec];
#pragma unroll
  for (int i = 0; i < kVec; i++) x[i] = whole ? in[i].get() : in[i].get_in(i0 + kEach * i, a.V);
  // (a NaN is neither the largest nor of any bin: no comparison holds for it)
  float top = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < kVec; i++)
#pragma unroll
    for (int e = 0; e < 4; e++) top = __builtin_fmaxf(top, x[i][e]);
  top = wave_max_fast(top);
  if ((tid & 63) == 0) wtop[tid >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; w++) top = __builtin_fmaxf(top, wtop[w]);
  ChunkHead* const head = a.heads + (int64_t)b * a.chunks + chunk;
  const bool none = top == -__builtin_inff();
  if (none || !(t > 0.0f)) {  // nothing here, or the largest is all that is asked for
    uint32_t idx = ~0u;
#pragma unroll
    for (int i = kVec - 1; i >= 0; i--)
#pragma unroll
      for (int e = 3; e >= 0; e--)
        if (x[i][e] == top) idx = (uint32_t)(i0 + kEach * i + e);
    for (int off = 32; off; off >>= 1) {
      const uint32_t o = __shfl_xor(idx, off);
      idx = o < idx ? o : idx;
    }
    if ((tid & 63) == 0) widx[tid >> 6] = idx;
    __syncthreads();
    if (tid == 0) {
      for (int w = 0; w < kWaves; w++) idx = min(idx, widx[w]);
      *head = ChunkHead{none ? -__builtin_inf() : 0.0, top, idx, kBins, 0};
    }
    return;
  }
  const bool inf = __builtin_amdgcn_readfirstlane((int)(top == __builtin_inff()));
  const PowerOf2 power;
  const double c = temperature_scale(t), R = inf ? 0.0 : __builtin_ceil(c * (double)top);
  int bin[kTops ? kVec : 1][4];  // of each logit
  if (inf)
#pragma unroll
    for (int i = 0; i < kVec; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) x[i][e] = x[i][e] == top ? 0.0f : -__builtin_inff();
#pragma unroll
  for (int i = 0; i < kVec; i++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
#pragma clang fp contract(off)
      const double y = c * (double)x[i][e], n = __builtin_ceil(y), d = R - n;
      const bool has = d < (double)kBins;
      if (has) atomicAdd(&bins[(int)d], (unsigned long long)power.mass(y - n) + (1ull << kCountShift));
      if constexpr (kTops) bin[i][e] = has ? (int)d : kBins;
    }
  if (tid == 0) depth = 0, listed = 0;
  __syncthreads();
  uint64_t* const to = a.bins + ((int64_t)b * a.chunks + chunk) * kBins;
  for (int i = tid; i < kBins; i += kThreads) to[i] = bins[i];
  if constexpr (kTops) {
    // as many of the first bins as hold no more than kTop tokens, two bins a thread
    const int lane = tid & 63, wave = tid >> 6, i = min(2 * tid, kBins - 2);
    const bool mine = 2 * tid < kBins;
    const int k0 = mine ? (int)(bins[i] >> kCountShift) : 0, k1 = mine ? (int)(bins[i + 1] >> kCountShift) : 0;
    int upto = scan_lanes(k0 + k1);
    if (lane == 63) wcount[wave] = upto;
    __syncthreads();
    for (int w = 0; w < wave; w++) upto += wcount[w];
    const uint64_t first = __ballot(mine && upto - k1 <= kTop), second = __ballot(mine && upto <= kTop);
    if (lane == 0) atomicMax(&depth, first ? 2 * 64 * wave + __popcll(first) + __popcll(second) : 0);
    __syncthreads();
    uint64_t* const tops = a.tops + ((int64_t)b * a.chunks + chunk) * kTop;
    const int d = depth;
    uint64_t set[kVec][4];
    int n = 0;
#pragma unroll
    for (int i = 0; i < kVec; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        set[i][e] = __ballot(bin[i][e] < d);
        n += __popcll(set[i][e]);
      }
    int at = 0;  // a place in the top for each of the wave's
    if (lane == 0) at = atomicAdd(&listed, n);
    at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
    for (int i = 0; i < kVec; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if (bin[i][e] < d)
          tops[at + __builtin_amdgcn_mbcnt_hi((uint32_t)(set[i][e] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)set[i][e], 0))] =
              (uint64_t)order_key(x[i][e]) << 32 | (uint32_t)~(i0 + kEach * i + e);
        at += __popcll(set[i][e]);
      }
    __syncthreads();
  }
  if (tid == 0) *head = ChunkHead{inf ? __builtin_inf() : R, top, 0, depth, listed};
}

// ---------------------------------------------------------------- the choice
enum Goal { kNth, kReach, kPass, kRatio };

// where a prefix ends
struct Ends {
  double mass;  // of the prefix
  double w;     // of its last token
  int idx;
};

template <int kSlots>
struct SampleLds {
  float value[kSlots][kSampleThreads];     // tokens taken from the row, of each thread its own
  uint16_t nth[kSlots][kSampleThreads];    // and which of the logits it has passed each is
  uint64_t some[kAll];  // those of one bin
  uint64_t small[kAll];  // in descending order
  double run[kAll];     // sums of their weights
  int place[kAll];      // places of those of s.some
  unsigned long long mass[kBins];
  uint32_t cnt[kBins];
  double before[kBins + 1];  // mass of the bins before
  int count[kBins + 1];      // tokens of the bins before
  double shift[kMaxChunks];  // of a chunk's bins; kBins or more: none of them counts
  int use[kMaxChunks];       // chunks to take tokens from
  int listed[kMaxChunks];    // tokens of a chunk's top
  double dsum[kSampleWaves];
  uint64_t key[kSampleWaves];
  uint32_t lo[kSampleWaves], hi[kSampleWaves];
  int n, m, at, bin, last, covered;
  Ends ends;
};

constexpr int kRanges = 2;

// one row, all threads of the workgroup; kPer: steps of a chunk, or of the row where the
// threads keep it (kKept)
template <bool kHalf, int kPer, bool kKept>
struct SampleRow {
  static constexpr int kSlots = kKept ? 4 * kPer : cia::kSlots;
  static constexpr int kCap = kKept ? 1 << 30 : cia::kCap;  // (as many as there are fit)
  SampleLds<kSlots>& s;
  const SampleArgs& a;
  const void* row;
  const ChunkHead* heads;
  const uint64_t* bins;
  double c;     // x = c l
  double R;     // ceil of the largest x
  double top_power, top_mass;  // 2^(f / 16) and its mass, of the largest logit
  float top;    // the largest logit
  bool inf;     // some are +inf: they count as 0, the others as -inf
  int tid, lane, wave;
  int taken;    // tokens that the thread has in the list
  int group_count;  // of bin_with
  double group_before;
  PowerOf2 power;
  f32x4 held[kKept ? kPer : 1];

  // what follows from the largest logit
  __device__ __forceinline__ void start(float largest, float temperature) {
    inf = __builtin_amdgcn_readfirstlane((int)(largest == __builtin_inff()));
    top = inf ? 0.0f : largest;
    c = temperature_scale(temperature);
    R = __builtin_ceil(x_of(top));
    top_mass = (double)mass_of(top);
    top_power = power_of(top);
  }

  // x of a logit, rounded.  (Fused with a difference, a product of 1e39 would be its
  // rounding away from its own ceil.)
  __device__ __forceinline__ double x_of(float l) const {
#pragma clang fp contract(off)
    return c * (double)l;
  }
  // w of a token of one of the bins, exactly 1 for the largest logit's
  __device__ __forceinline__ double weight(float l) const {
#pragma clang fp contract(off)
    const double x = x_of(l), n = __builtin_ceil(x);
    return power(x - n) / top_power * bin_edge((int)(R - n));
  }
  // the same for a sum of masses of tokens of one bin: whole for equals of the largest
  __device__ __forceinline__ double mass_in(int bin, unsigned long long m) const {
    return (double)m / top_mass * bin_edge(bin);
  }
  // the same without the bins' 2.5e-12
  __device__ __forceinline__ double ratio(float l) const { return exp2(((double)l - (double)top) * c * 0.0625); }
  __device__ __forceinline__ double power_of(float l) const {
#pragma clang fp contract(off)
    const double x = x_of(l);
    return power(x - __builtin_ceil(x));
  }
  __device__ __forceinline__ uint64_t mass_of(float l) const {
#pragma clang fp contract(off)
    const double x = x_of(l);
    return power.mass(x - __builtin_ceil(x));
  }

  // The row's largest logit, key << 32 | ~index, and each wave's first chunk's bins, two
  // of a lane's at a time, on their way.
  static constexpr int kPairs = (kBins / 2 + 63) / 64;
  struct Pairs {
    u32x4 v[kPairs];
  };
  __device__ __forceinline__ void load_pairs(int chunk, Pairs& p) const {
    const u32x4* const from = (const u32x4*)(bins + (int64_t)chunk * kBins);
#pragma unroll
    for (int i = 0; i < kPairs; i++) p.v[i] = from[min(64 * i + lane, kBins / 2 - 1)];
  }
  __device__ __forceinline__ uint64_t largest(Pairs& first) {
    load_pairs(min(wave, a.chunks - 1), first);
    for (int i = tid; i < kBins; i += kSampleThreads) s.mass[i] = 0, s.cnt[i] = 0;
    if (tid == 0) s.last = 0, s.covered = kBins;
    uint64_t best = 0;
    for (int i = tid; i < a.chunks; i += kSampleThreads) {
      const ChunkHead h = heads[i];
      if (h.n > -__builtin_inf()) {
        const uint64_t k = (uint64_t)order_key(h.top) << 32 | ~h.idx;
        best = k > best ? k : best;
      }
      s.shift[i] = h.n;
      s.use[i] = h.depth;
      s.listed[i] = h.listed;
    }
    for (int off = 32; off; off >>= 1) {
      const uint64_t o = __shfl_xor((unsigned long long)best, off);
      best = o > best ? o : best;
    }
    if (lane == 0) s.key[wave] = best;
    __syncthreads();
    for (int w = 0; w < kSampleWaves; w++) best = s.key[w] > best ? s.key[w] : best;
    return best;
  }

  // the row's bins: tokens and mass before each
  __device__ __forceinline__ void add_up(Pairs& p) {
    for (int i = tid; i < a.chunks; i += kSampleThreads) {
      const double n = s.shift[i];
      s.shift[i] = inf ? (n == __builtin_inf() ? 0.0 : (double)kBins) : fmin(R - n, (double)kBins);
      // (none of its tokens counts; of a chunk without +inf in a row that has some they are
      // the chunk's own logits, which may lie above the 0 that +inf stands for)
      if (s.shift[i] >= (double)kBins) s.listed[i] = 0;
      atomicMin(&s.covered, (int)s.shift[i] + s.use[i]);
    }
    __syncthreads();
    for (int chunk = wave; chunk < a.chunks; chunk += kSampleWaves) {
      if (chunk != wave) load_pairs(chunk, p);
      const int shift = (int)s.shift[chunk];
#pragma unroll
      for (int i = 0; i < kPairs; i++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const uint64_t v = (uint64_t)p.v[i][2 * e + 1] << 32 | p.v[i][2 * e];
          const int from = 2 * (64 * i + lane) + e, b = from + shift;
          // (the bins of a chunk without tokens are not written; they are past the last)
          if (from < kBins && b < kBins && v) {
            atomicAdd(&s.mass[b], (unsigned long long)(v & ((1ull << kCountShift) - 1)));
            atomicAdd(&s.cnt[b], (uint32_t)(v >> kCountShift));
          }
        }
    }
    __syncthreads();
    const int b = min(2 * tid, kBins - 2);
    scan(s.cnt[b], s.cnt[b + 1], s.mass[b], s.mass[b + 1]);
  }

  // the largest of the threads' numbers
  __device__ __forceinline__ float most(float v) const {
    v = wave_max_fast(v);
    if (lane == 0) s.lo[wave] = __builtin_bit_cast(uint32_t, v);
    __syncthreads();
    for (int w = 0; w < kSampleWaves; w++) v = __builtin_fmaxf(v, __builtin_bit_cast(float, s.lo[w]));
    return v;
  }
  // the first of the row's logits, kept by the threads, that is this one
  __device__ __forceinline__ int first_of(float l) const {
    int idx = 0x7fffffff;
#pragma unroll
    for (int i = kPer - 1; i >= 0; i--)
#pragma unroll
      for (int e = 3; e >= 0; e--)
        if (held[i][e] == l) idx = kStep * i + 4 * tid + e;
    for (int off = 32; off; off >>= 1) idx = min(idx, __shfl_xor(idx, off));
    if (lane == 0) s.hi[wave] = (uint32_t)idx;
    __syncthreads();
    for (int w = 0; w < kSampleWaves; w++) idx = min(idx, (int)s.hi[w]);
    return idx;
  }

  // The bins of a row that the threads keep, and the sums before each.
  __device__ __forceinline__ void bin_kept() {
#pragma unroll
    for (int i = 0; i < kPer; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
#pragma clang fp contract(off)
        if (inf) held[i][e] = held[i][e] == __builtin_inff() ? 0.0f : -__builtin_inff();
        const double y = c * (double)held[i][e], n = __builtin_ceil(y), d = R - n;
        if (d < (double)kBins)
          atomicAdd(&s.mass[(int)d], (unsigned long long)power.mass(y - n) + (1ull << kCountShift));
      }
    __syncthreads();
    const int b = min(2 * tid, kBins - 2);
    constexpr unsigned long long kMass = (1ull << kCountShift) - 1;
    const unsigned long long v0 = s.mass[b], v1 = s.mass[b + 1];
    scan((uint32_t)(v0 >> kCountShift), (uint32_t)(v1 >> kCountShift), v0 & kMass, v1 & kMass);
  }

  // first and what the waves before this one have
  template <typename T>
  __device__ __forceinline__ T before_wave(T first, const T (&of)[kSampleWaves]) const {
    T at[kSampleWaves];
#pragma unroll
    for (int w = 0; w < kSampleWaves; w++) at[w] = of[w];
#pragma unroll
    for (int w = 0; w < kSampleWaves - 1; w++) first += w < wave ? at[w] : T(0);
    return first;
  }

  // s.count and s.before, from two bins a thread: 2 tid and the next
  __device__ __forceinline__ void scan(uint32_t c0, uint32_t c1, unsigned long long u0, unsigned long long u1) {
    const int b = min(2 * tid, kBins - 2);
    const bool mine = 2 * tid < kBins;
    const int k0 = mine ? (int)c0 : 0, k1 = mine ? (int)c1 : 0;
    const double m0 = mine ? mass_in(b, u0) : 0.0, m1 = mine ? mass_in(b + 1, u1) : 0.0;
    double run = scan_lanes(m0 + m1);
    int upto = scan_lanes(k0 + k1);
    if (lane == 63) s.dsum[wave] = run, s.lo[wave] = (uint32_t)upto;
    const uint64_t any = __ballot(k0 + k1 > 0), odd = __ballot(k1 > 0);
    if (lane == 0 && any) {
      const int at = 63 - __builtin_clzll(any);
      atomicMax(&s.last, 2 * (64 * wave + at) + (int)(odd >> at & 1));
    }
    __syncthreads();
    run += before_wave(0.0, s.dsum), upto += (int)before_wave(0u, s.lo);
    if (mine) {
      s.before[b + 2] = run, s.count[b + 2] = upto;
      s.before[b + 1] = run - m1, s.count[b + 1] = upto - k1;
    }
    if (tid == 0) s.before[0] = 0.0, s.count[0] = 0;
    __syncthreads();
  }

  // the bin in which a prefix ends: the first whose sum satisfies the goal, the last
  // that holds any where none does; each wave looks by itself, in 56 groups of 12 bins,
  // whose sums it keeps (keep_groups), then in one of them
  static constexpr int kPart = kBins / 56;
  __device__ __forceinline__ void keep_groups() {
    const int b = min((lane + 1) * kPart, kBins);
    group_count = s.count[b], group_before = s.before[b];
  }
  __device__ __forceinline__ int bin_with(Goal how, int nth, double goal) const {
    const auto ends = [&](int count, double before) {
      return __ballot(how == kNth ? count >= nth : how == kReach ? before >= goal : before > goal);
    };
    uint64_t set = ends(group_count, group_before);
    if (!set) return __builtin_amdgcn_readfirstlane(s.last);
    const int at = __builtin_ctzll(set) * kPart, b = min(at + lane + 1, kBins);
    set = ends(s.count[b], s.before[b]);
    return min(at + __builtin_ctzll(set), kBins - 1);
  }

  // the chunks that may have a token in the bins up to `to`: whose largest is in one
  __device__ __forceinline__ void chunks_with(int to) {
    __syncthreads();
    if (tid == 0) s.m = 0;
    __syncthreads();
    for (int i = tid; i < a.chunks; i += kSampleThreads)
      if (s.shift[i] <= (double)to) s.use[atomicAdd(&s.m, 1)] = i;
    __syncthreads();
  }

  // The least key of the tokens of the bins up to `to`: x above R - to - 1.  It is within a
  // few of the quotient's, of which the lanes try 64.
  __device__ __forceinline__ uint32_t first_key(int to) const {
    if (!(c > 0.0)) return order_key(-3.402823466e38f);  // all tokens are in bin 0
    const uint32_t k = order_key((float)((R - (double)to - 1.0) / c)) - 32 + lane;
    const float v = key_value(k);
    const bool in = k > order_key(__builtin_inff()) || R - __builtin_ceil(x_of(v)) <= (double)to;
    const uint64_t set = __ballot(in);
    return __builtin_amdgcn_readfirstlane(k) + (set ? __builtin_ctzll(set) : 64);
  }
  // the keys of the bins from..to
  __device__ __forceinline__ void keys_of(int from, int to, uint32_t& lo, uint32_t& hi) const {
    lo = first_key(to);
    hi = from ? first_key(from - 1) - 1 : order_key(top);
    if (hi == 0x7fffffff) hi--;  // (-0, whose key is 0's)
  }

  // where the nth of the logits that a thread passes lies: four of a step, the steps of the
  // chunks in use in turn
  __device__ __forceinline__ int index_of(int nth) const {
    const int step = nth >> 2;
    if constexpr (kKept) return step * kStep + 4 * tid + (nth & 3);
    return s.use[step / kPer] * (kPer * kStep) + step % kPer * kStep + 4 * tid + (nth & 3);
  }

  // fn(nth, x): four neighbouring logits from the thread's nth on, of the s.m chunks in use
  template <typename F>
  __device__ __forceinline__ void each(F fn) {
    if constexpr (kKept) {
#pragma unroll
      for (int k = 0; k < kPer; k++) fn(4 * k, held[k]);
      return;
    }
    // kAhead steps' loads, of kAt chunks, are out while those before them are looked at
    constexpr int kAhead = 8, kAt = kAhead / (kKept ? 8 : kPer);
    const int m = __builtin_amdgcn_readfirstlane(s.m);
    Logits<kHalf> in[kAhead];
    int i[kAt];
    const auto load = [&](int c0) __attribute__((always_inline)) {
#pragma unroll
      for (int q = 0; q < kAt; q++)  // (past the last: it again, left out below)
        i[q] = __builtin_amdgcn_readfirstlane(s.use[min(c0 + q, m - 1)]) * (kPer * kStep);
#pragma unroll
      for (int k = 0; k < kAhead; k++) in[k].load_in(row, i[k / kPer] + k % kPer * kStep + 4 * tid, a.V);
    };
    load(0);
#pragma unroll 1
    for (int c0 = 0; c0 < m; c0 += kAt) {
      f32x4 x[kAhead];
      bool whole = true;
#pragma unroll
      for (int q = 0; q < kAt; q++) whole &= i[q] + kPer * kStep <= a.V;
      if (whole) {
#pragma unroll
        for (int k = 0; k < kAhead; k++) x[k] = in[k].get();
      } else {
#pragma unroll
        for (int k = 0; k < kAhead; k++) x[k] = in[k].get_in(i[k / kPer] + k % kPer * kStep + 4 * tid, a.V);
      }
      if (c0 + kAt < m) load(c0 + kAt);
#pragma unroll
      for (int k = 0; k < kAhead; k++) {
        if (c0 + k / kPer >= m) break;
        if (inf)
#pragma unroll
          for (int e = 0; e < 4; e++) x[k][e] = x[k][e] == __builtin_inff() ? 0.0f : -__builtin_inff();
        fn((c0 * kPer + k) * 4, x[k]);
      }
    }
  }

  // The tokens with keys in one of two ranges into the list: whether they fit.
  __device__ __forceinline__ bool take(const uint32_t (&from)[kRanges], const uint32_t (&upto)[kRanges]) {
    const float lo = key_value(__builtin_amdgcn_readfirstlane(from[0])), hi = key_value(__builtin_amdgcn_readfirstlane(upto[0]));
    const float lo1 = key_value(__builtin_amdgcn_readfirstlane(from[1])), hi1 = key_value(__builtin_amdgcn_readfirstlane(upto[1]));
    int have = 0;
    each([&](int nth, const f32x4& x) __attribute__((always_inline)) {
      bool in[4];
#pragma unroll
      for (int e = 0; e < 4; e++) in[e] = ((x[e] >= lo) & (x[e] <= hi)) | ((x[e] >= lo1) & (x[e] <= hi1));
      if (!__any(in[0] | in[1] | in[2] | in[3])) return;
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (in[e]) {
          const int at = min(have, kSlots - 1);
          s.value[at][tid] = x[e];
          s.nth[at][tid] = (uint16_t)(nth + e);
          have++;
        }
    });
    taken = min(have, kSlots);
    return !__syncthreads_or(have > kSlots);
  }

  // Places in s.some for a thread's `mine` tokens, in the threads' order: from which on;
  // n: of all.
  __device__ __forceinline__ int places(int mine, int& n) {
    int at = scan_lanes(mine);
    __syncthreads();
    if (lane == 63) s.lo[wave] = (uint32_t)at;
    __syncthreads();
    at += (int)before_wave(0u, s.lo) - mine;
    n = 0;
#pragma unroll
    for (int w = 0; w < kSampleWaves; w++) n += (int)s.lo[w];
    return at;
  }

  // The tokens in the list with keys lo..hi into s.some (kAll at most): how many.
  __device__ __forceinline__ int select(uint32_t lo, uint32_t hi) {
    uint64_t set = 0;  // which of the thread's
#pragma unroll 4
    for (int i = 0; i < taken; i++) {
      const uint32_t k = order_key(s.value[i][tid]);
      set |= (uint64_t)(k >= lo && k <= hi) << i;
    }
    int n, at = places(__popcll(set), n);
    for (; set && at < kAll; set &= set - 1, at++) {
      const int i = __builtin_ctzll(set);
      s.some[at] = (uint64_t)order_key(s.value[i][tid]) << 32 | (uint32_t)~index_of(s.nth[i][tid]);
    }
    __syncthreads();
    return n;
  }

  // The tokens that the threads keep with keys lo..hi into s.some (kAll at most): how many.
  __device__ __forceinline__ int select_held(uint32_t lo_key, uint32_t hi_key) {
    const float lo = key_value(__builtin_amdgcn_readfirstlane(lo_key)), hi = key_value(__builtin_amdgcn_readfirstlane(hi_key));
    int mine = 0;
    each([&](int, const f32x4& x) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 4; e++) mine += (x[e] >= lo) & (x[e] <= hi);
    });
    int n, at = places(mine, n);
    each([&](int nth, const f32x4& x) __attribute__((always_inline)) {
      if (__any((x[0] >= lo) | (x[1] >= lo) | (x[2] >= lo) | (x[3] >= lo)))
#pragma unroll
        for (int e = 0; e < 4; e++)
          if ((x[e] >= lo) & (x[e] <= hi)) s.some[min(at++, kAll - 1)] = (uint64_t)order_key(x[e]) << 32 | (uint32_t)~index_of(nth + e);
    });
    __syncthreads();
    return n;
  }

  // The tops of 8 chunks, one token of each a thread, on their way: those of the first 8
  // before it is known whether they are enough.
  static_assert(kTop == kSampleThreads);
  struct Tops {
    uint64_t v[8];
  };
  __device__ __forceinline__ void load_tops(const uint64_t* tops, int chunk, Tops& t) const {
#pragma unroll
    for (int i = 0; i < 8; i++) t.v[i] = tops[min(chunk + i, a.chunks - 1) * kTop + tid];
  }
  // The tokens of the chunks' tops with keys from lo on into s.some: how many.
  __device__ __forceinline__ int select_tops(const uint64_t* tops, Tops& t, uint32_t lo) {
    int n = 0;
    for (int chunk = 0; chunk < a.chunks; chunk += 8) {
      if (chunk) load_tops(tops, chunk, t);
      int mine = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const bool in = chunk + i < a.chunks && tid < s.listed[min(chunk + i, a.chunks - 1)] && (uint32_t)(t.v[i] >> 32) >= lo;
        if (!in) t.v[i] = 0;
        mine += in;
      }
      int more, at = n + places(mine, more);
      n += more;
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (t.v[i]) s.some[min(at++, kAll - 1)] = t.v[i];
    }
    __syncthreads();
    return n;
  }

  // n tokens of s.some, up to kSmall, into s.small in descending order, by one wave
  __device__ __forceinline__ void order_small(int n) {
    if (wave == 0) {
      const uint64_t mine = s.some[lane];
      int at = 0;
      for (int k = 0; k < n; k++) {
        const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), k) << 32 |
                               (uint32_t)__builtin_amdgcn_readlane((int)mine, k);
        at += other > mine;
      }
      if (lane < n) s.small[at] = mine;
    }
    __syncthreads();
  }

  // n tokens of s.some, with keys lo..hi, into s.small in descending order; n <= kAll.  A
  // token's place is how many have larger parts of the keys, of kSub, and how many of its
  // own part are larger.
  __device__ __forceinline__ void order(int n, uint32_t lo, uint32_t hi) {
    if (n <= kSmall) return order_small(n);
    const int shift = part_shift(lo, hi);
    __syncthreads();
    s.cnt[tid] = 0;
    __syncthreads();
    int nth[kAll / kSampleThreads];
#pragma unroll
    for (int e = 0; e < kAll / kSampleThreads; e++) {
      const int i = e * kSampleThreads + tid;
      if (i < n) nth[e] = (int)atomicAdd(&s.cnt[(hi - (uint32_t)(s.some[i] >> 32)) >> shift], 1u);
    }
    __syncthreads();
    const int c = (int)s.cnt[tid];
    int all;
    s.mass[tid] = (uint64_t)places(c, all);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kAll / kSampleThreads; e++) {
      const int i = e * kSampleThreads + tid;
      if (i >= n) continue;
      const uint64_t v = s.some[i];
      s.run[(int)s.mass[(hi - (uint32_t)(v >> 32)) >> shift] + nth[e]] = __builtin_bit_cast(double, v);
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kAll / kSampleThreads; e++) {
      const int i = e * kSampleThreads + tid;
      if (i >= n) continue;
      const uint64_t mine = __builtin_bit_cast(uint64_t, s.run[i]);
      const uint32_t part = (hi - (uint32_t)(mine >> 32)) >> shift;
      const int from = (int)s.mass[part], to = from + (int)s.cnt[part];
      int at = from;
#pragma unroll 4
      for (int k = from; k < to; k++) at += __builtin_bit_cast(uint64_t, s.run[k]) > mine;
      s.small[at] = mine;
    }
    __syncthreads();
  }
  // keys lo..hi in kSub parts, from hi on, of 2^this
  __device__ __forceinline__ static int part_shift(uint32_t lo, uint32_t hi) {
    return max(0, 32 - __clz((int)(hi - lo)) - __builtin_ctz(kSub));
  }

  // The same for all n tokens of the first bins: a token's place is what its bin starts at
  // and how many of the bin are larger.
  __device__ __forceinline__ void order_bins(int n) {
    __syncthreads();
    for (int i = tid; i < kBins; i += kSampleThreads) s.cnt[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kSampleThreads) {
      const uint64_t v = s.some[i];
      const int bin = (int)(R - __builtin_ceil(x_of(key_value((uint32_t)(v >> 32)))));
      const int at = s.count[bin] + (int)atomicAdd(&s.cnt[bin], 1u);
      s.run[at] = __builtin_bit_cast(double, v);
      s.place[at] = bin;
    }
    __syncthreads();
    for (int i = tid; i < n; i += kSampleThreads) {
      const uint64_t mine = __builtin_bit_cast(uint64_t, s.run[i]);
      const int from = s.count[s.place[i]], to = s.count[s.place[i] + 1];
      int at = from;
#pragma unroll 4
      for (int k = from; k < to; k++) at += __builtin_bit_cast(uint64_t, s.run[k]) > mine;
      s.small[at] = mine;
    }
    __syncthreads();
  }

  // sums of the weights of the n tokens in s.small, `mass` before them; s.some: the weights
  __device__ __forceinline__ void sums(int n, double mass) {
    for (int i0 = 0; i0 < n; i0 += kSampleThreads) {
      const int i = i0 + tid;
      const double w = i < n ? weight(key_value((uint32_t)(s.small[i] >> 32))) : 0.0, run = scan_lanes(w);
      if (i < n) s.some[i] = __builtin_bit_cast(uint64_t, w);
      if (lane == 63) s.dsum[wave] = run;
      __syncthreads();
      const double base = before_wave(mass, s.dsum);
      if (i < n) s.run[i] = base + run;
      if (i0 + kSampleThreads < n) {
        for (int w = 0; w < kSampleWaves; w++) mass += s.dsum[w];
      }
      __syncthreads();
    }
  }

  // the place in the ordered list of n at which a prefix ends, cnt tokens before the list;
  // its last where the sum stays below the goal by a rounding; kRatio: -1 if none is large
  // enough.  Each wave looks by itself: a 64th of the list, then the place in it.
  __device__ __forceinline__ int place(Goal how, int n, int cnt, int nth, double goal) const {
    if (how == kNth) return min(n, nth - cnt) - 1;
    constexpr int kLane = kAll / 64;
    auto past = [&](int i) {  // the prefix has ended at i (kRatio: before it)
      return how == kReach ? s.run[i] >= goal
             : how == kPass ? s.run[i] > goal : !(ratio(key_value((uint32_t)(s.small[i] >> 32))) >= goal);
    };
    uint64_t set = __ballot(lane * kLane < n && past(min(n - 1, lane * kLane + kLane - 1)));
    int at = n;
    if (set) {
      const int i = __builtin_ctzll(set) * kLane + lane;
      set = __ballot(lane < kLane && i < n && past(min(i, n - 1)));
      at = __builtin_amdgcn_readfirstlane(i) + __builtin_ctzll(set);
    }
    return how == kRatio ? at - 1 : min(at, n - 1);
  }

  // the token at a place of the ordered list, `mass` before the list
  __device__ __forceinline__ Ends ends_at(int at, double mass) const {
    if (at < 0) return Ends{mass, 0.0, -1};
    return Ends{s.run[at], __builtin_bit_cast(double, s.some[at]), (int)~(uint32_t)s.small[at]};
  }

  // One of kSub parts of the keys least..most, as `each` gives the tokens, in which the prefix ends:
  // keys lo..hi of it; cnt and mass move to what is before it.  Returns its tokens.
  template <typename E>
  __device__ __forceinline__ int divide(Goal how, int bin, int& cnt, double& mass, int nth, double goal, uint32_t least, uint32_t most,
                         uint32_t& lo, uint32_t& hi, E tokens) {
    const int shift = part_shift(least, most);
    __syncthreads();
    s.mass[tid] = 0, s.cnt[tid] = 0;
    if (tid == 0) s.at = kSub, s.bin = 0;
    __syncthreads();
    tokens([&](uint32_t k, float l) {
      const int p = (int)((most - k) >> shift);
      atomicAdd(&s.mass[p], (unsigned long long)mass_of(l));
      atomicAdd(&s.cnt[p], 1u);
    });
    __syncthreads();
    const int kc = (int)s.cnt[tid];
    const unsigned long long km = s.mass[tid];
    unsigned long long im = scan_lanes(km);
    int ik = scan_lanes(kc);
    if (lane == 63) s.key[wave] = im, s.lo[wave] = (uint32_t)ik;
    __syncthreads();
    im += before_wave((uint64_t)0, s.key), ik += (int)before_wave(0u, s.lo);
    const double after = mass + mass_in(bin, im);
    const uint32_t low = most - ((((uint32_t)tid + 1) << shift) - 1);  // the part's least key
    bool here = false;
    if (kc)
      here = how == kNth ? cnt + ik >= nth
             : how == kReach ? after >= goal
             : how == kPass ? after > goal : !(ratio(key_value(low < least || low > most ? least : low)) >= goal);
    const uint64_t ends = __ballot(here), any = __ballot(kc > 0);
    if (lane == 0 && ends) atomicMin(&s.at, 64 * wave + __builtin_ctzll(ends));
    if (lane == 0 && any) atomicMax(&s.bin, 64 * wave + 63 - __builtin_clzll(any));
    __syncthreads();
    const int at = s.at < kSub ? s.at : s.bin;
    if (tid == at) {
      s.ends.mass = mass + mass_in(bin, im - km);
      s.ends.idx = cnt + ik - kc;
      s.n = kc;
    }
    __syncthreads();
    mass = s.ends.mass;
    cnt = s.ends.idx;
    hi = most - ((uint32_t)at << shift);
    const uint32_t part = hi - ((1u << shift) - 1);
    lo = part < least || part > hi ? least : part;
    return s.n;
  }

  // Where in `bin` a prefix ends, the bins before it summed up: at its `nth` token,
  // where its sum reaches (kReach) or passes (kPass) `goal`, or at its last token of at
  // least `goal` times the largest weight (kRatio; none of the bin: idx -1).  listed:
  // whether the bin's tokens are in the list already.
  __device__ __forceinline__ Ends end_of(Goal how, int bin, int nth, double goal, bool listed) {
    int cnt = s.count[bin];
    double mass = s.before[bin];
    uint32_t lo, hi, least, most;
    keys_of(bin, bin, lo, hi);
    int n = s.count[bin + 1] - cnt;
    if (!kKept && !listed) {
      // divided where it lies until what is left can be taken
      chunks_with(bin);
      while (n > kCap || !take({lo, lo}, {hi, hi})) {
        if (lo == hi) return equals(how, cnt, mass, nth, goal, n, key_value(lo));
        least = lo, most = hi;
        n = divide(how, bin, cnt, mass, nth, goal, least, most, lo, hi, [&](auto add) {
          each([&](int, const f32x4& x) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const uint32_t k = order_key(x[e]);
              if (k >= least && k <= most) add(k, x[e]);
            }
          });
        });
      }
    }
    while (n > kAll && lo < hi) {
      least = lo, most = hi;
      n = divide(how, bin, cnt, mass, nth, goal, least, most, lo, hi, [&](auto add) {
        for (int i = 0; i < taken; i++) {
          const float l = s.value[i][tid];
          const uint32_t k = order_key(l);
          if (k >= least && k <= most) add(k, l);
        }
      });
    }
    n = select(lo, hi);
    if (n > kAll) return equals(how, cnt, mass, nth, goal, n, key_value(hi));
    order(n, lo, hi);
    sums(n, mass);
    return ends_at(place(how, n, cnt, nth, goal), mass);
  }

  // the same among n tokens of one logit l
  __device__ __forceinline__ Ends equals(Goal how, int cnt, double mass, int nth, double goal, int n, float l) {
    const double w = weight(l);
    int r;  // tokens of them in the prefix
    if (how == kNth) {
      r = nth - cnt;
    } else if (how == kRatio) {
      r = ratio(l) >= goal ? n : 0;
    } else {
      const double q = (goal - mass) / w;
      r = q >= (double)n ? n : (int)(how == kReach ? __builtin_ceil(q) : __builtin_floor(q) + 1.0);
    }
    if (how != kRatio) r = r < 1 ? 1 : r;
    r = r > n ? n : r;
    Ends e{mass + (double)r * w, w, -1};
    if (how != kPass) return e;
    // the r-th of them by index: each wave counts a part of the row, then walks its own
    const int per = (a.V + 64 * kSampleWaves - 1) / (64 * kSampleWaves) * 64;
    const int from = min(a.V, wave * per), to = min(a.V, from + per);
    int have = 0;
    for (int i = from + lane; i < to; i += 64) have += is(i, l);
    for (int off = 32; off; off >>= 1) have += __shfl_xor(have, off);
    __syncthreads();
    if (lane == 0) s.lo[wave] = (uint32_t)have;
    if (tid == 0) s.at = -1;
    __syncthreads();
    int before = 0;
    for (int v = 0; v < wave; v++) before += (int)s.lo[v];
    if (before < r && r <= before + have) {
      for (int i0 = from; i0 < to; i0 += 64) {
        const bool eq = i0 + lane < to && is(i0 + lane, l);
        const uint64_t set = __ballot(eq);
        const int k = __popcll(set);
        if (before + k >= r) {
          const int mine = before + __popcll(set & ((2ull << lane) - 1));
          if (eq && mine == r) s.at = i0 + lane;
          break;
        }
        before += k;
      }
    }
    __syncthreads();
    e.idx = s.at;
    return e;
  }
  __device__ __forceinline__ bool is(int i, float l) const {
    float x;
    if constexpr (kHalf)
      x = (float)((const _Float16*)row)[i];
    else
      x = ((const float*)row)[i];
    return inf ? x == __builtin_inff() : x == l;
  }

  // the row's token, after its bins
  __device__ __forceinline__ void choose(int row_at, int k, float tp, float mp, float u, const uint64_t* tops_at, Tops& first) {
    keep_groups();
    const int total = s.count[kBins];
    const double all = s.before[kBins], need = tp > 0.0f ? (double)tp : 0.0, least = mp < 1.0f ? (double)mp : 1.0;
    const bool by_k = k > 0 && k < total, by_p = tp < 1.0f;
    bool by_m = mp > 0.0f;
    // the bin of the last token that each filter can keep
    int bm = 0;
    if (by_m) {
      const double x = x_of(top) + 16 * log2(least), bin = R - __builtin_ceil(x);
      by_m = bin < (double)kBins;
      bm = by_m && bin > 0.0 ? (int)bin : 0;
    }
    u = u >= 0.0f ? (u < 1.0f ? u : 0x1.fffffep-1f) : 0.0f;
    // Bins in which the prefixes can end, by whole bins of what decides them: top-k's bk,
    // top-p's p0..p1 for the masses that bk leaves open, the draw's d0..d1 for the masses
    // that the filters can keep, from..to.  (One loop: its code is fetched once, which is
    // most of the time of code that runs once.)  Where all tokens up to a filter's bin are
    // few, they are put in order and the other bins not looked for.
    int bk = 0, p0 = 0, p1 = kBins - 1, d0 = 0, d1 = kBins - 1;
    // (top-p's goal is a part of top-k's mass: min-p does not end before it)
    int last = __builtin_amdgcn_readfirstlane(s.last);
    if (by_m && !(by_k && by_p)) last = min(last, bm);
    bool few = s.count[last + 1] <= kAll;
    double from = all, to = all;
#pragma unroll 1
    for (int i = by_k ? 0 : by_p ? 1 : 3; i < 5 && !few; i++) {
      if (i == 3 && by_m) from = fmin(from, s.before[bm]), to = fmin(to, s.before[bm + 1]);
      const double goal = i < 3 ? need * (i == 1 ? from : to) : (double)u * (i == 3 ? from : to);
      const int bin = bin_with(i == 0 ? kNth : i < 3 ? kReach : kPass, k, goal);
      if (i == 0) {
        bk = bin, from = s.before[bin], to = s.before[bin + 1];
      } else if (i == 1) {
        p0 = p1 = bin;
        if (!by_k) i = 2;  // (one goal)
      } else if (i == 2) {
        p1 = bin;
      } else if (i == 3) {
        d0 = d1 = bin;
        if (from == to) i = 4;
      } else {
        d1 = bin;
      }
      if (i == 2) from = fmin(from, s.before[p0]), to = fmin(to, s.before[p1 + 1]);
      if (i == 0 || i == 2) {
        const int upto = min(last, by_k ? bk : p1);
        few = s.count[upto + 1] <= kAll;
        if (few) last = upto;
        if (!by_p) i = 2;
      }
    }
    double kept = all;  // mass of what the filters keep
    Ends e;
    int f0 = kBins, f1 = 0;  // the bins of the filters, from the first to the last
    if (by_p) f0 = p0, f1 = p1;
    if (by_k) f0 = min(f0, bk), f1 = max(f1, bk);
    if (by_m) f0 = min(f0, bm), f1 = max(f1, bm);
    // few enough: all of them; else those bins and the draw's, if they fit
    bool listed = few || s.count[d1 + 1] - s.count[d0] + (f0 <= f1 ? s.count[f1 + 1] - s.count[f0] : 0) <= kCap;
    const bool tops = !kKept && kPer * kStep == kMinChunk && few && last < s.covered;  // they are at hand
    uint32_t lo[kRanges], hi[kRanges];
    if (listed && !tops) {
      keys_of(few ? 0 : d0, few ? last : d1, lo[0], hi[0]);
      lo[1] = lo[0], hi[1] = hi[0];
      if (!few && f0 <= f1) keys_of(f0, f1, lo[1], hi[1]);
      if constexpr (!kKept) chunks_with(few ? last : max(d1, f1));
      if (!kKept || !few) listed = take(lo, hi);
    }
    if (few && listed) {
      // every prefix among them, in order
      int n;
      if constexpr (kKept)
        n = select_held(lo[0], hi[0]);
      else
        n = tops ? select_tops(tops_at, first, first_key(last)) : select(0, ~0u);
      order_bins(n);
      sums(n, 0.0);
      if (by_k && k <= n) kept = s.run[k - 1];
      if (by_p) kept = fmin(kept, s.run[place(kReach, n, 0, 0, need * kept)]);
      // (all of them, where another filter ends before: its mass is less)
      if (by_m) kept = fmin(kept, s.run[max(0, place(kRatio, n, 0, 0, least))]);
      e = ends_at(place(kPass, n, 0, 0, (double)u * kept), 0.0);
    } else {
      for (int step = by_k ? 0 : 1; step < 4; step++) {  // top-k, top-p, min-p, the draw
        // (bins by masses that a rounding has moved past their range stay in it)
        Goal how = kPass;
        double goal = (double)u * kept;
        int bin;
        if (step == 0) {
          how = kNth, bin = few ? bin_with(kNth, k, 0.0) : bk;  // (few, but too many for one thread)
        } else if (step == 1) {
          if (!by_p) continue;
          how = kReach, goal = need * kept;
          bin = min(max(bin_with(kReach, 0, goal), p0), p1);
        } else if (step == 2) {
          if (!by_m) continue;
          how = kRatio, goal = least, bin = bm;
          if (s.count[bm + 1] == s.count[bm]) {  // bins before it are kept whole
            kept = fmin(kept, s.before[bm]);
            continue;
          }
        } else {
          bin = min(max(bin_with(kPass, 0, goal), d0), d1);
        }
        e = end_of(how, bin, k, goal, listed);
        if (step < 3) kept = fmin(kept, e.mass);
      }
    }
    put(row_at, e.idx, (float)(e.w / kept));
  }
  __device__ __forceinline__ void put(int row_at, int id, float p) const {
    if (tid) return;
    a.ids[row_at] = id;
    if (a.p) a.p[row_at] = p;
  }
};

// What a row's choice is given, on its way early.
struct Given {
  float t, tp, mp, u;
  int k;
  __device__ __forceinline__ Given(const SampleArgs& a, int b)
      : t(a.temperature ? a.temperature[b] : 1.0f),
        tp(a.top_p ? a.top_p[b] : 1.0f),
        mp(a.min_p ? a.min_p[b] : 0.0f),
        u(a.u[b]),
        k(a.top_k ? a.top_k[b] : 0) {}
};

// grid = rows, block = kSampleThreads: one workgroup a row, so that its steps meet at
// barriers.  us of them, of one row of 65 536 with all filters: the largest 2.4, bins added up 2.5,
// goals' bins 0.9, the few tokens 1.6, their order 0.8, sums 0.7, places 1.0.
template <bool kHalf, int kPer>
__global__ __launch_bounds__(kSampleThreads) void k_sample_pick(SampleArgs a) {
  using Row = SampleRow<kHalf, kPer, false>;
  __shared__ SampleLds<Row::kSlots> s;
  const int b = blockIdx.x, tid = threadIdx.x;
  const void* row = (const char*)a.logits + (int64_t)b * a.stride * (kHalf ? 2 : 4);
  Row r{s,   a,   row, a.heads + (int64_t)b * a.chunks, a.bins + (int64_t)b * a.chunks * kBins,
        0.0, 0.0, 1.0, 1.0, 0.0f, false, tid, tid & 63, tid >> 6, 0};
  const Given g(a, b);
  typename Row::Pairs first;
  typename Row::Tops tops;
  const uint64_t* const tops_at = a.tops + (int64_t)b * a.chunks * kTop;
  if constexpr (kPer * kStep == kMinChunk) r.load_tops(tops_at, 0, tops);
  const uint64_t best = r.largest(first);
  if (best == 0 || !(g.t > 0.0f)) {
    r.put(b, best ? (int)~(uint32_t)best : -1, best ? 1.0f : 0.0f);
    return;
  }
  r.start(key_value((uint32_t)(best >> 32)), g.t);
  r.add_up(first);
  r.choose(b, g.k, g.tp, g.mp, g.u, tops_at, tops);
}

// The same for a row of up to kPer * kStep logits by itself, which the threads keep in registers:
// one launch, no bins through memory, no second pass.  us of the two kernels / of this one:
//   logits                        1000         4000         8192        16 384
//   one row, top-k and top-p   16.8 / 7.8   13.6 / 8.1   14.0 / 8.7   14.6 / 11.6
//   256 rows, top-k and top-p  18.8 / 8.5   15.4 / 8.5   15.9 / 10.1  19.9 / 13.6
//   256 rows, broad top-p      18.4 / 8.5   24.4 / 15.1  24.8 / 17.2  31.0 / 21.0
// (Longer rows chunk by chunk in one workgroup: 5.7 us a chunk of 16384, even at 32 768 and 97
// for 92 with 256 rows of 131 072.)
template <bool kHalf, int kPer>
__global__ __launch_bounds__(kSampleThreads) void k_sample_row(SampleArgs a) {
  using Row = SampleRow<kHalf, kPer, true>;
  __shared__ SampleLds<Row::kSlots> s;
  const int b = blockIdx.x, tid = threadIdx.x;
  const void* row = (const char*)a.logits + (int64_t)b * a.stride * (kHalf ? 2 : 4);
  Row r{s,   a,   row, nullptr, nullptr, 0.0, 0.0, 1.0, 1.0, 0.0f, false, tid, tid & 63, tid >> 6, 0};
  Logits<kHalf> in[kPer];
  if (kPer == 1 && a.V < 4) {
    in[0].load_few(row, a.V);
  } else {
#pragma unroll
    for (int i = 0; i < kPer; i++) in[i].load_in(row, kStep * i + 4 * tid, a.V);
  }
  const Given g(a, b);
  for (int i = tid; i < kBins; i += kSampleThreads) s.mass[i] = 0;
  if (tid == 0) s.last = 0;
  float top = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    r.held[i] = in[i].get_in(kStep * i + 4 * tid, a.V);
#pragma unroll
    for (int e = 0; e < 4; e++) top = __builtin_fmaxf(top, r.held[i][e]);
  }
  top = r.most(top);
  const bool none = top == -__builtin_inff();
  if (none || !(g.t > 0.0f)) {
    const int id = none ? -1 : r.first_of(top);
    r.put(b, id, none ? 0.0f : 1.0f);
    return;
  }
  r.start(top, g.t);
  r.bin_kept();
  typename Row::Tops tops;
  r.choose(b, g.k, g.tp, g.mp, g.u, nullptr, tops);
}

}  // namespace cia

using namespace cia;

extern "C" int64_t cia_sample_workspace_bytes(int B, int V) {
  if (B < 0 || B > CIA_SAMPLE_MAX_ROWS || V < 1 || V > CIA_SAMPLE_MAX_VOCAB || (int64_t)B * V > CIA_SAMPLE_MAX_LOGITS)
    return 0;
  return sample_space_bytes(B, V);
}

template <bool kHalf>
static int sample_launch(const SampleArgs& a, hipStream_t s) {
  const dim3 rows((unsigned)a.B), block(kSampleThreads);
  if (a.V <= kMaxChunk) {
    if (a.V <= kStep)
      hipLaunchKernelGGL((k_sample_row<kHalf, 1>), rows, block, 0, s, a);
    else if (a.V <= 2 * kStep)
      hipLaunchKernelGGL((k_sample_row<kHalf, 2>), rows, block, 0, s, a);
    else if (a.V <= 4 * kStep)
      hipLaunchKernelGGL((k_sample_row<kHalf, 4>), rows, block, 0, s, a);
    else
      hipLaunchKernelGGL((k_sample_row<kHalf, kMaxChunk / kStep>), rows, block, 0, s, a);
    return launch_status();
  }
  const dim3 grid((unsigned)(a.B * a.chunks));
  if (a.chunk == kMinChunk)
    hipLaunchKernelGGL((k_sample_bins<kHalf, 512, kMinChunk / 2048>), grid, dim3(512), 0, s, a);
  else
    hipLaunchKernelGGL((k_sample_bins<kHalf, 512, kMaxChunk / 2048>), grid, dim3(512), 0, s, a);
  const int st = launch_status();
  if (st) return st;
  if (a.chunk == kMinChunk)
    hipLaunchKernelGGL((k_sample_pick<kHalf, kMinChunk / kStep>), dim3((unsigned)a.B), dim3(kSampleThreads), 0, s, a);
  else
    hipLaunchKernelGGL((k_sample_pick<kHalf, kMaxChunk / kStep>), dim3((unsigned)a.B), dim3(kSampleThreads), 0, s, a);
  return launch_status();
}

extern "C" int cia_sample(const void* logits, int type, int64_t stride, const float* temperature, const int32_t* top_k,
                          const float* top_p, const float* min_p, const float* u, int32_t* ids, float* p, int B, int V,
                          void* ws, int64_t ws_bytes, void* stream) {
  const int64_t need = cia_sample_workspace_bytes(B, V);
  CIA_REQUIRE(need > 0 && stride >= V && (type == CIA_LOGITS_F32 || type == CIA_LOGITS_F16), CIA_ERR_ARG);
  if (B == 0) return CIA_OK;
  CIA_REQUIRE(logits && u && ids && ws, CIA_ERR_NULL);
  CIA_REQUIRE(aligned(logits, type == CIA_LOGITS_F32 ? 4 : 2) && aligned(temperature, 4) && aligned(top_k, 4) &&
                  aligned(top_p, 4) && aligned(min_p, 4) && aligned(u, 4) && aligned(ids, 4) && aligned(p, 4) &&
                  aligned(ws, 16),
              CIA_ERR_ALIGN);
  CIA_REQUIRE(ws_bytes >= need, CIA_ERR_ARG);
  const SampleSpace at = sample_space(B, V);
  char* const space = (char*)ws;
  const SampleArgs a{logits, stride, temperature, top_k, top_p, min_p, u, ids, p, B, V, at.chunk, at.chunks,
                     (ChunkHead*)space, (uint64_t*)(space + at.bins), (uint64_t*)(space + at.tops)};
  return type == CIA_LOGITS_F16 ? sample_launch<true>(a, (hipStream_t)stream)
                                : sample_launch<false>(a, (hipStream_t)stream);
}
