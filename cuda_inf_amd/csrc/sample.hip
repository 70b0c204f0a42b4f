// sample.hip -- a token for each row of logits from a given random number, after
// temperature, top-k, top-p and min-p, on gfx950.
//
// In descending order of the logits (the lowest index first among equals) each filter
// keeps a prefix, and so does the draw: a prefix sum of w = exp((l - max) / T) that
// reaches a goal.  No row is sorted.  With x = 8 log2(e) l / T, a token's bin is
// ceil(x), an eighth of an octave of w, and the counts and masses of the 336 bins
// below the largest (42 octaves; what lies lower has no weight) say in which bin a
// prefix ends:
//   k_sample_bins  reads the logits once: the bins of each chunk of a row;
//   k_sample_pick  adds up a row's chunks, takes the few tokens that a filter or the
//                  draw can end at from the chunks that have them, and puts those in
//                  order.
// Bins lie at whole x, so that those of chunks with other maxima only need a shift.
// Masses are added as integers, 2^34 for a bin's upper edge, so that sums do not depend
// on the order of atomics.
#include <algorithm>

#include "common.h"
#include "cuda_inf_batch.h"

namespace cia {

constexpr int kSampleThreads = 1024;  // of k_sample_pick
constexpr int kSampleWaves = kSampleThreads / 64;
constexpr int kBins = 336;   // 42 octaves, 8 bins each
constexpr int kCap = 4096;   // tokens of a bin taken into LDS
constexpr int kSmall = 256;  // tokens put in order by counting the larger ones
constexpr int kAll = 1024;   // tokens put in order to find all prefixes among them
constexpr int kSub = 1024;   // parts of a bin that holds more than kSmall
constexpr int kTile = 4096;  // logits of a step: 4 a thread of k_sample_pick, 16 of k_sample_bins
constexpr int kMaxChunk = 4 * kTile;
constexpr int kMaxChunks = CIA_SAMPLE_MAX_VOCAB / kMaxChunk;  // 256
constexpr int kCountShift = 49;  // of a chunk's bin: count << 49 | mass; 2^14 tokens of 2^34

// of a chunk of a row; its bins follow the chunks of all rows
struct ChunkHead {
  double n;       // ceil of its largest x; -inf: no token, inf: logits of +inf
  float top;      // its largest logit
  uint32_t idx;   // the first token that has it
};

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
};

// order-preserving bits of a number; -0 as 0
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __builtin_bit_cast(float, k ^ ((uint32_t)((int32_t)~k >> 31) | 0x80000000u));
}

// four neighbouring logits from i on, -inf where NaN and past the row's end
template <bool kHalf>
__device__ __forceinline__ f32x4 load_logits(const void* row, int i, int V) {
  const float none = -__builtin_inff();
  f32x4 x{none, none, none, none};
  if constexpr (kHalf) {
    const _Float16* r = (const _Float16*)row;
    if (i + 4 <= V) {
      f16x4 h;
      __builtin_memcpy(&h, r + i, 8);
      for (int e = 0; e < 4; e++) x[e] = (float)h[e];
    } else {
      for (int e = 0; e < 4; e++)
        if (i + e < V) x[e] = (float)r[i + e];
    }
  } else {
    const float* r = (const float*)row;
    if (i + 4 <= V) {
      __builtin_memcpy(&x, r + i, 16);
    } else {
      for (int e = 0; e < 4; e++)
        if (i + e < V) x[e] = r[i + e];
    }
  }
  for (int e = 0; e < 4; e++) x[e] = x[e] == x[e] ? x[e] : none;
  return x;
}

// 2^(f / 8) in units of 2^-34 for f in (-1, 0]: the exponential's series to its 6th
// power (the next is 7e-12), rounded by an addition of 2^18
__device__ __forceinline__ uint64_t bin_mass(double f) {
  const double y = f * (0.69314718055994530942 / 8);
  double r = 1.0 / 720;
  r = __builtin_fma(r, y, 1.0 / 120);
  r = __builtin_fma(r, y, 1.0 / 24);
  r = __builtin_fma(r, y, 1.0 / 6);
  r = __builtin_fma(r, y, 0.5);
  r = __builtin_fma(r, y, 1.0);
  r = __builtin_fma(r, y, 1.0);
  return __builtin_bit_cast(uint64_t, r + 262144.0) - __builtin_bit_cast(uint64_t, 262144.0);
}
__device__ __forceinline__ double bin_unit(int bin) { return exp2((double)bin * -0.125 - 34.0); }

__device__ __forceinline__ double temperature_scale(float t) { return 8 * 1.44269504088896340736 / (double)t; }

// ---------------------------------------------------------------- the bins
// grid = rows * chunks, block = 256, kTiles * kTile logits a workgroup in registers
template <bool kHalf, int kTiles>
__global__ __launch_bounds__(256) void k_sample_bins(SampleArgs a) {
  __shared__ unsigned long long bins[kBins];
  __shared__ float wtop[4];
  __shared__ uint32_t widx[4];
  const int b = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks, tid = threadIdx.x;
  const void* row = (const char*)a.logits + (int64_t)b * a.stride * (kHalf ? 2 : 4);
  const int i0 = chunk * (kTiles * kTile) + 4 * tid;
  f32x4 x[4 * kTiles];
#pragma unroll
  for (int i = 0; i < 4 * kTiles; i++) x[i] = load_logits<kHalf>(row, i0 + 1024 * i, a.V);
  const float t = a.temperature ? a.temperature[b] : 1.0f;
  for (int i = tid; i < kBins; i += 256) bins[i] = 0;
  float top = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < 4 * kTiles; i++)
#pragma unroll
    for (int e = 0; e < 4; e++) top = __builtin_fmaxf(top, x[i][e]);
  top = wave_max_fast(top);
  if ((tid & 63) == 0) wtop[tid >> 6] = top;
  __syncthreads();
  top = __builtin_fmaxf(__builtin_fmaxf(wtop[0], wtop[1]), __builtin_fmaxf(wtop[2], wtop[3]));
  ChunkHead* const head = a.heads + (int64_t)b * a.chunks + chunk;
  const bool none = top == -__builtin_inff();
  if (none || !(t > 0.0f)) {  // nothing here, or the largest is all that is asked for
    uint32_t idx = ~0u;
#pragma unroll
    for (int i = 4 * kTiles - 1; i >= 0; i--)
#pragma unroll
      for (int e = 3; e >= 0; e--)
        if (x[i][e] == top) idx = (uint32_t)(i0 + 1024 * i + e);
    for (int off = 32; off; off >>= 1) {
      const uint32_t o = __shfl_xor(idx, off);
      idx = o < idx ? o : idx;
    }
    if ((tid & 63) == 0) widx[tid >> 6] = idx;
    __syncthreads();
    if (tid == 0) {
      idx = min(min(widx[0], widx[1]), min(widx[2], widx[3]));
      *head = ChunkHead{none ? -__builtin_inf() : 0.0, top, idx};
    }
    return;
  }
  const bool inf = top == __builtin_inff();
  const double c = temperature_scale(t), R = inf ? 0.0 : __builtin_ceil(c * (double)top);
#pragma unroll
  for (int i = 0; i < 4 * kTiles; i++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
#pragma clang fp contract(off)
      float l = x[i][e];
      if (inf) l = l == top ? 0.0f : -__builtin_inff();
      const double y = c * (double)l, n = __builtin_ceil(y), d = R - n;
      if (d < (double)kBins)
        atomicAdd(&bins[(int)d], (unsigned long long)bin_mass(y - n) + (1ull << kCountShift));
    }
  __syncthreads();
  uint64_t* const to = a.bins + ((int64_t)b * a.chunks + chunk) * kBins;
  for (int i = tid; i < kBins; i += 256) to[i] = bins[i];
  if (tid == 0) *head = ChunkHead{inf ? __builtin_inf() : R, top, 0};
}

// ---------------------------------------------------------------- the choice
enum Goal { kNth, kReach, kPass, kRatio };

// where a prefix ends
struct Ends {
  double mass;  // of the prefix, the largest bin's upper edge being 1
  double w;     // of its last token
  int idx;
};

struct SampleLds {
  uint64_t list[kCap];  // key << 32 | ~index
  uint64_t small[kAll];
  double run[kAll];     // sums of the ordered list
  unsigned long long mass[kSub];
  uint32_t cnt[kSub];
  double before[kBins + 1];  // mass of the bins before
  int count[kBins + 1];      // tokens of the bins before
  double shift[kMaxChunks];  // of a chunk's bins; kBins or more: none of them counts
  int use[kMaxChunks];       // chunks to take tokens from
  double dsum[kSampleWaves];
  uint64_t key[kSampleWaves];
  uint32_t lo[kSampleWaves], hi[kSampleWaves];
  int n, m, at, bin;
  Ends ends;
};

// one row, all threads of the workgroup
template <bool kHalf>
struct SampleRow {
  SampleLds& s;
  const SampleArgs& a;
  const void* row;
  const ChunkHead* heads;
  const uint64_t* bins;
  double c;     // x = c l
  double R;     // ceil of the largest x
  float top;    // the largest logit
  bool inf;     // some are +inf: they count as 0, the others as -inf
  int tid, lane, wave;

  __device__ __forceinline__ f32x4 load(int i) const {
    f32x4 x = load_logits<kHalf>(row, i, a.V);
    if (inf)
      for (int e = 0; e < 4; e++) x[e] = x[e] == __builtin_inff() ? 0.0f : -__builtin_inff();
    return x;
  }
  // x of a logit, rounded.  (Fused with a difference, a product of 1e39 would be its
  // rounding away from its own ceil.)
  __device__ __forceinline__ double x_of(float l) const {
#pragma clang fp contract(off)
    return c * (double)l;
  }
  __device__ __forceinline__ double weight(float l) const {
#pragma clang fp contract(off)
    return exp2((x_of(l) - R) * 0.125);
  }
  // w over the largest
  __device__ __forceinline__ double ratio(float l) const { return exp2(((double)l - (double)top) * c * 0.125); }
  __device__ __forceinline__ uint64_t mass_of(float l) const {
#pragma clang fp contract(off)
    const double x = x_of(l);
    return bin_mass(x - __builtin_ceil(x));
  }

  // the row's largest logit: key << 32 | ~index
  __device__ uint64_t largest() {
    uint64_t best = 0;
    for (int i = tid; i < a.chunks; i += kSampleThreads) {
      const ChunkHead h = heads[i];
      if (h.n > -__builtin_inf()) {
        const uint64_t k = (uint64_t)order_key(h.top) << 32 | ~h.idx;
        best = k > best ? k : best;
      }
      s.shift[i] = h.n;
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
  __device__ void add_up() {
    constexpr int kWays = kSampleThreads / kBins;  // threads of a bin
    for (int i = tid; i < a.chunks; i += kSampleThreads) {
      const double n = s.shift[i];
      s.shift[i] = inf ? (n == __builtin_inf() ? 0.0 : (double)kBins) : R - n;
    }
    __syncthreads();
    const int b = tid % kBins, way = tid / kBins;
    unsigned long long m = 0;
    uint32_t k = 0;
    if (way < kWays)
#pragma unroll 8
      for (int i = way; i < a.chunks; i += kWays) {
        const double d = (double)b - s.shift[i];
        const uint64_t v = d >= 0.0 ? bins[(int64_t)i * kBins + (int)d] : 0;
        m += v & ((1ull << kCountShift) - 1);
        k += (uint32_t)(v >> kCountShift);
      }
    if (way < kWays) s.list[tid] = m, s.cnt[tid] = k;  // (tid = way * kBins + b)
    __syncthreads();
    if (wave == 0) {  // 6 bins a lane
      double dm[6], im = 0.0;
      int dk[6], ik = 0;
      for (int j = 0; j < 6; j++) {
        const int i = lane * 6 + j;
        dm[j] = im, dk[j] = ik;
        if (i < kBins) {
          unsigned long long q = 0;
          for (int w = 0; w < kWays; w++) q += s.list[w * kBins + i], ik += (int)s.cnt[w * kBins + i];
          im += (double)q * bin_unit(i);
        }
      }
      const double own = im;
      const int owk = ik;
      for (int off = 1; off < 64; off <<= 1) {
        const double um = __shfl_up(im, off);
        const int uk = __shfl_up(ik, off);
        if (lane >= off) im += um, ik += uk;
      }
      for (int j = 0; j < 6; j++) {
        const int i = lane * 6 + j;
        if (i <= kBins) s.before[i] = (im - own) + dm[j], s.count[i] = (ik - owk) + dk[j];
      }
    }
    __syncthreads();
  }

  // the bin in which a prefix ends: the first whose sum satisfies the goal, the last
  // that holds any where none does
  __device__ int bin_with(Goal how, int nth, double goal) {
    __syncthreads();
    if (tid == 0) s.bin = kBins, s.at = 0;
    __syncthreads();
    if (tid < kBins && s.count[tid + 1] > s.count[tid]) {
      const bool here = how == kNth ? s.count[tid + 1] >= nth
                        : how == kReach ? s.before[tid + 1] >= goal : s.before[tid + 1] > goal;
      if (here) atomicMin(&s.bin, tid);
      atomicMax(&s.at, tid);
    }
    __syncthreads();
    return s.bin < kBins ? s.bin : s.at;
  }

  // the chunks that have tokens in the bins from `b0` to `b1`: how many
  __device__ int chunks_with(int b0, int b1) {
    __syncthreads();
    if (tid == 0) s.m = 0;
    __syncthreads();
    for (int i = tid; i < a.chunks; i += kSampleThreads) {
      const double sh = s.shift[i];
      // (its first bin has a token, its largest)
      if (sh > (double)b1) continue;
      if (b0 == b1) {
        const uint64_t v = bins[(int64_t)i * kBins + (b1 - (int)sh)];
        if (!(v >> kCountShift)) continue;
      }
      s.use[atomicAdd(&s.m, 1)] = i;
    }
    __syncthreads();
    return s.m;
  }

  // fn(key, logit, index) for the tokens of the bins from b0 to b1, of the s.m chunks in use
  template <typename F>
  __device__ __forceinline__ void each(int b0, int b1, F fn) {
    const int steps = s.m * (a.chunk / kTile);
    for (int k = 0; k < steps; k++) {
      const int i = s.use[k / (a.chunk / kTile)] * a.chunk + k % (a.chunk / kTile) * kTile + 4 * tid;
      const f32x4 x = load(i);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const double d = R - __builtin_ceil(x_of(x[e]));
        if (d >= (double)b0 && d <= (double)b1) fn(order_key(x[e]), x[e], i + e);
      }
    }
  }

  // The tokens of the bins b0..b1 with keys lo..hi into the list: how many there are
  // (the list holds kCap at most), and their least and largest key.
  __device__ int gather(int b0, int b1, uint32_t lo, uint32_t hi, uint32_t& least, uint32_t& most) {
    __syncthreads();
    if (tid == 0) s.n = 0;
    __syncthreads();
    least = ~0u, most = 0;
    each(b0, b1, [&](uint32_t k, float, int i) {
      if (k < lo || k > hi) return;
      least = k < least ? k : least;
      most = k > most ? k : most;
      const int n = atomicAdd(&s.n, 1);
      if (n < kCap) s.list[n] = (uint64_t)k << 32 | (uint32_t)~i;
    });
    for (int off = 32; off; off >>= 1) {
      const uint32_t u = __shfl_xor(least, off), v = __shfl_xor(most, off);
      least = u < least ? u : least;
      most = v > most ? v : most;
    }
    if (lane == 0) s.lo[wave] = least, s.hi[wave] = most;
    __syncthreads();
    for (int w = 0; w < kSampleWaves; w++) {
      least = s.lo[w] < least ? s.lo[w] : least;
      most = s.hi[w] > most ? s.hi[w] : most;
    }
    return s.n;
  }

  // n tokens of `from` into s.small in descending order; n <= kAll
  __device__ void order(const uint64_t* from, int n) {
    __syncthreads();
    if (n <= kSmall) {
      // a token's place is how many are larger: 4 threads a token, each a quarter of them
      const int i = tid & (kSmall - 1), quarter = tid / kSmall, per = (n + 3) / 4;
      if (tid < kSmall) s.cnt[tid] = 0;
      __syncthreads();
      const uint64_t mine = i < n ? from[i] : ~0ull;
      int larger = 0;
      for (int k = quarter * per; k < min(n, quarter * per + per); k++) larger += from[k] > mine;
      if (i < n && larger) atomicAdd(&s.cnt[i], (uint32_t)larger);
      __syncthreads();
      if (tid < n) s.small[s.cnt[tid]] = mine;
      __syncthreads();
      return;
    }
    int size = 2 * kSmall;
    while (size < n) size *= 2;
    if (tid < size) s.small[tid] = tid < n ? from[tid] : 0;
    __syncthreads();
    for (int k = 2; k <= size; k *= 2)
      for (int j = k / 2; j; j /= 2) {
        if (tid < size / 2) {
          const int u = (tid / j) * 2 * j + tid % j, v = u + j;
          const uint64_t x = s.small[u], y = s.small[v];
          if ((x < y) == ((u & k) == 0)) s.small[u] = y, s.small[v] = x;
        }
        __syncthreads();
      }
  }

  // sums of the weights of the n tokens in s.small, `mass` before them; a thread's own weight
  __device__ double sums(int n, double mass) {
    double w = tid < n ? weight(key_value((uint32_t)(s.small[tid] >> 32))) : 0.0, run = w;
    for (int off = 1; off < 64; off <<= 1) {
      const double o = __shfl_up(run, off);
      if (lane >= off) run += o;
    }
    if (lane == 63) s.dsum[wave] = run;
    __syncthreads();
    double base = mass;
    for (int v = 0; v < wave; v++) base += s.dsum[v];
    if (tid < n) s.run[tid] = base + run;
    __syncthreads();
    return w;
  }

  // the place in the ordered list of n at which a prefix ends, cnt tokens before the list;
  // its last where the sum stays below the goal by a rounding; kRatio: -1 if none is large enough
  __device__ int place(Goal how, int n, int cnt, int nth, double goal) {
    __syncthreads();
    if (tid == 0) s.at = n - 1;
    __syncthreads();
    if (tid < n) {
      const bool stop = how == kNth ? cnt + tid + 1 >= nth
                        : how == kReach ? s.run[tid] >= goal
                        : how == kPass ? s.run[tid] > goal
                                       : !(ratio(key_value((uint32_t)(s.small[tid] >> 32))) >= goal);
      if (stop) atomicMin(&s.at, how == kRatio ? tid - 1 : tid);
    }
    __syncthreads();
    return s.at;
  }

  // One of kSub parts of the keys least..most, as `each` gives the tokens, in which the prefix ends:
  // keys lo..hi of it; cnt and mass move to what is before it.
  template <typename E>
  __device__ void divide(Goal how, int bin, int& cnt, double& mass, int nth, double goal, uint32_t least, uint32_t most,
                         uint32_t& lo, uint32_t& hi, E tokens) {
    int shift = 0;
    while ((most - least) >> shift >= kSub) shift++;
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
    unsigned long long im = km;
    int ik = kc;
    for (int off = 1; off < 64; off <<= 1) {
      const unsigned long long um = __shfl_up(im, off);
      const int uk = __shfl_up(ik, off);
      if (lane >= off) im += um, ik += uk;
    }
    if (lane == 63) s.key[wave] = im, s.lo[wave] = (uint32_t)ik;
    __syncthreads();
    for (int w = 0; w < wave; w++) im += s.key[w], ik += (int)s.lo[w];
    const double unit = bin_unit(bin), after = mass + (double)im * unit;
    const uint32_t low = most - ((((uint32_t)tid + 1) << shift) - 1);  // the part's least key
    if (kc) {
      const bool here = how == kNth ? cnt + ik >= nth
                        : how == kReach ? after >= goal
                        : how == kPass ? after > goal
                                       : !(ratio(key_value(low < least || low > most ? least : low)) >= goal);
      if (here) atomicMin(&s.at, tid);
      atomicMax(&s.bin, tid);
    }
    __syncthreads();
    const int at = s.at < kSub ? s.at : s.bin;
    if (tid == at) {
      s.ends.mass = mass + (double)(im - km) * unit;
      s.ends.idx = cnt + ik - kc;
    }
    __syncthreads();
    mass = s.ends.mass;
    cnt = s.ends.idx;
    hi = most - ((uint32_t)at << shift);
    const uint32_t part = hi - ((1u << shift) - 1);
    lo = part < least || part > hi ? least : part;
  }

  // Where in `bin` a prefix ends, cnt tokens and mass before it: at its `nth` token,
  // where its sum reaches (kReach) or passes (kPass) `goal`, or at its last token of
  // at least `goal` times the largest weight (kRatio; none of the bin: idx -1).
  __device__ Ends end_of(Goal how, int bin, int cnt, double mass, int nth, double goal) {
    uint32_t lo = 0, hi = ~0u, least, most;
    chunks_with(bin, bin);
    int n = gather(bin, bin, lo, hi, least, most);
    while (n > kCap && least < most) {
      divide(how, bin, cnt, mass, nth, goal, least, most, lo, hi, [&](auto add) {
        each(bin, bin, [&](uint32_t k, float l, int) {
          if (k >= least && k <= most) add(k, l);
        });
      });
      n = gather(bin, bin, lo, hi, least, most);
    }
    if (n > kCap) return equals(how, cnt, mass, nth, goal, n, key_value(most));
    const uint64_t* from = s.list;
    while (n > kSmall && least < most) {
      divide(how, bin, cnt, mass, nth, goal, least, most, lo, hi, [&](auto add) {
        for (int i = tid; i < n; i += kSampleThreads) {
          const uint32_t k = (uint32_t)(s.list[i] >> 32);
          if (k >= least && k <= most) add(k, key_value(k));
        }
      });
      // its tokens to the front (a step's are read before any is written)
      if (tid == 0) s.m = 0;
      uint32_t l2 = ~0u, m2 = 0;
      for (int i0 = 0; i0 < n; i0 += kSampleThreads) {
        const uint64_t v = i0 + tid < n ? s.list[i0 + tid] : 0;
        const uint32_t k = (uint32_t)(v >> 32);
        __syncthreads();
        if (i0 + tid < n && k >= lo && k <= hi) {
          s.list[atomicAdd(&s.m, 1)] = v;
          l2 = k < l2 ? k : l2;
          m2 = k > m2 ? k : m2;
        }
      }
      for (int off = 32; off; off >>= 1) {
        const uint32_t u = __shfl_xor(l2, off), v = __shfl_xor(m2, off);
        l2 = u < l2 ? u : l2;
        m2 = v > m2 ? v : m2;
      }
      __syncthreads();
      if (lane == 0) s.lo[wave] = l2, s.hi[wave] = m2;
      __syncthreads();
      n = s.m;
      least = ~0u, most = 0;
      for (int w = 0; w < kSampleWaves; w++) {
        least = s.lo[w] < least ? s.lo[w] : least;
        most = s.hi[w] > most ? s.hi[w] : most;
      }
      __syncthreads();
    }
    if (n > kAll) return equals(how, cnt, mass, nth, goal, n, key_value(most));
    order(from, n);
    const double w = sums(n, mass);
    const int at = place(how, n, cnt, nth, goal);
    if (tid == 0) s.ends = Ends{mass, 0.0, -1};
    __syncthreads();
    if (tid == at) s.ends = Ends{s.run[tid], w, (int)~(uint32_t)s.small[tid]};
    __syncthreads();
    return s.ends;
  }
  __device__ Ends end(Goal how, int nth, double goal) {
    const int b = bin_with(how, nth, goal);
    return end_of(how, b, s.count[b], s.before[b], nth, goal);
  }

  // the same among n tokens of one logit l
  __device__ Ends equals(Goal how, int cnt, double mass, int nth, double goal, int n, float l) {
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
};

// grid = rows, block = 1024
template <bool kHalf>
__global__ __launch_bounds__(kSampleThreads) void k_sample_pick(SampleArgs a) {
  __shared__ SampleLds s;
  const int b = blockIdx.x, tid = threadIdx.x;
  const void* row = (const char*)a.logits + (int64_t)b * a.stride * (kHalf ? 2 : 4);
  SampleRow<kHalf> r{s,   a,   row, a.heads + (int64_t)b * a.chunks, a.bins + (int64_t)b * a.chunks * kBins,
                     0.0, 0.0, 0.0f, false, tid, tid & 63, tid >> 6};
  const float t = a.temperature ? a.temperature[b] : 1.0f;
  const int k = a.top_k ? a.top_k[b] : 0;
  const float tp = a.top_p ? a.top_p[b] : 1.0f, mp = a.min_p ? a.min_p[b] : 0.0f;
  float u = a.u[b];
  const uint64_t best = r.largest();
  if (best == 0 || !(t > 0.0f)) {
    if (tid == 0) {
      a.ids[b] = best ? (int)~(uint32_t)best : -1;
      if (a.p) a.p[b] = best ? 1.0f : 0.0f;
    }
    return;
  }
  r.top = key_value((uint32_t)(best >> 32));
  r.inf = r.top == __builtin_inff();
  if (r.inf) r.top = 0.0f;
  r.c = temperature_scale(t);
  r.R = __builtin_ceil(r.x_of(r.top));
  r.add_up();
  const int total = s.count[kBins];
  const double all = s.before[kBins], need = tp > 0.0f ? (double)tp : 0.0, least = mp < 1.0f ? (double)mp : 1.0;
  const bool by_k = k > 0 && k < total, by_p = tp < 1.0f;
  bool by_m = mp > 0.0f;
  // the bin of the last token that each filter can keep
  int bm = 0;
  if (by_m) {
    const double x = r.x_of(r.top) + 8 * log2(least), bin = r.R - __builtin_ceil(x);
    by_m = bin < (double)kBins;
    bm = by_m && bin > 0.0 ? (int)bin : 0;
  }
  const int bk = by_k ? r.bin_with(kNth, k, 0.0) : kBins - 1;
  const int bp = by_p ? r.bin_with(kReach, 0, need * s.before[bk + 1]) : kBins - 1;
  u = u >= 0.0f ? (u < 1.0f ? u : 0x1.fffffep-1f) : 0.0f;
  double kept = all;  // mass of what the filters keep
  Ends e;
  // top-p's goal is a part of top-k's mass
  const int last = by_k && by_p ? bk : min(min(bk, bp), by_m ? bm : kBins - 1);
  if ((by_k || by_p || by_m) && s.count[last + 1] <= kAll) {
    // few enough: all of them in order, and every prefix among them
    r.chunks_with(0, last);
    uint32_t lo, hi;
    const int n = r.gather(0, last, 0, ~0u, lo, hi);
    r.order(s.list, n);
    const double w = r.sums(n, 0.0);
    if (by_k && k <= n) kept = s.run[k - 1];
    if (by_p) {
      const double m = s.run[r.place(kReach, n, 0, 0, need * kept)];
      kept = m < kept ? m : kept;
    }
    if (by_m) {
      // (all of them, where another filter ends before: its mass is less)
      const double m = s.run[max(0, r.place(kRatio, n, 0, 0, least))];
      kept = m < kept ? m : kept;
    }
    const int at = r.place(kPass, n, 0, 0, (double)u * kept);
    if (tid == at) s.ends = Ends{s.run[tid], w, (int)~(uint32_t)s.small[tid]};
    __syncthreads();
    e = s.ends;
  } else {
    if (by_k) kept = r.end(kNth, k, 0.0).mass;
    if (by_p) {
      const double m = r.end(kReach, 0, need * kept).mass;
      kept = m < kept ? m : kept;
    }
    if (by_m) {
      // bins before the one of `least` times the largest weight are kept whole
      const double m = s.count[bm + 1] > s.count[bm] ? r.end_of(kRatio, bm, s.count[bm], s.before[bm], 0, least).mass
                                                     : s.before[bm];
      kept = m < kept ? m : kept;
    }
    e = r.end(kPass, 0, (double)u * kept);
  }
  if (tid == 0) {
    a.ids[b] = e.idx;
    if (a.p) a.p[b] = (float)(e.w / kept);
  }
}

// Chunks of 16384 logits where that makes two workgroups a compute unit, or a row more than 64
// of the smaller ones; else of 4096.
static int sample_chunk(int B, int V) {
  return (int64_t)B * ((V + kMaxChunk - 1) / kMaxChunk) >= 512 || V > 64 * kTile ? kMaxChunk : kTile;
}

}  // namespace cia

using namespace cia;

extern "C" int64_t cia_sample_workspace_bytes(int B, int V) {
  if (B < 0 || B > CIA_SAMPLE_MAX_ROWS || V < 1 || V > CIA_SAMPLE_MAX_VOCAB) return 0;
  // (the most that B rows or fewer need: a smaller batch may have smaller chunks)
  const int64_t big = (V + kMaxChunk - 1) / kMaxChunk, small = (V + kTile - 1) / kTile;
  int64_t n = (int64_t)B * (sample_chunk(B, V) == kTile ? small : big);
  if (sample_chunk(1, V) == kTile) n = std::max(n, std::min<int64_t>(B, 511 / big) * small);
  return 16 + n * (int64_t)(sizeof(ChunkHead) + kBins * sizeof(uint64_t));
}

template <bool kHalf>
static int sample_launch(const SampleArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.B * a.chunks));
  if (a.chunk == kTile)
    hipLaunchKernelGGL((k_sample_bins<kHalf, 1>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((k_sample_bins<kHalf, kMaxChunk / kTile>), grid, dim3(256), 0, s, a);
  const int st = launch_status();
  if (st) return st;
  hipLaunchKernelGGL((k_sample_pick<kHalf>), dim3((unsigned)a.B), dim3(kSampleThreads), 0, s, a);
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
  const int chunk = sample_chunk(B, V), chunks = (V + chunk - 1) / chunk;
  ChunkHead* const heads = (ChunkHead*)ws;
  const SampleArgs a{logits, stride, temperature, top_k, top_p, min_p, u, ids, p, B, V, chunk, chunks, heads,
                     (uint64_t*)(heads + (int64_t)B * chunks)};
  return type == CIA_LOGITS_F16 ? sample_launch<true>(a, (hipStream_t)stream)
                                : sample_launch<false>(a, (hipStream_t)stream);
}
