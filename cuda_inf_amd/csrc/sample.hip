// sample.hip -- a token for each row of logits from a given random number, after
// temperature, top-k, top-p and min-p, on gfx950.
//
// In descending order of the logits (the lowest index first among equals) each filter
// keeps a prefix, and so does the draw: a prefix sum of w = exp((l - max) / T) that
// reaches a goal.  No row is sorted: with x = 8 log2(e) l / T, a token's bin is
// ceil(x), an eighth of an octave of w, and the counts and masses of the 336 bins
// below the largest (42 octaves; what lies lower has no weight) say in which bin a
// prefix ends.  The tokens of that bin alone are gathered, put in order and summed; a
// bin that holds more of them than fit is divided by its keys first.
//
// Masses are added as integers, 2^34 for the upper edge of a bin, so their sums do not
// depend on the order of the atomics.
#include "common.h"
#include "cuda_inf_batch.h"

namespace cia {

constexpr int kSampleThreads = 1024;
constexpr int kSampleWaves = kSampleThreads / 64;
constexpr int kBins = 336;   // 42 octaves, 8 bins each
constexpr int kCap = 4096;   // tokens of a bin put in order in LDS
constexpr int kSub = 1024;   // parts of a bin that holds more
constexpr int kTile = 4 * kSampleThreads;  // logits of a step of the workgroup

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

enum Goal { kNth, kReach, kPass, kRatio };

// where a prefix ends
struct Ends {
  double mass;  // of the prefix, the largest bin's upper edge being 1
  double w;     // of its last token
  int idx;
};

struct SampleLds {
  union {
    uint64_t list[kCap];  // key << 32 | ~index, in descending order
    struct {
      unsigned long long mass[kSub];
      uint32_t cnt[kSub];
    } sub;
  };
  unsigned long long mass[kBins];
  uint32_t cnt[kBins];
  double before[kBins + 1];  // mass of the bins before
  int count[kBins + 1];      // tokens of the bins before
  double dsum[kSampleWaves];
  uint64_t key[kSampleWaves];
  uint32_t lo[kSampleWaves], hi[kSampleWaves];
  int n, at, bin;
  Ends ends;
};

// one row, all threads of the workgroup
template <bool kHalf>
struct SampleRow {
  SampleLds& s;
  const void* row;
  int V;
  double c;     // x = c l
  double R;     // ceil of the largest x
  float top;    // the largest logit
  bool inf;     // some are +inf: they count as 0, the others as -inf
  int tid, lane, wave;

  __device__ __forceinline__ f32x4 load(int i) const {
    f32x4 x = load_logits<kHalf>(row, i, V);
    if (inf)
      for (int e = 0; e < 4; e++) x[e] = x[e] == __builtin_inff() ? 0.0f : -__builtin_inff();
    return x;
  }
  // bin of a logit (kBins: none), and its place in it.  (x is rounded before R is taken
  // off: fused, a product of 1e39 would be its rounding away from its own ceil.)
  __device__ __forceinline__ int bin_of(float l, double& f) const {
#pragma clang fp contract(off)
    if (!(l > -__builtin_inff())) return kBins;
    const double x = c * (double)l, n = __builtin_ceil(x), b = R - n;
    f = x - n;
    return b < (double)kBins ? (int)b : kBins;
  }
  __device__ __forceinline__ double weight(float l) const {
#pragma clang fp contract(off)
    const double x = c * (double)l;
    return exp2((x - R) * 0.125);
  }

  // the largest logit, lowest index first: key << 32 | ~index
  __device__ uint64_t largest() {
    uint64_t best = 0;
    for (int i = 4 * tid; i < V; i += kTile) {
      const f32x4 x = load_logits<kHalf>(row, i, V);
      for (int e = 0; e < 4; e++)
        if (x[e] > -__builtin_inff()) {
          const uint64_t k = (uint64_t)order_key(x[e]) << 32 | (uint32_t)~(i + e);
          best = k > best ? k : best;
        }
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

  __device__ void histogram() {
    for (int b = tid; b < kBins; b += kSampleThreads) s.mass[b] = 0, s.cnt[b] = 0;
    __syncthreads();
    for (int i = 4 * tid; i < V; i += kTile) {
      const f32x4 x = load(i);
      for (int e = 0; e < 4; e++) {
        double f;
        const int b = bin_of(x[e], f);
        if (b < kBins) {
          atomicAdd(&s.mass[b], (unsigned long long)bin_mass(f));
          atomicAdd(&s.cnt[b], 1u);
        }
      }
    }
    __syncthreads();
    if (wave == 0) {  // the sums of the bins before each, 6 bins a lane
      double m[6], dm = 0.0;
      int k[6], dk = 0;
      for (int j = 0; j < 6; j++) {
        const int b = lane * 6 + j;
        m[j] = dm;
        k[j] = dk;
        if (b < kBins) dm += (double)s.mass[b] * bin_unit(b), dk += (int)s.cnt[b];
      }
      double im = dm;
      int ik = dk;
      for (int off = 1; off < 64; off <<= 1) {
        const double um = __shfl_up(im, off);
        const int uk = __shfl_up(ik, off);
        if (lane >= off) im += um, ik += uk;
      }
      for (int j = 0; j < 6; j++) {
        const int b = lane * 6 + j;
        if (b <= kBins) s.before[b] = (im - dm) + m[j], s.count[b] = (ik - dk) + k[j];
      }
    }
    __syncthreads();
  }

  // the tokens of `bin` with keys lo..hi into the list: how many there are (the list
  // holds kCap at most), and their least and largest key
  __device__ int gather(int bin, uint32_t lo, uint32_t hi, uint32_t& least, uint32_t& most) {
    __syncthreads();
    if (tid == 0) s.n = 0;
    __syncthreads();
    least = ~0u, most = 0;
    for (int i = 4 * tid; i < V; i += kTile) {
      const f32x4 x = load(i);
      for (int e = 0; e < 4; e++) {
        double f;
        const uint32_t k = order_key(x[e]);
        if (k < lo || k > hi || bin_of(x[e], f) != bin) continue;
        least = k < least ? k : least;
        most = k > most ? k : most;
        const int n = atomicAdd(&s.n, 1);
        if (n < kCap) s.list[n] = (uint64_t)k << 32 | (uint32_t)~(i + e);
      }
    }
    for (int off = 32; off; off >>= 1) {
      const uint32_t a = __shfl_xor(least, off), b = __shfl_xor(most, off);
      least = a < least ? a : least;
      most = b > most ? b : most;
    }
    if (lane == 0) s.lo[wave] = least, s.hi[wave] = most;
    __syncthreads();
    for (int w = 0; w < kSampleWaves; w++) {
      least = s.lo[w] < least ? s.lo[w] : least;
      most = s.hi[w] > most ? s.hi[w] : most;
    }
    return s.n;
  }

  // the first n of the list in descending order
  __device__ void order(int n) {
    int size = 64;
    while (size < n) size *= 2;
    for (int i = n + tid; i < size; i += kSampleThreads) s.list[i] = 0;
    __syncthreads();
    for (int k = 2; k <= size; k *= 2)
      for (int j = k / 2; j; j /= 2) {
        for (int i = tid; i < size / 2; i += kSampleThreads) {
          const int a = (i / j) * 2 * j + i % j, b = a + j;
          const uint64_t u = s.list[a], v = s.list[b];
          if ((u < v) == ((a & k) == 0)) s.list[a] = v, s.list[b] = u;
        }
        __syncthreads();
      }
  }

  // Where in `bin` a prefix ends, cnt tokens and mass before it: at its `nth` token,
  // where its sum reaches (kReach) or passes (kPass) `goal`, or at its last token of
  // at least `goal` times the largest weight (kRatio; none of the bin: idx -1).  The
  // bin's last token where its sum stays below the goal by a rounding.
  __device__ Ends end_of(Goal how, int bin, int cnt, double mass, int nth, double goal) {
    uint32_t lo = 0, hi = ~0u, least, most;
    int n = gather(bin, lo, hi, least, most);
    while (n > kCap && least < most) {
      // divide its keys: hist of (most - key) >> shift, the part in which it ends
      int shift = 0;
      while ((most - least) >> shift >= kSub) shift++;
      __syncthreads();
      for (int i = tid; i < kSub; i += kSampleThreads) s.sub.mass[i] = 0, s.sub.cnt[i] = 0;
      if (tid == 0) s.at = kSub;
      __syncthreads();
      for (int i = 4 * tid; i < V; i += kTile) {
        const f32x4 x = load(i);
        for (int e = 0; e < 4; e++) {
          double f;
          const uint32_t k = order_key(x[e]);
          if (k < least || k > most || bin_of(x[e], f) != bin) continue;
          const int b = (int)((most - k) >> shift);
          atomicAdd(&s.sub.mass[b], (unsigned long long)bin_mass(f));
          atomicAdd(&s.sub.cnt[b], 1u);
        }
      }
      __syncthreads();
      // the sums before each part (a part a thread, in order)
      const int kc = (int)s.sub.cnt[tid];
      const unsigned long long km = s.sub.mass[tid];
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
      bool here = false;
      if (kc)
        here = how == kNth ? cnt + ik >= nth
               : how == kReach ? after >= goal
               : how == kPass ? after > goal
                              : !(ratio(key_value(low < least || low > most ? least : low)) >= goal);
      if (here) atomicMin(&s.at, tid);
      __syncthreads();
      int at = s.at;
      if (at == kSub) {  // by a rounding in none: the last
        if (kc) atomicMax(&s.n, 0x40000000 + tid);
        __syncthreads();
        at = s.n - 0x40000000;
      }
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
      n = gather(bin, lo, hi, least, most);
    }
    if (n > kCap) return equals(how, cnt, mass, nth, goal, n, key_value(most));
    order(n);
    // four tokens a thread, in order
    double w[4], run = 0.0;
    const int i0 = 4 * tid;
    for (int e = 0; e < 4; e++) {
      w[e] = i0 + e < n ? weight(key_value((uint32_t)(s.list[i0 + e] >> 32))) : 0.0;
      run += w[e];
    }
    const double own = run;
    for (int off = 1; off < 64; off <<= 1) {
      const double o = __shfl_up(run, off);
      if (lane >= off) run += o;
    }
    if (lane == 63) s.dsum[wave] = run;
    if (tid == 0) s.at = kCap, s.ends = Ends{mass, 0.0, -1};
    __syncthreads();
    run -= own;
    for (int v = 0; v < wave; v++) run += s.dsum[v];
    run += mass;
    double upto[4];
    int mine = kCap;
    for (int e = 3; e >= 0; e--) {
      double r = run;
      for (int k = 0; k <= e; k++) r += w[k];
      upto[e] = r;
    }
    for (int e = 3; e >= 0; e--) {
      const int i = i0 + e;
      if (i >= n) continue;
      bool stop;
      if (how == kRatio)  // the last one that is large enough
        stop = i + 1 == n || !(ratio(key_value((uint32_t)(s.list[i + 1] >> 32))) >= goal);
      else
        stop = i + 1 == n || (how == kNth ? cnt + i + 1 >= nth : how == kReach ? upto[e] >= goal : upto[e] > goal);
      if (stop) mine = i;
    }
    if (mine < kCap) atomicMin(&s.at, mine);
    __syncthreads();
    const int at = s.at;
    if (at / 4 == tid && at < n) {
      const int e = at & 3;
      const float l = key_value((uint32_t)(s.list[at] >> 32));
      if (!(how == kRatio && !(ratio(l) >= goal)))
        s.ends = Ends{upto[e], w[e], (int)~(uint32_t)s.list[at]};
    }
    __syncthreads();
    return s.ends;
  }

  // w over the largest
  __device__ __forceinline__ double ratio(float l) const { return exp2(((double)l - (double)top) * c * 0.125); }

  // the same among n tokens of one logit l, more than the list holds
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
    if (how != kPass || r == 0) return e;
    // the r-th of them by index: each wave counts a part of the row, then walks its own
    const int per = (V + 64 * kSampleWaves - 1) / (64 * kSampleWaves) * 64;
    const int a = min(V, wave * per), b = min(V, a + per);
    int have = 0;
    for (int i = a + lane; i < b; i += 64) have += is(i, l);
    for (int off = 32; off; off >>= 1) have += __shfl_xor(have, off);
    __syncthreads();
    if (lane == 0) s.lo[wave] = (uint32_t)have;
    if (tid == 0) s.at = -1;
    __syncthreads();
    int before = 0;
    for (int v = 0; v < wave; v++) before += (int)s.lo[v];
    if (before < r && r <= before + have) {
      for (int i0 = a; i0 < b; i0 += 64) {
        const bool eq = i0 + lane < b && is(i0 + lane, l);
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
  __device__ Ends end(Goal how, int nth, double goal) {
    const int b = bin_with(how, nth, goal);
    return end_of(how, b, s.count[b], s.before[b], nth, goal);
  }
};

// grid = rows, block = 1024
template <bool kHalf>
__global__ __launch_bounds__(kSampleThreads) void k_sample(SampleArgs a) {
  __shared__ SampleLds lds;
  const int b = blockIdx.x, tid = threadIdx.x;
  const void* row = (const char*)a.logits + (int64_t)b * a.stride * (kHalf ? 2 : 4);
  SampleRow<kHalf> r{lds, row, a.V, 0.0, 0.0, 0.0f, false, tid, tid & 63, tid >> 6};
  const uint64_t best = r.largest();
  const float t = a.temperature ? a.temperature[b] : 1.0f;
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
  r.c = 8 * 1.44269504088896340736 / (double)t;
  r.R = __builtin_ceil(r.c * (double)r.top);
  r.histogram();
  const int total = lds.count[kBins];
  const double all = lds.before[kBins];
  double kept = all;  // mass of what the filters keep
  const int k = a.top_k ? a.top_k[b] : 0;
  if (k > 0 && k < total) kept = r.end(kNth, k, 0.0).mass;
  const float tp = a.top_p ? a.top_p[b] : 1.0f;
  if (tp < 1.0f) {
    const double m = r.end(kReach, 0, (tp > 0.0f ? (double)tp : 0.0) * kept).mass;
    kept = m < kept ? m : kept;
  }
  const float mp = a.min_p ? a.min_p[b] : 0.0f;
  if (mp > 0.0f) {
    const double least = mp < 1.0f ? (double)mp : 1.0;
    // bins before the one of least times the largest weight are kept whole
    const double x = r.c * (double)r.top + 8 * log2(least), bin = r.R - __builtin_ceil(x);
    if (bin < (double)kBins) {
      const int i = bin > 0.0 ? (int)bin : 0;
      const double m = lds.count[i + 1] > lds.count[i] ? r.end_of(kRatio, i, lds.count[i], lds.before[i], 0, least).mass
                                                       : lds.before[i];
      kept = m < kept ? m : kept;
    }
  }
  float u = a.u[b];
  u = u >= 0.0f ? (u < 1.0f ? u : 0x1.fffffep-1f) : 0.0f;
  const Ends e = r.end(kPass, 0, (double)u * kept);
  if (tid == 0) {
    a.ids[b] = e.idx;
    if (a.p) a.p[b] = (float)(e.w / kept);
  }
}

}  // namespace cia

using namespace cia;

extern "C" int64_t cia_sample_workspace_bytes(int B, int V) {
  if (B < 0 || B > CIA_SAMPLE_MAX_ROWS || V < 1 || V > CIA_SAMPLE_MAX_VOCAB) return 0;
  return 16;
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
  const SampleArgs a{logits, stride, temperature, top_k, top_p, min_p, u, ids, p, B, V};
  hipStream_t s = (hipStream_t)stream;
  if (type == CIA_LOGITS_F16)
    hipLaunchKernelGGL((k_sample<true>), dim3((unsigned)B), dim3(kSampleThreads), 0, s, a);
  else
    hipLaunchKernelGGL((k_sample<false>), dim3((unsigned)B), dim3(kSampleThreads), 0, s, a);
  return launch_status();
}
