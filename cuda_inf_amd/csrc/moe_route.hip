// moe_route.hip -- the router of a layer of experts: logits, scores, choice of
// k experts and their weights (of engine.cu:869-905, which copies the logits to
// the host at 880 and chooses there), on the device.
//
//   l = gate x,  s = 1 / (1 + exp(-l)) or softmax(l),  c = s + bias
//   groups: those topk_group of n_group whose two best c have the largest sum
//   ids = the k largest c among the experts of those groups, largest first,
//   the lowest index first among equals;  w = s[ids]
//   renorm: w / (sum w + eps);  then times scale
//
// The experts chosen are those of logits summed in 64 bits: fp16 products are
// exact there and the order of their sum does not matter (an fp32 sum of 2048
// products is 1e-7 off, which moves a choice in one token of some 1e5), so a
// token's experts do not depend on the batch around it.  Few tokens have their sums
// in 64 bits; of many the matrix cores' fp32 sums decide where their error cannot
// matter, and 64 bits the rest.
#include "common.h"
#include "cuda_inf_ffn.h"

namespace cia {

constexpr int kRouteMaxE = CIA_MOE_MAX_EXPERTS;
constexpr int kRouteMaxK = CIA_MOE_MAX_TOP_K;

struct RouteArgs {
  const uint16_t* x;      // fp16 [S][H], or null: logits are given
  const uint16_t* gate;   // fp16 [E][H]
  const float* logits_in; // fp32 [S][E]
  const float* bias;      // fp32 [E], or null
  int32_t* ids;
  float* weights;
  float* logits;          // fp32 [S][E], or null
  int S, H, E, k, softmax, n_group, topk_group, renorm;
  float eps, scale;
};

typedef double f64x2 __attribute__((ext_vector_type(2)));
typedef double f64x4 __attribute__((ext_vector_type(4)));

// Sums and maxima over the wave without the LDS unit, in 64 bits; every lane gets
// the same value.
__device__ __forceinline__ double f64_of(uint32_t lo, uint32_t hi) {
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int kN>
__device__ __forceinline__ double row_ror_f64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  return f64_of((uint32_t)__builtin_amdgcn_mov_dpp((int)u, 0x120 + kN, 0xF, 0xF, true),
                (uint32_t)__builtin_amdgcn_mov_dpp((int)(u >> 32), 0x120 + kN, 0xF, 0xF, true));
}
// the value of the lane 16 (32) on or back
template <bool k32>
__device__ __forceinline__ f64x2 swap_f64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)u, hi = (uint32_t)(u >> 32);
  if constexpr (k32) {
    const auto a = __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
    return f64x2{f64_of(a[0], b[0]), f64_of(a[1], b[1])};
  } else {
    const auto a = __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
    const auto b = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
    return f64x2{f64_of(a[0], b[0]), f64_of(a[1], b[1])};
  }
}
template <class F>
__device__ __forceinline__ double wave_fold(double v, const F& f) {
  v = f(v, row_ror_f64<8>(v));
  v = f(v, row_ror_f64<4>(v));
  v = f(v, row_ror_f64<2>(v));
  v = f(v, row_ror_f64<1>(v));
  f64x2 r = swap_f64<false>(v);
  v = f(r[0], r[1]);
  r = swap_f64<true>(v);
  return f(r[0], r[1]);
}
__device__ __forceinline__ double wave_sum_f64(double v) {
  return wave_fold(v, [](double a, double b) { return a + b; });
}
// (of values that are numbers)
__device__ __forceinline__ double wave_max_f64(double v) {
  return wave_fold(v, [](double a, double b) { return a > b ? a : b; });
}

// A token's choice by one wave: lg, its logits in LDS; ch, E doubles of LDS for
// the wave.  Lane l has experts l, l + 64, .., kPer of them.  (A template of kPer:
// the code of experts that are not there is fetched all the same, and at a few
// tokens fetching code is much of the time.)  far: how far a logit may be off;
// where logits that near could choose otherwise, the choice is not written, and
// false returned; doubt[i] then has a bit for each expert 64 i + .. whose exact
// logit the choice needs.
template <int kPer>
__device__ __forceinline__ bool choose(const RouteArgs& a, int s, const double* lg, double* ch, double far,
                                       uint64_t* doubt) {
  const int l = threadIdx.x & 63;
  const double ninf = -__builtin_inf();
  double sc[kPer], c[kPer];
  bool bad = false;
  double m = ninf;
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    const int e = l + 64 * i;
    sc[i] = e < a.E ? lg[e] : ninf;
    if (e < a.E && a.logits) a.logits[(size_t)s * a.E + e] = (float)sc[i];
    bad = bad || sc[i] != sc[i];
    m = sc[i] > m ? sc[i] : m;
  }
  // How far a choice may be off: a sigmoid's slope is at most 1/4; a softmax moves by
  // s (dl - sum s dl), at most 2 s |dl| and its square; and what 64 bits round.
  auto off = [&](double score, double choice) __attribute__((always_inline)) {
    return (a.softmax ? 2.05 * score : 0.25) * far + 1e-14 + (choice > ninf ? 1e-15 * __builtin_fabs(choice) : 0.0);
  };
  double largest = 1.0;  // no score is above it
  bool safe = far == 0.0 || !(__any(bad) || !(far < (a.softmax ? 0.01 : 1e30)));
  if (a.softmax) {
    m = wave_max_f64(m);
    // no number among infinities (inf - inf) or beside a NaN; all -inf: scores of 0
    bad = __any(bad || m == __builtin_inf());
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      if (i > 0 && 64 * i >= a.E) break;
      sc[i] = sc[i] > ninf ? exp(sc[i] - m) : 0.0;
      sum += sc[i];
    }
    sum = wave_sum_f64(sum);
    largest = 1.0 / sum;  // (the largest logit's)
#pragma unroll
    for (int i = 0; i < kPer; i++) sc[i] = bad ? __builtin_nan("") : (sum == 0.0 ? 0.0 : sc[i] / sum);
  } else {
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      if (i > 0 && 64 * i >= a.E) break;
      sc[i] = 1.0 / (1.0 + exp(-sc[i]));
    }
  }
  // a choice that is not a number ranks with the last
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    const int e = l + 64 * i;
    c[i] = ninf;
    if (e < a.E) {
      c[i] = sc[i] + (a.bias ? (double)a.bias[e] : 0.0);
      if (c[i] != c[i]) c[i] = ninf;
      ch[e] = c[i];
    }
  }
  uint32_t real = 0;  // bit i: there is an expert l + 64 i
#pragma unroll
  for (int i = 0; i < kPer; i++) real |= (l + 64 * i < a.E ? 1u : 0u) << i;
  uint32_t in = real;     // that may be chosen
  uint32_t again = real;  // that may turn out to be, where the choice is in doubt
  bool groups_safe = true;
  if (a.n_group > 1) {
    // lane l has groups l, l + 64, ..: the sum of a group's two best choices
    const int per = a.E / a.n_group;
    double best[kPer];
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const int g = l + 64 * i;
      double b0 = ninf, b1 = ninf;
      if (g < a.n_group)
#pragma unroll 8
        for (int j = 0; j < per; j++) {
          const double v = ch[g * per + j];
          b1 = v > b0 ? b0 : (v > b1 ? v : b1);
          b0 = v > b0 ? v : b0;
        }
      best[i] = per > 1 ? b0 + b1 : b0;
      if (best[i] != best[i]) best[i] = ninf;
    }
    // (the choices are read: their place takes the groups' sums, then which are in)
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < kPer; i++)
      if (l + 64 * i < a.n_group) ch[l + 64 * i] = best[i];
    uint32_t keep = 0, open = 0;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const int g = l + 64 * i;
      if (64 * i >= a.n_group) break;
      int rank = 0, sure = 0;  // groups that are before it, and that are so for sure
      bool near = false;       // another group's sum of two
      const double o = 4.0 * off(largest, best[i]);
#pragma unroll 8
      for (int j = 0; j < a.n_group; j++) {
        rank += ch[j] > best[i] || (ch[j] == best[i] && j < g);
        sure += ch[j] - best[i] > o;
        near = near || (j != g && __builtin_fabs(ch[j] - best[i]) <= o);
      }
      keep |= (g < a.n_group && rank < a.topk_group ? 1u : 0u) << i;
      open |= (g < a.n_group && sure < a.topk_group ? 1u : 0u) << i;
      // (only the last one in and the first one out matter)
      if (far != 0.0)
        groups_safe = groups_safe && !__any(g < a.n_group && near && rank >= a.topk_group - 1 && rank <= a.topk_group);
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < kPer; i++)
      if (l + 64 * i < a.n_group) ch[l + 64 * i] = keep >> i & 1 ? 2.0 : open >> i & 1 ? 1.0 : 0.0;
    in = again = 0;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const double of = l + 64 * i < a.E ? ch[(l + 64 * i) / per] : 0.0;
      in |= (of == 2.0 ? 1u : 0u) << i;
      again |= (of != 0.0 ? 1u : 0u) << i;
    }
    if (groups_safe) again = in;
  }
  // Beside a bias the distance of two scores hangs on the sum over all experts.  Where
  // the groups are in doubt, all of those that are not out for sure are looked at
  // again: the last one kept is then compared with exact sums, or with sums that stay
  // below it by more than they may be off.
  if (!safe || (a.softmax && a.bias)) again = real;
  safe = safe && groups_safe;
  const bool all = !safe || (a.softmax && a.bias);  // of again are in doubt, if any
  // k rounds (and one more for how near the next one is): the best choice left, the
  // lowest index among equals; lane j keeps round j's
  int id = 0;
  double w = 0.0, above = __builtin_inf(), above_off = 0.0;
  for (int j = 0; j < a.k + (far != 0.0 ? 1 : 0); j++) {
    double v = ninf;
#pragma unroll
    for (int i = 0; i < kPer; i++)
      if (in >> i & 1 && c[i] > v) v = c[i];
    const double top = wave_max_f64(v);
    uint64_t at = 0;
    int wi = 0;
    double vs = 0.0;
#pragma unroll
    for (int i = kPer - 1; i >= 0; i--) {
      const uint64_t b = __ballot(in >> i & 1 && c[i] == top);
      if (b) {
        at = b;
        wi = i;
        vs = sc[i];
      }
    }
    if (!at) break;  // (the choice was all of them)
    const int lane = __builtin_ctzll(at);
    const uint64_t u = __builtin_bit_cast(uint64_t, vs);
    const double ws = f64_of((uint32_t)__builtin_amdgcn_readlane((int)u, lane),
                             (uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), lane));
    if (far != 0.0) {
      const double o = off(ws, top);
      safe = safe && !(above - top <= above_off + o);
      above = top;
      above_off = o;
      if (j == a.k) break;
    }
    if (l == lane) in &= ~(1u << wi);
    if (l == j) {
      id = lane + 64 * wi;
      w = ws;
    }
  }
  if (!safe) {
    // what is sure to stay below the last one looked at is not in doubt
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const uint64_t b = __ballot(again >> i & 1 && (all || !(c[i] + off(sc[i], c[i]) < above - above_off)));
      if (l == 0) doubt[i] = b;
    }
    return false;
  }
  double f = (double)a.scale;
  if (a.renorm) {
    const double sum = wave_sum_f64(l < a.k ? w : 0.0) + (double)a.eps;
    f = sum == 0.0 ? 0.0 : f / sum;
  }
  if (l < a.k) {
    a.ids[(size_t)s * a.k + l] = id;
    a.weights[(size_t)s * a.k + l] = (float)(w * f);
  }
  return true;
}

// Few tokens: kT a workgroup, its waves every 8th (of many experts every 16th)
// expert each, so that a token's gate is read by all of a compute unit.  x lies in
// LDS in 64 bits, a lane's 8 elements in four 16-byte pieces kSpan / 8 lanes apart.
//   Bound by what the conversions to 64 bits and their products take of a compute
// unit, and by latency: a token of 32 experts, H = 2048, 6.5 us, 300 of 128, H =
// 1280, in 8 groups, 18.8 us a call (20.8 with 8 waves; of 32 experts 16 waves take
// 10.1 instead of 8.3).
constexpr int tok_waves(int kT, int kPer) { return kT <= 2 && kPer > 1 ? 16 : 8; }

template <int kT, int kPer>
__global__ __launch_bounds__(64 * tok_waves(kT, kPer)) void k_route_tok(RouteArgs a) {
  constexpr int kTokWaves = tok_waves(kT, kPer);
  constexpr int kSpan = 4096 / kT;  // elements of a row in LDS at a time
  __shared__ f64x2 xs[kT][4][kSpan / 8];
  __shared__ double lg[kT][kRouteMaxE];
  __shared__ double ch[kT][kRouteMaxE];
  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, s0 = blockIdx.x * kT;
  if (kT <= 2 && a.x) {  // (8 tokens bring their logits)
    for (int h0 = 0; h0 < a.H; h0 += kSpan) {
      const int n8 = (a.H - h0 < kSpan ? a.H - h0 : kSpan) / 8;
      if (h0) __syncthreads();
      for (int i = tid; i < kT * n8; i += 64 * kTokWaves) {
        const int t = kT > 1 ? i / n8 : 0, c = i - t * n8;
        const int s = s0 + t < a.S ? s0 + t : a.S - 1;
        const f16x8 v = *(const f16x8*)(a.x + (size_t)s * a.H + h0 + 8 * c);
#pragma unroll
        for (int p = 0; p < 4; p++) xs[t][p][c] = f64x2{(double)(float)v[2 * p], (double)(float)v[2 * p + 1]};
      }
      __syncthreads();
      // 4 experts at a time, w, w + 8, .., a step's 8 elements of each fetched a
      // step ahead, across experts too
      const int steps = (n8 + 63) / 64, rounds = (a.E + 4 * kTokWaves - 1) / (4 * kTokWaves);
      f16x8 g[4], gn[4];
      auto fetch = [&](int round, int step, f16x8 (&o)[4]) __attribute__((always_inline)) {
        const int c = 64 * step + l;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int e = 4 * kTokWaves * round + kTokWaves * j + w;
          o[j] = *(const f16x8*)(a.gate + (size_t)(e < a.E ? e : a.E - 1) * a.H + h0 + 8 * (c < n8 ? c : n8 - 1));
        }
      };
      fetch(0, 0, gn);
      for (int round = 0; round < rounds; round++) {
        double acc[kT][4][2] = {};
        for (int step = 0; step < steps; step++) {
#pragma unroll
          for (int j = 0; j < 4; j++) g[j] = gn[j];
          const bool last = step + 1 == steps;
          if (!last || round + 1 < rounds) fetch(last ? round + 1 : round, last ? 0 : step + 1, gn);
          const int c = 64 * step + l;
          if (c < n8)
#pragma unroll
            for (int p = 0; p < 4; p++) {
              f64x2 xv[kT];
#pragma unroll
              for (int t = 0; t < kT; t++) xv[t] = xs[t][p][c];
#pragma unroll
              for (int j = 0; j < 4; j++) {
                const double g0 = (double)(float)g[j][2 * p], g1 = (double)(float)g[j][2 * p + 1];
#pragma unroll
                for (int t = 0; t < kT; t++) {
                  acc[t][j][0] = __builtin_fma(xv[t][0], g0, acc[t][j][0]);
                  acc[t][j][1] = __builtin_fma(xv[t][1], g1, acc[t][j][1]);
                }
              }
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int e = 4 * kTokWaves * round + kTokWaves * j + w;
#pragma unroll
          for (int t = 0; t < kT; t++) {
            const double v = wave_sum_f64(acc[t][j][0] + acc[t][j][1]);
            if (l == 0 && e < a.E) lg[t][e] = h0 ? lg[t][e] + v : v;
          }
        }
      }
    }
    __syncthreads();
  } else {
    for (int i = tid; i < kT * a.E; i += 64 * kTokWaves) {
      const int t = i / a.E, e = i - t * a.E;
      lg[t][e] = s0 + t < a.S ? (double)a.logits_in[(size_t)(s0 + t) * a.E + e] : 0.0;
    }
    __syncthreads();
  }
  if (w < kT && s0 + w < a.S) choose<kPer>(a, s0 + w, lg[w], ch[w], 0.0, nullptr);
}

// More tokens: 16 a workgroup on the fp16 matrix cores, 16 experts a tile, the 16
// waves a part of H each.  32 products are summed in fp32, the rest in 64 bits; a
// second product, of the magnitudes, bounds what the fp32 sums have lost.  Tokens
// whose choice hangs on that (1 of 200 of 32 experts, H = 2048) have the logits that
// it hangs on taken again, in 64 bits, by all the waves; the others' logits and weights
// keep the fp32 sums' accuracy (4096 tokens: 5.1e-8 off on average, 2.7e-8 where the
// sums are in 64 bits and only rounded).
// (4096 tokens of 32 experts, H = 2048: 16.4 us on the 64-bit matrix cores.)
constexpr int kTileToks = 16, kMfmaWaves = 16;

template <int kPer>
__global__ __launch_bounds__(64 * kMfmaWaves) void k_route_mfma(RouteArgs a) {
  constexpr int kTiles = 2, kAhead = 4;  // tiles of experts at a time, steps whose operands are fetched together
  __shared__ double part[kMfmaWaves][kTiles][256];  // in the end the waves' choices
  __shared__ double lg[kTileToks][kRouteMaxE];
  __shared__ u32x4 stage[kMfmaWaves][1 + kTiles][64];
  __shared__ float mag[kMfmaWaves][kTileToks];
  __shared__ int again;  // bit t: token t
  __shared__ uint64_t doubt[kTileToks][kPer];
  static_assert(kTiles * 256 >= kRouteMaxE && kTileToks == kMfmaWaves, "a wave's choices; a wave a token");
  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, r16 = l & 15, q = l >> 4;
  const int s0 = blockIdx.x * kTileToks;
  const int n32 = (a.H + 31) / 32;  // steps of 32 elements
  // Operands are fetched 4 lanes to a row's 64 bytes (16 bytes a lane in rows of
  // their own take four times as long) and change lanes in the wave's LDS.
  const int row = l >> 2, to = (l & ~3) | ((l & 3) ^ ((l >> 4) & 3)), from = 4 * r16 + (q ^ ((r16 >> 2) & 3));
  const uint16_t* const xr = a.x + (size_t)(s0 + row < a.S ? s0 + row : a.S - 1) * a.H;
  if (tid == 0) again = 0;
  f32x4 most = {};  // of this wave's sums of magnitudes, tokens 4q .. 4q + 3
  for (int e0 = 0; e0 < a.E; e0 += 16 * kTiles) {
    double acc[kTiles][4] = {};
    f32x4 mags[kTiles] = {};
    const uint16_t* gr[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; t++) {
      const int e = e0 + 16 * t + row;
      gr[t] = a.gate + (size_t)(e < a.E ? e : a.E - 1) * a.H;
    }
    auto abs8 = [](f16x8 v) __attribute__((always_inline)) {
      u32x4 u = __builtin_bit_cast(u32x4, v);
#pragma unroll
      for (int i = 0; i < 4; i++) u[i] &= 0x7FFF7FFFu;
      return __builtin_bit_cast(f16x8, u);
    };
    for (int i0 = w; i0 < n32; i0 += kMfmaWaves * kAhead) {
      u32x4 x[kAhead], g[kAhead][kTiles];
#pragma unroll
      for (int i = 0; i < kAhead; i++) {
        // (elements past H: the last ones of the row, and zeros for them)
        const int k0 = 32 * (i0 + kMfmaWaves * i) + 8 * (l & 3), k = k0 < a.H ? k0 : a.H - 8;
        x[i] = *(const u32x4*)(xr + k);
#pragma unroll
        for (int t = 0; t < kTiles; t++) g[i][t] = *(const u32x4*)(gr[t] + k);
      }
#pragma unroll
      for (int i = 0; i < kAhead; i++) {
        const bool in = 32 * (i0 + kMfmaWaves * i) + 8 * (l & 3) < a.H;
        stage[w][0][to] = in ? x[i] : u32x4{0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < kTiles; t++) stage[w][1 + t][to] = in ? g[i][t] : u32x4{0, 0, 0, 0};
        const f16x8 xi = __builtin_bit_cast(f16x8, stage[w][0][from]);
#pragma unroll
        for (int t = 0; t < kTiles; t++) {
          const f16x8 gi = __builtin_bit_cast(f16x8, stage[w][1 + t][from]);
          const f32x4 p = __builtin_amdgcn_mfma_f32_16x16x32_f16(xi, gi, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
          mags[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(abs8(xi), abs8(gi), mags[t], 0, 0, 0);
#pragma unroll
          for (int j = 0; j < 4; j++) acc[t][j] += (double)p[j];
        }
      }
    }
    // lane holds tokens 4q + j, j = 0 .. 3, of expert r16
#pragma unroll
    for (int t = 0; t < kTiles; t++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        part[w][t][16 * (4 * q + j) + r16] = acc[t][j];
        most[j] = mags[t][j] > most[j] ? mags[t][j] : most[j];
      }
    __syncthreads();
    for (int i = tid; i < 256 * kTiles; i += 64 * kMfmaWaves) {
      const int t = i >> 8, j = i & 255, e = e0 + 16 * t + (j & 15);
      double v = 0.0;
#pragma unroll
      for (int k = 0; k < kMfmaWaves; k++) v += part[k][t][j];
      if (e < a.E) lg[j >> 4][e] = v;
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < 4; j++) {
    float v = most[j];
    v = __builtin_fmaxf(v, row_ror<8>(v));
    v = __builtin_fmaxf(v, row_ror<4>(v));
    v = __builtin_fmaxf(v, row_ror<2>(v));
    v = __builtin_fmaxf(v, row_ror<1>(v));
    if (r16 == 0) mag[w][4 * q + j] = v;
  }
  __syncthreads();
  // A step's 32 additions lose at most half an fp32 step each of the magnitudes'
  // sum; twice that, as the magnitudes' sums lose as much.  (What is no number shows
  // in the logits.)
  double far = 0.0;
#pragma unroll
  for (int k = 0; k < kMfmaWaves; k++) far += (double)mag[k][w];
  far *= 0x1p-18;
  bool todo = s0 + w < a.S;
  for (int pass = 0;; pass++) {  // (all waves take the same turns)
    if (todo && !choose<kPer>(a, s0 + w, lg[w], part[w][0], far, doubt[w]) && l == 0) atomicOr(&again, 1 << w);
    __syncthreads();
    const int bits = again;
    if (pass == 1 || !bits) break;
    for (int left = bits; left; left &= left - 1) {
      const int t = __builtin_ctz(left);
      const uint16_t* xt = a.x + (size_t)(s0 + t) * a.H;
      uint64_t of[kPer];
#pragma unroll
      for (int i = 0; i < kPer; i++) of[i] = doubt[t][i];
      // the n-th of them is wave n's
      auto take = [&](int n) __attribute__((always_inline)) {
        int e = -1;
#pragma unroll
        for (int i = 0; i < kPer; i++) {
          const int c = __popcll(of[i]);
          if (e < 0 && n >= 0 && n < c) {
            uint64_t b = of[i];
            for (int k = 0; k < n; k++) b &= b - 1;
            e = 64 * i + __builtin_ctzll(b);
          }
          n -= c;
        }
        return e;
      };
      for (int n = w, e; (e = take(n)) >= 0; n += kMfmaWaves) {
        const uint16_t* gr = a.gate + (size_t)e * a.H;
        double v = 0.0;
#pragma unroll 4
        for (int c = 8 * l; c < a.H; c += 512) {
          const f16x8 xv = *(const f16x8*)(xt + c), gv = *(const f16x8*)(gr + c);
#pragma unroll
          for (int j = 0; j < 8; j++) v = __builtin_fma((double)(float)xv[j], (double)(float)gv[j], v);
        }
        v = wave_sum_f64(v);
        if (l == 0) lg[t][e] = v;
      }
    }
    __syncthreads();
    todo = todo && bits >> w & 1;
    far = 0.0;
  }
}

template <int kPer>
static void route_launch(const RouteArgs& a, hipStream_t s) {
  // Calls in us, 1 token a workgroup / 2 / 16 in tiles: 32 experts, H = 2048, 256
  // tokens 8.1 / 9.2 / 13.9, 512 10.1 / 9.1 / 14.0, 1024 15.7 / 12.2 / 14.1, 2048
  // 26.3 / 20.6 / 15.6; 128 experts, H = 1280, 256 15.0 / 18.3 / 28.3, 512 22.8 /
  // 19.1 / 28.5, 1024 36.3 / 28.9 / 29.0, 2048 65 / 50 / 30.  (256 experts, H = 4096, 512
  // tokens 64, 1024 123, and 1100 in tiles 86: for so many the border lies too high.)
  if (a.x && a.S > 1024)
    hipLaunchKernelGGL(k_route_mfma<kPer>, dim3((unsigned)((a.S + kTileToks - 1) / kTileToks)), dim3(64 * kMfmaWaves), 0, s, a);
  else if (!a.x && a.S >= 64)  // (nothing but the choice: a wave a token)
    hipLaunchKernelGGL((k_route_tok<8, kPer>), dim3((unsigned)((a.S + 7) / 8)), dim3(64 * tok_waves(8, kPer)), 0, s, a);
  else if (a.S <= 256)
    hipLaunchKernelGGL((k_route_tok<1, kPer>), dim3((unsigned)a.S), dim3(64 * tok_waves(1, kPer)), 0, s, a);
  else
    hipLaunchKernelGGL((k_route_tok<2, kPer>), dim3((unsigned)((a.S + 1) / 2)), dim3(64 * tok_waves(2, kPer)), 0, s, a);
}

static int route_run(const RouteArgs& a, hipStream_t s) {
  if (a.E <= 64)
    route_launch<1>(a, s);
  else
    route_launch<kRouteMaxE / 64>(a, s);
  return launch_status();
}

// the choice's parameters into a; CIA_ERR_ARG where they contradict each other
static int route_args(RouteArgs& a, const cia_moe_gating* g, int S) {
  CIA_REQUIRE(g, CIA_ERR_NULL);
  CIA_REQUIRE(g->n_experts >= 1 && g->n_experts <= kRouteMaxE && g->top_k >= 1 && g->top_k <= kRouteMaxK &&
                  g->top_k <= g->n_experts && S >= 0 && S <= CIA_FFN_MAX_TOKENS,
              CIA_ERR_ARG);
  CIA_REQUIRE(g->score == CIA_SCORE_SIGMOID || g->score == CIA_SCORE_SOFTMAX, CIA_ERR_ARG);
  CIA_REQUIRE(g->n_group >= 1 && g->n_experts % g->n_group == 0 && g->topk_group >= 1 &&
                  g->topk_group <= g->n_group && g->n_experts / g->n_group * g->topk_group >= g->top_k,
              CIA_ERR_ARG);
  CIA_REQUIRE(g->eps >= 0.0f && g->eps < __builtin_inff() && g->scale - g->scale == 0.0f, CIA_ERR_ARG);
  a.S = S;
  a.E = g->n_experts;
  a.k = g->top_k;
  a.softmax = g->score == CIA_SCORE_SOFTMAX;
  a.n_group = g->n_group;
  a.topk_group = g->topk_group;
  a.renorm = g->renorm != 0;
  a.eps = g->eps;
  a.scale = g->scale;
  return CIA_OK;
}

}  // namespace cia

using namespace cia;

extern "C" int cia_moe_route(const uint16_t* x, const uint16_t* gate, const float* bias,
                             const cia_moe_gating* g, int32_t* ids, float* weights, float* logits,
                             int S, int H, void* stream) {
  RouteArgs a{};
  const int st = route_args(a, g, S);
  if (st) return st;
  CIA_REQUIRE(H > 0 && H <= CIA_FFN_MAX_WIDTH && H % 8 == 0, CIA_ERR_ARG);
  if (S == 0) return CIA_OK;
  CIA_REQUIRE(x && gate && ids && weights, CIA_ERR_NULL);
  CIA_REQUIRE(aligned(x, 16) && aligned(gate, 16) && aligned(bias, 4) && aligned(ids, 4) &&
                  aligned(weights, 4) && aligned(logits, 4),
              CIA_ERR_ALIGN);
  a.x = x;
  a.gate = gate;
  a.bias = bias;
  a.ids = ids;
  a.weights = weights;
  a.logits = logits;
  a.H = H;
  return route_run(a, (hipStream_t)stream);
}

extern "C" int cia_moe_select(const float* logits, const float* bias, const cia_moe_gating* g,
                              int32_t* ids, float* weights, int S, void* stream) {
  RouteArgs a{};
  const int st = route_args(a, g, S);
  if (st) return st;
  if (S == 0) return CIA_OK;
  CIA_REQUIRE(logits && ids && weights, CIA_ERR_NULL);
  CIA_REQUIRE(aligned(logits, 4) && aligned(bias, 4) && aligned(ids, 4) && aligned(weights, 4), CIA_ERR_ALIGN);
  a.logits_in = logits;
  a.bias = bias;
  a.ids = ids;
  a.weights = weights;
  return route_run(a, (hipStream_t)stream);
}
