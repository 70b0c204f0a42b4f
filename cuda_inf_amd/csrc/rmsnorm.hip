// rmsnorm.hip -- residual addition and hidden-state RMSNorm (add_f32_inplace,
// engine.cu:527-559, and rmsnorm, engine.cu:131-144) in one pass on gfx950.
//
//   hsum = h + add,   out = fp16(hsum * rsqrt(mean(hsum^2) + eps) * w)
//
// Bound by memory: 6 bytes an element, 14 with the addition.  A row stays in
// registers between its sum of squares and its outputs, so h is read once.  4096
// rows of 2048 with the addition: 27 us, 4.35 TB/s, where a large copy reaches 4.78;
// one row 2.1 us, little more than an empty launch.
#include "common.h"
#include "cuda_inf_ffn.h"

namespace cia {

struct NormArgs {
  const float* h;
  const float* add;   // or null
  const uint16_t* w;  // fp16 [H]
  float* hsum;        // h + add, or null
  uint16_t* out;
  int S, H;
  float eps;
};

// 8 consecutive elements a lane and step: two 16-byte loads, one 16-byte store
constexpr int kNormVec = 8;

__device__ __forceinline__ void norm_load(const NormArgs& a, size_t at, f32x4& u, f32x4& v) {
  u = *(const f32x4*)(a.h + at);
  v = *(const f32x4*)(a.h + at + 4);
  if (a.add) {
    u += *(const f32x4*)(a.add + at);
    v += *(const f32x4*)(a.add + at + 4);
  }
}

__device__ __forceinline__ void norm_store(const NormArgs& a, size_t at, int c, float inv, const f32x4& u,
                                           const f32x4& v) {
  const f16x8 wv = *(const f16x8*)(a.w + c);
  f16x8 o;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    o[e] = (_Float16)(u[e] * inv * (float)wv[e]);
    o[4 + e] = (_Float16)(v[e] * inv * (float)wv[4 + e]);
  }
  *(f16x8*)(a.out + at) = o;
  if (a.hsum) {
    *(f32x4*)(a.hsum + at) = u;
    *(f32x4*)(a.hsum + at + 4) = v;
  }
}

// kWaves waves a row, kSteps steps of 512 kWaves elements held in registers
// (H up to kSteps * 512 * kWaves).  block = 256: 4 / kWaves rows.  A wave a row
// while a row's 32 values a lane fit, as its sum then needs no meeting of waves.
template <int kWaves, int kSteps>
__global__ __launch_bounds__(256) void k_rmsnorm(NormArgs a) {
  __shared__ float part[4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int row = blockIdx.x * (4 / kWaves) + wave / kWaves;
  const int c0 = ((wave % kWaves) * 64 + lane) * kNormVec;
  const bool live = row < a.S;
  const size_t base = (size_t)(live ? row : 0) * a.H;
  f32x4 u[kSteps], v[kSteps];
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < kSteps; i++) {
    const int c = c0 + i * 512 * kWaves;
    u[i] = v[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (c < a.H) norm_load(a, base + c, u[i], v[i]);
  }
#pragma unroll
  for (int i = 0; i < kSteps; i++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      ss = __builtin_fmaf(u[i][e], u[i][e], ss);
      ss = __builtin_fmaf(v[i][e], v[i][e], ss);
    }
  ss = wave_sum_fast(ss);
  if constexpr (kWaves > 1) {
    if (lane == 0) part[wave] = ss;
    __syncthreads();
    ss = 0.0f;
#pragma unroll
    for (int i = 0; i < kWaves; i++) ss += part[wave / kWaves * kWaves + i];
  }
  if (!live) return;
  const float inv = 1.0f / sqrtf(ss / (float)a.H + a.eps);
#pragma unroll
  for (int i = 0; i < kSteps; i++) {
    const int c = c0 + i * 512 * kWaves;
    if (c < a.H) norm_store(a, base + c, c, inv, u[i], v[i]);
  }
}

// Rows longer than the registers: summed, then read again.  A lane's steps are added
// up in 64 bits: 65536 squares in one fp32 chain (H = 2^24) were up to 1e-3 off
// where the elements are alike, as each addition rounds the same way.  (4096 rows
// of 16384 with the addition: 225 us, 4.2 TB/s, the second read from the caches;
// with fp32 chains the same.  One row of 2^24 is one workgroup's: 5.3 ms.)
__global__ __launch_bounds__(256) void k_rmsnorm_long(NormArgs a) {
  __shared__ float part[4];
  const size_t base = (size_t)blockIdx.x * a.H;
  double sum = 0.0;
  for (int c = threadIdx.x * kNormVec; c < a.H; c += 256 * kNormVec) {
    f32x4 u, v;
    norm_load(a, base + c, u, v);
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      ss = __builtin_fmaf(u[e], u[e], ss);
      ss = __builtin_fmaf(v[e], v[e], ss);
    }
    sum += (double)ss;
  }
  const float ss = wave_sum_fast((float)sum);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = ss;
  __syncthreads();
  const float inv = 1.0f / sqrtf((part[0] + part[1] + part[2] + part[3]) / (float)a.H + a.eps);
  for (int c = threadIdx.x * kNormVec; c < a.H; c += 256 * kNormVec) {
    f32x4 u, v;
    norm_load(a, base + c, u, v);
    norm_store(a, base + c, c, inv, u, v);
  }
}

}  // namespace cia

using namespace cia;

extern "C" int cia_add_rmsnorm(const float* h, const float* add, const uint16_t* w, float eps,
                               float* hsum, uint16_t* out, int S, int H, void* stream) {
  CIA_REQUIRE(S >= 0 && S <= CIA_FFN_MAX_TOKENS && H > 0 && H <= CIA_FFN_MAX_WIDTH && H % kNormVec == 0 && eps >= 0.0f, CIA_ERR_ARG);
  if (S == 0) return CIA_OK;
  CIA_REQUIRE(h && w && out, CIA_ERR_NULL);
  CIA_REQUIRE(aligned(h, 16) && aligned(add, 16) && aligned(w, 16) && aligned(hsum, 16) && aligned(out, 16),
              CIA_ERR_ALIGN);
  const NormArgs a{h, add, w, hsum, out, S, H, eps};
  hipStream_t s = (hipStream_t)stream;
  if (H <= 2048)
    hipLaunchKernelGGL((k_rmsnorm<1, 4>), dim3((unsigned)((S + 3) / 4)), dim3(256), 0, s, a);
  else if (H <= 8192)
    hipLaunchKernelGGL((k_rmsnorm<4, 4>), dim3((unsigned)S), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(k_rmsnorm_long, dim3((unsigned)S), dim3(256), 0, s, a);
  return launch_status();
}
