// moe_int4.hip -- the experts' INT4 group-128 products (the expert loop of
// engine.cu:894-905: w1, w3, swiglu, w2, acc_scaled) on gfx950, for all the
// tokens of a call and the experts each has chosen.
//
//   up    act[s][j] = fp16(silu(g) * u),  g = W1[e] x[s], u = W3[e] x[s],
//         e = ids[s][j], silu(g) = g / (1 + exp(-g))
//   down  out[s] = res[s] + sum over j of weights[s][j] * (W2[e] act[s][j])
//
// Weights as in gemv_int4.hip: w = (nibble - 8) * scale[row][k / 128].  The
// products of a scale group are exact fp16 inputs to the matrix cores, summed
// in fp32 and scaled in fp32.
//
// A pair (s, j) is row s * k + j.  A pair whose id is not an expert's takes no
// part: its act row is left as it is, and it adds nothing to out.
#include "common.h"
#include "cuda_inf_ffn.h"

namespace cia {

constexpr int kMoeMaxE = CIA_MOE_MAX_EXPERTS;
constexpr int kMoeMaxK = CIA_MOE_MAX_TOP_K;
constexpr int kMoeMaxPairs = 1 << 24;

struct MoeArgs {
  const uint16_t* x;      // fp16: [S][K] (up), [S k][K] (down)
  const int32_t* ids;     // [S k], or null: every row is expert 0's
  const uint8_t* packed[2];  // up: W1, W3; down: W2 twice
  const uint16_t* scales[2];
  int64_t pstride[2], sstride[2];  // of an expert: bytes, elements
  int K, N;               // inputs and outputs (up: of each of the two)
  int S, k, E;
  uint16_t* act;          // up: [S k][N]
  float* y;               // down: [S k][N]
  const int* plan;        // offs[E + 1], rows[S k]
};

// ---------------------------------------------------------------- plan
// Rows by expert: offs[e] .. offs[e + 1] - 1 of rows are expert e's.  Their order
// within an expert does not matter: a row's results do not depend on its
// neighbours.
__global__ __launch_bounds__(1024) void k_moe_plan(const int32_t* ids, int P, int E, int* plan) {
  __shared__ int cnt[kMoeMaxE], at[kMoeMaxE];
  const int tid = threadIdx.x;
  if (tid < kMoeMaxE) cnt[tid] = 0;
  __syncthreads();
  for (int i = tid; i < P; i += 1024) {
    const int e = ids ? ids[i] : 0;
    if ((unsigned)e < (unsigned)E) atomicAdd(&cnt[e], 1);
  }
  __syncthreads();
  if (tid < E) {
    int o = 0;
    for (int j = 0; j < tid; j++) o += cnt[j];
    at[tid] = o;
    plan[tid] = o;
    if (tid == E - 1) plan[E] = o + cnt[tid];
  }
  __syncthreads();
  int* rows = plan + E + 1;
  for (int i = tid; i < P; i += 1024) {
    const int e = ids ? ids[i] : 0;
    if ((unsigned)e < (unsigned)E) rows[atomicAdd(&at[e], 1)] = i;
  }
}

// ---------------------------------------------------------------- products
// 8 nibbles (k even in the low one) -> 8 fp16 (nibble - 8), exact: byte b twice
// into a word, its low nibble under the exponent of 1024 and its high one, not
// shifted, 16 fold; one fma takes {1, 1/16} and the offsets back out.
__device__ __forceinline__ f16x8 nib8(uint32_t u) {
  const f16x2 mul = {(_Float16)1.0f, (_Float16)0.0625f}, off = {(_Float16)-1032.0f, (_Float16)-72.0f};
  f16x8 r;
#pragma unroll
  for (int b = 0; b < 4; b++) {
    const uint32_t t = __builtin_amdgcn_perm(u, u, 0x0C000C00u | (uint32_t)b << 16 | (uint32_t)b);
    const f16x2 h = __builtin_elementwise_fma(
        __builtin_bit_cast(f16x2, (t & 0x00F0000Fu) | 0x64006400u), mul, off);
    r[2 * b] = h[0];
    r[2 * b + 1] = h[1];
  }
  return r;
}

__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.0f + fast_exp(-g)) * u; }

// the value of the neighbouring lane (l ^ 1)
__device__ __forceinline__ float lane_pair(float v) {
  return __builtin_bit_cast(
      float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, false));
}

// Column c of a tile: up interleaves the two matrices (even W1, odd W3), so
// that a gate and its up product are in neighbouring lanes.
template <bool kUp>
struct Col {
  const uint8_t* w;
  const uint16_t* s;
  __device__ __forceinline__ Col(const MoeArgs& a, int e, int c) {
    const int m = kUp ? c & 1 : 0, n0 = kUp ? c >> 1 : c, n = n0 < a.N ? n0 : a.N - 1;
    w = (m ? a.packed[1] : a.packed[0]) + (size_t)e * (m ? a.pstride[1] : a.pstride[0]) + (size_t)n * (a.K >> 1);
    s = (m ? a.scales[1] : a.scales[0]) + (size_t)e * (m ? a.sstride[1] : a.sstride[0]) + (size_t)n * (a.K >> 7);
  }
};

// One wave: 16 rows x 32 columns, operands straight from memory.
template <bool kUp>
__global__ __launch_bounds__(64) void k_moe_simple(MoeArgs a) {
  const int l = threadIdx.x, n16 = l & 15, q = l >> 4, ng = a.K >> 7;
  const int nct = (kUp ? 2 * a.N : a.N) / 32;
  int e = 0, t = blockIdx.x / nct;
  for (; e < a.E; e++) {
    const int nt = (a.plan[e + 1] - a.plan[e] + 15) >> 4;
    if (t < nt) break;
    t -= nt;
  }
  if (e == a.E) return;
  const int r0 = a.plan[e] + 16 * t, r1 = a.plan[e + 1];
  const int* rows = a.plan + a.E + 1;
  const int ra = rows[r0 + n16 < r1 ? r0 + n16 : r1 - 1];
  const uint16_t* xr = a.x + (size_t)(kUp ? ra / a.k : ra) * a.K;
  const int c0 = blockIdx.x % nct * 32;
  f32x4 acc[2] = {};
  const Col<kUp> col[2] = {Col<kUp>(a, e, c0 + n16), Col<kUp>(a, e, c0 + 16 + n16)};
  for (int g = 0; g < ng; g++)
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const u32x4 wq = *(const u32x4*)(col[j].w + 64 * g + 16 * q);
      f32x4 p = {};
#pragma unroll
      for (int s = 0; s < 4; s++)
        p = __builtin_amdgcn_mfma_f32_16x16x32_f16(*(const f16x8*)(xr + 128 * g + 32 * q + 8 * s), nib8(wq[s]), p, 0, 0, 0);
      const float sc = h2f(col[j].s[g]);
#pragma unroll
      for (int i = 0; i < 4; i++) acc[j][i] = __builtin_fmaf(p[i], sc, acc[j][i]);
    }
#pragma unroll
  for (int j = 0; j < 2; j++) {
    const int c = c0 + 16 * j + n16;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int r = r0 + 4 * q + i;
      const float v = acc[j][i], o = lane_pair(v);
      if constexpr (kUp) {
        if (!(c & 1) && r < r1 && (c >> 1) < a.N)
          a.act[(size_t)rows[r] * a.N + (c >> 1)] = f2h(silu_mul(v, o));
      } else if (r < r1 && c < a.N) {
        a.y[(size_t)rows[r] * a.N + c] = v;
      }
    }
  }
}

// ---------------------------------------------------------------- combine
struct CombineArgs {
  const float* y;
  const int32_t* ids;
  const float* weights;  // or null: 1
  const float* res;
  float* out;
  int S, k, E, H;
};

// out = res + the k weighted rows of each token, in the order of j
__global__ __launch_bounds__(256) void k_moe_combine(CombineArgs a) {
  const int nc = (a.H + 1023) / 1024;
  const int s = blockIdx.x / nc, c = (blockIdx.x % nc * 256 + threadIdx.x) * 4;
  if (c >= a.H) return;
  f32x4 v = *(const f32x4*)(a.res + (size_t)s * a.H + c);
  for (int j = 0; j < a.k; j++) {
    const int p = s * a.k + j, e = a.ids ? a.ids[p] : 0;
    if ((unsigned)e >= (unsigned)a.E) continue;
    const float w = a.weights ? a.weights[p] : 1.0f;
    const f32x4 y = *(const f32x4*)(a.y + (size_t)p * a.H + c);
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = __builtin_fmaf(w, y[i], v[i]);
  }
  *(f32x4*)(a.out + (size_t)s * a.H + c) = v;
}

// ---------------------------------------------------------------- host
static int64_t plan_bytes(int64_t P, int E) { return ((E + 1 + P) * 4 + 255) / 256 * 256; }

static int moe_check(int S, int k, int E, int H, int F, const int32_t* ids) {
  CIA_REQUIRE(S >= 0 && k >= 1 && k <= kMoeMaxK && E >= 1 && E <= kMoeMaxE && H > 0 && F > 0 &&
                  H % 128 == 0 && F % 128 == 0 && H <= (1 << 20) && F <= (1 << 20) &&
                  (int64_t)S * k <= kMoeMaxPairs,
              CIA_ERR_ARG);
  // without ids there is nothing to choose from
  CIA_REQUIRE(ids || (E == 1 && k == 1), CIA_ERR_ARG);
  return CIA_OK;
}

// an expert's strides hold its rows
static int q4_check(const cia_q4_experts* w, int E, int64_t rows, int64_t cols) {
  CIA_REQUIRE(w && w->packed && w->scales, CIA_ERR_NULL);
  CIA_REQUIRE(aligned(w->packed, 16) && aligned(w->scales, 2) && w->packed_stride % 16 == 0, CIA_ERR_ALIGN);
  CIA_REQUIRE(E == 1 || (w->packed_stride >= rows * cols / 2 && w->scales_stride >= rows * cols / 128), CIA_ERR_ARG);
  return CIA_OK;
}

static void set_w(MoeArgs& a, int i, const cia_q4_experts* w) {
  a.packed[i] = w->packed;
  a.scales[i] = w->scales;
  a.pstride[i] = w->packed_stride;
  a.sstride[i] = w->scales_stride;
}

template <bool kUp>
static int products(MoeArgs& a, void* ws, hipStream_t s) {
  const int P = a.S * a.k;
  a.plan = (const int*)ws;
  hipLaunchKernelGGL(k_moe_plan, dim3(1), dim3(1024), 0, s, a.ids, P, a.E, (int*)ws);
  const int nv = kUp ? 2 * a.N : a.N;
  hipLaunchKernelGGL((k_moe_simple<kUp>), dim3((unsigned)(nv / 32) * (unsigned)(P / 16 + a.E)), dim3(64), 0, s, a);
  return launch_status();
}

}  // namespace cia

using namespace cia;

extern "C" int64_t cia_moe_workspace_bytes(int S, int k, int E, int H, int F) {
  if (S < 0 || k < 1 || E < 1 || H < 1 || F < 1) return 0;
  const int64_t P = (int64_t)S * k;
  return plan_bytes(P, E) + P * H * 4;
}

extern "C" int cia_moe_up_int4(const uint16_t* x, const int32_t* ids, const cia_q4_experts* w1,
                               const cia_q4_experts* w3, uint16_t* act, int S, int k, int E, int H,
                               int F, void* ws, int64_t ws_bytes, void* stream) {
  int st = moe_check(S, k, E, H, F, ids);
  if (st) return st;
  if (S == 0) return CIA_OK;
  CIA_REQUIRE(x && act && ws, CIA_ERR_NULL);
  if ((st = q4_check(w1, E, F, H)) || (st = q4_check(w3, E, F, H))) return st;
  CIA_REQUIRE(aligned(x, 16) && aligned(ids, 4) && aligned(act, 16) && aligned(ws, 16), CIA_ERR_ALIGN);
  CIA_REQUIRE(ws_bytes >= cia_moe_workspace_bytes(S, k, E, H, F), CIA_ERR_ARG);
  MoeArgs a{};
  a.x = x;
  a.ids = ids;
  set_w(a, 0, w1);
  set_w(a, 1, w3);
  a.K = H;
  a.N = F;
  a.S = S;
  a.k = k;
  a.E = E;
  a.act = act;
  return products<true>(a, ws, (hipStream_t)stream);
}

extern "C" int cia_moe_down_int4(const uint16_t* act, const int32_t* ids, const float* weights,
                                 const cia_q4_experts* w2, const float* res, float* out, int S, int k,
                                 int E, int H, int F, void* ws, int64_t ws_bytes, void* stream) {
  int st = moe_check(S, k, E, H, F, ids);
  if (st) return st;
  if (S == 0) return CIA_OK;
  CIA_REQUIRE(act && res && out && ws, CIA_ERR_NULL);
  if ((st = q4_check(w2, E, H, F))) return st;
  CIA_REQUIRE(aligned(act, 16) && aligned(ids, 4) && aligned(weights, 4) && aligned(res, 16) &&
                  aligned(out, 16) && aligned(ws, 16),
              CIA_ERR_ALIGN);
  CIA_REQUIRE(ws_bytes >= cia_moe_workspace_bytes(S, k, E, H, F), CIA_ERR_ARG);
  MoeArgs a{};
  a.x = act;
  a.ids = ids;
  set_w(a, 0, w2);
  set_w(a, 1, w2);
  a.K = F;
  a.N = H;
  a.S = S;
  a.k = k;
  a.E = E;
  a.y = (float*)((char*)ws + plan_bytes((int64_t)S * k, E));
  hipStream_t s = (hipStream_t)stream;
  if ((st = products<false>(a, ws, s))) return st;
  const CombineArgs c{a.y, ids, weights, res, out, S, k, E, H};
  hipLaunchKernelGGL(k_moe_combine, dim3((unsigned)((H + 1023) / 1024) * (unsigned)S), dim3(256), 0, s, c);
  return launch_status();
}

// ---------------------------------------------------------------- the branch
namespace {

// The pieces of a branch's scratch, each 256-byte aligned within it
struct BlockWs {
  int64_t x, ids, weights, act, moe, end;
};

BlockWs block_ws(const cia_moe* M, int S) {
  const int64_t k = M->gate ? M->gating.top_k : 1;
  const int E = M->gate ? M->gating.n_experts : 1;
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  BlockWs b;
  b.x = 0;
  b.ids = b.x + up((int64_t)S * M->H * 2);
  b.weights = b.ids + up(S * k * 4);
  b.act = b.weights + up(S * k * 4);
  b.moe = b.act + up(S * k * M->F * 2);
  b.end = b.moe + cia_moe_workspace_bytes(S, (int)k, E, M->H, M->F);
  return b;
}

}  // namespace

extern "C" int64_t cia_moe_block_workspace_bytes(const cia_moe* M, int cap) {
  if (!M || cap < 0 || M->H < 1 || M->F < 1 || (M->gate && (M->gating.top_k < 1 || M->gating.n_experts < 1)))
    return 0;
  return block_ws(M, cap).end;
}

extern "C" int cia_moe_block_forward(const cia_moe* M, float* h, int S, void* stream) {
  CIA_REQUIRE(M && h, CIA_ERR_NULL);
  CIA_REQUIRE(S >= 0 && S <= M->cap, CIA_ERR_ARG);
  if (S == 0) return CIA_OK;
  const int k = M->gate ? M->gating.top_k : 1, E = M->gate ? M->gating.n_experts : 1;
  CIA_REQUIRE(M->ws, CIA_ERR_NULL);
  CIA_REQUIRE(aligned(M->ws, 16), CIA_ERR_ALIGN);
  // all of the branch's arguments before its first launch
  int st = moe_check(S, k, E, M->H, M->F, M->gate ? (const int32_t*)M->ws : nullptr);
  if (st) return st;
  CIA_REQUIRE(M->ws_bytes >= cia_moe_block_workspace_bytes(M, S), CIA_ERR_ARG);
  if ((st = q4_check(&M->w1, E, M->F, M->H)) || (st = q4_check(&M->w3, E, M->F, M->H)) ||
      (st = q4_check(&M->w2, E, M->H, M->F)))
    return st;
  const BlockWs b = block_ws(M, S);
  char* ws = (char*)M->ws;
  uint16_t* x = (uint16_t*)(ws + b.x);
  int32_t* ids = M->gate ? (int32_t*)(ws + b.ids) : nullptr;
  float* weights = M->gate ? (float*)(ws + b.weights) : nullptr;
  uint16_t* act = (uint16_t*)(ws + b.act);
  if (M->gate && (st = cia_moe_route(x, M->gate, M->bias, &M->gating, ids, weights, nullptr, 0, M->H, stream)))
    return st;  // (no tokens: its checks alone)
  if ((st = cia_add_rmsnorm(h, nullptr, M->norm_w, M->norm_eps, nullptr, x, S, M->H, stream))) return st;
  if (M->gate && (st = cia_moe_route(x, M->gate, M->bias, &M->gating, ids, weights, nullptr, S, M->H, stream)))
    return st;
  if ((st = cia_moe_up_int4(x, ids, &M->w1, &M->w3, act, S, k, E, M->H, M->F, ws + b.moe,
                            M->ws_bytes - b.moe, stream)))
    return st;
  return cia_moe_down_int4(act, ids, weights, &M->w2, h, h, S, k, E, M->H, M->F, ws + b.moe,
                           M->ws_bytes - b.moe, stream);
}
