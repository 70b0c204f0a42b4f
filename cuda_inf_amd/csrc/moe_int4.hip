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
  const int* plan;        // offs[E + 1], tiles, (expert, first) of each, rows[S k]
  int splits;             // down: parts of K, each into its own y
};

// Rows of a row tile.  The plan lists the tiles: expert e's are its rows 128 at a time.
constexpr int kTileRows = 128;

// The most row tiles P pairs of E experts can make
__host__ __device__ constexpr int64_t max_tiles(int64_t P, int E) { return P / kTileRows + (P < E ? P : E); }
__host__ __device__ constexpr int64_t plan_rows_at(int64_t P, int E) { return E + 2 + 2 * max_tiles(P, E); }

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
    int o = 0, t = 0;
    for (int j = 0; j < tid; j++) {
      o += cnt[j];
      t += (cnt[j] + kTileRows - 1) / kTileRows;
    }
    at[tid] = o;
    plan[tid] = o;
    for (int i = 0; i < cnt[tid]; i += kTileRows, t++) {
      plan[E + 2 + 2 * t] = tid;
      plan[E + 3 + 2 * t] = o + i;
    }
    if (tid == E - 1) {
      plan[E] = o + cnt[tid];
      plan[E + 1] = t;
    }
  }
  __syncthreads();
  int* rows = plan + plan_rows_at(P, E);
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

// The product is rounded to fp32 before its caller rounds it to fp16.  (Left to
// itself the compiler multiplies and converts in one instruction at some places
// and in two at others, and a row's bits would depend on its place in a tile.)
__device__ __forceinline__ float silu_mul(float g, float u) {
  float v = g / (1.0f + fast_exp(-g)) * u;
  asm("" : "+v"(v));
  return v;
}

// the value of the neighbouring lane (l ^ 1)
__device__ __forceinline__ float lane_pair(float v) {
  return __builtin_bit_cast(
      float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, false));
}

// A kernel argument as a scalar value.  (Left visible, the choice below between
// the two matrices' arguments becomes a choice of address in the argument
// segment, and a vector load from it.)
template <class T>
__device__ __forceinline__ T arg(T v) {
  uint64_t u = (uint64_t)v;
  asm("" : "+s"(u));
  return (T)u;
}

// Column c of a tile: up interleaves the two matrices (even W1, odd W3), so
// that a gate and its up product are in neighbouring lanes.
template <bool kUp>
struct Col {
  const uint8_t* w;
  const uint16_t* s;
  __device__ __forceinline__ Col(const MoeArgs& a, int e, int c) {
    const int n0 = kUp ? c >> 1 : c, n = n0 < a.N ? n0 : a.N - 1;
    const uint8_t* w0 = arg(a.packed[0]) + (size_t)e * a.pstride[0];
    const uint16_t* s0 = arg(a.scales[0]) + (size_t)e * a.sstride[0];
    if constexpr (kUp) {
      const uint8_t* w1 = arg(a.packed[1]) + (size_t)e * arg(a.pstride[1]);
      const uint16_t* s1 = arg(a.scales[1]) + (size_t)e * arg(a.sstride[1]);
      w0 = c & 1 ? w1 : w0;
      s0 = c & 1 ? s1 : s0;
    }
    w = w0 + (size_t)n * (a.K >> 1);
    s = s0 + (size_t)n * (a.K >> 7);
  }
};

// ---------------------------------------------------------------- tiles
// Many rows an expert: a workgroup of 8 waves computes 128 rows x (128 kNT)
// columns, a wave all the rows of its own 16 kNT columns, so that a dequantised
// operand serves 128 rows and no column is dequantised twice.  The K loop runs
// over the scale groups in two LDS slots, filled by DMA one group ahead:
//   X  128 rows x 16 chunks of 16 bytes, fetched from the rows of the tile
//      wherever they are (a row's address is the lane's own).  Row r's chunk c at
//      c ^ xsw(r): a 16-byte read is served 32 lanes, 512 bytes of banks, at a
//      time, and so reaches 32 different places.
//   W  each wave's own columns, 4 chunks of nibbles; column c's chunk q at
//      q ^ ((c >> 2) & 3).
// Inside a group lane q = l >> 4 of an operand holds k = 32q + 8s .. + 7 at step
// s, so one 16-byte read brings a column's nibbles for all four steps.
// Scales lie in an LDS table, filled once for up to kTabGroups groups.
typedef __attribute__((address_space(3))) void lds_void_t;
typedef __attribute__((address_space(1))) void gbl_void_t;

constexpr int kTileWaves = 8;
constexpr int kTabGroups = 32;

__device__ __forceinline__ int xsw(int r) { return ((r >> 1) & 3) | ((r & 1) << 2) | (r & 8); }

__device__ __forceinline__ void dma16(const void* src, void* dst) {
  __builtin_amdgcn_global_load_lds((gbl_void_t*)src, (lds_void_t*)dst, 16, 0, 0);
}

template <bool kUp, int kNT>
struct Tile {
  static constexpr int kCols = 16 * kNT;  // of a wave
  static constexpr int kX = kTileRows * 256, kW = kTileWaves * kCols * 64, kSlot = kX + kW;
  static constexpr int kTab = kTileWaves * kTabGroups * kCols * 2;
  static constexpr int kLds = 2 * kSlot + kTab + kTileRows * 4;
};

// A lane's DMA sources in group 0
template <int kNT>
struct TileSrc {
  const uint8_t *x0, *x1, *x2, *x3, *w0, *w1, *w2;
  __device__ __forceinline__ const uint8_t* x(int t) const { return t == 0 ? x0 : t == 1 ? x1 : t == 2 ? x2 : x3; }
  __device__ __forceinline__ const uint8_t* w(int t) const { return t == 0 ? w0 : t == 1 ? w1 : w2; }
};

template <bool kUp, int kNT, int kPR>
__device__ __forceinline__ void tile_fetch(uint8_t* slot, const TileSrc<kNT>& src, int w, int g) {
  using T = Tile<kUp, kNT>;
#pragma unroll
  for (int t = 0; t < 4; t++)
    if (kPR == 4 || 16 * w + 4 * t < 32 * kPR) dma16(src.x(t) + 256 * (size_t)g, slot + (4 * w + t) * 1024);
#pragma unroll
  for (int t = 0; t < kNT; t++)
    dma16(src.w(t) + 64 * (size_t)g, slot + T::kX + w * T::kCols * 64 + t * 1024);
}

// One scale group: group g + 1 (if more) is fetched into next while cur is
// multiplied.
template <bool kUp, int kNT, int kPR>
__device__ __forceinline__ void tile_group(const uint8_t* cur, uint8_t* next, const uint16_t* scales, const TileSrc<kNT>& src, int w, int g,
                                           bool more, f32x4 (&C)[2 * kPR][kNT]) {
  using T = Tile<kUp, kNT>;
  const int l = threadIdx.x & 63, n16 = l & 15, q = l >> 4;
  if (more) tile_fetch<kUp, kNT, kPR>(next, src, w, g + 1);
  const uint16_t* xs = (const uint16_t*)cur + n16 * 128;
  const uint8_t* ws = cur + T::kX + w * T::kCols * 64;
  // Units of two row tiles x two k steps: a unit's x operands are requested
  // before the products of the unit before it.
  f16x8 A[2][4];
  auto load_a = [&](int u, f16x8 (&o)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int s = 0; s < 2; s++)
        o[2 * i + s] = *(const f16x8*)(xs + 16 * (2 * (u >> 1) + i) * 128 + 8 * ((4 * q + 2 * (u & 1) + s) ^ xsw(n16)));
  };
  u32x4 wq[kNT];
  float scl[kNT];
#pragma unroll
  for (int j = 0; j < kNT; j++) {
    const int c = 16 * j + n16;
    wq[j] = *(const u32x4*)(ws + c * 64 + 16 * (q ^ ((c >> 2) & 3)));
    scl[j] = h2f(scales[c]);
  }
  load_a(0, A[0]);
  f16x8 B[kNT][4];
  f32x4 P[2][2][kNT];  // of a pair of row tiles, and of the pair before
  auto scale_add = [&](int pr) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int j = 0; j < kNT; j++)
#pragma unroll
        for (int r = 0; r < 4; r++)
          C[2 * pr + i][j][r] = __builtin_fmaf(P[pr & 1][i][j][r], scl[j], C[2 * pr + i][j][r]);
  };
#pragma unroll
  for (int u = 0; u < 2 * kPR; u++) {
    if (u + 1 < 2 * kPR) load_a(u + 1, A[(u + 1) & 1]);
    __builtin_amdgcn_sched_barrier(0);
    const int s0 = 2 * (u & 1), pr = u >> 1;
    if (u < 2)
#pragma unroll
      for (int j = 0; j < kNT; j++) {
        B[j][s0] = nib8(wq[j][s0]);
        B[j][s0 + 1] = nib8(wq[j][s0 + 1]);
      }
#pragma unroll
    for (int s = 0; s < 2; s++)
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < kNT; j++)
          P[pr & 1][i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
              A[u & 1][2 * i + s], B[j][s0 + s], s0 + s == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : P[pr & 1][i][j], 0, 0, 0);
    // the pair before is scaled between this pair's first products
    if (pr > 0 && (u & 1) == 0) {
      scale_add(pr - 1);
#pragma unroll
      for (int k = 0; k < 4 * kNT; k++) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // one MFMA
        __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);  // two vector instructions
      }
    }
  }
  scale_add(kPR - 1);
}

// The K loop of a tile of up to 32 kPR rows
template <bool kUp, int kNT, int kPR>
__device__ __forceinline__ void tile_loop(const MoeArgs& a, uint8_t* lds, uint16_t* tab, TileSrc<kNT> src, int e, int c0,
                                          int g0, int g1, f32x4 (&C)[2 * kPR][kNT]) {
  using T = Tile<kUp, kNT>;
  const int l = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  tile_fetch<kUp, kNT, kPR>(lds, src, w, g0);
#pragma unroll
  for (int i = 0; i < 2 * kPR; i++)
#pragma unroll
    for (int j = 0; j < kNT; j++) C[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int g = g0; g < g1; g++) {
    const int i = g - g0, slot = (i & 1) * T::kSlot;
    if (i % kTabGroups == 0)  // this wave's scales of the next groups
      for (int k = l; k < T::kCols * kTabGroups; k += 64) {
        const int c = k / kTabGroups, gg = g + k % kTabGroups;
        if (gg < g1) tab[(k % kTabGroups) * T::kCols + c] = Col<kUp>(a, e, c0 + c).s[gg];
      }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0): this wave's DMA and scales landed
    __builtin_amdgcn_s_barrier();        // every wave's did; the other slot is read
    asm volatile("" ::: "memory");
    tile_group<kUp, kNT, kPR>(lds + slot, lds + (T::kSlot - slot), tab + i % kTabGroups * T::kCols, src, w, g,
                              g + 1 < g1, C);
  }
}

template <bool kUp, int kNT, int kPR>
__device__ __forceinline__ void tile_run(const MoeArgs& a, uint8_t* lds, uint16_t* tab, TileSrc<kNT> src,
                                         const int* rows, int nrows, int e, int c0,
                                         int g0, int g1, float* y) {
  const int l = threadIdx.x & 63, n16 = l & 15, q = l >> 4;
  f32x4 C[2 * kPR][kNT];
  tile_loop<kUp, kNT, kPR>(a, lds, tab, src, e, c0, g0, g1, C);
  // lane holds rows 4q .. 4q + 3 of row tile i, column n16 of column tile j
#pragma unroll
  for (int i = 0; i < 2 * kPR; i++) {
    auto row = [&](int r) __attribute__((always_inline)) {
      const int t = 16 * i + 4 * q + r;
      return t < nrows ? rows[t] : -1;
    };
    const int p0 = row(0), p1 = row(1), p2 = row(2), p3 = row(3);
#pragma unroll
    for (int j = 0; j < kNT; j++) {
      const int c = c0 + 16 * j + n16;
      const f32x4 v = C[i][j];
      if constexpr (kUp) {
        // the even lane takes rows 0 and 1 of the pair's column, the odd one 2, 3
        const bool odd = c & 1;
        const int n = c >> 1, pa = odd ? p2 : p0, pb = odd ? p3 : p1;
        const float o0 = lane_pair(v[0]), o1 = lane_pair(v[1]), o2 = lane_pair(v[2]), o3 = lane_pair(v[3]);
        const float va = silu_mul(odd ? o2 : v[0], odd ? v[2] : o0), vb = silu_mul(odd ? o3 : v[1], odd ? v[3] : o1);
        if (n < a.N) {
          if (pa >= 0) a.act[(size_t)pa * a.N + n] = f2h(va);
          if (pb >= 0) a.act[(size_t)pb * a.N + n] = f2h(vb);
        }
      } else if (c < a.N) {
        if (p0 >= 0) y[(size_t)p0 * a.N + c] = v[0];
        if (p1 >= 0) y[(size_t)p1 * a.N + c] = v[1];
        if (p2 >= 0) y[(size_t)p2 * a.N + c] = v[2];
        if (p3 >= 0) y[(size_t)p3 * a.N + c] = v[3];
      }
    }
  }
}

// grid = max_tiles x column tiles x splits, up to a multiple of 8; block = 512
template <bool kUp, int kNT>
__global__ __launch_bounds__(64 * kTileWaves) void k_moe_tile(MoeArgs a) {
  using T = Tile<kUp, kNT>;
  // (one LDS variable: with two the compiler tells their accesses apart, takes the
  // DMA's target for known, and waits for it before any read of that variable)
  __shared__ __attribute__((aligned(16))) uint8_t lds[T::kLds];
  int* const srows = (int*)(lds + T::kLds) - kTileRows;
  const int tid = threadIdx.x, l = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nv = kUp ? 2 * a.N : a.N, nct = (nv + T::kCols * kTileWaves - 1) / (T::kCols * kTileWaves);
  // Workgroups go to the 8 XCDs in turn: each takes a run of tiles, row tiles
  // slowest, so that its L2 holds what neighbours share.
  const int ntiles = a.plan[a.E + 1] * nct * a.splits, per = (ntiles + 7) >> 3;
  int tile = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || tile >= ntiles) return;
  const int ct = tile % nct;
  tile /= nct;
  const int sp = tile % a.splits;
  tile /= a.splits;
  const int e = a.plan[a.E + 2 + 2 * tile], r0 = a.plan[a.E + 3 + 2 * tile];
  const int left = a.plan[e + 1] - r0, nrows = left < kTileRows ? left : kTileRows;
  if (tid < kTileRows) {
    const int* rows = a.plan + plan_rows_at((int64_t)a.S * a.k, a.E);
    srows[tid] = rows[r0 + (tid < nrows ? tid : nrows - 1)];
  }
  __syncthreads();
  const int c0 = ct * T::kCols * kTileWaves + w * T::kCols;
  const int ng = a.K >> 7, g0 = ng * sp / a.splits, g1 = ng * (sp + 1) / a.splits;
  auto xsrc = [&](int t) {
    const int r = 16 * w + 4 * t + (l >> 4), p = srows[r];
    return (const uint8_t*)(a.x + (size_t)(kUp ? p / a.k : p) * a.K) + 16 * ((l & 15) ^ xsw(r));
  };
  auto wsrc = [&](int t) {
    const int c = 16 * t + (l >> 2);
    return Col<kUp>(a, e, c0 + c).w + 16 * ((l & 3) ^ ((c >> 2) & 3));
  };
  const TileSrc<kNT> src = {xsrc(0), xsrc(1), xsrc(2), xsrc(3), wsrc(0), wsrc(1), kNT > 2 ? wsrc(2) : nullptr};
  uint16_t* tab = (uint16_t*)(lds + 2 * T::kSlot) + w * kTabGroups * T::kCols;
  float* y = kUp ? nullptr : a.y + (size_t)sp * a.S * a.k * a.N;
  switch ((nrows + 31) >> 5) {
    case 1: return tile_run<kUp, kNT, 1>(a, lds, tab, src, srows, nrows, e, c0, g0, g1, y);
    case 2: return tile_run<kUp, kNT, 2>(a, lds, tab, src, srows, nrows, e, c0, g0, g1, y);
    case 3: return tile_run<kUp, kNT, 3>(a, lds, tab, src, srows, nrows, e, c0, g0, g1, y);
    default: return tile_run<kUp, kNT, 4>(a, lds, tab, src, srows, nrows, e, c0, g0, g1, y);
  }
}

// ---------------------------------------------------------------- combine
struct CombineArgs {
  const float* y;
  const int32_t* ids;
  const float* weights;  // or null: 1
  const float* res;
  float* out;
  int S, k, E, H, splits;
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
    f32x4 y = *(const f32x4*)(a.y + (size_t)p * a.H + c);
    for (int i = 1; i < a.splits; i++) y += *(const f32x4*)(a.y + ((size_t)i * a.S * a.k + p) * a.H + c);
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = __builtin_fmaf(w, y[i], v[i]);
  }
  *(f32x4*)(a.out + (size_t)s * a.H + c) = v;
}

// ---------------------------------------------------------------- host
static int64_t plan_bytes(int64_t P, int E) { return ((plan_rows_at(P, E) + P) * 4 + 255) / 256 * 256; }

// Rows of y: P, and room for parts of K where few pairs leave the chip empty
static int64_t y_rows(int64_t P) { return P >= 4096 ? P : (8 * P < 4096 ? 8 * P : 4096); }

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
  constexpr int kNT = 2;
  const int P = a.S * a.k;
  a.plan = (const int*)ws;
  hipLaunchKernelGGL(k_moe_plan, dim3(1), dim3(1024), 0, s, a.ids, P, a.E, (int*)ws);
  const int nv = kUp ? 2 * a.N : a.N, cols = 128 * kNT;
  const int64_t tiles = max_tiles(P, a.E) * ((nv + cols - 1) / cols) * a.splits;
  hipLaunchKernelGGL((k_moe_tile<kUp, kNT>), dim3((unsigned)((tiles + 7) / 8 * 8)), dim3(64 * kTileWaves), 0, s, a);
  return launch_status();
}

}  // namespace cia

using namespace cia;

extern "C" int64_t cia_moe_workspace_bytes(int S, int k, int E, int H, int F) {
  if (S < 0 || k < 1 || E < 1 || H < 1 || F < 1) return 0;
  const int64_t P = (int64_t)S * k;
  return plan_bytes(P, E) + y_rows(P) * H * 4;
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
  a.splits = 1;
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
  a.splits = 1;
  hipStream_t s = (hipStream_t)stream;
  if ((st = products<false>(a, ws, s))) return st;
  const CombineArgs c{a.y, ids, weights, res, out, S, k, E, H, a.splits};
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
