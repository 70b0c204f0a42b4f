// moe_int4.hip -- the experts' INT4 group-128 products (w1, w3, swiglu, w2 and
// acc_scaled of engine.cu:869-905) on gfx950, for all the tokens of a call and the
// experts each has chosen.
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
#include "moe_shape.h"

namespace cia {

constexpr int kMoeMaxE = CIA_MOE_MAX_EXPERTS;
constexpr int kMoeMaxK = CIA_MOE_MAX_TOP_K;
constexpr int kMoeMaxPairs = CIA_MOE_MAX_PAIRS, kMoeMaxCols = CIA_MOE_MAX_WIDTH;

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
  const int* plan;        // k_moe_plan's; null: every workgroup finds its tile
  int splits;             // down: parts of K, each into its own y
  const float* res;       // down in tiles of a dense layer, one part: straight into out
  float* out;             // null: into y
};

// Row tiles of kTileRows are in the order of the whole ones of all experts, then
// the experts' last, partly filled ones, those of the most rows first, as the last
// round of workgroups ends with the shortest.  (4 of 32 experts of 1792, H = 2048, up:
// 500 tokens 62 us, 77 with these in the order of the experts and a run of them on
// each XCD.)

// An expert's n rows: its whole tiles (if whole), and its partly filled one under how
// many times 32 rows it has, 4 first, in fields of kBits from the lowest.  256 experts'
// sums fit 12 bits where all have fewer than 4096 tiles.
template <int kBits>
__device__ __forceinline__ uint64_t tile_counts(int n, bool whole) {
  const int c = (n % kTileRows + 31) >> 5;  // 0: none
  uint64_t v = c ? 1ull << kBits * (whole ? 5 - c : 4 - c) : 0;
  return whole ? v + (uint64_t)(n / kTileRows) : v;
}
// Of the wave's lanes up to this one
__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {
  const int l = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t u = __shfl_up(v, d);
    if (l >= d) v += u;
  }
  return v;
}

// plan: offs[E + 1], whole tiles, tiles, (expert, first) of each, rows[P]
// (rows 16-byte aligned, and written 4 at a time)
__host__ __device__ constexpr int64_t plan_rows_at(int64_t P, int E) { return (E + 3 + 2 * max_tiles(P, E) + 3) / 4 * 4; }

// ---------------------------------------------------------------- plan
// Rows by expert: offs[e] .. offs[e + 1] - 1 of rows are expert e's.  Their order
// within an expert does not matter: a row's results do not depend on its
// neighbours.
//   Bound by latency.  One workgroup; up to 16384 pairs are read once, 16 to a
// thread, and counted by wave: the count before is a pair's rank.  They are put in
// order in LDS and leave it 16 bytes a lane.  (16384 pairs: 16.3 us with two reads
// and shared counts, 10.8 with each pair stored on its own.)
constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;

__global__ __launch_bounds__(kPlanThreads) void k_moe_plan(const int32_t* ids, int P, int E, int* plan) {
  __shared__ int cnt[kPlanWaves][kMoeMaxE];  // of a wave, then the first place of its pairs
  __shared__ uint64_t part[2][4];  // of 64 experts: pairs and whole tiles, the others
  __shared__ __attribute__((aligned(16))) int order[16 * kPlanThreads];
  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63;
  int* rows = plan + plan_rows_at(P, E);
  constexpr int kPer = 16;
  const bool once = P <= kPer * kPlanThreads;
  for (int i = tid; i < kPlanWaves * kMoeMaxE; i += kPlanThreads) (&cnt[0][0])[i] = 0;
  __syncthreads();
  // pair i = 1024 j + tid
  int id[kPer], rank[kPer];
  if (!ids) {
    if (tid == 0) cnt[0][0] = P;
  } else if (once) {
#pragma unroll
    for (int j = 0; j < kPer; j++) {
      const int i = kPlanThreads * j + tid;
      id[j] = i < P ? ids[i] : -1;
    }
#pragma unroll
    for (int j = 0; j < kPer; j++)
      if ((unsigned)id[j] < (unsigned)E) rank[j] = atomicAdd(&cnt[w][id[j]], 1);
  } else {
    for (int i = tid; i < P; i += kPlanThreads) {
      const int e = ids[i];
      if ((unsigned)e < (unsigned)E) atomicAdd(&cnt[w][e], 1);
    }
  }
  __syncthreads();
  // thread e: its pairs and whole tiles (in the halves of a word), its partly filled
  // tile, and how many of each the experts before it have
  int n = 0;
  uint64_t own[2] = {}, before[2] = {};
  if (tid < kMoeMaxE) {
    for (int i = 0; i < kPlanWaves; i++) n += cnt[i][tid];
    own[0] = (uint64_t)(n / kTileRows) << 32 | (uint32_t)n;
    own[1] = tile_counts<16>(n, false);
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const uint64_t v = wave_scan(own[k]);
      before[k] = v - own[k];
      if (l == 63) part[k][w] = v;
    }
  }
  __syncthreads();
  uint64_t total[2] = {};
#pragma unroll
  for (int k = 0; k < 2; k++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (i < w) before[k] += part[k][i];
      total[k] += part[k][i];
    }
  if (tid < kMoeMaxE) {
    const int whole = (int)(total[0] >> 32), first = (int)(uint32_t)before[0];
    if (tid < E) {
      plan[tid] = first;
      int* tiles = plan + E + 3;
      const int full = n / kTileRows;
      for (int i = 0; i < full; i++) {
        const int at = (int)(before[0] >> 32) + i;
        tiles[2 * at] = tid;
        tiles[2 * at + 1] = first + i * kTileRows;
      }
      int others = 0;
#pragma unroll
      for (int c = 0; c < 4; c++) {
        if (own[1] >> 16 * c & 1) {
          const int at = whole + others + (int)(before[1] >> 16 * c & 0xFFFF);
          tiles[2 * at] = tid;
          tiles[2 * at + 1] = first + full * kTileRows;
        }
        others += (int)(total[1] >> 16 * c & 0xFFFF);
      }
      if (tid == E - 1) {
        plan[E] = first + n;
        plan[E + 1] = whole;
        plan[E + 2] = whole + others;
      }
    }
    int at = first;
    for (int i = 0; i < kPlanWaves; i++) {
      const int c = cnt[i][tid];
      cnt[i][tid] = at;
      at += c;
    }
  }
  __syncthreads();
  if (!ids) {
    for (int i = tid; i < P; i += kPlanThreads) rows[i] = i;
  } else if (once) {
#pragma unroll
    for (int j = 0; j < kPer; j++)
      if ((unsigned)id[j] < (unsigned)E) order[cnt[w][id[j]] + rank[j]] = kPlanThreads * j + tid;
    __syncthreads();
    const int quads = ((int)(uint32_t)total[0] + 3) / 4;
    for (int i = tid; i < quads; i += kPlanThreads) ((u32x4*)rows)[i] = ((const u32x4*)order)[i];
  } else {
    for (int i = tid; i < P; i += kPlanThreads) {
      const int e = ids[i];
      if ((unsigned)e < (unsigned)E) rows[atomicAdd(&cnt[w][e], 1)] = i;
    }
  }
}

// ---------------------------------------------------------------- products
// 8 nibbles (k even in the low one) -> 8 fp16 (nibble - 8), exact, in 12
// instructions: a permute puts byte b under the exponent of 1024 in both halves
// of a word, an and leaves the low half its low nibble and the high half its high
// one, not shifted and so 16 fold, and one fma takes {1, 1/16} and the offsets
// back out.
__device__ __forceinline__ f16x8 nib8(uint32_t u) {
  const f16x2 mul = {(_Float16)1.0f, (_Float16)0.0625f}, off = {(_Float16)-1032.0f, (_Float16)-72.0f};
  f16x8 r;
#pragma unroll
  for (int b = 0; b < 4; b++) {
    const uint32_t t = __builtin_amdgcn_perm(0x64646464u, u, 0x04000400u | (uint32_t)b << 16 | (uint32_t)b);
    const f16x2 h = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, t & 0x64F0640Fu), mul, off);
    r[2 * b] = h[0];
    r[2 * b + 1] = h[1];
  }
  return r;
}

// The product is rounded to fp32 before its caller rounds it to fp16.  (Left to
// itself the compiler multiplies and converts in one instruction at some places
// and in two at others, and a row's bits would depend on its place in a tile.)
__device__ __forceinline__ float silu_mul(float g, float u) {
  float v = g * __builtin_amdgcn_rcpf(1.0f + fast_exp(-g)) * u;
  asm("" : "+v"(v));
  return v;
}

// the value of the neighbouring lane (l ^ 1)
__device__ __forceinline__ float lane_pair(float v) {
  return __builtin_bit_cast(
      float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, true));
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

// Columns of a tile: up interleaves the two matrices (even W1, odd W3), so that a
// gate and its up product are in neighbouring lanes.  A lane's columns are all
// even or all odd.
template <bool kUp>
struct Cols {
  const uint8_t* w;
  const uint16_t* s;
  int last, ng;
  __device__ __forceinline__ Cols(const MoeArgs& a, int e, bool odd) {
    w = arg(a.packed[0]) + (size_t)e * a.pstride[0];
    s = arg(a.scales[0]) + (size_t)e * a.sstride[0];
    if constexpr (kUp) {
      const uint8_t* w1 = arg(a.packed[1]) + (size_t)e * arg(a.pstride[1]);
      const uint16_t* s1 = arg(a.scales[1]) + (size_t)e * arg(a.sstride[1]);
      w = odd ? w1 : w;
      s = odd ? s1 : s;
    }
    last = a.N - 1;
    ng = a.K >> 7;
  }
  // (an expert's bytes and scales: at most 2^29 and 2^23)
  __device__ __forceinline__ size_t row(int c) const {
    const int n = kUp ? c >> 1 : c;
    return (size_t)((uint64_t)(uint32_t)(n < last ? n : last) * (uint32_t)ng);
  }
  __device__ __forceinline__ const uint8_t* packed(int c) const { return w + row(c) * 64; }
  __device__ __forceinline__ const uint16_t* scales(int c) const { return s + row(c); }
  // (through a pointer to global memory: the choice of matrix hides where it points)
  __device__ __forceinline__ uint16_t scale(int c, int g) const {
    return ((const __attribute__((address_space(1))) uint16_t*)s)[row(c) + g];
  }
};

// ---------------------------------------------------------------- tiles
// Many rows an expert: a workgroup of 4 waves computes 128 rows x (64 kNT)
// columns, a wave all the rows of its own 16 kNT columns, so that a dequantised
// operand serves 128 rows and no column is dequantised twice.  Two workgroups a
// compute unit, so that one's first loads, dequantisation and outputs lie under
// the other's products.  The K loop runs over the scale groups, operands through
// LDS by DMA:
//   X  half a group, 64 rows x 16 chunks of 16 bytes, a slot, three slots; fetched
//      from the rows of the tile wherever they are (a row's address is the lane's
//      own).  Row r's chunk c at c ^ xsw(r): a 16-byte read is served 32 lanes,
//      512 bytes of banks, at a time, and so reaches 32 different places.
//   W  each wave's own columns, 4 chunks of nibbles, two slots; column c's chunk q
//      at q ^ ((c >> 2) & 3).
// Inside a group lane q = l >> 4 of an operand holds k = 32q + 8s .. + 7 at step
// s, so one 16-byte read brings a column's nibbles for all four steps.
//   One barrier a half: past the one before half h, h has landed, and all have
// read h - 1, whose slot h + 2 takes.
//   4096 tokens of 4 of 32 experts of 1792, H = 2048, up: 246-252 us, 955-978 TFLOP/s,
// where a large fp16 product reaches 1140-1306.  The matrix cores are busy 49 % of it: 3.7
// vector instructions (dequantisation, scales) go with a product, and the operands'
// LDS reads alone take 32 % of the cycles at 128 bytes each.  Few rows an expert are bound by memory: 45 tokens, down,
// 16 us for 59 MB.  (W and X fetched 3 groups ahead instead, where 32 rows leave the
// slots room: 1 % slower.)
typedef __attribute__((address_space(3))) void lds_void_t;
typedef __attribute__((address_space(1))) void gbl_void_t;

constexpr int kTileWaves = 4;
constexpr int kTabGroups = 16;  // groups whose scales the LDS table holds

__device__ __forceinline__ int xsw(int r) { return ((r >> 1) & 3) | ((r & 1) << 2) | (r & 8); }

__device__ __forceinline__ void dma16(const void* src, void* dst) {
  __builtin_amdgcn_global_load_lds((gbl_void_t*)src, (lds_void_t*)dst, 16, 0, 0);
}

template <int kNT>
struct Tile {
  static constexpr int kCols = 16 * kNT;  // of a wave
  static constexpr int kX = 64 * 256, kW = kTileWaves * kCols * 64;  // of a slot
  static constexpr int kTab = kTileWaves * kTabGroups * kCols * 2;
  static constexpr int kLds = 3 * kX + 2 * kW + kTab + 2 * kTileRows * 4;
};

// A lane's DMA sources in group 0: X of the first and second half, W
template <int kNT>
struct TileSrc {
  const uint8_t *x0, *x1, *x2, *x3, *y0, *y1, *y2, *y3, *w0, *w1, *w2;
  __device__ __forceinline__ const uint8_t* x(int half, int t) const {
    return half == 0 ? (t == 0 ? x0 : t == 1 ? x1 : t == 2 ? x2 : x3) : (t == 0 ? y0 : t == 1 ? y1 : t == 2 ? y2 : y3);
  }
  __device__ __forceinline__ const uint8_t* w(int t) const { return t == 0 ? w0 : t == 1 ? w1 : w2; }
};

// The K loop of a wave over up to 32 kPR rows, in kHalves halves of a group.
template <int kNT, int kPR>
struct TileLoop {
  static_assert(kNT <= 3, "the columns' sources");
  using T = Tile<kNT>;
  static constexpr int kUnits = 2 * kPR;  // of a row tile
  static constexpr int kHalves = kPR > 2 ? 2 : 1;
  static constexpr int kLast = kPR > 2 ? 2 * (kPR - 2) : 2 * kPR;  // DMA instructions a wave in the last half: its row tiles
  uint8_t* lds;
  uint16_t* tab;  // this wave's scales
  TileSrc<kNT> src;
  int w, n16, q, g1;
  f32x4 C[kUnits][kNT];
  f32x4 P[2][kNT];  // of a row tile, and of the one before
  f16x8 A[2][4];    // of a row tile, and of the next
  f16x8 B[kNT][4];
  float scl[kNT], scl_old[kNT];  // of a group, and of the one before

  // Half of group g into the slot at byte at; past the last group that one again
  // (a branch here would part the block that products and vector instructions are
  // mixed in)
  template <int kHalf>
  __device__ __forceinline__ void fetch_x(int at, int g) const {
    constexpr int n = kHalf == kHalves - 1 ? kLast : 4;
    g = g < g1 ? g : g1 - 1;
#pragma unroll
    for (int t = 0; t < n; t++) dma16(src.x(kHalf, t) + 256 * (size_t)g, lds + at + (n * w + t) * 1024);
  }
  __device__ __forceinline__ uint8_t* wslot(int i) const { return lds + 3 * T::kX + (i & 1) * T::kW + w * T::kCols * 64; }
  __device__ __forceinline__ void fetch_w(int i, int g) const {
    g = g < g1 ? g : g1 - 1;
#pragma unroll
    for (int t = 0; t < kNT; t++) dma16(src.w(t) + 64 * (size_t)g, wslot(i) + t * 1024);
  }
  __device__ __forceinline__ void load_a(int at, int u, f16x8 (&o)[4]) const {
    const uint16_t* xs = (const uint16_t*)(lds + at) + n16 * 128;
#pragma unroll
    for (int s = 0; s < 4; s++) o[s] = *(const f16x8*)(xs + 16 * (u & 3) * 128 + 8 * ((4 * q + s) ^ xsw(n16)));
  }
  __device__ __forceinline__ void scale(int row_tile, int p, const float (&sc)[kNT]) {
#pragma unroll
    for (int j = 0; j < kNT; j++)
#pragma unroll
      for (int r = 0; r < 4; r++) C[row_tile][j][r] = __builtin_fmaf(P[p][j][r], sc[j], C[row_tile][j][r]);
  }
  __device__ __forceinline__ static int after(int at) { return at == 2 * T::kX ? 0 : at + T::kX; }
  // All but the last kLeft fetches have landed, and every LDS read has its data:
  // products are not held by the barrier, and the wait of the last ones for their
  // operands could follow it, with the operands' slot already being fetched into.
  template <int kLeft>
  __device__ __forceinline__ static void meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070 | kLeft);  // vmcnt(kLeft) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }

  // The i-th group, group g, its first half in the slot at at; returns the next's.
  __device__ __forceinline__ int group(int i, int g, int at) {
    u32x4 wq[kNT];
#pragma unroll
    for (int u = 0; u < kUnits; u++) {
      if (u == 0) {
        // what may be in flight: the half after this one, fetched last
        meet<kLast>();
        fetch_w(i + 1, g + 1);
        __builtin_amdgcn_sched_barrier(0);
        fetch_x<0>(after(after(at)), kHalves == 2 ? g + 1 : g + 2);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < kNT; j++) {
          const int c = 16 * j + n16;
          wq[j] = *(const u32x4*)(wslot(i) + c * 64 + 16 * (q ^ ((c >> 2) & 3)));
          scl_old[j] = scl[j];
          scl[j] = h2f(tab[i % kTabGroups * T::kCols + c]);
          asm("" : "+v"(scl[j]));  // (an fp32 register: no conversion in every fma)
        }
        load_a(at, 0, A[0]);
      }
      if (u == 4) {
        meet<kNT + 4>();
        at = after(at);
        fetch_x<1>(after(after(at)), g + 1);
        __builtin_amdgcn_sched_barrier(0);
        load_a(at, 0, A[0]);
      }
      __builtin_amdgcn_sched_barrier(0);
      // (the wave with products before the one that dequantises: 2 %)
      if (u == 0) __builtin_amdgcn_s_setprio(0);
      if (u == 1) __builtin_amdgcn_s_setprio(1);
      if (u + 1 < kUnits && u != 3) load_a(at, u + 1, A[(u + 1) & 1]);
#pragma unroll
      for (int s = 0; s < 4; s++)
#pragma unroll
        for (int j = 0; j < kNT; j++) {
          if (u == 0) B[j][s] = nib8(wq[j][s]);
          P[u & 1][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A[u & 1][s], B[j][s],
                                                               s == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : P[u & 1][j], 0, 0, 0);
        }
      // the row tile before (of the group before, at a group's start)
      if (u == 0)
        scale(kUnits - 1, 1, scl_old);
      else
        scale(u - 1, (u - 1) & 1, scl);
    }
    return after(at);
  }

  // groups g0 .. g1 - 1; scales(c, g) is column c's
  template <class F>
  __device__ __forceinline__ void run(int g0, const F& scales) {
    auto refill = [&](int g, int l) __attribute__((always_inline)) {
      constexpr int n = T::kCols * kTabGroups / 64;  // 16 neighbouring lanes a column
      const int gg = g + l % kTabGroups;
      uint16_t v[n];
#pragma unroll
      for (int k = 0; k < n; k++) v[k] = scales((64 * k + l) / kTabGroups, gg < g1 ? gg : g1 - 1);
#pragma unroll
      for (int k = 0; k < n; k++) tab[l % kTabGroups * T::kCols + (64 * k + l) / kTabGroups] = v[k];
    };
    fetch_w(0, g0);
    fetch_x<0>(0, g0);
    if constexpr (kHalves == 2)
      fetch_x<1>(T::kX, g0);
    else
      fetch_x<0>(T::kX, g0 + 1);
    refill(g0, threadIdx.x & 63);
#pragma unroll
    for (int j = 0; j < kNT; j++) {
#pragma unroll
      for (int i = 0; i < kUnits; i++) C[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      P[1][j] = f32x4{0.f, 0.f, 0.f, 0.f};  // (of the group before the first)
      scl[j] = 0.f;
    }
    int at = 0;
    for (int i = 0; g0 + i < g1; i++) {
      if (i > 0 && i % kTabGroups == 0) {
        // (worked out anew: kept over the loop its addresses go to scratch, and loads from
        // there into the count that meet() waits for)
        int l = threadIdx.x & 63;
        asm volatile("" : "+v"(l));
        refill(g0 + i, l);
      }
      at = group(i, g0 + i, at);
    }
    scale(kUnits - 1, 1, scl);
  }
};

template <bool kUp, int kNT, int kPR>
__device__ __forceinline__ void tile_run(const MoeArgs& a, uint8_t* lds, uint16_t* tab, const int* rows, int nrows, int e,
                                         int c0, int g0, int g1, float* y) {
  using T = Tile<kNT>;
  const int l = threadIdx.x & 63, n16 = l & 15, q = l >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  TileLoop<kNT, kPR> loop;
  // X instruction t of wave w fills rows 4 (n w + t) .. + 3 of its half, n
  // instructions a wave; W instruction t this wave's columns 16 t .. + 15
  auto xsrc = [&](int half, int t) __attribute__((always_inline)) {
    const int n = half == loop.kHalves - 1 ? loop.kLast : 4;
    const int r = half >= loop.kHalves || t >= n ? 0 : 64 * half + 4 * (n * w + t) + (l >> 4);
    return (const uint8_t*)(a.x + (uint64_t)(uint32_t)rows[kTileRows + r] * (uint32_t)a.K) + 16 * ((l & 15) ^ xsw(r));
  };
  const Cols<kUp> wcols(a, e, (l >> 2) & 1), scols(a, e, (l >> 4) & 1);
  auto wsrc = [&](int t) __attribute__((always_inline)) {
    const int c = 16 * t + (l >> 2);
    return wcols.packed(c0 + c) + 16 * ((l & 3) ^ ((c >> 2) & 3));
  };
  loop.lds = lds;
  loop.tab = tab;
  loop.src = {xsrc(0, 0), xsrc(0, 1), xsrc(0, 2), xsrc(0, 3), xsrc(1, 0), xsrc(1, 1),
              xsrc(1, 2), xsrc(1, 3), wsrc(0),    wsrc(kNT > 1 ? 1 : 0), wsrc(kNT > 2 ? 2 : 0)};
  loop.w = w;
  loop.n16 = n16;
  loop.q = q;
  loop.g1 = g1;
  loop.run(g0, [&](int c, int g) { return scols.scale(c0 + c, g); });
  // Lane holds rows 4q .. 4q + 3 of row tile i, column n16 of column tile j.  They
  // change places in LDS, where all have read, and go out 16 bytes a lane.
  loop.template meet<0>();
  uint8_t* const out = lds + w * ((3 * T::kX + 2 * T::kW) / kTileWaves);
  if constexpr (kUp) {
    constexpr int kN = T::kCols / 2;  // outputs of a row
    uint16_t* st = (uint16_t*)out + (4 * q + (n16 & 1) * 2) * kN + (n16 >> 1);
#pragma unroll
    for (int i = 0; i < 2 * kPR; i++)
#pragma unroll
      for (int j = 0; j < kNT; j++) {
        // the even lane takes rows 0 and 1 of the pair's column, the odd one 2, 3
        const f32x4 v = loop.C[i][j];
        const bool odd = n16 & 1;
        const float o0 = lane_pair(v[0]), o1 = lane_pair(v[1]), o2 = lane_pair(v[2]), o3 = lane_pair(v[3]);
        st[16 * i * kN + 8 * j] = f2h(silu_mul(odd ? o2 : v[0], odd ? v[2] : o0));
        st[(16 * i + 1) * kN + 8 * j] = f2h(silu_mul(odd ? o3 : v[1], odd ? v[3] : o1));
      }
#pragma unroll
    for (int k = 0; k < (32 * kPR * kNT + 63) / 64; k++) {
      const int i = 64 * k + l, r = i / kNT, n = c0 / 2 + 8 * (i % kNT);
      if (r < nrows && n < a.N)
        *(u32x4*)(a.act + (uint64_t)(uint32_t)rows[r] * (uint32_t)a.N + n) = *(const u32x4*)(out + 16 * i);
    }
  } else {
    constexpr int kRow = T::kCols + 4;  // floats: the four row groups of a store on different banks
#pragma unroll
    for (int half = 0; half < (kPR + 1) / 2; half++) {  // 64 rows at a time
      float* st = (float*)out + 4 * q * kRow + n16;
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (4 * half + i < 2 * kPR)
#pragma unroll
          for (int j = 0; j < kNT; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) st[(16 * i + r) * kRow + 16 * j] = loop.C[4 * half + i < 2 * kPR ? 4 * half + i : 0][j][r];
#pragma unroll
      for (int k = 0; k < 4 * kNT; k++) {
        const int i = 64 * k + l, r = i / (4 * kNT), ch = i % (4 * kNT), n = c0 + 4 * ch;
        if (64 * half + r < nrows && n < a.N) {
          const uint64_t o = (uint64_t)(uint32_t)rows[64 * half + r] * (uint32_t)a.N + n;
          f32x4 v = *(const f32x4*)((const float*)out + r * kRow + 4 * ch);
          if (a.out) v += *(const f32x4*)(a.res + o);
          *(f32x4*)((a.out ? a.out : y) + o) = v;
        }
      }
    }
  }
}

// A workgroup's tile: its expert, rows and their rows of x, in rows[128] and
// rows[128 + ..].  From the plan, or from up to kOwnPairs ids by itself.
struct TileOf {
  int e, n;  // n = 0: none
  int ct, sp;
};

// Workgroups go to the 8 XCDs in turn: each takes a run of the whole tiles, row tiles
// slowest, so that its L2 holds what neighbours share.  The others, whose neighbours
// share few rows and no weights, in their order.  Returns the row tile, or -1.
__device__ __forceinline__ int tile_index(int whole, int others, int nct, int splits, TileOf& t) {
  const int n0 = whole * nct * splits, n1 = others * nct * splits, per0 = (n0 + 7) >> 3;
  int i = blockIdx.x >> 3;
  if (i < per0) {
    i += (blockIdx.x & 7) * per0;
    if (i >= n0) return -1;
  } else {
    i = blockIdx.x - 8 * per0;
    if (i >= n1) return -1;
    i += n0;
  }
  t.ct = i % nct;
  i /= nct;
  t.sp = i % splits;
  return i / splits;
}

template <bool kUp>
__device__ __forceinline__ TileOf planned_tile(const MoeArgs& a, int nct, int* rows) {
  const int tid = threadIdx.x, whole = a.plan[a.E + 1];
  TileOf t{};
  const int tile = tile_index(whole, a.plan[a.E + 2] - whole, nct, a.splits, t);
  if (tile < 0) return t;
  t.e = a.plan[a.E + 3 + 2 * tile];
  const int r0 = a.plan[a.E + 4 + 2 * tile], left = a.plan[t.e + 1] - r0;
  t.n = left < kTileRows ? left : kTileRows;
  if (tid < kTileRows) {
    const int p = a.plan[plan_rows_at((int64_t)a.S * a.k, a.E) + r0 + (tid < t.n ? tid : t.n - 1)];
    rows[tid] = p;
    rows[kTileRows + tid] = kUp ? p / a.k : p;
  }
  __syncthreads();
  return t;
}

// scratch: LDS that the tile's loop takes afterwards
template <bool kUp>
__device__ __forceinline__ TileOf own_tile(const MoeArgs& a, int nct, int* rows, int* scratch) {
  constexpr int kPer = kOwnPairs / (64 * kTileWaves);
  static_assert(kMoeMaxE <= 64 * kTileWaves, "a thread an expert");
  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, P = a.S * a.k;
  int* const cnt = scratch;               // [256]
  uint64_t* const part = (uint64_t*)(scratch + kMoeMaxE);  // [4]: tiles of 64 experts
  int* const found = (int*)(part + kTileWaves);
  int* const wave = found + 2;            // [kPer][4]: pairs of the expert
  int id[kPer];
#pragma unroll
  for (int j = 0; j < kPer; j++) {
    const int i = 64 * kTileWaves * j + tid;
    id[j] = i < P ? (a.ids ? a.ids[i] : 0) : -1;
    if ((unsigned)id[j] >= (unsigned)a.E) id[j] = -1;
  }
  cnt[tid] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kPer; j++)
    if (id[j] >= 0) atomicAdd(&cnt[id[j]], 1);
  __syncthreads();
  static_assert(kOwnPairs / kTileRows < 4096 && kMoeMaxE < 4096, "tile_counts in 12 bits");
  const int mine = cnt[tid];
  const uint64_t own = tile_counts<12>(mine, true), upto = wave_scan(own);
  uint64_t before = upto - own, total = 0;
  if (l == 63) part[w] = upto;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kTileWaves; i++) {
    if (i < w) before += part[i];
    total += part[i];
  }
  const int whole = (int)(total & 0xFFF), full = mine / kTileRows;
  int others = 0;
#pragma unroll
  for (int c = 1; c <= 4; c++) others += (int)(total >> 12 * c & 0xFFF);
  TileOf t{};
  const int tile = tile_index(whole, others, nct, a.splits, t);
  if (tile < 0) return t;
  const int first = (int)(before & 0xFFF);
  if (tile >= first && tile < first + full) {
    found[0] = tid;
    found[1] = (tile - first) * kTileRows;
  }
  int at = whole;
#pragma unroll
  for (int c = 1; c <= 4; c++) {
    if ((own >> 12 * c & 1) && tile == at + (int)(before >> 12 * c & 0xFFF)) {
      found[0] = tid;
      found[1] = full * kTileRows;
    }
    at += (int)(total >> 12 * c & 0xFFF);
  }
  __syncthreads();
  t.e = __builtin_amdgcn_readfirstlane(found[0]);
  const int r0 = __builtin_amdgcn_readfirstlane(found[1]), left = __builtin_amdgcn_readfirstlane(cnt[t.e]) - r0;
  t.n = left < kTileRows ? left : kTileRows;
  // its rows from r0 on, in the order of the pairs, the same in every workgroup
  uint64_t b[kPer];
#pragma unroll
  for (int j = 0; j < kPer; j++) {
    b[j] = __ballot(id[j] == t.e);
    if (l == 0) wave[kTileWaves * j + w] = __popcll(b[j]);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kPer; j++) {
    int r = __popcll(b[j] & ((1ull << l) - 1)) - r0;
    for (int i = 0; i < kTileWaves * j + w; i++) r += wave[i];
    const int p = 64 * kTileWaves * j + tid;
    if (id[j] == t.e && r >= 0 && r < kTileRows) {
      rows[r] = p;
      rows[kTileRows + r] = kUp ? p / a.k : p;
    }
  }
  __syncthreads();
  if (tid >= t.n && tid < kTileRows) rows[kTileRows + tid] = rows[kTileRows];  // (read, and not used)
  __syncthreads();
  return t;
}

// grid = max_tiles x column tiles x splits, up to a multiple of 8, and 8; block = 256
template <bool kUp, int kNT>
__global__ __launch_bounds__(64 * kTileWaves, 2) void k_moe_tile(MoeArgs a) {
  using T = Tile<kNT>;
  // (one LDS variable: with two the compiler tells their accesses apart, takes the
  // DMA's target for known, and waits for it before any read of that variable)
  __shared__ __attribute__((aligned(16))) uint8_t lds[T::kLds];
  int* const srows = (int*)(lds + T::kLds) - 2 * kTileRows;  // rows, and their rows of x
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nv = kUp ? 2 * a.N : a.N, nct = (nv + T::kCols * kTileWaves - 1) / (T::kCols * kTileWaves);
  const TileOf t = a.plan ? planned_tile<kUp>(a, nct, srows) : own_tile<kUp>(a, nct, srows, (int*)lds);
  if (t.n == 0) return;
  const int c0 = t.ct * T::kCols * kTileWaves + w * T::kCols;
  const int ng = a.K >> 7, g0 = ng * t.sp / a.splits, g1 = ng * (t.sp + 1) / a.splits;
  uint16_t* tab = (uint16_t*)(lds + 3 * T::kX + 2 * T::kW) + w * kTabGroups * T::kCols;
  float* y = kUp ? nullptr : a.y + (size_t)t.sp * a.S * a.k * a.N;
  switch ((t.n + 31) >> 5) {
    case 1: return tile_run<kUp, kNT, 1>(a, lds, tab, srows, t.n, t.e, c0, g0, g1, y);
    case 2: return tile_run<kUp, kNT, 2>(a, lds, tab, srows, t.n, t.e, c0, g0, g1, y);
    case 3: return tile_run<kUp, kNT, 3>(a, lds, tab, srows, t.n, t.e, c0, g0, g1, y);
    default: return tile_run<kUp, kNT, 4>(a, lds, tab, srows, t.n, t.e, c0, g0, g1, y);
  }
}

// ---------------------------------------------------------------- streams
// Few rows an expert: the experts' weights are read once, at the memory's rate,
// and everything else lies under that.  A workgroup of 8 waves takes a run of
// column tiles (16 columns) of one expert; its waves split K, each keeping its
// scale groups' x of up to 16 kMT rows in registers for the whole run, so that
// x is fetched once a run and a weight passes through one wave only.
//   W     4 lanes to a column's 64 bytes of a group, as a load is quick (a lane's
//         16 bytes in a line of its own takes four times as long), kRing tiles
//         ahead in registers; then through the wave's own LDS into operand order.
//   sums  a wave's products are scaled in its registers; the 8 waves' sums of
//         kRing tiles meet in LDS and are added there in the order of the groups.
// A token of 4 of 32 experts of 1792, H = 2048, up: 7.5-8.2 us, of them 2 the launch
// and 3.2 the weights at a copy's rate; 12 such tokens 17.4 us.
// Rows by expert are found by the workgroup itself, from up to kStreamPairs ids:
// no launch before this one.
template <int kG, int kMT>
struct Stream {
  static constexpr int kRing = kG <= 2 ? 4 : 2;
  static constexpr int kMaxMT = kMT, kRows = 16 * kMT;
  // row tiles x tiles that the LDS holds of each wave; operand slots of a wave
  static constexpr int kPart = kRing * kMT > 8 ? 16 : 8, kStage = kMT == 1 ? 1 : 2;
  // 16 rows: registers and LDS for two workgroups a compute unit
  static constexpr int kPerUnit = kMT == 1 && kG <= 2 ? 2 : 1;
  struct Lds {
    f32x4 part[kPart][kStreamWaves][64];
    u32x4 stage[kStreamWaves][kStage][64];
    int cnt[kMoeMaxE], seg[kMoeMaxE];
    int sum[4], wave[kStreamWaves], rows[kRows], expert[2];
  };
};

// tiles t0 .. t1 - 1 of expert e, part part_k of K, for its n rows in L.rows
template <bool kUp, int kG, int kMT, class St>
__device__ __forceinline__ void stream_run(const MoeArgs& a, typename St::Lds& L, int e, int part_k, int n, int t0, int t1) {
  constexpr int kRing = St::kRing;
  constexpr bool kTwo = 2 * kRing * kMT <= St::kPart;  // two batches fit
  const int tid = threadIdx.x, l = tid & 63, n16 = l & 15, q = l >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ng = a.K >> 7, k0 = kUp ? 0 : ng * part_k / a.splits, nk = (kUp ? ng : ng * (part_k + 1) / a.splits) - k0;
  const int g0 = k0 + w * nk / kStreamWaves, mine = k0 + (w + 1) * nk / kStreamWaves - g0;  // <= kG
  float* const y = kUp ? nullptr : a.y + (size_t)part_k * a.S * a.k * a.N;
  const Cols<kUp> wc(a, e, (l >> 2) & 1), sc(a, e, n16 & 1);
  typedef const __attribute__((address_space(1))) uint16_t* gs_t;
  typedef const __attribute__((address_space(1))) u32x4* gw_t;
  const uint8_t* wp = wc.packed(16 * t0 + (l >> 2)) + 64 * (size_t)g0 + 16 * (l & 3);
  const uint16_t* sp = sc.scales(16 * t0 + n16) + g0;
  const size_t step = (size_t)(kUp ? 8 : 16) * ng;  // groups from a tile to the next
  u32x4 wr[kRing][kG];
  uint32_t sr[kRing][kG];
  auto fetch = [&](int t, int d) __attribute__((always_inline)) {
    const size_t o = step * (size_t)((t < t1 ? t : t1 - 1) - t0);
#pragma unroll
    for (int g = 0; g < kG; g++) {
      const int gg = g < mine ? g : 0;
      wr[d][g] = *(gw_t)(wp + 64 * (o + gg));
      sr[d][g] = *(gs_t)(sp + o + gg);
    }
  };
  if (mine > 0)
#pragma unroll
    for (int d = 0; d < kRing; d++) fetch(t0 + d, d);
  // x of this wave's groups: lane (n16, q) holds row 16 i + n16, k = 32q + 8s .. + 7
  f16x8 A[kMT][kG][4];
#pragma unroll
  for (int i = 0; i < kMT; i++) {
    const int r = 16 * i + n16;
    const int p = L.rows[r < n ? r : 0];
    const uint16_t* xr = a.x + (uint64_t)(uint32_t)(kUp ? p / a.k : p) * (uint32_t)a.K + 128 * g0 + 32 * q;
#pragma unroll
    for (int g = 0; g < kG; g++)
#pragma unroll
      for (int s = 0; s < 4; s++) {
        A[i][g][s] = f16x8{};
        if (r < n && g < mine) A[i][g][s] = *(const f16x8*)(xr + 128 * g + 8 * s);
      }
  }
  for (int tb = t0, batch = 0; tb < t1; tb += kRing, batch++) {
    f32x4(*part)[kStreamWaves][64] = L.part + (kTwo && (batch & 1) ? kRing * kMT : 0);
#pragma unroll
    for (int d = 0; d < kRing; d++) {
      if (tb + d >= t1) break;
      f32x4 acc[kMT] = {};
      if (mine > 0) {
        float scl[kG];
#pragma unroll
        for (int g = 0; g < kG; g++) scl[g] = g < mine ? h2f((uint16_t)sr[d][g]) : 0.f;
        u32x4 wq[kG];
#pragma unroll
        for (int g = 0; g < kG; g++) {
          u32x4* st = L.stage[w][g % St::kStage];
          // column l >> 2's chunk l & 3 at chunk ^ (column >> 2) & 3: a read's 16 columns on all banks
          st[(l & ~3) | ((l & 3) ^ ((l >> 4) & 3))] = wr[d][g];
          wq[g] = st[4 * n16 + (q ^ ((n16 >> 2) & 3))];
        }
        fetch(tb + d + kRing, d);
#pragma unroll
        for (int g = 0; g < kG; g++) {
          f32x4 P[kMT];
#pragma unroll
          for (int s = 0; s < 4; s++) {
            const f16x8 B = nib8(wq[g][s]);
#pragma unroll
            for (int i = 0; i < kMT; i++)
              P[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A[i][g][s], B, s == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : P[i], 0, 0, 0);
          }
#pragma unroll
          for (int i = 0; i < kMT; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) acc[i][r] = __builtin_fmaf(P[i][r], scl[g], acc[i][r]);
        }
      }
#pragma unroll
      for (int i = 0; i < kMT; i++) part[d * kMT + i][w][l] = acc[i];
    }
    __syncthreads();
    // sums of tile d, row tile i: wave d kMT + i, 4 on in every second batch
#pragma unroll
    for (int u = 0; u < (kRing * kMT + 7) / 8; u++) {
      const int it = ((w + (kRing * kMT <= 4 ? 4 * (batch & 1) : 0)) & 7) + 8 * u, d = it / kMT, i = it % kMT;
      if (it >= kRing * kMT || tb + d >= t1) continue;
      f32x4 v = {};
#pragma unroll
      for (int k = 0; k < kStreamWaves; k++) v += part[it][k][l];
      const int c = 16 * (tb + d) + n16, r = 16 * i + 4 * q;
      if constexpr (kUp) {
        // the even lane takes rows 0 and 1 of the pair's column, the odd one 2, 3
        const bool odd = n16 & 1;
        const float o0 = lane_pair(v[0]), o1 = lane_pair(v[1]), o2 = lane_pair(v[2]), o3 = lane_pair(v[3]);
        const float va = silu_mul(odd ? o2 : v[0], odd ? v[2] : o0), vb = silu_mul(odd ? o3 : v[1], odd ? v[3] : o1);
        const int ra = r + (odd ? 2 : 0);
        if (ra < n) a.act[(uint64_t)(uint32_t)L.rows[ra] * (uint32_t)a.N + (c >> 1)] = f2h(va);
        if (ra + 1 < n) a.act[(uint64_t)(uint32_t)L.rows[ra + 1] * (uint32_t)a.N + (c >> 1)] = f2h(vb);
      } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (r + k < n) y[(uint64_t)(uint32_t)L.rows[r + k] * (uint32_t)a.N + c] = v[k];
      }
    }
    if (!kTwo) __syncthreads();  // the sums are read
  }
}

template <bool kUp, int kG, class St>
__device__ __forceinline__ void stream_rows(const MoeArgs& a, typename St::Lds& L, int e, int part_k, int n, int t0, int t1) {
  constexpr int kMax = St::kMaxMT;
  if (kMax >= 4 && n > 32)
    stream_run<kUp, kG, kMax >= 4 ? 4 : 1, St>(a, L, e, part_k, n, t0, t1);
  else if (kMax >= 2 && n > 16)
    stream_run<kUp, kG, kMax >= 2 ? 2 : 1, St>(a, L, e, part_k, n, t0, t1);
  else
    stream_run<kUp, kG, 1, St>(a, L, e, part_k, n, t0, t1);
  __syncthreads();  // the sums and rows are read
}

// grid = any, block = 512; S k <= kStreamPairs (64 if kMT > 1), a part of K at most
// 1024 kG
template <bool kUp, int kG, int kMT>
__global__ __launch_bounds__(64 * kStreamWaves, (2 * Stream<kG, kMT>::kPerUnit)) void k_moe_stream(MoeArgs a) {
  using St = Stream<kG, kMT>;
  __shared__ typename St::Lds L;
  const int tid = threadIdx.x, l = tid & 63, w = tid >> 6, P = a.S * a.k;
  const int nct = (kUp ? 2 * a.N : a.N) >> 4, parts = kUp ? 1 : a.splits;
  // Segments: an expert's rows kRows at a time, in the order of the pairs, the same
  // in every workgroup.  Each takes an equal run of all the segments' column tiles.
  if (kMT > 1 || P <= 64) {  // (more pairs are 16 rows at a time)
    // every wave finds its own, lane i with pair i, and waits for no other
    int id = l < P ? (a.ids ? a.ids[l] : 0) : -1;
    if ((unsigned)id >= (unsigned)a.E) id = -1;
    uint64_t same = __ballot(id >= 0);
#pragma unroll
    for (int b = 0; b < 8; b++) {
      const uint64_t v = __ballot(id >> b & 1);
      same &= id >> b & 1 ? v : ~v;
    }
    const uint64_t below = (1ull << l) - 1;
    const bool first = id >= 0 && !(same & below);  // of its expert
    const int segs = first ? (__popcll(same) + St::kRows - 1) / St::kRows : 0;
    int before = 0, nseg = 0;
#pragma unroll
    for (int k = 1; k <= 64 / St::kRows; k++) {
      const uint64_t v = __ballot(segs >= k);
      before += __popcll(v & below);
      nseg += __popcll(v);
    }
    int u0 = (int)((int64_t)nseg * parts * nct * blockIdx.x / gridDim.x);
    const int u1 = (int)((int64_t)nseg * parts * nct * (blockIdx.x + 1) / gridDim.x);
    while (u0 < u1) {
      int sg = u0 / nct;
      const int t0 = u0 - sg * nct, t1 = u1 - u0 < nct - t0 ? t0 + (u1 - u0) : nct;
      u0 += t1 - t0;
      const int part_k = sg % parts;
      sg /= parts;
      const int at = __builtin_ctzll(__ballot(segs > 0 && sg >= before && sg < before + segs));
      const int e = __builtin_amdgcn_readlane(id, at);
      const int r0 = (sg - __builtin_amdgcn_readlane(before, at)) * St::kRows;
      const uint64_t rows = __ballot(id == e);
      const int r = __popcll(rows & below) - r0, left = __popcll(rows) - r0;
      if (id == e && r >= 0 && r < St::kRows) L.rows[r] = l;  // (all waves the same)
      stream_rows<kUp, kG, St>(a, L, e, part_k, left < St::kRows ? left : St::kRows, t0, t1);
    }
    return;
  }
  int id = tid < P ? (a.ids ? a.ids[tid] : 0) : -1;
  if ((unsigned)id >= (unsigned)a.E) id = -1;
  if (tid < kMoeMaxE) L.cnt[tid] = 0;
  __syncthreads();
  if (id >= 0) atomicAdd(&L.cnt[id], 1);
  __syncthreads();
  const int segs = tid < kMoeMaxE ? (L.cnt[tid] + St::kRows - 1) / St::kRows : 0;
  int before = segs;
  if (tid < kMoeMaxE) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int u = __shfl_up(before, d);
      if (l >= d) before += u;
    }
    if (l == 63) L.sum[w] = before;
  }
  __syncthreads();
  before -= segs;
  if (tid < kMoeMaxE)
    for (int i = 0; i < w; i++) before += L.sum[i];
  const int64_t all = (int64_t)(L.sum[0] + L.sum[1] + L.sum[2] + L.sum[3]) * parts * nct;
  int64_t u0 = all * blockIdx.x / gridDim.x;
  const int64_t u1 = all * (blockIdx.x + 1) / gridDim.x;
  while (u0 < u1) {
    int sg = (int)(u0 / nct);
    const int t0 = (int)(u0 - (int64_t)sg * nct), t1 = u1 - u0 < nct - t0 ? t0 + (int)(u1 - u0) : nct;
    u0 += t1 - t0;
    const int part_k = sg % parts;
    sg /= parts;
    if (segs > 0 && sg >= before && sg < before + segs) {
      L.expert[0] = tid;
      L.expert[1] = sg - before;
    }
    __syncthreads();
    const int e = __builtin_amdgcn_readfirstlane(L.expert[0]);
    const int r0 = __builtin_amdgcn_readfirstlane(L.expert[1]) * St::kRows;
    const uint64_t b = __ballot(id == e);
    if (l == 0) L.wave[w] = __popcll(b);
    __syncthreads();
    int r = __popcll(b & ((1ull << l) - 1)) - r0;
    for (int k = 0; k < w; k++) r += L.wave[k];
    if (id == e && r >= 0 && r < St::kRows) L.rows[r] = tid;
    __syncthreads();
    const int left = L.cnt[e] - r0, n = __builtin_amdgcn_readfirstlane(left < St::kRows ? left : St::kRows);
    stream_rows<kUp, kG, St>(a, L, e, part_k, n, t0, t1);
  }
}

// Down for up to kFewPairs pairs: a workgroup takes 16 columns of out through all
// the experts that have a row, so that it can weight the rows and add them to the
// residual itself, and no launch follows.  The waves split K as above, the weights
// of the next kRing experts in flight; all the experts' sums meet in LDS at once.
//   Bound by latency: ids, then weights and x, then two meetings of the waves.  16
// waves where K has more than 8 groups: 1 token of 4 of 32 experts of 1792, H =
// 2048, 8.1 us with 8 waves, 7.4 with 16; 6 of 64 of 768 6.8 / 7.4.  (Calls in us,
// in two launches / so: the first 11.8 / 8.8, 4 such tokens, 16 pairs, 16.4 / 19.2.)
static_assert(kFewPairs <= 8, "a wave an expert's sums; an expert's rows in a row tile");

struct FewArgs {
  MoeArgs m;
  const float* weights;  // or null: 1
  const float* res;
  float* out;
};

// grid = N / 16, block = 64 kWaves; K <= 128 kWaves kG
template <int kWaves, int kG>
__global__ __launch_bounds__(64 * kWaves) void k_moe_few(FewArgs f) {
  constexpr int kRing = kG == 1 ? 4 : 2;
  const MoeArgs& a = f.m;
  __shared__ f32x4 part[kFewPairs][kWaves][64];
  __shared__ u32x4 stage[kWaves][64];
  __shared__ float sums[kFewPairs][16];
  __shared__ int rows[kWaves][kFewPairs][kFewPairs];
  const int tid = threadIdx.x, l = tid & 63, n16 = l & 15, q = l >> 4, P = a.S * a.k;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c0 = 16 * blockIdx.x;
  // the rows by expert, lane i with pair i; an expert's first pair stands for it
  int id = l < P ? (a.ids ? a.ids[l] : 0) : -1;
  if ((unsigned)id >= (unsigned)a.E) id = -1;
  // this thread's output: column tid & 15 of token tid >> 4
  static_assert(kFewPairs <= 32, "a thread an output");
  const int so = tid >> 4;
  const float old = f.res[(size_t)(so < a.S ? so : 0) * a.N + c0 + (tid & 15)];
  const float wt = l < P && f.weights ? f.weights[l] : 1.0f;
  uint64_t same = __ballot(id >= 0);
  const uint64_t live = same;
#pragma unroll
  for (int b = 0; b < 8; b++) {
    const uint64_t v = __ballot(id >> b & 1);
    same &= id >> b & 1 ? v : ~v;
  }
  const uint64_t below = (1ull << l) - 1;
  const uint64_t firsts = __ballot(id >= 0 && !(same & below));
  const int nexp = __popcll(firsts);
  const int ng = a.K >> 7, g0 = w * ng / kWaves, mine = (w + 1) * ng / kWaves - g0;
  typedef const __attribute__((address_space(1))) uint16_t* gs_t;
  typedef const __attribute__((address_space(1))) u32x4* gw_t;
  u32x4 wr[kRing][kG];
  uint32_t sr[kRing][kG];
  // the n-th expert with a row
  auto expert = [&](int n) __attribute__((always_inline)) {
    uint64_t m = firsts;
    for (int i = 0; i < n; i++) m &= m - 1;
    return __builtin_amdgcn_readlane(id, __builtin_ctzll(m));
  };
  // its weights, scales and x rows of this wave's groups
  f16x8 A[kRing][kG][4];
  auto fetch = [&](int n, int d) __attribute__((always_inline)) {
    if (n >= nexp) return;
    const int e = expert(n);
    const uint64_t m = __ballot(id == e);
    const int left = __popcll(m);
    int* const list = rows[w][n];
    if (id == e) list[__popcll(m & below)] = l;
    if (mine == 0) return;
    const Cols<false> col(a, e, false);
    const gw_t wp = (gw_t)(col.packed(c0 + (l >> 2)) + 64 * (size_t)g0 + 16 * (l & 3));
    const gs_t sp = (gs_t)(col.scales(c0 + n16) + g0);
#pragma unroll
    for (int g = 0; g < kG; g++) {
      const int gg = g < mine ? g : 0;
      wr[d][g] = wp[4 * gg];
      sr[d][g] = sp[gg];
    }
    // (rows past the last one: the first, its products are not read)
    const int p = list[n16 < left ? n16 : 0];
    const gw_t xr = (gw_t)(a.x + (uint64_t)(uint32_t)p * (uint32_t)a.K + 128 * g0 + 32 * q);
    if (n16 < left)
#pragma unroll
      for (int g = 0; g < kG; g++)
#pragma unroll
        for (int s = 0; s < 4; s++) A[d][g][s] = __builtin_bit_cast(f16x8, xr[16 * (g < mine ? g : 0) + s]);
  };
#pragma unroll
  for (int d = 0; d < kRing; d++) {
#pragma unroll
    for (int g = 0; g < kG; g++)
#pragma unroll
      for (int s = 0; s < 4; s++) A[d][g][s] = f16x8{};
    fetch(d, d);
  }
#pragma unroll
  for (int n = 0; n < kFewPairs; n++) {
    const int d = n % kRing;
    if (n >= nexp) break;
    f32x4 acc = {};
    if (mine > 0) {
      u32x4 wq[kG];
      float scl[kG];
#pragma unroll
      for (int g = 0; g < kG; g++) {
        u32x4* st = stage[w];
        st[(l & ~3) | ((l & 3) ^ ((l >> 4) & 3))] = wr[d][g];
        wq[g] = st[4 * n16 + (q ^ ((n16 >> 2) & 3))];
        scl[g] = g < mine ? h2f((uint16_t)sr[d][g]) : 0.f;
      }
#pragma unroll
      for (int g = 0; g < kG; g++) {
        f32x4 Pg = {};
#pragma unroll
        for (int s = 0; s < 4; s++) Pg = __builtin_amdgcn_mfma_f32_16x16x32_f16(A[d][g][s], nib8(wq[g][s]), Pg, 0, 0, 0);
        if (g < mine)
#pragma unroll
          for (int i = 0; i < 4; i++) acc[i] = __builtin_fmaf(Pg[i], scl[g], acc[i]);
      }
    }
    fetch(n + kRing, d);
    part[n][w][l] = acc;
  }
  __syncthreads();
  // wave n adds up the n-th expert's (its own list of its rows)
  if (w < nexp) {
    f32x4 v = {};
#pragma unroll
    for (int k = 0; k < kWaves; k++) v += part[w][k][l];
    const int left = __popcll(__ballot(id == expert(w)));
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (4 * q + i < left) sums[rows[w][w][4 * q + i]][n16] = v[i];
  }
  __syncthreads();
  float v = old;
  for (int j = 0; j < a.k; j++) {
    const int p = so < a.S ? so * a.k + j : 0;
    const float wp = __shfl(wt, p);
    if (live >> p & 1) v = __builtin_fmaf(wp, sums[p][tid & 15], v);
  }
  if (so < a.S) f.out[(size_t)so * a.N + c0 + (tid & 15)] = v;
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

// out = res + the k weighted rows of each token, in the order of j, each the sum of
// its parts of K.  A thread takes 4 columns; bound by memory (4096 tokens of 2048, k =
// 4: 200 MB, 30 us).  4 loads together, of whichever rows and parts come next; without
// ids and weights (kDense) nothing stands between them (20 rows, 4 parts of 7168: the
// call 14.7 us with the other code, 12.9 so).
constexpr unsigned kCombineGrid = 1u << 20;

template <bool kDense>
__global__ __launch_bounds__(256) void k_moe_combine(CombineArgs a) {
  const unsigned nc = (a.H + 1023) / 1024;
  const size_t part = (size_t)a.S * a.k * a.H;
  for (unsigned b = blockIdx.x; b < (unsigned)a.S * nc; b += gridDim.x) {
    const int s = b / nc, c = (b % nc * 256 + threadIdx.x) * 4;
    if (c >= a.H) continue;
    f32x4 v = *(const f32x4*)(a.res + (size_t)s * a.H + c), sum = {};
    int j = 0, i = 0;  // the next row and part
    while (j < a.k) {
      f32x4 y[4];
      float w[4];
      bool live[4], last[4];
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const int p = s * a.k + (j < a.k ? j : a.k - 1), e = kDense || !a.ids ? 0 : a.ids[p];
        live[u] = j < a.k && (unsigned)e < (unsigned)a.E;
        last[u] = i == a.splits - 1;
        w[u] = kDense || !a.weights ? 1.0f : a.weights[p];
        y[u] = *(const f32x4*)(a.y + i * part + (size_t)p * a.H + c);  // (in ws whether written or not)
        i = last[u] ? 0 : i + 1;
        j += last[u];
      }
#pragma unroll
      for (int u = 0; u < 4; u++) {
        sum += y[u];
        if (!last[u]) continue;
#pragma unroll
        for (int q = 0; q < 4; q++)
          if (live[u]) v[q] = __builtin_fmaf(w[u], sum[q], v[q]);
        sum = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
    *(f32x4*)(a.out + (size_t)s * a.H + c) = v;
  }
}

// ---------------------------------------------------------------- host
static int64_t plan_bytes(int64_t P, int E) { return ((plan_rows_at(P, E) + P + 3) * 4 + 255) / 256 * 256; }

static int moe_check(int S, int k, int E, int H, int F, const int32_t* ids) {
  CIA_REQUIRE(S >= 0 && k >= 1 && k <= kMoeMaxK && E >= 1 && E <= kMoeMaxE && H > 0 && F > 0 &&
                  H % 128 == 0 && F % 128 == 0 && H <= kMoeMaxCols && F <= kMoeMaxCols &&
                  (int64_t)S * k <= kMoeMaxPairs,
              CIA_ERR_ARG);
  // without ids there is nothing to choose from
  CIA_REQUIRE(ids || (E == 1 && k == 1), CIA_ERR_ARG);
  return CIA_OK;
}

// an expert's strides hold its rows
static int q4_check(const cia_q4_experts* w, int E, int64_t rows, int64_t cols) {
  CIA_REQUIRE(w && w->packed && w->scales, CIA_ERR_NULL);
  CIA_REQUIRE(aligned(w->packed, 16) && aligned(w->scales, 2) && (E == 1 || w->packed_stride % 16 == 0), CIA_ERR_ALIGN);
  CIA_REQUIRE(E == 1 || (w->packed_stride >= rows * cols / 2 && w->scales_stride >= rows * cols / 128), CIA_ERR_ARG);
  return CIA_OK;
}

static void set_w(MoeArgs& a, int i, const cia_q4_experts* w) {
  a.packed[i] = w->packed;
  a.scales[i] = w->scales;
  a.pstride[i] = w->packed_stride;
  a.sstride[i] = w->scales_stride;
}

static_assert(2 * kMoeMaxE <= kStreamPairs && 64 <= kStreamPairs, "a thread a pair");

// (16 rows at a time: two workgroups a compute unit)
template <bool kUp, int kG>
static void stream_launch(const MoeArgs& a, int mt, hipStream_t s) {
  const dim3 block(64 * kStreamWaves);
  const int64_t P = (int64_t)a.S * a.k;
  if (kUp && mt > 1) {
    hipLaunchKernelGGL((k_moe_stream<kUp, kG, kUp ? stream_mt(kG) : 1>), dim3(kUnits), block, 0, s, a);
    return;
  }
  // (as many workgroups as tiles to take 4 of)
  const int64_t tiles = (P < a.E ? P : a.E) * ((kUp ? 2 * a.N : a.N) >> 4) * (kUp ? 1 : a.splits);
  const int n = tiles <= 4 * kUnits ? kUnits : kUnits * Stream<kG, 1>::kPerUnit;
  hipLaunchKernelGGL((k_moe_stream<kUp, kG, 1>), dim3(n), block, 0, s, a);
}

template <bool kUp, int kNT>
static void tile_launch(const MoeArgs& a, hipStream_t s) {
  const int nv = kUp ? 2 * a.N : a.N, cols = 16 * kNT * kTileWaves;
  const int64_t tiles = max_tiles((int64_t)a.S * a.k, a.E) * ((nv + cols - 1) / cols) * a.splits;
  hipLaunchKernelGGL((k_moe_tile<kUp, kNT>), dim3((unsigned)((tiles + 7) / 8 * 8 + 8)), dim3(64 * kTileWaves), 0, s, a);
}

// planned: ws holds the plan of these ids already
template <bool kUp>
static int products(MoeArgs& a, const MoeShape& shape, void* ws, bool planned, hipStream_t s) {
  if (shape.kernel == kMoeStream) {
    switch (shape.a) {
      case 1: stream_launch<kUp, 1>(a, shape.b, s); break;
      case 2: stream_launch<kUp, 2>(a, shape.b, s); break;
      default: stream_launch<kUp, 4>(a, shape.b, s);
    }
    return launch_status();
  }
  a.plan = shape.b ? (const int*)ws : nullptr;
  if (a.plan && !planned)
    hipLaunchKernelGGL(k_moe_plan, dim3(1), dim3(kPlanThreads), 0, s, a.ids, a.S * a.k, a.E, (int*)ws);
  switch (shape.a) {
    case 1: tile_launch<kUp, 1>(a, s); break;
    case 2: tile_launch<kUp, 2>(a, s); break;
    default: tile_launch<kUp, 3>(a, s);
  }
  return launch_status();
}

}  // namespace cia

using namespace cia;

extern "C" int64_t cia_moe_workspace_bytes(int S, int k, int E, int H, int F) {
  if (S < 0 || k < 1 || k > kMoeMaxK || E < 1 || E > kMoeMaxE || H < 1 || H > kMoeMaxCols || H % 128 || F < 1 ||
      F > kMoeMaxCols || F % 128)
    return 0;
  const int64_t P = (int64_t)S * k;
  return plan_bytes(P, E) + y_rows(P) * H * 4;
}

static int moe_up(const uint16_t* x, const int32_t* ids, const cia_q4_experts* w1, const cia_q4_experts* w3,
                  uint16_t* act, int S, int k, int E, int H, int F, void* ws, int64_t ws_bytes, void* stream) {
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
  const MoeShape shape = moe_shape(true, (int64_t)S * k, E, H, F);
  a.splits = shape.splits;
  return products<true>(a, shape, ws, false, (hipStream_t)stream);
}

extern "C" int cia_moe_up_int4(const uint16_t* x, const int32_t* ids, const cia_q4_experts* w1,
                               const cia_q4_experts* w3, uint16_t* act, int S, int k, int E, int H,
                               int F, void* ws, int64_t ws_bytes, void* stream) {
  return moe_up(x, ids, w1, w3, act, S, k, E, H, F, ws, ws_bytes, stream);
}

// planned: ws holds these ids' plan (moe_up's in tiles)
static int moe_down(const uint16_t* act, const int32_t* ids, const float* weights, const cia_q4_experts* w2,
                    const float* res, float* out, int S, int k, int E, int H, int F, void* ws, int64_t ws_bytes,
                    bool planned, void* stream) {
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
  const MoeShape shape = moe_shape(false, (int64_t)S * k, E, F, H);
  a.splits = shape.splits;
  hipStream_t s = (hipStream_t)stream;
  if (shape.kernel == kMoeFew) {
    const FewArgs f{a, weights, res, out};
    const dim3 grid((unsigned)(H / 16));
    if (shape.a == 8)
      hipLaunchKernelGGL((k_moe_few<8, 1>), grid, dim3(512), 0, s, f);
    else if (shape.b == 1)
      hipLaunchKernelGGL((k_moe_few<16, 1>), grid, dim3(1024), 0, s, f);
    else
      hipLaunchKernelGGL((k_moe_few<16, 2>), grid, dim3(1024), 0, s, f);
    return launch_status();
  }
  if (!ids && !weights && a.splits == 1 && shape.kernel == kMoeTile) {
    a.res = res;
    a.out = out;
    return products<false>(a, shape, ws, planned, s);
  }
  if ((st = products<false>(a, shape, ws, planned, s))) return st;
  const CombineArgs c{a.y, ids, weights, res, out, S, k, E, H, a.splits};
  const unsigned blocks = (unsigned)((H + 1023) / 1024) * (unsigned)S;
  const dim3 grid(blocks < kCombineGrid ? blocks : kCombineGrid);
  if (!ids && !weights)
    hipLaunchKernelGGL(k_moe_combine<true>, grid, dim3(256), 0, s, c);
  else
    hipLaunchKernelGGL(k_moe_combine<false>, grid, dim3(256), 0, s, c);
  return launch_status();
}

extern "C" int cia_moe_down_int4(const uint16_t* act, const int32_t* ids, const float* weights,
                                 const cia_q4_experts* w2, const float* res, float* out, int S, int k,
                                 int E, int H, int F, void* ws, int64_t ws_bytes, void* stream) {
  return moe_down(act, ids, weights, w2, res, out, S, k, E, H, F, ws, ws_bytes, false, stream);
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
  if (!M || cap < 0) return 0;
  const int k = M->gate ? M->gating.top_k : 1, E = M->gate ? M->gating.n_experts : 1;
  if (!cia_moe_workspace_bytes(0, k, E, M->H, M->F) || (int64_t)cap * k > kMoeMaxPairs) return 0;
  return block_ws(M, cap).end;
}

extern "C" int cia_moe_block_forward(const cia_moe* M, float* h, int S, void* stream) {
  CIA_REQUIRE(M, CIA_ERR_NULL);
  CIA_REQUIRE(S >= 0 && S <= M->cap, CIA_ERR_ARG);
  if (S == 0) return CIA_OK;
  CIA_REQUIRE(h, CIA_ERR_NULL);
  const int k = M->gate ? M->gating.top_k : 1, E = M->gate ? M->gating.n_experts : 1;
  CIA_REQUIRE(M->ws, CIA_ERR_NULL);
  CIA_REQUIRE(aligned(M->ws, 16) && aligned(M->gate, 16) && (!M->gate || aligned(M->bias, 4)), CIA_ERR_ALIGN);
  // the branch's arguments before its first launch (the norm checks its own, and is
  // the first; h is written by the last)
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
  if ((st = moe_up(x, ids, &M->w1, &M->w3, act, S, k, E, M->H, M->F, ws + b.moe, M->ws_bytes - b.moe, stream)))
    return st;
  return moe_down(act, ids, weights, &M->w2, h, h, S, k, E, M->H, M->F, ws + b.moe, M->ws_bytes - b.moe,
                  !streams(true, (int64_t)S * k, E, M->H), stream);
}
