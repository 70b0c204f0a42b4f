// attn_pages.hip -- attention of one query token per row over a paged key-value
// cache on gfx950: per row t and query head h
//   s_j = scale q . k_j,   out = sum_j exp(s_j - max s) v_j / sum_j exp(s_j - max s)
// over the tokens of the row's sequence up to its position, each K and V row read once.
//
// Bound by memory: 2 D + 4 bytes a token and kv head in e4m3, 4 D in fp16.  32 query heads
// on 8 kv heads of 64 in e4m3: 256 rows of 900 to 2048 tokens take 78 us (380 MB, 4.9 TB/s; a
// large copy reaches 5.1), 58 of 9 to 9000 21.3 (89 MB, 4.2 TB/s), one of 32 768
// 12.7 (35 MB in about 6, launch and first loads 4, the join 3), one of 700 6.4.
//
// Work.  A row's tokens are units of 128, and the units of all rows one list, of which
// each of the P workgroups of a kv head takes an equal part, whatever rows it falls
// into: batches of very different lengths keep every compute unit busy to the end.  A
// row's start counts as some units more, or workgroups of many short rows end last (with
// a better join and fewer parts 27.9 -> 23.5 us for 58 ragged rows).  The
// list follows from the positions on the device, so a captured call can be replayed with
// others.  A row in one workgroup's part is finished there; the parts of a longer one are
// joined by the workgroup that ends last (it counts itself in, nothing waits).
//
// A tile is 32 tokens of a wave, both products on the matrix cores with no pass through
// LDS: S^T = K Q^T leaves a lane (column n, block g) with tokens of rows 4 g + r, and
// which token a row is may be chosen: token 4 r + g, so that lane block g has the tokens
// g, 4 + g, .., 28 + g of the tile, in the order in which the second product's lanes
// take 8 of them, and eight loads of V rows are each of 4 neighbouring rows.  Fewer than
// 16 query heads fill the 16 columns several times over (kNB): column block j keeps the
// scores of r = j alone, so a lane has two exponentials a tile instead of eight, and
// its products' other places are zeros; the blocks' sums are added at the row's end.
// Matrix cores are busy 9 % of the time, vector units 33 % (256 rows): neither bounds.
#include "decode_wave.h"
#include "pages.h"

namespace cia {

constexpr int kUnit = 128;        // tokens of a unit: 32 a wave
constexpr int kRowCost = 2;       // units that a row's start and end take the time of
// Workgroups of a call, two a compute unit.  (Three: even for 256 rows, 15.5 us for 13.1 for one
// of 32 768 tokens, whose join has more parts.)
constexpr int kGroups = 512;
constexpr int kMaxParts = 256;    // of them for one kv head
constexpr int kTicketStride = 16;  // uint32 between two counters
constexpr int64_t kTicketBytes = (int64_t)kGroups * kTicketStride * 4;
constexpr float kLow = -3.0e38f;  // max of no scores: finite, so that exp2(-inf - kLow) is 0
// The largest numerator of a column is 2^12, and up to 2^15 until the rest is scaled down to
// it: fp16's least step is then 2^-36 of it.  (With 1 for the largest, 12 000 tokens of 4e-8
// of its weight were 1/40 off in their sum.)
constexpr float kLift = 12.0f, kMost = 15.0f;
// Scores from here on have steps of 1/2 and more in fp32, and less kLift they are rounded: by
// steps of 4 to 16 about 2^26, which made numerators of 2^16 and more, that fp16 has not.  Of
// these the largest score itself is taken off, which leaves numerators of at most V's scale;
// the bits of small weights are lost in the scores' steps there.
constexpr float kFar = 0x1p22f;

struct AttnPagesArgs {
  Pages P;
  const uint16_t* q;
  int64_t q_stride;
  const int32_t* seq;  // or null
  const int32_t* pos;
  int T, n_q, group;  // group: query heads of a kv head
  int cols;           // parts of 16 query heads of a kv head
  int parts;          // workgroups of a kv head (and part of 16)
  float scale;        // times log2 e
  int window;
  uint16_t* out;
  uint32_t* tickets;
  float* partial;
};

// the tokens [first, len) of a row
struct Span {
  int seq, first, len;
};
__device__ __forceinline__ Span row_span(const AttnPagesArgs& a, int t) {
  const int s = a.seq ? a.seq[t] : t, pos = a.pos[t];
  Span r{s, 0, 0};
  if (s >= 0 && s < a.P.n_seq && pos >= 0) {
    r.len = min(pos, a.P.max_tokens - 1) + 1;
    if (a.window > 0) r.first = max(0, pos - a.window + 1);
    if (r.first >= r.len) r.len = 0;
  }
  return r;
}
// a row's cost: its units, and kRowCost for its start
__device__ __forceinline__ int span_cost(const Span& r) {
  return r.len ? (r.len + kUnit - 1) / kUnit - r.first / kUnit + kRowCost : 0;
}

template <int kD, bool kF8, int kNB>
struct AttnTile {
  static constexpr int kRowB = kD * (kF8 ? 1 : 2);
  static constexpr int kK = kRowB / 64;   // 16-byte loads of a K row's part, a lane
  static constexpr int kV = kRowB / 64;   // dwords of a V row, a lane
  static constexpr int kR = 4 / kNB;      // scores of a lane in 16 tokens
  u32x4 k[2][kK];
  uint32_t v[8][kV];
  uint16_t ks[2][kR], vs[2][kR];
};

template <int kV>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[kV]) {
  if constexpr (kV == 1) {
    w[0] = *(const uint32_t*)p;
  } else if constexpr (kV == 2) {
    const u32x2 x = *(const u32x2*)p;
    w[0] = x[0], w[1] = x[1];
  } else {
    const u32x4 x = *(const u32x4*)p;
    w[0] = x[0], w[1] = x[1], w[2] = x[2], w[3] = x[3];
  }
}

__device__ __forceinline__ uint32_t f16_bits(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }

// Partials cross the XCDs: coherent stores and loads, the workgroup's address plus a
// uniform offset in floats and a lane's.
__device__ __forceinline__ void put4(__amdgpu_buffer_rsrc_t ws, int at, int lane_at, const f32x4& x) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), ws, lane_at * 4, at * 4, kCoherent);
}
__device__ __forceinline__ f32x4 take4(__amdgpu_buffer_rsrc_t ws, int at, int lane_at) {
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(ws, lane_at * 4, at * 4, kCoherent));
}

// grid = kv heads * cols * parts, block = 256, LDS: T rows
template <int kD, bool kF8, int kNB>
__global__ __launch_bounds__(256, 2) void k_attn_pages(AttnPagesArgs a) {
  using Tile = AttnTile<kD, kF8, kNB>;
  constexpr int kRp = 16 / kNB;        // query heads of a workgroup
  constexpr int kRowB = Tile::kRowB, kR = Tile::kR, kO = kD / 16;
  constexpr int kPart = kRp * (kD + 4);  // floats of a partial: o, then (max, sum, -, -) of each head
  constexpr int kVecs = kRp * kD / 4;    // fours of a row's outputs
  extern __shared__ Span spans[];  // of the rows, and then the cost before each
  int* const pre = (int*)(spans + a.T);
  __shared__ union {
    struct {
      float o[4][kRp][kD];
      float m[4][kRp], l[4][kRp];
    } w;
    struct {
      float weight[kRp][kMaxParts];
      float o[256 * 4];
      float l[kRp];
    } j;
  } s;
  __shared__ int wsum[4], last;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n_vh = a.P.n_kv * a.cols, vh = blockIdx.x % n_vh, part = blockIdx.x / n_vh;
  const int head = vh / a.cols, h0 = head * a.group + vh % a.cols * 16;  // kv head, first query head
  const int heads = min(kRp, a.group - vh % a.cols * 16);

  // ---- the list of the rows' costs; rows without any units are zeros
  auto put_row = [&](int t, const Span& r, int before, int cost) __attribute__((always_inline)) {
    pre[t] = before;
    spans[t] = r;
    if (cost == 0 && t % a.parts == part)
      for (int i = 0; i < heads * kD / 8; i++)
        *(u32x4*)(a.out + ((int64_t)t * a.n_q + h0) * kD + 8 * i) = u32x4{0, 0, 0, 0};
  };
  int total = 0, start = 0x7fffffff;  // start: of row `lane`, up to 64 rows
  if (a.T <= 64) {
    // every wave for itself: what it reads of the list, it has written
    const Span r = lane < a.T ? row_span(a, lane) : Span{0, 0, 0};
    const int cost = span_cost(r), upto = scan_lanes(cost);
    if (lane < a.T) put_row(lane, r, start = upto - cost, cost);
    total = __builtin_amdgcn_readlane(upto, 63);
    if (lane == 0) pre[a.T] = total;
  } else {
    for (int base = 0; base < a.T; base += 256) {
      const int t = base + tid;
      const Span r = t < a.T ? row_span(a, t) : Span{0, 0, 0};
      const int cost = span_cost(r), upto = scan_lanes(cost);
      if (lane == 63) wsum[wave] = upto;
      __syncthreads();
      int before = total;
      for (int w = 0; w < 4; w++) {
        if (w < wave) before += wsum[w];
        total += wsum[w];
      }
      if (t < a.T) put_row(t, r, before + upto - cost, cost);
      __syncthreads();
    }
    if (tid == 0) pre[a.T] = total;
    __syncthreads();
  }
  if (total == 0) return;
  // as few parts as make the largest no larger
  const int most = (total + a.parts - 1) / a.parts, parts = (total + most - 1) / most;
  if (part >= parts) return;
  // (exact: the quotients' fractions are at least 2^-8, in numbers below 2^31)
  const int from = (int)((double)total * part / parts), to = (int)((double)total * (part + 1) / parts);

  // ---- the lane's places
  const int n = lane & 15, g = lane >> 4, j = n / kRp;
  const int mine = n & (kRp - 1);  // query head of the column
  const uint32_t k_lane = (uint32_t)((4 * (n & 3) + (n >> 2)) * kRowB + 16 * g);
  const uint32_t v_lane = (uint32_t)(g * kRowB + n * (kRowB / 16));
  const int page_mask = (1 << a.P.shift) - 1;

  // the last row that starts at or before `from`, among 64 rows or groups of them at once
  int row;
  if (a.T <= 64) {
    row = __popcll(__ballot(start <= from)) - 1;
  } else {
    const int per = (a.T + 63) / 64;
    row = (__popcll(__ballot(lane * per < a.T && pre[min(lane * per, a.T)] <= from)) - 1) * per;
    row += __popcll(__ballot(lane < per && row + lane < a.T && pre[min(row + lane, a.T)] <= from)) - 1;
  }
  for (; row < a.T && pre[row] < to; row++) {
    // the units [u0, u1) of the row's
    const int r0 = pre[row] + kRowCost, r1 = pre[row + 1];
    const int u0 = max(from - r0, 0), u1 = min(to, r1) - r0, count = u1 - u0;
    if (count <= 0) continue;
    const Span span = spans[row];
    const int base = (span.first / kUnit + u0) * kUnit + 32 * wave;  // the wave's first token

    f16x8 Q[kD / 32];
#pragma unroll
    for (int i = 0; i < kD / 32; i++) {
      const int d = kF8 ? 64 * (i >> 1) + 16 * g + 8 * (i & 1) : 32 * i + 8 * g;
      u32x4 w{0, 0, 0, 0};
      if (mine < heads) w = *(const u32x4*)(a.q + row * a.q_stride + (h0 + mine) * kD + d);
      Q[i] = __builtin_bit_cast(f16x8, w);
    }
    float m = kLow, l = 0.0f;
    f32x4 O[kO];
#pragma unroll
    for (int i = 0; i < kO; i++) O[i] = f32x4{0.f, 0.f, 0.f, 0.f};

    for (int chunk = 0; chunk < count; chunk += 32) {
      // page ids of the next 32 tiles: lane 2 i + b, 16 tokens b of tile i
      int pids = -1;
      {
        const int i = chunk + (lane >> 1), tok = base + i * kUnit + 16 * (lane & 1);
        if (i < count && tok < span.len && tok + 16 > span.first) pids = page_of(a.P, span.seq, tok);
      }
      const int tiles = min(32, count - chunk);
      auto load = [&](Tile& x, int i) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < 2; b++) {
          const int pid = max(0, __builtin_amdgcn_readlane(pids, 2 * i + b));  // (none: masked, any page)
          const int tok = (base + (chunk + i) * kUnit + 16 * b) & page_mask;
          const int64_t r = (((int64_t)pid * a.P.n_kv + head) << a.P.shift) + tok;
          const uint8_t* kp = (const uint8_t*)a.P.k + r * kRowB;
          const uint8_t* vp = (const uint8_t*)a.P.v + r * kRowB;
#pragma unroll
          for (int c = 0; c < Tile::kK; c++) x.k[b][c] = *(const u32x4*)(kp + k_lane + 64 * c);
#pragma unroll
          for (int e = 0; e < 4; e++) load_words(vp + v_lane + 4 * e * kRowB, x.v[4 * b + e]);
          if constexpr (kF8) {
#pragma unroll
            for (int e = 0; e < kR; e++) {
              x.ks[b][e] = a.P.ks[r + 4 * (j * kR + e) + g];
              x.vs[b][e] = a.P.vs[r + 4 * (j * kR + e) + g];
            }
          }
        }
      };
      auto compute = [&](Tile& x, int i) __attribute__((always_inline)) {
        const int tok = base + (chunk + i) * kUnit;
        const int p0 = __builtin_amdgcn_readlane(pids, 2 * i), p1 = __builtin_amdgcn_readlane(pids, 2 * i + 1);
        const bool whole = p0 >= 0 && p1 >= 0 && tok >= span.first && tok + 32 <= span.len;
        float y[2][kR], vs[2][kR];
#pragma unroll
        for (int b = 0; b < 2; b++) {
          f32x4 S{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < Tile::kK; c++) {
            if constexpr (kF8) {
              S = __builtin_amdgcn_mfma_f32_16x16x32_f16(cvt8(x.k[b][c][0], x.k[b][c][1]), Q[2 * c], S, 0, 0, 0);
              S = __builtin_amdgcn_mfma_f32_16x16x32_f16(cvt8(x.k[b][c][2], x.k[b][c][3]), Q[2 * c + 1], S, 0, 0, 0);
            } else {
              S = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x.k[b][c]), Q[c], S, 0, 0, 0);
            }
          }
          if constexpr (kNB == 4) {
            y[b][0] = j < 2 ? (j == 0 ? S[0] : S[1]) : (j == 2 ? S[2] : S[3]);
          } else if constexpr (kNB == 2) {
            y[b][0] = j ? S[2] : S[0];
            y[b][1] = j ? S[3] : S[1];
          } else {
#pragma unroll
            for (int e = 0; e < 4; e++) y[b][e] = S[e];
          }
#pragma unroll
          for (int e = 0; e < kR; e++) {
            if constexpr (kF8) {
              y[b][e] *= h2f(x.ks[b][e]) * a.scale;
              vs[b][e] = h2f(x.vs[b][e]);
            } else {
              y[b][e] *= a.scale;
              vs[b][e] = 1.0f;
            }
          }
        }
        if (!whole) {
          // tokens outside the span or without a page: no weight, and zeros for V, whose
          // bytes may be anything
#pragma unroll
          for (int b = 0; b < 2; b++) {
            const int first = (b ? p1 : p0) >= 0 ? span.first : 0x7fffffff;
#pragma unroll
            for (int e = 0; e < kR; e++) {
              const int u = tok + 16 * b + 4 * (j * kR + e) + g;
              if (u < first || u >= span.len) y[b][e] = -__builtin_inff(), vs[b][e] = 0.0f;
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const int u = tok + 16 * b + 4 * e + g;
              if (u < first || u >= span.len)
#pragma unroll
                for (int c = 0; c < Tile::kV; c++) x.v[4 * b + e][c] = 0;
            }
          }
        }
        // The numerators are those of weight times V's scale, so that they fill fp16's
        // range whatever the scales are: m is the max of s + log2 vs, less kLift.  It is let
        // lag: a rescaling only where a numerator would be 2^kMost or more.  (With steps of
        // u there, top is off by u / 2 and so is the sum with kMost; of two numbers in these
        // steps the smaller is less by u: what is not rescaled is below 2^kMost or at it.)
        float top = -__builtin_inff();
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
          for (int e = 0; e < kR; e++)
            top = __builtin_fmaxf(
                top, kF8 ? y[b][e] + __builtin_amdgcn_logf(__builtin_fmaxf(vs[b][e], 0x1p-24f)) : y[b][e]);
        if (__any(top >= m + kMost)) {
          float score = -__builtin_inff();
#pragma unroll
          for (int b = 0; b < 2; b++)
#pragma unroll
            for (int e = 0; e < kR; e++) score = __builtin_fmaxf(score, y[b][e]);
          score = col4_max(score), top = col4_max(top);
          const float now = __builtin_fmaxf(m, __builtin_fabsf(top) < kFar ? top - kLift : score);
          const float f = __builtin_amdgcn_exp2f(m - now);
          m = now;
          l *= f;
#pragma unroll
          for (int i = 0; i < kO; i++) O[i] *= f;
        }
        // numerators as two fp16: 22 bits (256 rows 80.2 us, with one of 11 bits 79.8)
        uint32_t hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
#pragma unroll
        for (int b = 0; b < 2; b++) {
          uint32_t ph[kR], pl[kR];
#pragma unroll
          for (int e = 0; e < kR; e++) {
            const float p = __builtin_amdgcn_exp2f(y[b][e] - m);
            l += p;
            const float w = kF8 ? p * vs[b][e] : p;
            ph[e] = f16_bits(w);
            pl[e] = f16_bits(w - h2f((uint16_t)ph[e]));
          }
          if constexpr (kNB == 4) {
            const uint32_t sh = 16 * (j & 1), low = j < 2 ? ~0u : 0u;
            hi[2 * b] = (ph[0] << sh) & low;
            hi[2 * b + 1] = (ph[0] << sh) & ~low;
            lo[2 * b] = (pl[0] << sh) & low;
            lo[2 * b + 1] = (pl[0] << sh) & ~low;
          } else if constexpr (kNB == 2) {
            const uint32_t h = ph[0] | ph[1] << 16, w = pl[0] | pl[1] << 16;
            hi[2 * b] = j ? 0 : h;
            hi[2 * b + 1] = j ? h : 0;
            lo[2 * b] = j ? 0 : w;
            lo[2 * b + 1] = j ? w : 0;
          } else {
            hi[2 * b] = ph[0] | ph[1] << 16;
            hi[2 * b + 1] = ph[2] | ph[3] << 16;
            lo[2 * b] = pl[0] | pl[1] << 16;
            lo[2 * b + 1] = pl[2] | pl[3] << 16;
          }
        }
        const f16x8 H = __builtin_bit_cast(f16x8, u32x4{hi[0], hi[1], hi[2], hi[3]});
        const f16x8 L = __builtin_bit_cast(f16x8, u32x4{lo[0], lo[1], lo[2], lo[3]});
        // a lane's words are neighbouring dimensions of a token; a product takes 8 tokens
        // of one
#pragma unroll
        for (int c = 0; c < Tile::kV; c++) {
          if constexpr (kF8) {
            u32x4 A[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const uint32_t u = __builtin_amdgcn_perm(x.v[2 * e + 1][c], x.v[2 * e][c], 0x05010400);
              const uint32_t w = __builtin_amdgcn_perm(x.v[2 * e + 1][c], x.v[2 * e][c], 0x07030602);
              A[0][e] = __builtin_bit_cast(uint32_t, (f16x2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(u, 1.0f, false));
              A[1][e] = __builtin_bit_cast(uint32_t, (f16x2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(u, 1.0f, true));
              A[2][e] = __builtin_bit_cast(uint32_t, (f16x2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
              A[3][e] = __builtin_bit_cast(uint32_t, (f16x2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const f16x8 V = __builtin_bit_cast(f16x8, A[i]);
              O[4 * c + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(V, H, O[4 * c + i], 0, 0, 0);
              O[4 * c + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(V, L, O[4 * c + i], 0, 0, 0);
            }
          } else {
            u32x4 A[2];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              A[0][e] = __builtin_amdgcn_perm(x.v[2 * e + 1][c], x.v[2 * e][c], 0x05040100);
              A[1][e] = __builtin_amdgcn_perm(x.v[2 * e + 1][c], x.v[2 * e][c], 0x07060302);
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const f16x8 V = __builtin_bit_cast(f16x8, A[i]);
              O[2 * c + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(V, H, O[2 * c + i], 0, 0, 0);
              O[2 * c + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(V, L, O[2 * c + i], 0, 0, 0);
            }
          }
        }
      };
      if constexpr (kRowB == 256) {
        // (16 KiB of loads a wave: two tiles of them do not fit the registers beside O)
        Tile x;
        for (int i = 0; i < tiles; i++) {
          load(x, i);
          compute(x, i);
        }
      } else {
        Tile x0, x1;
        load(x0, 0);
        for (int i = 0; i < tiles; i += 2) {
          if (i + 1 < tiles) load(x1, i + 1);
          compute(x0, i);
          if (i + 1 < tiles) {
            if (i + 2 < tiles) load(x0, i + 2);
            compute(x1, i + 1);
          }
        }
      }
    }

    // ---- a head's column blocks, then the waves
    float M = m;
    if constexpr (kNB >= 2) M = __builtin_fmaxf(M, row_ror<8>(M));
    if constexpr (kNB == 4) M = __builtin_fmaxf(M, row_ror<4>(M));
    const float f = __builtin_amdgcn_exp2f(m - M);
    l = col4_sum(l) * f;
    if constexpr (kNB >= 2) l += row_ror<8>(l);
    if constexpr (kNB == 4) l += row_ror<4>(l);
#pragma unroll
    for (int i = 0; i < kO; i++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        float o = O[i][r] * f;
        if constexpr (kNB >= 2) o += row_ror<8>(o);
        if constexpr (kNB == 4) o += row_ror<4>(o);
        O[i][r] = o;
      }
    __syncthreads();
    if (j == 0) {
      // O[i][r]: dimension kO (4 g + r) + i
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int i = 0; i < kO; i += 4)
          *(f32x4*)&s.w.o[wave][mine][kO * (4 * g + r) + i] = f32x4{O[i][r], O[i + 1][r], O[i + 2][r], O[i + 3][r]};
      if (g == 0) s.w.m[wave][mine] = M, s.w.l[wave][mine] = l;
    }
    __syncthreads();
    const bool ends = u0 == 0 && r0 + u1 == r1;  // the whole row
    const __amdgpu_buffer_rsrc_t ws = buf_rsrc(a.partial + (int64_t)vh * a.parts * 2 * kPart);
    for (int i = tid; i < kVecs; i += 256) {
      const int h = i / (kD / 4), d = i % (kD / 4) * 4;
      float top = s.w.m[0][h];
#pragma unroll
      for (int w = 1; w < 4; w++) top = __builtin_fmaxf(top, s.w.m[w][h]);
      float sum = 0.0f;
      f32x4 o{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; w++) {
        const float e = __builtin_amdgcn_exp2f(s.w.m[w][h] - top);
        sum = __builtin_fmaf(s.w.l[w][h], e, sum);
        const f32x4 x = *(const f32x4*)&s.w.o[w][h][d];
#pragma unroll
        for (int c = 0; c < 4; c++) o[c] = __builtin_fmaf(x[c], e, o[c]);
      }
      if (ends) {
        if (h < heads) {
          const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
          *(f16x4*)(a.out + ((int64_t)row * a.n_q + h0 + h) * kD + d) =
              f16x4{(_Float16)(o[0] * inv), (_Float16)(o[1] * inv), (_Float16)(o[2] * inv), (_Float16)(o[3] * inv)};
        }
      } else {
        const int to = (part * 2 + (u0 == 0 ? 1 : 0)) * kPart;
        put4(ws, to, h * kD + d, o);
        if (d == 0) put4(ws, to, kRp * kD + 4 * h, f32x4{top, sum, 0.f, 0.f});
      }
    }
    if (!ends) {
      // the row's parts: the workgroups that have a unit of it, from that of its first
      // (exact as above: fractions of at least 2^-31, in numbers up to 256)
      const double N = total, W = parts;
      const int first = (int)(((r0 + 1) * W - 1) / N), fin = (int)((r1 * W - 1) / N);
      const int pieces = fin - first + 1;
      stores_acked();
      __syncthreads();
      if (tid == 0) {
        uint32_t* const c = a.tickets + (int64_t)(vh * a.parts + first) * kTicketStride;
        const uint32_t had = __hip_atomic_fetch_add(c, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = had + 1 == (uint32_t)pieces;
        if (last) __hip_atomic_store(c, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      __syncthreads();
      if (last) {
        auto piece = [&](int i) { return ((first + i) * 2 + (i == 0 ? 1 : 0)) * kPart; };
        constexpr int kSplit = kVecs < 256 ? 256 / kVecs : 1;  // ways that share a four's pieces
        constexpr int kFours = kVecs > 256 ? kVecs / 256 : 1;  // fours of a thread
        // a thread's first pieces are on their way while the weights are made
        constexpr int kEarly = 8 / kFours, kHeads = kRp / 4;
        const int way = __builtin_amdgcn_readfirstlane(tid / kVecs);
        f32x4 early[kFours][kEarly];
#pragma unroll
        for (int f = 0; f < kFours; f++)
#pragma unroll
          for (int c = 0; c < kEarly; c++) {
            early[f][c] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (way + c * kSplit < pieces)
              early[f][c] = take4(ws, piece(way + c * kSplit), 4 * (tid % kVecs + 256 * f));
          }
        // a wave's heads, a piece a lane
        float pm[kHeads][kMaxParts / 64], pl[kHeads][kMaxParts / 64];
#pragma unroll
        for (int c = 0; c < kMaxParts / 64; c++)
#pragma unroll
          for (int e = 0; e < kHeads; e++) {
            pm[e][c] = kLow, pl[e][c] = 0.0f;
            if (64 * c < pieces && lane + 64 * c < pieces) {
              const f32x4 x = take4(ws, 0, piece(lane + 64 * c) + kRp * kD + 4 * (wave + 4 * e));
              pm[e][c] = x[0], pl[e][c] = x[1];
            }
          }
#pragma unroll
        for (int e = 0; e < kHeads; e++) {
          float top = pm[e][0], sum = 0.0f;
#pragma unroll
          for (int c = 1; c < kMaxParts / 64; c++) top = __builtin_fmaxf(top, pm[e][c]);
          top = wave_max_fast(top);
#pragma unroll
          for (int c = 0; c < kMaxParts / 64; c++) {
            const float w = __builtin_amdgcn_exp2f(pm[e][c] - top);
            sum = __builtin_fmaf(pl[e][c], w, sum);
            s.j.weight[wave + 4 * e][lane + 64 * c] = w;
          }
          sum = wave_sum_fast(sum);
          if (lane == 0) s.j.l[wave + 4 * e] = sum;
        }
        __syncthreads();
#pragma unroll
        for (int f = 0; f < kFours; f++) {
          const int i4 = tid % kVecs + 256 * f, h = i4 / (kD / 4), d = i4 % (kD / 4) * 4;
          f32x4 o{0.f, 0.f, 0.f, 0.f};
          auto add = [&](const f32x4& x, int i) __attribute__((always_inline)) {
            const float e = s.j.weight[h][i];
#pragma unroll
            for (int c = 0; c < 4; c++) o[c] = __builtin_fmaf(x[c], e, o[c]);
          };
#pragma unroll
          for (int c = 0; c < kEarly; c++) add(early[f][c], way + c * kSplit);  // (0 past the last)
#pragma unroll 1
          for (int i = way + kEarly * kSplit; i < pieces; i += kEarly * kSplit) {
            f32x4 x[kEarly];
#pragma unroll
            for (int c = 0; c < kEarly; c++)
              if (i + c * kSplit < pieces) x[c] = take4(ws, piece(i + c * kSplit), 4 * i4);
#pragma unroll
            for (int c = 0; c < kEarly; c++)
              if (i + c * kSplit < pieces) add(x[c], i + c * kSplit);
          }
          if constexpr (kSplit > 1) {
            *(f32x4*)&s.j.o[4 * tid] = o;
            __syncthreads();
            if (tid < kVecs)
#pragma unroll
              for (int c = 1; c < kSplit; c++) o += *(const f32x4*)&s.j.o[4 * (tid + c * kVecs)];
          }
          if (tid < kVecs && h < heads) {
            const float inv = s.j.l[h] == 0.0f ? 0.0f : 1.0f / s.j.l[h];
            *(f16x4*)(a.out + ((int64_t)row * a.n_q + h0 + h) * kD + d) =
                f16x4{(_Float16)(o[0] * inv), (_Float16)(o[1] * inv), (_Float16)(o[2] * inv), (_Float16)(o[3] * inv)};
          }
        }
      }
    }
  }
}

// workgroups of a kv head (and part of 16 query heads)
static int attn_parts(int vheads) { return std::max(1, std::min(kMaxParts, kGroups / vheads)); }
static int attn_columns(int group) { return group <= 4 ? 4 : group <= 8 ? 8 : 16; }

template <int kD, bool kF8>
static void attn_launch(const AttnPagesArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.P.n_kv * a.cols * a.parts));
  const size_t lds = (size_t)a.T * (sizeof(Span) + sizeof(int)) + sizeof(int);
  switch (attn_columns(a.group)) {
    case 4: hipLaunchKernelGGL((k_attn_pages<kD, kF8, 4>), grid, dim3(256), lds, s, a); break;
    case 8: hipLaunchKernelGGL((k_attn_pages<kD, kF8, 2>), grid, dim3(256), lds, s, a); break;
    default: hipLaunchKernelGGL((k_attn_pages<kD, kF8, 1>), grid, dim3(256), lds, s, a); break;
  }
}

}  // namespace cia

using namespace cia;

extern "C" int64_t cia_attn_pages_workspace_bytes(int n_q, int n_kv, int head_dim) {
  if (n_kv < 1 || n_kv > CIA_PAGES_MAX_KV || (head_dim != 64 && head_dim != 128) || n_q < n_kv || n_q % n_kv ||
      n_q / n_kv > CIA_PAGES_MAX_GROUP)
    return 0;
  const int group = n_q / n_kv, vheads = n_kv * ((group + 15) / 16);
  return kTicketBytes + (int64_t)vheads * attn_parts(vheads) * 2 * attn_columns(group) * (head_dim + 4) * sizeof(float);
}

extern "C" int cia_attn_pages(const cia_kv_pages* p, const uint16_t* q, int64_t q_stride, const int32_t* seq,
                              const int32_t* pos, int T, int n_q, float scale, int window, uint16_t* out, void* ws,
                              int64_t ws_bytes, void* stream) {
  int st = pages_check(p);
  if (st) return st;
  const int64_t need = cia_attn_pages_workspace_bytes(n_q, p->n_kv, p->head_dim);
  CIA_REQUIRE(need > 0 && T >= 0 && T <= CIA_PAGES_MAX_ROWS && (seq || T <= p->n_seq), CIA_ERR_ARG);
  CIA_REQUIRE(q_stride >= (int64_t)n_q * p->head_dim && q_stride % 8 == 0 && window >= 0, CIA_ERR_ARG);
  // (scores of finite q and K are below 2^48, so that they stay above kLow times log2 e; no NaN)
  CIA_REQUIRE(__builtin_fabsf(scale) <= 0x1p64f, CIA_ERR_ARG);
  if (T == 0) return CIA_OK;
  if ((st = pages_check_ptr(p))) return st;
  CIA_REQUIRE(q && pos && out && ws, CIA_ERR_NULL);
  CIA_REQUIRE(aligned(q, 16) && aligned(seq, 4) && aligned(pos, 4) && aligned(out, 16) && aligned(ws, 16),
              CIA_ERR_ALIGN);
  CIA_REQUIRE(ws_bytes >= need, CIA_ERR_ARG);
  const int group = n_q / p->n_kv, cols = (group + 15) / 16;
  const AttnPagesArgs a{pages_of(p), q,    q_stride, seq,           pos,    T,   n_q,
                        group,       cols, attn_parts(p->n_kv * cols), scale * kLog2e, window, out,
                        (uint32_t*)ws, (float*)((char*)ws + kTicketBytes)};
  hipStream_t s = (hipStream_t)stream;
  if (p->head_dim == 64) {
    if (p->type == CIA_KV_E4M3)
      attn_launch<64, true>(a, s);
    else
      attn_launch<64, false>(a, s);
  } else {
    if (p->type == CIA_KV_E4M3)
      attn_launch<128, true>(a, s);
    else
      attn_launch<128, false>(a, s);
  }
  return launch_status();
}
