// kv_pages.hip -- tokens into the paged cache, quantised on the way, and back, on
// gfx950.  The rows are kv_quant_write's (engine.cu:317-333): per token and kv head
// s = amax / 448 + 1e-12, bytes e4m3(x / s), fp16(s).
//
// Bound by memory: 4 D bytes of K and V in fp16, 2 D + 4 in the cache, a token and head.
// 8192 tokens of 8 heads of 64 read back take 6.0-6.4 us (4.0-4.2 TB/s; a large copy
// reaches 5.1), 5001 written 5.8-7.0 (2.2-2.7 TB/s), one token 3.2-3.6, an empty kernel
// 2.0-2.2: what is left beside the bytes is a chain of three loads, position, page id and
// row, of which the write has its rows' out before the other two.
#include "pages.h"

namespace cia {

struct MoveArgs {
  Pages P;
  uint16_t* k;  // fp16 rows: read by the write, written by the read
  uint16_t* v;
  int64_t k_stride, v_stride;
  const int32_t* seq;  // or null: token t is sequence t's
  const int32_t* pos;
  int T;
};

// max over the kD / 8 lanes of a row (8 or 16 neighbours): within quads, then quads
// of 8, then the halves of 16
template <int kCtrl>
__device__ __forceinline__ float dpp_max(float v) {
  return __builtin_fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), kCtrl, 0xF, 0xF, false)));
}
template <int kD>
__device__ __forceinline__ float row_max(float v) {
  v = dpp_max<0xB1>(v);   // quad_perm 1,0,3,2
  v = dpp_max<0x4E>(v);   // quad_perm 2,3,0,1
  v = dpp_max<0x141>(v);  // row_half_mirror
  if (kD == 128) v = dpp_max<0x140>(v);  // row_mirror
  return v;
}

// 8 values of a row of K or V into the cache; every lane of the row is here
template <int kD>
__device__ __forceinline__ void store_e4m3(const u32x4& w, uint8_t* rows, uint16_t* scales, int64_t row, int c, bool live) {
  const f16x8 h = __builtin_bit_cast(f16x8, w);
  float m = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; e++) m = __builtin_fmaxf(m, __builtin_fabsf((float)h[e]));
  const float s = quant_scale(row_max<kD>(m)), r = 1.0f / s, d = quant_div_s(s);
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; e++) y[e] = quant_div((float)h[e], d, r);
  if (!live) return;
  *(u32x2*)(rows + row * kD + 8 * c) = u32x2{e4m3x4(y[0], y[1], y[2], y[3]), e4m3x4(y[4], y[5], y[6], y[7])};
  if (c == 0) scales[row] = f2h(s);
}

__device__ __forceinline__ u32x4 load_e4m3(const uint8_t* rows, const uint16_t* scales, int64_t at, int64_t row) {
  const u32x2 w = *(const u32x2*)(rows + at);
  const float s = h2f(scales[row]);
  f16x8 h;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const f32x2 a = e4m3x2_to_f32<false>(w[i]), b = e4m3x2_to_f32<true>(w[i]);
    h[4 * i] = (_Float16)(a[0] * s);
    h[4 * i + 1] = (_Float16)(a[1] * s);
    h[4 * i + 2] = (_Float16)(b[0] * s);
    h[4 * i + 3] = (_Float16)(b[1] * s);
  }
  return __builtin_bit_cast(u32x4, h);
}

// grid = (tokens / (2048 / kD), kv heads), block = 256: kD / 8 lanes a token, 8 values
// each of K and of V, so that a token's amax stays in a DPP row and every load and store
// of fp16 is 16 bytes.  Neighbouring tokens of one head are neighbouring rows of a
// page, so a workgroup's stores fill whole lines though a row is 64 bytes.
template <int kD, bool kF8, bool kWrite>
__global__ __launch_bounds__(256) void k_pages_move(MoveArgs a) {
  constexpr int kLanes = kD / 8;
  const int t = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes, c = threadIdx.x % kLanes, head = blockIdx.y;
  const bool here = t < a.T;
  uint16_t* const k = a.k + (here ? t : 0) * a.k_stride + head * kD + 8 * c;
  uint16_t* const v = a.v + (here ? t : 0) * a.v_stride + head * kD + 8 * c;
  u32x4 kw{0, 0, 0, 0}, vw{0, 0, 0, 0};
  if constexpr (kWrite) kw = *(const u32x4*)k, vw = *(const u32x4*)v;  // (before the place is known)
  int page = -1, pos = -1;
  if (here) {
    pos = a.pos[t];
    const int s = a.seq ? a.seq[t] : t;
    if (s >= 0 && s < a.P.n_seq && pos >= 0 && pos < a.P.max_tokens) page = page_of(a.P, s, pos);
  }
  const bool live = page >= 0;
  const int64_t row = live ? page_row(a.P, page, head, pos) : 0;
  if constexpr (kWrite) {
    if constexpr (kF8) {
      store_e4m3<kD>(kw, (uint8_t*)a.P.k, a.P.ks, row, c, live);
      store_e4m3<kD>(vw, (uint8_t*)a.P.v, a.P.vs, row, c, live);
    } else if (live) {
      *(u32x4*)((uint16_t*)a.P.k + row * kD + 8 * c) = kw;
      *(u32x4*)((uint16_t*)a.P.v + row * kD + 8 * c) = vw;
    }
  } else if (live) {
    const int64_t at = row * kD + 8 * c;
    if constexpr (kF8) {
      kw = load_e4m3((const uint8_t*)a.P.k, a.P.ks, at, row);
      vw = load_e4m3((const uint8_t*)a.P.v, a.P.vs, at, row);
    } else {
      kw = *(const u32x4*)((const uint16_t*)a.P.k + at);
      vw = *(const u32x4*)((const uint16_t*)a.P.v + at);
    }
    *(u32x4*)k = kw;
    *(u32x4*)v = vw;
  }
}

template <bool kWrite>
static int pages_move(const cia_kv_pages* p, uint16_t* k, int64_t k_stride, uint16_t* v, int64_t v_stride,
                      const int32_t* seq, const int32_t* pos, int T, void* stream) {
  int st = pages_check(p);
  if (st) return st;
  const int64_t width = (int64_t)p->n_kv * p->head_dim;
  CIA_REQUIRE(T >= 0 && T <= CIA_PAGES_MAX_CALL && (seq || T <= p->n_seq), CIA_ERR_ARG);
  CIA_REQUIRE(k_stride >= width && v_stride >= width && k_stride % 8 == 0 && v_stride % 8 == 0, CIA_ERR_ARG);
  if (T == 0) return CIA_OK;
  if ((st = pages_check_ptr(p))) return st;
  CIA_REQUIRE(k && v && pos, CIA_ERR_NULL);
  CIA_REQUIRE(aligned(k, 16) && aligned(v, 16) && aligned(seq, 4) && aligned(pos, 4), CIA_ERR_ALIGN);
  const MoveArgs a{pages_of(p), k, v, k_stride, v_stride, seq, pos, T};
  const int per = 2048 / p->head_dim;
  const dim3 grid((unsigned)((T + per - 1) / per), (unsigned)p->n_kv);
  hipStream_t s = (hipStream_t)stream;
  if (p->head_dim == 64) {
    if (p->type == CIA_KV_E4M3)
      hipLaunchKernelGGL((k_pages_move<64, true, kWrite>), grid, dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((k_pages_move<64, false, kWrite>), grid, dim3(256), 0, s, a);
  } else {
    if (p->type == CIA_KV_E4M3)
      hipLaunchKernelGGL((k_pages_move<128, true, kWrite>), grid, dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((k_pages_move<128, false, kWrite>), grid, dim3(256), 0, s, a);
  }
  return launch_status();
}

}  // namespace cia

using namespace cia;

extern "C" int cia_kv_pages_write(const cia_kv_pages* P, const uint16_t* k, int64_t k_stride, const uint16_t* v,
                                  int64_t v_stride, const int32_t* seq, const int32_t* pos, int T, void* stream) {
  return pages_move<true>(P, const_cast<uint16_t*>(k), k_stride, const_cast<uint16_t*>(v), v_stride, seq, pos, T,
                          stream);
}

extern "C" int cia_kv_pages_read(const cia_kv_pages* P, uint16_t* k, int64_t k_stride, uint16_t* v, int64_t v_stride,
                                 const int32_t* seq, const int32_t* pos, int T, void* stream) {
  return pages_move<false>(P, k, k_stride, v, v_stride, seq, pos, T, stream);
}
