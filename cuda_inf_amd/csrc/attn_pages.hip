// attn_pages.hip -- attention of one query token per row over a paged key-value
// cache on gfx950: per row t and query head h
//   s_j = scale q . k_j,   out = sum_j exp(s_j - max s) v_j / sum_j exp(s_j - max s)
// over the tokens of the row's sequence up to its position.
//
// Bound by memory: every K and V row once, 2 D + 4 bytes a token and kv head in e4m3.
#include "pages.h"

namespace cia {

struct AttnPagesArgs {
  Pages P;
  const uint16_t* q;
  int64_t q_stride;
  const int32_t* seq;  // or null
  const int32_t* pos;
  int T, n_q, group;  // group: query heads of a kv head
  float scale;
  int window;
  uint16_t* out;
};

constexpr int kTok = 256;  // tokens a step: one a thread

// grid = (query heads, rows), block = 256.  Scores with a token a thread, then the
// step's V rows with a dimension a thread.
template <int kD, bool kF8>
__global__ __launch_bounds__(256) void k_attn_pages(AttnPagesArgs a) {
  constexpr int kParts = 256 / kD;
  __shared__ float sq[kD], sp[kTok], red[8], so[kParts][kD];
  __shared__ int64_t srow[kTok];
  const int h = blockIdx.x, t = blockIdx.y, g = h / a.group, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int s = a.seq ? a.seq[t] : t;
  const int pos = a.pos[t];
  const int len = s >= 0 && s < a.P.n_seq && pos >= 0 ? min(pos, a.P.max_tokens - 1) + 1 : 0;
  const int first = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
  if (tid < kD) sq[tid] = h2f(a.q[t * a.q_stride + h * kD + tid]);
  float m = -__builtin_inff(), l = 0.0f, o = 0.0f;
  const int d = tid % kD, part = tid / kD;
  for (int base = first & ~(kTok - 1); base < len; base += kTok) {
    const int j = base + tid;
    const int page = j >= first && j < len ? page_of(a.P, s, j) : -1;
    const int64_t row = page >= 0 ? page_row(a.P, page, g, j) : -1;
    __syncthreads();
    srow[tid] = row;
    float x = -__builtin_inff();
    if (row >= 0) {
      float dot = 0.0f;
      if constexpr (kF8) {
        const uint32_t* w = (const uint32_t*)((const uint8_t*)a.P.k + row * kD);
#pragma unroll 4
        for (int i = 0; i < kD / 4; i++) {
          const f32x2 u = e4m3x2_to_f32<false>(w[i]), v = e4m3x2_to_f32<true>(w[i]);
          dot = __builtin_fmaf(sq[4 * i], u[0], dot);
          dot = __builtin_fmaf(sq[4 * i + 1], u[1], dot);
          dot = __builtin_fmaf(sq[4 * i + 2], v[0], dot);
          dot = __builtin_fmaf(sq[4 * i + 3], v[1], dot);
        }
        dot *= h2f(a.P.ks[row]);
      } else {
        const uint16_t* w = (const uint16_t*)a.P.k + row * kD;
#pragma unroll 8
        for (int i = 0; i < kD; i++) dot = __builtin_fmaf(sq[i], h2f(w[i]), dot);
      }
      x = dot * a.scale;
    }
    float top = wave_max(x);
    if (lane == 0) red[wave] = top;
    __syncthreads();
    top = __builtin_fmaxf(__builtin_fmaxf(red[0], red[1]), __builtin_fmaxf(red[2], red[3]));
    const float now = __builtin_fmaxf(m, top);
    const float keep = now > -__builtin_inff() ? __expf(m - now) : 1.0f;
    const float p = row >= 0 ? __expf(x - now) : 0.0f;
    m = now;
    sp[tid] = p;
    const float sum = wave_sum(p);
    if (lane == 0) red[4 + wave] = sum;
    __syncthreads();
    l = l * keep + ((red[4] + red[5]) + (red[6] + red[7]));
    o *= keep;
    for (int i = part; i < kTok; i += kParts) {
      const int64_t r = srow[i];
      if (r < 0) continue;
      float v;
      if constexpr (kF8)
        v = e4m3_to_f32<0>(((const uint8_t*)a.P.v)[r * kD + d]) * h2f(a.P.vs[r]);
      else
        v = h2f(((const uint16_t*)a.P.v)[r * kD + d]);
      o = __builtin_fmaf(sp[i], v, o);
    }
  }
  so[part][d] = o;
  __syncthreads();
  if (tid < kD) {
    float sum = 0.0f;
    for (int i = 0; i < kParts; i++) sum += so[i][tid];
    a.out[((int64_t)t * a.n_q + h) * kD + tid] = f2h(l == 0.0f ? 0.0f : sum / l);
  }
}

}  // namespace cia

using namespace cia;

extern "C" int64_t cia_attn_pages_workspace_bytes(int n_q, int n_kv, int head_dim) {
  if (n_kv < 1 || n_kv > CIA_PAGES_MAX_KV || (head_dim != 64 && head_dim != 128) || n_q < n_kv || n_q % n_kv ||
      n_q / n_kv > CIA_PAGES_MAX_GROUP)
    return 0;
  return 16;
}

extern "C" int cia_attn_pages(const cia_kv_pages* p, const uint16_t* q, int64_t q_stride, const int32_t* seq,
                              const int32_t* pos, int T, int n_q, float scale, int window, uint16_t* out, void* ws,
                              int64_t ws_bytes, void* stream) {
  int st = pages_check(p);
  if (st) return st;
  const int64_t need = cia_attn_pages_workspace_bytes(n_q, p->n_kv, p->head_dim);
  CIA_REQUIRE(need > 0 && T >= 0 && T <= CIA_PAGES_MAX_ROWS && (seq || T <= p->n_seq), CIA_ERR_ARG);
  CIA_REQUIRE(q_stride >= (int64_t)n_q * p->head_dim && q_stride % 8 == 0 && window >= 0, CIA_ERR_ARG);
  CIA_REQUIRE(scale - scale == 0.0f, CIA_ERR_ARG);  // finite
  if (T == 0) return CIA_OK;
  if ((st = pages_check_ptr(p))) return st;
  CIA_REQUIRE(q && pos && out && ws, CIA_ERR_NULL);
  CIA_REQUIRE(aligned(q, 16) && aligned(seq, 4) && aligned(pos, 4) && aligned(out, 16) && aligned(ws, 16),
              CIA_ERR_ALIGN);
  CIA_REQUIRE(ws_bytes >= need, CIA_ERR_ARG);
  const AttnPagesArgs a{pages_of(p), q, q_stride, seq, pos, T, n_q, n_q / p->n_kv, scale, window, out};
  const dim3 grid((unsigned)n_q, (unsigned)T);
  hipStream_t s = (hipStream_t)stream;
  if (p->head_dim == 64) {
    if (p->type == CIA_KV_E4M3)
      hipLaunchKernelGGL((k_attn_pages<64, true>), grid, dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((k_attn_pages<64, false>), grid, dim3(256), 0, s, a);
  } else {
    if (p->type == CIA_KV_E4M3)
      hipLaunchKernelGGL((k_attn_pages<128, true>), grid, dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((k_attn_pages<128, false>), grid, dim3(256), 0, s, a);
  }
  return launch_status();
}
