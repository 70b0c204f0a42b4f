// pages.h -- what the kernels of the paged cache share: the cache as they take
// it, a token's place, and the host's checks.
#pragma once

#include "common.h"
#include "cuda_inf_batch.h"

namespace cia {

struct Pages {
  void* k;
  void* v;
  uint16_t* ks;
  uint16_t* vs;
  const int32_t* table;
  int64_t table_stride;
  int n_pages, shift, n_kv, n_seq;  // page = 1 << shift
  int max_tokens;                   // of a sequence: max_pages << shift
};

// the page of token pos (in [0, max_tokens)) of sequence s, -1: none
__device__ __forceinline__ int page_of(const Pages& P, int s, int pos) {
  const int id = P.table[(int64_t)s * P.table_stride + (pos >> P.shift)];
  return id >= 0 && id < P.n_pages ? id : -1;
}

// row of (page, kv head, token) among all rows of the cache, as the scales count them
__device__ __forceinline__ int64_t page_row(const Pages& P, int page, int head, int pos) {
  return ((((int64_t)page * P.n_kv + head) << P.shift)) + (pos & ((1 << P.shift) - 1));
}

// ---------------------------------------------------------------- host side
inline int pages_check(const cia_kv_pages* p) {
  CIA_REQUIRE(p, CIA_ERR_NULL);
  CIA_REQUIRE(p->type == CIA_KV_E4M3 || p->type == CIA_KV_F16, CIA_ERR_ARG);
  CIA_REQUIRE(p->n_pages >= 1 && p->n_seq >= 1 && p->max_pages >= 1, CIA_ERR_ARG);
  CIA_REQUIRE(p->page >= CIA_PAGE_MIN && p->page <= CIA_PAGE_MAX && !(p->page & (p->page - 1)), CIA_ERR_ARG);
  CIA_REQUIRE(p->n_kv >= 1 && p->n_kv <= CIA_PAGES_MAX_KV, CIA_ERR_ARG);
  CIA_REQUIRE(p->head_dim == 64 || p->head_dim == 128, CIA_ERR_ARG);
  CIA_REQUIRE((int64_t)p->max_pages * p->page <= CIA_PAGES_MAX_TOKENS && p->table_stride >= p->max_pages, CIA_ERR_ARG);
  return CIA_OK;
}
// the pointers, where a call has work
inline int pages_check_ptr(const cia_kv_pages* p) {
  const bool q = p->type == CIA_KV_E4M3;
  CIA_REQUIRE(p->k && p->v && p->table && (!q || (p->ks && p->vs)), CIA_ERR_NULL);
  CIA_REQUIRE(aligned(p->k, 16) && aligned(p->v, 16) && aligned(p->table, 4), CIA_ERR_ALIGN);
  CIA_REQUIRE(!q || (aligned(p->ks, 2) && aligned(p->vs, 2)), CIA_ERR_ALIGN);
  return CIA_OK;
}
inline Pages pages_of(const cia_kv_pages* p) {
  return Pages{p->k,       p->v,
               p->ks,      p->vs,
               p->table,   p->table_stride,
               p->n_pages, __builtin_ctz((unsigned)p->page),
               p->n_kv,    p->n_seq,
               p->max_pages * p->page};
}

}  // namespace cia
