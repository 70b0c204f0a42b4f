/*
 * cuda_inf_batch.h -- a decode step of many sequences on MI355X (gfx950): a
 * paged key-value cache that they share, attention over it, and the choice of
 * each row's next token.  The reference engine (g023/cuda_inf) runs one
 * sequence, whose cache is one buffer a layer, and chooses by argmax
 * (src/engine.cu:562-572); these have no kernel of its own to replace.
 *
 * The conventions are cuda_inf_attn.h's: device pointers owned by the caller,
 * fp16 tensors as uint16_t*; every call is enqueued on `stream` and returns a
 * cia_status; nothing allocates device memory, synchronises or copies to the
 * host, so all of it can be captured into a graph.  Structs are read on the
 * host during the call.  Work runs on the current device.
 */
#ifndef CUDA_INF_BATCH_H
#define CUDA_INF_BATCH_H

#include <stdint.h>

#include "cuda_inf_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define CIA_KV_E4M3 0
#define CIA_KV_F16 1

#define CIA_PAGE_MIN 16                /* tokens of a page: a power of two */
#define CIA_PAGE_MAX 1024
#define CIA_PAGES_MAX_KV 128           /* kv heads */
#define CIA_PAGES_MAX_GROUP 64         /* query heads of a kv head */
#define CIA_PAGES_MAX_TOKENS (1 << 25) /* max_pages * page: a sequence's tokens */
#define CIA_PAGES_MAX_CALL (1 << 22)   /* tokens of a write or read */
#define CIA_PAGES_MAX_ROWS 4096        /* rows of an attention call */
#define CIA_SAMPLE_MAX_ROWS (1 << 16)
#define CIA_SAMPLE_MAX_VOCAB (1 << 22)
#define CIA_SAMPLE_MAX_LOGITS ((int64_t)1 << 34) /* B * V */

/* One layer's cache for many sequences.  Token `pos` of sequence `s` is row
 * pos % page of page table[s * table_stride + pos / page].  A token has no
 * place where s is outside [0, n_seq), pos outside [0, max_pages * page) or
 * the page's id outside [0, n_pages): it takes no part in a call, so that
 * empty places of a batch are marked with pos -1 and pages that are not there
 * with -1.
 *   CIA_KV_E4M3: a row of x is stored as kv_quant_write (engine.cu:317-333)
 *   stores it, per kv head: s = amax / 448 + 1e-12 in fp32, the bytes
 *   e4m3(x / s) and fp16(s); it stands for byte * fp16(s).
 *   CIA_KV_F16: the fp16 values.
 * k, v and their scales are written by cia_kv_pages_write alone; the table is
 * the caller's, and may change between calls. */
typedef struct cia_kv_pages {
  void* k;                /* [n_pages][n_kv][page][head_dim], 16-byte aligned */
  void* v;
  uint16_t* ks;           /* e4m3: fp16 [n_pages][n_kv][page]; fp16: not read */
  uint16_t* vs;
  int type;               /* CIA_KV_E4M3 or CIA_KV_F16 */
  int n_pages;            /* >= 1 */
  int page;               /* tokens: a power of two, CIA_PAGE_MIN..CIA_PAGE_MAX */
  int n_kv;               /* 1..CIA_PAGES_MAX_KV */
  int head_dim;           /* 64 or 128 */
  int n_seq;              /* rows of the table, >= 1 */
  int max_pages;          /* its columns, >= 1 */
  const int32_t* table;   /* [n_seq][table_stride] */
  int64_t table_stride;   /* >= max_pages */
} cia_kv_pages;

/* T tokens' K and V into their places, quantised on the way.
 * k, v: fp16, token t's [n_kv][head_dim] at k + t * k_stride, v + t * v_stride
 * (elements; multiples of 8, n_kv * head_dim at least; 16-byte aligned).  seq:
 * int32 [T], the tokens' sequences, NULL: token t is sequence t's (T <= n_seq).
 * pos: int32 [T].  Two tokens of a call must not have the same place: what it
 * then holds is not defined.  T at most CIA_PAGES_MAX_CALL. */
int cia_kv_pages_write(const cia_kv_pages* P, const uint16_t* k,
                       int64_t k_stride, const uint16_t* v, int64_t v_stride,
                       const int32_t* seq, const int32_t* pos, int T,
                       void* stream);

/* The reverse: k and v rows of T tokens from their places, fp16(byte *
 * fp16(s)) of an e4m3 cache.  Rows of tokens without a place are left as they
 * were. */
int cia_kv_pages_read(const cia_kv_pages* P, uint16_t* k, int64_t k_stride,
                      uint16_t* v, int64_t v_stride, const int32_t* seq,
                      const int32_t* pos, int T, void* stream);

/* Attention of T rows, each one query token, over the pages of its sequence:
 * for query head h of kv head g = h / (n_q / n_kv),
 *   out[t][h] = sum_j softmax_j(scale * q[t][h] . k_j) v_j
 * over the tokens j <= pos[t] of sequence seq[t] (NULL: t) that have a place,
 * the last `window` positions of them if window > 0.  The token at pos[t]
 * itself is read from the cache: it is written before.  Rows with nothing to
 * attend to (pos < 0, no pages) are 0.
 * q: fp16, row t's [n_q][head_dim] at q + t * q_stride (a multiple of 8, n_q *
 * head_dim at least); out: fp16 [T][n_q][head_dim]; both 16-byte aligned.  n_q
 * a multiple of n_kv, at most CIA_PAGES_MAX_GROUP times it; T at most
 * CIA_PAGES_MAX_ROWS; |scale| <= 2^64.  Softmax and sums are fp32.  A NaN or an
 * infinity in what a row attends to makes its kv head's outputs NaN or
 * infinite (one in V: those of its dimension), but for a score of -inf, which
 * has no weight; elsewhere in the cache they do nothing.
 * ws: device scratch of at least cia_attn_pages_workspace_bytes, 16-byte
 * aligned, zeroed before its first use; every call leaves its counters at
 * zero.  Calls that share one must be ordered, captured graphs included. */
int cia_attn_pages(const cia_kv_pages* P, const uint16_t* q, int64_t q_stride,
                   const int32_t* seq, const int32_t* pos, int T, int n_q,
                   float scale, int window, uint16_t* out, void* ws,
                   int64_t ws_bytes, void* stream);

/* Workspace bytes of cia_attn_pages for any T; 0 where it refuses the heads. */
int64_t cia_attn_pages_workspace_bytes(int n_q, int n_kv, int head_dim);

#define CIA_LOGITS_F32 0
#define CIA_LOGITS_F16 1

/* A token for each of B rows of V logits, from the given random numbers:
 *   w_i = exp((l_i - max l) / temperature), in order of descending l, the
 *   lowest index first among equals;
 *   K = the first top_k of the order;  P = its shortest prefix whose sum is at
 *   least top_p * sum(K), within K;  M = those of P with w >= min_p;
 *   ids = the first of the order whose running sum exceeds u * sum(M);
 *   p = w[ids] / sum(M).
 * logits: row b at logits + b * stride (elements, >= V), of `type`.
 * temperature, top_p, min_p: fp32 [B]; top_k: int32 [B]; each may be NULL (1,
 * and no filter).  A temperature of 0 (or less, or NaN) takes the first of the
 * order, with p = 1.  No filter: top_k <= 0, top_p >= 1 or NaN, min_p <= 0 or
 * NaN; a top_p <= 0 and a min_p > 1 leave one token, or its equals with
 * min_p.  u: fp32 [B] in [0, 1), other values are taken as the nearest of
 * them, NaN as 0.  ids: int32 [B]; p: fp32 [B], may be NULL.
 * A NaN logit counts as -inf; -inf is never chosen; where logits are +inf they
 * alone are, all alike; a row of none gives id -1 and p 0.  Weights below
 * 2^-41 of the largest may count as 0: all V of them are up to V 2^-41 of a sum.
 * Sums are 64 bits wide: weights are good to 2^-34 + |l| / temperature 2^-52 of
 * themselves in them.  A u within about the sum of these (2^-34 to 2^-33 for an
 * ordinary row of up to 128 tokens below 2^-41, 2^-24 for 131 072 of them) of a
 * border can fall on its other side, and p is as far off.
 * logits aligned to their type, ws to 16 bytes; ws_bytes at least
 * cia_sample_workspace_bytes(B, V); ws holds nothing between calls; calls that
 * share one must be ordered, captured graphs included.  B at most
 * CIA_SAMPLE_MAX_ROWS, V from 1 to CIA_SAMPLE_MAX_VOCAB, B * V at most
 * CIA_SAMPLE_MAX_LOGITS. */
int cia_sample(const void* logits, int type, int64_t stride,
               const float* temperature, const int32_t* top_k,
               const float* top_p, const float* min_p, const float* u,
               int32_t* ids, float* p, int B, int V, void* ws, int64_t ws_bytes,
               void* stream);

/* Workspace bytes of cia_sample for up to B rows of V; 0 where it refuses. */
int64_t cia_sample_workspace_bytes(int B, int V);

#ifdef __cplusplus
}
#endif
#endif
