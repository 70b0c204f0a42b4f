/*
 * cuda_inf_ffn.h -- the feed-forward half of a layer of the cuda_inf engine on
 * MI355X (gfx950): residual addition with RMSNorm, the router, the experts'
 * INT4 products and the branch that runs them (g023/cuda_inf,
 * src/engine.cu:869-905).
 *
 * The conventions are cuda_inf_attn.h's: device pointers owned by the caller,
 * fp16 tensors as uint16_t*, contiguous; every call is enqueued on `stream`
 * and returns a cia_status; nothing allocates device memory, synchronises or
 * copies to the host, so all of it can be captured into a graph.  Structs are
 * read on the host during the call.  Work runs on the current device.
 *
 * Workspaces (ws) hold nothing from one call to the next; calls that share one
 * must be ordered (same stream, or events), captured graphs included.
 */
#ifndef CUDA_INF_FFN_H
#define CUDA_INF_FFN_H

#include <stdint.h>

#include "cuda_inf_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define CIA_MOE_MAX_EXPERTS 256
#define CIA_MOE_MAX_TOP_K 16
#define CIA_MOE_MAX_WIDTH 32768     /* H and F of the experts */
#define CIA_MOE_MAX_PAIRS (1 << 20) /* S * k of a call */
#define CIA_FFN_MAX_TOKENS (1 << 22) /* S of the norm and the router */
#define CIA_FFN_MAX_WIDTH (1 << 24)  /* their H */

/* add_f32_inplace and rmsnorm (engine.cu:527-559, 131-144; launched at 867 and
 * 870): hsum = h + add, out = fp16(hsum * rsqrt(mean(hsum^2) + eps) * w) for
 * each of the S rows of H.
 * h, add, hsum: fp32 [S][H]; add may be NULL (nothing is added); hsum may be
 * NULL (the sum is not kept), h or add (in place).  w: fp16 [H].  out: fp16
 * [S][H].  H a multiple of 8 and at most CIA_FFN_MAX_WIDTH, S at most
 * CIA_FFN_MAX_TOKENS; all pointers 16-byte aligned.  Sums are fp32, a lane's
 * part of a row above 8192 in 64 bits. */
int cia_add_rmsnorm(const float* h, const float* add, const uint16_t* w,
                    float eps, float* hsum, uint16_t* out, int S, int H,
                    void* stream);

#define CIA_SCORE_SIGMOID 0
#define CIA_SCORE_SOFTMAX 1

/* How a router chooses. */
typedef struct cia_moe_gating {
  int n_experts;   /* 1 .. CIA_MOE_MAX_EXPERTS */
  int top_k;       /* experts per token: 1 .. min(CIA_MOE_MAX_TOP_K, n_experts) */
  int score;       /* CIA_SCORE_SIGMOID, or CIA_SCORE_SOFTMAX over all experts */
  int n_group;     /* groups of n_experts / n_group neighbours; 1: no groups */
  int topk_group;  /* groups a token may choose from; they hold top_k experts */
  int renorm;      /* nonzero: weights are divided by their sum + eps */
  float eps;       /* >= 0 */
  float scale;     /* every weight is multiplied by it; finite */
} cia_moe_gating;

/* The router (of engine.cu:869-905, which copies the logits to the host at 880
 * and chooses there):
 *   l = gate x;  s = score(l);  c = s + bias;
 *   of the groups, the topk_group whose two best c have the largest sum;
 *   ids = the top_k largest c among the experts of those groups, largest
 *   first, the lowest index first among equals;  weights = s[ids], divided by
 *   (their sum + eps) if renorm, times scale.
 * x: fp16 [S][H]; gate: fp16 [n_experts][H]; bias: fp32 [n_experts], may be
 * NULL, used for the choice alone.  ids: int32 [S][top_k]; weights: fp32
 * [S][top_k]; logits: fp32 [S][n_experts], may be NULL.  H a multiple of 8
 * and at most CIA_FFN_MAX_WIDTH; x and gate 16-byte aligned.
 * The choice is the one of logits summed in 64 bits, so a token's experts do
 * not depend on the other tokens of the call.  Logits are at most 2^-19 of
 * sum |gate x| and half an fp32 step off, in calls of up to 1024 tokens the half
 * step alone; weights as far as that moves them.
 * A c that is not a number ranks with -inf; a softmax over logits that are all
 * -inf gives scores of 0, one with a NaN or +inf among them NaN; a sum + eps
 * of 0 gives weights of 0.  S at most CIA_FFN_MAX_TOKENS. */
int cia_moe_route(const uint16_t* x, const uint16_t* gate, const float* bias,
                  const cia_moe_gating* g, int32_t* ids, float* weights,
                  float* logits, int S, int H, void* stream);

/* The same from logits fp32 [S][n_experts] that the caller has, in 64 bits up
 * to one rounding of the weights. */
int cia_moe_select(const float* logits, const float* bias,
                   const cia_moe_gating* g, int32_t* ids, float* weights, int S,
                   void* stream);

/* INT4 group-128 weights of E experts, each [rows][cols] in the format of
 * cia_gemv_int4: expert e's packed bytes [rows][cols/2] at
 * packed + e * packed_stride and its fp16 scales [rows][cols/128] at
 * scales + e * scales_stride (elements).  packed 16-byte aligned;
 * scales 2-byte aligned.  Strides are read only where E > 1: packed_stride is
 * then a multiple of 16, and they hold an expert, rows * cols / 2 bytes and
 * rows * cols / 128 elements at least. */
typedef struct cia_q4_experts {
  const uint8_t* packed;
  const uint16_t* scales;
  int64_t packed_stride;
  int64_t scales_stride;
} cia_q4_experts;

/* The experts' gate and up products with SwiGLU (of engine.cu:869-905, for every
 * token and chosen expert): act[s][j] = fp16(g / (1 + exp(-g)) * u) with
 * g = W1[e] x[s], u = W3[e] x[s], e = ids[s][j].
 * x: fp16 [S][H]; ids: int32 [S][k]; w1, w3: E experts of [F][H];
 * act: fp16 [S][k][F].  A pair whose id is outside [0, E) takes no part (a
 * place of a padded batch, another device's expert): its act row is left as it
 * was.  An id may repeat within a token.  ids NULL: every row is expert 0's
 * (E = k = 1, a dense layer).  H and F multiples of 128, at most
 * CIA_MOE_MAX_WIDTH; k at most CIA_MOE_MAX_TOP_K, S * k at most
 * CIA_MOE_MAX_PAIRS.  x, act and ws 16-byte aligned;
 * ws_bytes at least cia_moe_workspace_bytes(S, k, E, H, F). */
int cia_moe_up_int4(const uint16_t* x, const int32_t* ids,
                    const cia_q4_experts* w1, const cia_q4_experts* w3,
                    uint16_t* act, int S, int k, int E, int H, int F, void* ws,
                    int64_t ws_bytes, void* stream);

/* The experts' down products, weighted and added to the residual
 * (of engine.cu:869-905): out[s] = res[s] + sum over j, in order, of
 * weights[s][j] * (W2[e] act[s][j]).
 * act: fp16 [S][k][F]; weights: fp32 [S][k], NULL: 1; w2: E experts of [H][F];
 * res, out: fp32 [S][H], out may be res.  Pairs outside [0, E) add nothing,
 * whatever their act rows and weights hold.  The rest as cia_moe_up_int4;
 * act, res, out and ws 16-byte aligned. */
int cia_moe_down_int4(const uint16_t* act, const int32_t* ids,
                      const float* weights, const cia_q4_experts* w2,
                      const float* res, float* out, int S, int k, int E, int H,
                      int F, void* ws, int64_t ws_bytes, void* stream);

/* Workspace bytes of cia_moe_up_int4 and cia_moe_down_int4 for up to S tokens;
 * 0 where S is negative, or k, E, H or F is one that they refuse.  (More than
 * CIA_MOE_MAX_PAIRS pairs have a size as well, though no call takes them.) */
int64_t cia_moe_workspace_bytes(int S, int k, int E, int H, int F);

/* The feed-forward branch of one layer. */
typedef struct cia_moe {
  const uint16_t* norm_w;  /* ffn_norm's weight, fp16 [H] */
  float norm_eps;
  int H, F;
  const uint16_t* gate;    /* the router, fp16 [n_experts][H]; NULL: a dense
                              layer (one expert, no router; gating is not read) */
  const float* bias;       /* fp32 [n_experts], may be NULL */
  cia_moe_gating gating;
  cia_q4_experts w1, w3;   /* experts of [F][H] */
  cia_q4_experts w2;       /* experts of [H][F] */
  void* ws;                /* device scratch, 16-byte aligned */
  int64_t ws_bytes;        /* at least cia_moe_block_workspace_bytes(this, cap) */
  int cap;                 /* tokens a call may bring */
} cia_moe;

/* Scratch bytes of a branch for calls of up to cap tokens; 0 where cap is
 * negative, cap tokens make more than CIA_MOE_MAX_PAIRS pairs, or top_k,
 * n_experts, H or F is one that cia_moe_workspace_bytes gives 0 for. */
int64_t cia_moe_block_workspace_bytes(const cia_moe* M, int cap);

/* The feed-forward branch (engine.cu:869-905) for S <= M->cap tokens, from the
 * residual to the residual: x = cia_add_rmsnorm(h), cia_moe_route,
 * cia_moe_up_int4, cia_moe_down_int4 into h (fp32 [S][H], in place). */
int cia_moe_block_forward(const cia_moe* M, float* h, int S, void* stream);

#ifdef __cplusplus
}
#endif
#endif
