/* Launchers of the float-side kernels (ops_kernels.hip). Internal to the library. */
#ifndef SDY_OPS_H
#define SDY_OPS_H
#include <stddef.h>
#include <stdint.h>

#include "sdy_shim.h"

#ifdef __cplusplus
extern "C" {
#endif
int sdy_rmsnorm(const float *x, const float *w, float *out, int n, float eps, int n_rows, long x_stride,
                long out_stride, sdy_stream s);
/* KV-cache element types (kv_type arguments): f32, or f16 with each value rounded to nearest even
 * when written (the reference's f32 -> f16 rules). A layer's cache is [n_kv_head][max_seq][hd]
 * elements; head_stride counts elements. */
enum { SDY_KV_F32 = 0, SDY_KV_F16 = 1 };
size_t sdy_kv_elt_bytes(int kv_type); /* 4, 2, or 0 for an unknown type */
int sdy_qk_rope_kv(float *q, float *k, const float *v, const float *qn, const float *kn, float eps,
                   const float *rope_cos, const float *rope_sin, int pos0, int n_tok, int n_head, int n_kv_head, int hd,
                   int interleaved, void *k_cache, void *v_cache, int kv_type, long head_stride, sdy_stream s);
/* the same with token rows t * q_stride, t * k_stride, t * v_stride floats apart (q|k|v of one GEMM) */
int sdy_qk_rope_kv_strided(float *q, float *k, const float *v, long q_stride, long k_stride, long v_stride,
                           const float *qn, const float *kn, float eps, const float *rope_cos, const float *rope_sin,
                           int pos0, int n_tok, int n_head, int n_kv_head, int hd, int interleaved, void *k_cache,
                           void *v_cache, int kv_type, long head_stride, sdy_stream s);
/* Causal attention of n_tok tokens at positions n_kv0 - 1 + t (q rotated, K/V in the cache) in the
 * reference's arithmetic; scores: sdy_attn_scores_floats(n_tok, n_head, n_kv0 + n_tok - 1) floats of
 * device scratch. head_dim 32, 64, 128 or 256. */
size_t sdy_attn_scores_floats(int n_tok, int n_head, int max_kv);
int sdy_attention(const float *q, const void *k_cache, const void *v_cache, int kv_type, int n_tok, int n_head,
                  int n_kv_head, int hd, int n_kv0, long head_stride, long q_stride, float *scores, float *out,
                  long out_stride, sdy_stream s);
/* The same attention in flash form on the f32 matrix cores (attn_flash.hip): within tolerance of the
 * reference, not its bits; no scratch. head_dim 64 or 128; q rows and both strides 16-byte aligned. */
int sdy_attention_flash_ok(int n_head, int n_kv_head, int hd);
int sdy_attention_flash(const float *q, const void *k_cache, const void *v_cache, int kv_type, int n_tok,
                        int n_head, int n_kv_head, int hd, int n_kv0, long head_stride, long q_stride, float *out,
                        long out_stride, sdy_stream s);
int sdy_silu_mul(float *gate, const float *up, long n, sdy_stream s);
int sdy_add(const float *a, const float *b, float *out, long n, sdy_stream s);
int sdy_axpy(float *y, float a, const float *x, long n, sdy_stream s);
int sdy_dot(const float *a, const float *b, int n, float *out, sdy_stream s);
int sdy_f16_to_f32(const uint16_t *x, float *out, long n, sdy_stream s);
int sdy_f32_to_f16(const float *x, uint16_t *out, long n, sdy_stream s);
int sdy_softmax(float *x, int n, int n_rows, long stride, sdy_stream s);
/* RoPE cos/sin tables [n_pos][hd/2], computed on the host (libm, double) into host memory */
void sdy_rope_table_host(float *cos_out, float *sin_out, int n_pos, int hd, float theta);
int sdy_rope(float *x, int n_heads, int hd, const float *cs, const float *sn, int interleaved, sdy_stream s);
int sdy_moe_route(float *probs, int n_tok, int n_expert, int k, int32_t *top, float *wts, sdy_stream s);
/* The routed (token, slot) pairs of top ([n_tok][k] expert ids) grouped by expert, stably: sorted row
 * r is pair out_row[r] = t * k + s of token src_tok[r]; expert e owns rows grp_tok[e] ..
 * grp_tok[e + 1] - 1 and the bn-row tiles grp_tile[e] .. grp_tile[e + 1] - 1 (arrays of n_expert + 1). */
int sdy_moe_sort(const int32_t *top, int n_tok, int k, int n_expert, int bn, int *grp_tok, int *grp_tile,
                 int32_t *src_tok, int32_t *out_row, sdy_stream s);
int sdy_gather_rows(const float *src, const int32_t *idx, int n, int dim, float *dst, sdy_stream s);
int sdy_moe_combine(const float *y, const int32_t *top, const float *wts, int n_tok, int k, int dim, float *out,
                    const float *resid, sdy_stream s);
/* RMSNorm of n_rows rows of n floats, then the activation quantiser vtype (SDY_Q8_K / SDY_Q8_0)
 * into xq, or vtype SDY_F32: normalise only. xb receives the f32 rows (may be NULL when
 * quantising). Bytes equal sdy_rmsnorm followed by sdy_quantize. */
int sdy_norm_quant(const float *x, const float *w, float eps, int n, int n_rows, float *xb, int vtype, void *xq,
                   sdy_stream s);
/* One-token decode attention at the position held in step_dev[1] (read on the device, so that a
 * recorded step replays for every position): q/k norm + RoPE, the KV-cache write of that position,
 * the scores (scores: sdy_attn_scores_floats(1, n_head, max_seq) floats of scratch), the softmax and
 * the weighted V into out (n_head * hd floats), and with xq_q8k also out's Q8_K row. */
int sdy_attn_decode_ok(int n_head, int n_kv_head, int hd, int max_seq);
int sdy_attn_decode(const float *q, const float *k, const float *v, const float *q_norm, const float *k_norm,
                    float eps, const float *rope_cos, const float *rope_sin, const int32_t *step_dev, int n_head,
                    int n_kv_head, int hd, int interleaved, void *k_cache, void *v_cache, int kv_type,
                    long head_stride, int max_seq, float *scores, float *out, void *xq_q8k, sdy_stream s);
/* One-token decode attention in two launches, split over spans of positions (64, or more for
 * caches beyond 8192 positions) with a deterministic merge in span order (within tolerance of the
 * reference; sdy_attn_decode is the bit-exact form): the same inputs and outputs as
 * sdy_attn_decode, with part (sdy_attn_chunked_floats floats) as scratch. xq_q8k needs
 * n_head * hd % 256 == 0. head_dim 64, 128 or 256, at most 16 query heads per kv head. */
int sdy_attn_chunked_ok(int n_head, int n_kv_head, int hd);
size_t sdy_attn_chunked_floats(int n_head, int hd, int max_seq);
int sdy_attn_decode_chunked(const float *q, const float *k, const float *v, const float *q_norm, const float *k_norm,
                            float eps, const float *rope_cos, const float *rope_sin, const int32_t *step_dev,
                            int n_head, int n_kv_head, int hd, int interleaved, void *k_cache, void *v_cache,
                            int kv_type, long head_stride, int max_seq, float *part, float *out, void *xq_q8k,
                            sdy_stream s);
/* One-token decode attention in one launch, split over 32-position chunks with a deterministic
 * merge (within tolerance of the reference; sdy_attn_decode is the bit-exact form): the same
 * inputs and outputs as sdy_attn_decode (f32 cache only), with part (sdy_attn_decode_split_floats floats) and count
 * (n_kv_head unsigned, zero before the first call; each call leaves them zero) as scratch. xq_q8k
 * needs whole Q8_K blocks per kv group ((n_head / n_kv_head) * hd % 256 == 0). head_dim 64 or 128,
 * at most 16 query heads per kv head. */
int sdy_attn_decode_split_ok(int n_head, int n_kv_head, int hd);
size_t sdy_attn_decode_split_floats(int n_head, int hd, int max_seq);
int sdy_attn_decode_split(const float *q, const float *k, const float *v, const float *q_norm, const float *k_norm,
                          float eps, const float *rope_cos, const float *rope_sin, const int32_t *step_dev, int n_head,
                          int n_kv_head, int hd, int interleaved, float *k_cache, float *v_cache, long head_stride,
                          int max_seq, float *part, unsigned *count, float *out, void *xq_q8k, sdy_stream s);
/* ---- one step of speculative decoding: a drafted tree of tokens evaluated together. Node t of n_tok has the parent
 * parent[t] (device int32), a lower index; one outside [0, t) makes t a root, and below -1 marks a place without a node (so
 * that a recorded step of a fixed size replays for smaller trees). The calls are asynchronous on s, allocate nothing and
 * keep nothing between calls; every array is device memory of the calling thread's current device. */

/* Scaling of rotary positions for contexts beyond the original one */
enum { SDY_ROPE_PLAIN = 0, SDY_ROPE_LINEAR = 1, SDY_ROPE_YARN = 2, SDY_ROPE_LLAMA3 = 3 };
typedef struct {
    int kind;                    /* SDY_ROPE_* */
    float factor;                /* the context's growth (not PLAIN) */
    int orig_ctx;                /* YARN, LLAMA3: the context of training */
    float beta_fast, beta_slow;  /* YARN: turns over orig_ctx that keep, or take the whole of, the scaling (32, 1) */
    float attn_factor;           /* YARN: the factor on cos and sin; 0: 0.1 ln(factor) + 1 */
    float low_freq, high_freq;   /* LLAMA3: turns over orig_ctx between which the scaling fades (1, 4) */
} sdy_rope_scaling;
/* Host only: freq[n_rot / 2] and *mscale of sdy_qk_rope_at for base theta; sc may be NULL (PLAIN). */
int sdy_rope_freqs(double *freq, float *mscale, int n_rot, float theta, const sdy_rope_scaling *sc);

/* Rotary positions of tokens with a position and a slot each (drafted trees, several conversations' tokens, prompts that
 * go to scattered slots): the q heads' rotated rows to q_out, the rotated k and the v rows to slots of K/V memory. */
typedef struct {
    const float *q, *k, *v;      /* token rows t * q_stride ... floats apart; q or k (with v) may be NULL */
    long q_stride, k_stride, v_stride;
    float *q_out;                /* rows q_out_stride apart; may be q with the same stride, no other overlap */
    long q_out_stride;
    void *k_rows, *v_rows;       /* [n_kv_head][n_slot][hd] of kv_type, heads head_stride elements apart */
    long head_stride;
    int kv_type, n_slot;
    const int32_t *pos, *slot;   /* [n_tok]; slot NULL: pos. A slot outside [0, n_slot): no row is written; of several
                                    tokens with one slot the last one's row is (found by comparing all: give
                                    tens of thousands of tokens in several calls). Any int32 position */
    const double *freq;          /* [n_rot / 2] (sdy_rope_freqs): angle pos * freq[i] */
    float mscale;                /* the factor on cos and sin */
    int n_rot, interleaved;      /* dims of a head that turn, the first; pairs (2i, 2i+1) or (i, i + n_rot/2) */
    const float *q_norm, *k_norm; /* [hd] RMSNorm weights of a head before it turns, or NULL */
    float eps;
    int n_tok, n_head, n_kv_head, hd; /* hd even, at most 512 */
} sdy_rope_at_args;
int sdy_qk_rope_at(const sdy_rope_at_args *a, sdy_stream s);

/* Attention of the nodes: node t sees every cached position below *n_past, itself and the nodes above it. K/V rows of the
 * nodes are in memory of their own (as sdy_qk_rope_at writes them with slot = node), so the cache holds accepted
 * positions only. Within tolerance (f32 sums in the kernel's order), the same on every call. An infinity or NaN in a K or V
 * row makes the outputs of the nodes that see it NaN, and of no others. An unused place's output row, and with *n_past
 * outside [0, max_past] every row, is left as it was. */
typedef struct {
    const float *q;              /* rotated queries, rows q_stride floats apart */
    long q_stride;
    const void *k_cache, *v_cache; /* [n_kv_head][..][hd] of kv_type, heads head_stride elements apart */
    long head_stride;
    const void *k_draft, *v_draft; /* node t's rows at t * hd of each kv head, heads draft_stride elements apart */
    long draft_stride;
    int kv_type;
    const int32_t *parent;       /* [n_tok] */
    const int32_t *n_past;       /* device int: the number of cached positions */
    int max_past;                /* bound on *n_past (the scratch's size and the launch's), at most 2^28 */
    int n_tok, n_head, n_kv_head, hd; /* n_tok at most 256; hd 64, 128 or 256 */
    float *out;                  /* rows out_stride floats apart */
    long out_stride;
    float *part;                 /* scratch of sdy_attn_tree_floats floats; not for two calls at once */
} sdy_attn_tree_args;
int sdy_attn_tree_ok(int n_tok, int n_head, int n_kv_head, int hd);
size_t sdy_attn_tree_floats(int n_tok, int n_head, int n_kv_head, int hd, int max_past);
int sdy_attn_tree(const sdy_attn_tree_args *a, sdy_stream s);

/* A token per row of logits. In the order of a row's logits, the greatest first and of equal ones the lowest index: the
 * first top_k tokens stay (<= 0: all); of these the shortest prefix whose probabilities (at temperature temp) reach top_p of
 * their sum (>= 1: all, <= 0: the first); of these the ones with at least min_p times the first one's probability; the first
 * always. The token is the first by index at which the running sum of the kept probabilities exceeds u of their whole
 * (u in [0, 1), clamped). temp <= 0: the first token. -inf and NaN logits are never chosen; a row of nothing else gives
 * token -1 and prob 0; beside +inf logits no others count. Probabilities below 2^(ceil log2 n_vocab - 62) of the greatest count as 0. */
typedef struct {
    const float *logits;         /* rows stride floats apart */
    long stride;
    int n_rows, n_vocab;         /* at most 65535, 2^22 */
    const float *temp;           /* [n_rows] each, or NULL: temperature 1, no top-k, no top-p, no min-p (NaN: temp as 0,
                                    the others as if not given) */
    const int32_t *top_k;
    const float *top_p, *min_p;
    const float *u;              /* [n_rows] uniform numbers */
    int32_t *token;              /* [n_rows] */
    float *prob;                 /* [n_rows] the token's probability among the kept, or NULL */
    void *ws;                    /* scratch of sdy_sample_ws_bytes bytes; not for two calls at once */
} sdy_sample_args;
size_t sdy_sample_ws_bytes(int n_rows, int n_vocab);
int sdy_sample(const sdy_sample_args *a, sdy_stream s);

/* The accepted path: node 0 (the step's own token), then from each node the lowest child whose token is the one sampled at
 * its parent. Node path[i]'s K/V rows go to position *n_past + i of every layer's cache; nodes beyond max_seq are not
 * accepted. With *n_past outside [0, max_seq) or no node 0, nothing is (n_acc 0, step and caches left as they were). */
typedef struct {
    const int32_t *token, *parent, *sampled; /* [n_tok] the drafted tokens, their parents, the token sampled at each node */
    int n_tok;                   /* at most 256 */
    const int32_t *n_past;       /* device int */
    const void *k_draft, *v_draft; /* [n_layer][n_kv_head][..][hd] of kv_type, strides in elements; not in the cache */
    long draft_stride, draft_layer_stride;
    void *k_cache, *v_cache;     /* [n_layer][n_kv_head][max_seq][hd] */
    long head_stride, layer_stride;
    int kv_type, max_seq, n_layer, n_kv_head, hd;
    int32_t *path;               /* [n_tok] the accepted nodes in order, then -1 */
    int32_t *n_acc;              /* [1] */
    int32_t *step;               /* [2] the next token and its position, as the one-token steps read them; path, n_acc and step
                                    share memory with nothing else */
} sdy_tree_commit_args;
int sdy_tree_commit(const sdy_tree_commit_args *a, sdy_stream s);
#ifdef __cplusplus
}
#endif
#endif
