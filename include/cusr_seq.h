/* cusr_seq.h -- C ABI of the sequence operators (libcusr_seq.so): what a
 * learned proposer of expressions needs next to the constant fitter. A
 * population's prefix programs are token sequences packed end to end with
 * offsets (pop_format.h); a causal model over them proposes expressions, the
 * fitter returns their losses, and a policy gradient trains the model on
 * those. No counterpart in the reference.
 *
 * Every entry point takes device pointers and a HIP stream, launches on that
 * stream and returns without waiting; nothing is allocated, and nothing is
 * kept from one call for the next. The calling thread's current device must
 * be the stream's. Arguments are checked on the host first: a refusal launches
 * nothing. Offsets, lengths, tokens and positions live on the device and are
 * checked there, by the kernels: a value out of range never leads to an access
 * out of range (each entry says what it gives instead).
 *
 * Return codes are cusr_co.h's: CO_OK, CO_ERR_NULLARG (null pointer, negative
 * size, struct of another size), CO_ERR_BOUNDS (a size beyond the bounds
 * below), CO_ERR_DATA (alignment, stride or workspace that does not fit; a
 * scale, temperature, clip width or coefficient out of range), CO_ERR_CUDA (a
 * HIP error at launch). */
#ifndef CUSR_SEQ_H
#define CUSR_SEQ_H

#include <stddef.h>
#include <stdint.h>

#include "cusr_co.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SEQ_FP32 0
#define SEQ_BF16 1
#define SEQ_FP16 2

#define SEQ_MAX_HEAD 128          /* head size of attention, a multiple of 8 */
#define SEQ_MAX_ROWS 2147000000LL /* query rows times heads, key rows, tokens */
#define SEQ_LEAST 1e-30f          /* least and largest scale and temperature */
#define SEQ_MOST 1e30f

/* Causal attention over packed sequences, bf16 or fp16.
 *
 * q [tq, hq, d], k and v [tk, hkv, d], o [tq, hq, d]: strides of rows and
 * heads in elements, the last dimension contiguous; hq a multiple of hkv, and
 * query head h reads key head h / (hq / hkv). Sequence b's queries are rows
 * cu_q[b] .. cu_q[b+1]-1, its keys start at row cu_k[b] and number
 * cu_k[b+1] - cu_k[b], or k_lens[b] of them when k_lens is given (a cache
 * whose segments have room to spare; rows beyond a length are never used).
 * cu_q[0] is 0. Queries are the last ones of the keys: query i of lq sees
 * keys 0 .. i + lk - lq. A query that sees no key, and a query row in no
 * sequence, give o = 0 and lse = -inf. Offsets out of order or out of range
 * are clamped into the tensors. A key or value that is not finite reaches only
 * queries that see it, and in the gradient a query or output gradient only keys
 * that it sees; near one a call takes longer.
 *
 * lse (may be null for the forward) [hq, tq] fp32: log of the sum of
 * exp(scale q.k) over the visible keys. o_low (may be null): what rounding o to
 * its type took away, itself rounded to it, in the rows whose gradient reads it (the
 * others are not written). A gradient needs sum(o * d_o) of each
 * row; from o alone its error is that of o's rounding and goes into every key of
 * the row alike. */
typedef struct SeqAttention {
    int32_t struct_size;
    int32_t dtype;
    int32_t n_seq, hq, hkv, d;
    int64_t tq, tk;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;
    float scale;
    int32_t reserved;
    const void *q, *k, *v;
    void *o;
    float *lse;
    void *o_low;              /* null, or [tq, hq, d], contiguous */
    const int32_t *cu_q, *cu_k, *k_lens;
    void *workspace;          /* seq_attention_workspace bytes, 256-aligned */
    int64_t workspace_bytes;
} SeqAttention;

/* Bytes of workspace of a call (0: none; negative: a refusal's code).
 * Depends on the sizes in the struct only, not on the offsets. */
int64_t seq_attention_workspace(const SeqAttention *a);
int seq_attention(const SeqAttention *a, void *stream);

/* Gradient of seq_attention: a's q, k, v, o, lse, o_low and offsets as the forward
 * call had them; d_o is the gradient of o. dq, dk, dv as q, k, v. Rows of dk and dv
 * that no query sees are 0. No atomics: the same call gives the same bits. */
typedef struct SeqAttentionGrad {
    int32_t struct_size;
    int32_t reserved;
    int64_t do_row, do_head, dq_row, dq_head, dk_row, dk_head, dv_row, dv_head;
    const void *d_o;
    void *dq, *dk, *dv;
} SeqAttentionGrad;

int64_t seq_attention_grad_workspace(const SeqAttention *a);
int seq_attention_grad(const SeqAttention *a, const SeqAttentionGrad *g, void *stream);

/* Rotary positions of q [tokens, hq, d] and k [tokens, hkv, d] (hkv 0: q
 * alone) in one launch. table [table_len, rot/2, 2] fp32 holds (cos, sin);
 * the first rot elements of each head turn, the rest is copied. Pairs are
 * (i, i + rot/2), or (2i, 2i + 1) when interleaved. inverse turns by the opposite
 * angles: the gradient (and the way back where cos^2 + sin^2 is 1 in the table).
 * In place (q_out == q with equal strides, every element of q and k in memory of
 * its own) is allowed. A position outside the table gives NaN in the turned
 * elements of its token. */
typedef struct SeqRotary {
    int32_t struct_size;
    int32_t dtype;            /* SEQ_FP32, SEQ_BF16 or SEQ_FP16 */
    int32_t hq, hkv, d, rot;
    int32_t interleaved, inverse;
    int64_t tokens, table_len;
    int64_t q_row, q_head, k_row, k_head, qo_row, qo_head, ko_row, ko_head;
    const void *q, *k;
    void *q_out, *k_out;
    const void *positions;    /* [tokens], int32_t, or int64_t when positions_64 */
    const float *table;
    int32_t positions_64, reserved;
} SeqRotary;

int seq_rotary(const SeqRotary *r, void *stream);

/* Clipped policy loss with a KL term over logits [tokens, vocab] (rows
 * `row` elements apart): z = logits / temperature,
 *   logp = z[action] - logsumexp z,   ratio = exp(logp - logp_old),
 *   l = -min(ratio A, clip(ratio, 1 - clip_lo, 1 + clip_hi) A)
 *       + kl_coef (exp(logp_ref - logp) - (logp_ref - logp) - 1),
 *   loss = sum over tokens of weight * l.
 * logp_ref null or kl_coef 0: no KL term. A token of weight 0 takes no part,
 * whatever its logits: logp = 0, its gradient row is 0. A row whose action has the
 * logit -inf has logp = -inf, ratio 0 and no gradient (and with a KL term an
 * infinite loss), whatever logp_old and logp_ref, -inf among them. An action
 * outside the vocabulary gives logp = NaN.
 * dlogits (may be null: loss and logp alone) [tokens, vocab] like logits,
 * rows `drow` apart: d loss / d logits, times *dloss when dloss is given.
 * loss is one fp32. */
typedef struct SeqPolicyLoss {
    int32_t struct_size;
    int32_t dtype;
    int64_t tokens, vocab, row, drow;
    float clip_lo, clip_hi, kl_coef, temperature;
    const void *logits;
    const int64_t *actions;
    const float *logp_old, *logp_ref, *advantages, *weights;
    const float *dloss;
    float *loss, *logp;
    void *dlogits;
    void *workspace;
    int64_t workspace_bytes;
} SeqPolicyLoss;

int64_t seq_policy_loss_workspace(const SeqPolicyLoss *p);
int seq_policy_loss(const SeqPolicyLoss *p, void *stream);

#ifdef __cplusplus
}
#endif
#endif
