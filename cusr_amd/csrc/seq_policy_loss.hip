// seq_policy_loss.hip -- clipped policy loss with a KL term and its gradient
// (include/cusr_seq.h, seq_policy_loss).
//
// Each token needs the log-sum-exp of its row of logits and one logit of it;
// the gradient is a multiple of (one-hot(action) - softmax) per row. The bound
// is memory: a row is read, and its gradient written, once.
#include "seq_common.h"

namespace seq {

// the token's loss term and d term / d logp
struct Term { float loss, slope; };
__device__ inline Term policy_term(const SeqPolicyLoss &p, int64_t t, float logp) {
    Term r;
    const float A = p.advantages[t];
    const float ratio = __expf(logp - p.logp_old[t]);
    const float free_ = ratio * A;
    // comparisons rather than fminf and fmaxf, which would drop a NaN
    const float lo = 1.0f - p.clip_lo, hi = 1.0f + p.clip_hi;
    const float held = (ratio < lo ? lo : (ratio > hi ? hi : ratio)) * A;
    r.loss = -(free_ <= held ? free_ : held);
    r.slope = free_ <= held ? -free_ : (held < free_ ? 0.0f : held);
    if (p.logp_ref) {
        const float gap = p.logp_ref[t] - logp;
        const float e = expm1f(gap);
        r.loss += p.kl_coef * (gap > 80.0f ? e : e - gap);   // no inf - inf
        r.slope -= p.kl_coef * e;
    }
    return r;
}

template <typename T>
__global__ __launch_bounds__(256) void policy_rows(SeqPolicyLoss p, float *terms) {
    const int64_t t = blockIdx.x;
    const T *x = (const T *)p.logits + t * p.row;
    T *dx = p.dlogits ? (T *)p.dlogits + t * p.drow : nullptr;
    const float w = p.weights[t];
    if (w == 0.0f) {
        if (threadIdx.x == 0) { p.logp[t] = 0.0f; terms[t] = 0.0f; }
        if (dx) for (int64_t j = threadIdx.x; j < p.vocab; j += 256) dx[j] = (T)0.0f;
        return;
    }
    const float inv_t = 1.0f / p.temperature;
    __shared__ float red[8];
    float m = neg_inf();
    for (int64_t j = threadIdx.x; j < p.vocab; j += 256) m = fmaxf(m, (float)x[j]);
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float m0 = m == neg_inf() ? 0.0f : m;
    float sum = 0.0f;
    for (int64_t j = threadIdx.x; j < p.vocab; j += 256)
        sum += exp2_fast(((float)x[j] - m0) * inv_t * kLog2e);
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if ((threadIdx.x & 63) == 0) red[4 + (threadIdx.x >> 6)] = sum;
    __syncthreads();
    sum = (red[4] + red[5]) + (red[6] + red[7]);
    const int64_t a = p.actions[t];
    const bool in = a >= 0 && a < p.vocab;
    const float xa = in ? (float)x[a] : __builtin_nanf("");
    const float logp = xa == neg_inf() ? neg_inf() : (xa - m0) * inv_t - logf(sum);
    const Term term = policy_term(p, t, logp);
    if (threadIdx.x == 0) { p.logp[t] = logp; terms[t] = w * term.loss; }
    if (!dx) return;
    float g = logp == neg_inf() ? 0.0f : w * term.slope * inv_t;
    if (p.dloss) g *= *p.dloss;
    const float gs = g == 0.0f ? 0.0f : -g / sum;
    for (int64_t j = threadIdx.x; j < p.vocab; j += 256) {
        const float e = exp2_fast(((float)x[j] - m0) * inv_t * kLog2e);
        dx[j] = (T)((j == a ? g : 0.0f) + gs * e);
    }
}

// the tokens' terms in one fixed order
__global__ __launch_bounds__(1024) void policy_sum(const float *terms, int64_t n, float *loss) {
    __shared__ double red[16];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) s += terms[i];
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int i = 0; i < 16; i++) t += red[i];
        *loss = (float)t;
    }
}

int check_policy(const SeqPolicyLoss *p) {
    if (!p || p->struct_size != (int32_t)sizeof(SeqPolicyLoss)) return CO_ERR_NULLARG;
    if (p->tokens < 0 || p->vocab < 1) return CO_ERR_NULLARG;
    if (p->tokens > SEQ_MAX_ROWS || p->vocab > SEQ_MAX_ROWS) return CO_ERR_BOUNDS;
    if (p->dtype < SEQ_FP32 || p->dtype > SEQ_FP16) return CO_ERR_DATA;
    return CO_OK;
}

template <typename T>
int launch_policy(const SeqPolicyLoss &p, hipStream_t s) {
    float *terms = (float *)p.workspace;
    policy_rows<T><<<dim3((unsigned)p.tokens), 256, 0, s>>>(p, terms);
    return launch_status();
}

}  // namespace seq

extern "C" int64_t seq_policy_loss_workspace(const SeqPolicyLoss *p) {
    const int rc = seq::check_policy(p);
    if (rc != CO_OK) return rc > 0 ? -rc : rc;
    return 4 * p->tokens;
}

extern "C" int seq_policy_loss(const SeqPolicyLoss *p, void *stream) {
    int rc = seq::check_policy(p);
    if (rc != CO_OK) return rc;
    if (!p->loss) return CO_ERR_NULLARG;
    if (!(p->temperature > 0.0f)) return CO_ERR_DATA;
    hipStream_t s = (hipStream_t)stream;
    if (p->tokens) {
        if (!p->logits || !p->actions || !p->logp_old || !p->advantages || !p->weights ||
            !p->logp || !p->workspace)
            return CO_ERR_NULLARG;
        if (p->workspace_bytes < 4 * p->tokens) return CO_ERR_DATA;
        switch (p->dtype) {
            case SEQ_FP32: rc = seq::launch_policy<float>(*p, s); break;
            case SEQ_BF16: rc = seq::launch_policy<__bf16>(*p, s); break;
            default: rc = seq::launch_policy<_Float16>(*p, s); break;
        }
        if (rc != CO_OK) return rc;
    }
    seq::policy_sum<<<1, 1024, 0, s>>>((const float *)p->workspace, p->tokens, p->loss);
    return seq::launch_status();
}
