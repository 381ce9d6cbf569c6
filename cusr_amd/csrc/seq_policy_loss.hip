// seq_policy_loss.hip -- clipped policy loss with a KL term and its gradient
// (include/cusr_seq.h, seq_policy_loss).
//
// Each token needs the log-sum-exp of its row of logits and one logit of it;
// the gradient is a multiple of (one-hot(action) - softmax) per row. The bound
// is memory: a row is read, and its gradient written, once.
#include "seq_common.h"

namespace seq {

// exp(x / temperature) for x <= 0 as a power of two. The factor has two parts, for what
// 32 bits round away would be the same relative error in every exponent of every
// token and so reach the loss undiminished. Both are positive: -inf stays itself. `two`:
// the second part is a quarter of a rounding or more (at temperature 1 it is a fifth).
// The branch on it splits the sums of a long row by pieces, which the compiler
// otherwise runs into each other: 8,192 rows of 131,071 in bf16 take 0.75 ms with it
// at either temperature, 0.90 with the second part always, 0.85 with none.
struct Scale {
    float high, low, nearest;
    bool two;
    double inverse;                          // 1 / temperature
    __device__ float exp(float x) const { return exp2_fast(__builtin_fmaf(x, high, x * low)); }
    // for a gradient, whose errors are its own
    __device__ float exp_nearest(float x) const { return exp2_fast(x * nearest); }
};
struct Policy : SeqPolicyLoss { Scale scale; };

Policy make_policy(const SeqPolicyLoss *p) {
    Policy r;
    static_cast<SeqPolicyLoss &>(r) = *p;
    const double k = 1.4426950408889634 / (double)p->temperature;
    r.scale.high = r.scale.nearest = (float)k;
    if ((double)r.scale.high > k) r.scale.high = nextafterf(r.scale.high, 0.0f);
    r.scale.two = fabs(k - (double)r.scale.nearest) > k * 0x1p-26;
    r.scale.inverse = 1.0 / (double)p->temperature;
    r.scale.low = fmaxf((float)(k - (double)r.scale.high), 1e-37f);
    return r;
}

// what a token brings beside its logits: read before them, so as not to wait after
struct Token { float weight, advantage, old, ref; int64_t action; };
__device__ inline Token token_of(const Policy &p, int64_t t) {
    return {p.weights[t], p.advantages[t], p.logp_old[t], p.logp_ref ? p.logp_ref[t] : 0.0f,
            p.actions[t]};
}

// the token's loss term and d term / d logp
struct Term { float loss, slope; };
__device__ inline Term policy_term(const Policy &p, const Token &k, double logp) {
    Term r;
    const float A = k.advantage;
    // a forbidden action's logp is -inf: its ratio is 0 and its KL term infinite also
    // where the other policies forbid it and the differences would be inf - inf
    const double none = -__builtin_inf();
    const bool old_none = logp == none && (double)k.old == none;
    const bool ref_none = logp == none && (double)k.ref == none;
    const float ratio = old_none ? 0.0f : expf((float)(logp - (double)k.old));
    const float free_ = ratio * A;
    // comparisons rather than fminf and fmaxf, which would drop a NaN
    const float lo = 1.0f - p.clip_lo, hi = 1.0f + p.clip_hi;
    const float held = (ratio < lo ? lo : (ratio > hi ? hi : ratio)) * A;
    r.loss = -(free_ <= held ? free_ : held);
    r.slope = free_ <= held ? -free_ : (held < free_ ? 0.0f : held);
    if (p.logp_ref && p.kl_coef != 0.0f) {   // a coefficient of 0 is no term: no 0 * inf
        const float gap = ref_none ? __builtin_inff() : (float)((double)k.ref - logp);
        const float e = expm1f(gap);
        r.loss += p.kl_coef * (gap > 80.0f ? e : e - gap);   // no inf - inf
        r.slope -= p.kl_coef * e;
    }
    return r;
}

// 16 bytes of a row: 8 values of a 16-bit type, 4 of fp32
template <typename T> struct Vec;
template <> struct Vec<__bf16> {
    static constexpr int n = 8;
    static __device__ float get(const uint4v &v, int j) {
        return j & 1 ? Bf16::hi(v[j / 2]) : Bf16::lo(v[j / 2]);
    }
    static __device__ uint4v pack(const float *f) {
        return {Bf16::pack(f[0], f[1]), Bf16::pack(f[2], f[3]), Bf16::pack(f[4], f[5]),
                Bf16::pack(f[6], f[7])};
    }
};
template <> struct Vec<_Float16> {
    static constexpr int n = 8;
    static __device__ float get(const uint4v &v, int j) {
        return j & 1 ? Fp16::hi(v[j / 2]) : Fp16::lo(v[j / 2]);
    }
    static __device__ uint4v pack(const float *f) {
        return {Fp16::pack(f[0], f[1]), Fp16::pack(f[2], f[3]), Fp16::pack(f[4], f[5]),
                Fp16::pack(f[6], f[7])};
    }
};
template <> struct Vec<float> {
    static constexpr int n = 4;
    static __device__ float get(const uint4v &v, int j) { return __uint_as_float(v[j]); }
    static __device__ uint4v pack(const float *f) {
        return {__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                __float_as_uint(f[3])};
    }
};

// Running maximum m and sum of exp((x - m) / temperature) of a thread.
struct Running {
    float m = neg_inf(), s = 0.0f;
    template <int N> __device__ void add(const float *x, Scale k) {
        float c = x[0];
#pragma unroll
        for (int j = 1; j < N; j++) c = fmaxf(c, x[j]);
        const float mn = fmaxf(m, c), m0 = mn == neg_inf() ? 0.0f : mn;
        s *= k.exp(m - m0);
        if (k.two)
#pragma unroll
            for (int j = 0; j < N; j++) s += k.exp(x[j] - m0);
        else
#pragma unroll
            for (int j = 0; j < N; j++) s += k.exp_nearest(x[j] - m0);
        m = mn;
    }
};

// The maximum and the sum of a block's running pairs, in one order, on every
// thread. red holds 2 * waves floats.
template <int WAVES>
__device__ inline void block_softmax(Running r, Scale k, float *red, float &m0, float &sum) {
    float m = r.m;
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    const int w = threadIdx.x >> 6;
    if (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) red[w] = m;
        __syncthreads();
        m = red[0];
#pragma unroll
        for (int i = 1; i < WAVES; i++) m = fmaxf(m, red[i]);
    }
    m0 = m == neg_inf() ? 0.0f : m;
    // a thread without a finite value has r.m = -inf and s = 0 (or NaN)
    float s = r.s * (r.m == neg_inf() ? 1.0f : k.exp(r.m - m0));
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    if (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) red[WAVES + w] = s;
        __syncthreads();
        s = red[WAVES];
#pragma unroll
        for (int i = 1; i < WAVES; i++) s += red[WAVES + i];
    }
    sum = s;
}

// What a row's gradient needs: dlogits_j = gs exp((x_j - m0) / temperature), plus g at
// the action.
struct RowGrad { float g, gs; };
template <typename T>
__device__ inline RowGrad finish_row(const Policy &p, const Token &k, float xa, float m0,
                                     float sum, float &term, float &logp) {
    const float inv_t = 1.0f / p.temperature;
    // in 64 bits but for the mantissa's logarithm: differences from the other policies'
    // follow, which are small beside the terms
    int e;
    const float mantissa = frexpf(sum, &e);
    double l = ((double)xa - (double)m0) * p.scale.inverse -
               ((double)e * 0.69314718055994531 + (double)logf(mantissa));
    if (xa == neg_inf()) l = -__builtin_inf();
    logp = (float)l;
    const Term q = policy_term(p, k, l);
    term = k.weight * q.loss;
    RowGrad r;
    r.g = logp == neg_inf() ? 0.0f : k.weight * q.slope * inv_t;
    if (p.dloss) r.g *= *p.dloss;
    r.gs = r.g == 0.0f ? 0.0f : -r.g / sum;
    return r;
}

// A row per block, any size, stride and alignment: reads the row once for the
// sums and, for the gradient, once more (mostly from the last cache). The loss
// alone of 64 rows of 32,001 in fp32 takes 16 us with its sum, which is two
// launches.
template <typename T>
__global__ __launch_bounds__(1024) void policy_stream(Policy p, double *terms) {
    constexpr int N = Vec<T>::n;
    const int64_t t = block_number();
    if (t >= p.tokens) return;
    const T *x = (const T *)p.logits + t * p.row;
    T *dx = p.dlogits ? (T *)p.dlogits + t * p.drow : nullptr;
    const Token of = token_of(p, t);
    if (of.weight == 0.0f) {
        if (threadIdx.x == 0) { p.logp[t] = 0.0f; terms[t] = 0.0; }
        if (dx) for (int64_t j = threadIdx.x; j < p.vocab; j += 1024) dx[j] = (T)0.0f;
        return;
    }
    __shared__ float red[32];
    const Scale k = p.scale;
    const int64_t a = of.action;
    const float xa = a >= 0 && a < p.vocab ? (float)x[a] : __builtin_nanf("");
    Running r;
    // whole 16-byte pieces between the row's first and last aligned address
    const int64_t head = (int64_t)((-(uintptr_t)x & 15) / sizeof(T));
    const int64_t pieces = p.vocab > head ? (p.vocab - head) / N : 0;
    for (int64_t i = threadIdx.x; i < pieces; i += 1024) {
        const uint4v v = *(const uint4v *)(x + head + i * N);
        float f[N];
#pragma unroll
        for (int j = 0; j < N; j++) f[j] = Vec<T>::get(v, j);
        r.add<N>(f, k);
    }
    const int64_t edge = p.vocab - pieces * N;        // values outside the pieces
    for (int64_t i = threadIdx.x; i < edge; i += 1024) {
        const float f = (float)x[i < head ? i : pieces * N + i];
        r.add<1>(&f, k);
    }
    float m0, sum, term, logp;
    block_softmax<16>(r, k, red, m0, sum);
    const RowGrad g = finish_row<T>(p, of, xa, m0, sum, term, logp);
    if (threadIdx.x == 0) { p.logp[t] = logp; terms[t] = term; }
    if (dx)
        for (int64_t j = threadIdx.x; j < p.vocab; j += 1024)
            dx[j] = (T)((j == a ? g.g : 0.0f) + g.gs * k.exp_nearest((float)x[j] - m0));
}

// A row per block of THREADS, kept in registers as NV pieces of 16 bytes a
// thread: read once, written once; memory bounds it (8,192 rows of 131,071 in bf16,
// a fifth of them without weight: 0.75 ms, 5.2 TB/s). Pieces are the aligned ones
// inside the row; the few values before and after them go one to a thread.
template <typename T, int THREADS, int NV>
__global__ __launch_bounds__(THREADS) void policy_row(Policy p, double *terms) {
    constexpr int N = Vec<T>::n, WAVES = THREADS / 64;
    const int64_t t = block_number();
    if (t >= p.tokens) return;
    const T *x = (const T *)p.logits + t * p.row;
    T *dx = (T *)p.dlogits + t * p.drow;
    const int V = (int)p.vocab, tid = (int)threadIdx.x;
    const int head = min(V, (int)((-(uintptr_t)x & 15) / sizeof(T)));
    const int pieces = (V - head) / N, edge = V - pieces * N;
    const int je = tid < head ? tid : pieces * N + tid;     // this thread's edge value
    const uint4v *x4 = (const uint4v *)(x + head);
    uint4v *d4 = (uint4v *)(dx + head);
    const Token of = token_of(p, t);
    if (of.weight == 0.0f) {
        if (tid == 0) { p.logp[t] = 0.0f; terms[t] = 0.0; }
        const uint4v z = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (i * THREADS + tid < pieces) (d4 + i * THREADS)[tid] = z;
        if (tid < edge) dx[je] = (T)0.0f;
        return;
    }
    const Scale k = p.scale;
    uint4v v[NV];
    const float ninf[8] = {neg_inf(), neg_inf(), neg_inf(), neg_inf(),
                           neg_inf(), neg_inf(), neg_inf(), neg_inf()};
    const uint4v none = Vec<T>::pack(ninf);
#pragma unroll
    for (int i = 0; i < NV; i++) {
        v[i] = none;
        if (i * THREADS + tid < pieces) v[i] = (x4 + i * THREADS)[tid];
    }
    const float xe = tid < edge ? (float)x[je] : neg_inf();
    const int64_t a = of.action;
    const float xa = a >= 0 && a < V ? (float)x[a] : __builtin_nanf("");
    __shared__ float red[2 * WAVES];
    Running r;
    r.add<1>(&xe, k);
#pragma unroll
    for (int i = 0; i < NV; i++) {
        float f[N];
#pragma unroll
        for (int j = 0; j < N; j++) f[j] = Vec<T>::get(v[i], j);
        r.add<N>(f, k);
    }
    float m0, sum, term, logp;
    block_softmax<WAVES>(r, k, red, m0, sum);
    const RowGrad g = finish_row<T>(p, of, xa, m0, sum, term, logp);
    if (tid == 0) { p.logp[t] = logp; terms[t] = term; }
    const int act = a >= 0 && a < V ? (int)a : -1;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int j0 = head + (i * THREADS + tid) * N;
        float f[N];
        // the unpacked values of the first pass are not to be kept: twice the registers
        asm volatile("" : "+v"(v[i]));
#pragma unroll
        for (int j = 0; j < N; j++) f[j] = g.gs * k.exp_nearest(Vec<T>::get(v[i], j) - m0);
        if (act >= j0 && act < j0 + N)
#pragma unroll
            for (int j = 0; j < N; j++) f[j] += j0 + j == act ? g.g : 0.0f;
        if (i * THREADS + tid < pieces) (d4 + i * THREADS)[tid] = Vec<T>::pack(f);
    }
    if (tid < edge) dx[je] = (T)((je == act ? g.g : 0.0f) + g.gs * k.exp_nearest(xe - m0));
}

// Few symbols: a block takes R rows through LDS, in 16-byte pieces when they
// lie end to end (`joined`); a thread owns a row. TURN: a thread starts its row at a
// column of its own, so that rows of a multiple of 16 bytes spread over the banks;
// others do by themselves, and save half of the vector instructions, which fill the
// time: 1.3 M rows of 21 in bf16 take 34 us with their sum, 4.2 TB/s,
// with turns 40 us. Unrolled loops take 61: the compiler joins columns to wider reads
// off their alignment.
template <typename T, int R, bool TURN>
__global__ __launch_bounds__(R) void policy_symbols(Policy p, bool joined, double *terms) {
    extern __shared__ __align__(16) unsigned char lds[];
    __shared__ double red[R / 64];
    constexpr int N = Vec<T>::n;
    const int V = (int)p.vocab;
    const int64_t t0 = (int64_t)blockIdx.x * R;
    const int rows = (int)(p.tokens - t0 < R ? p.tokens - t0 : R);
    const T *x = (const T *)p.logits + t0 * p.row;
    T *row = (T *)lds;
    const int n = rows * V, pieces = joined ? n / N : 0;
    const int64_t t = t0 + ((int)threadIdx.x < rows ? threadIdx.x : 0);
    const Token of = token_of(p, t);
    for (int i = threadIdx.x; i < pieces; i += R * 4) {
        uint4v v[4];                         // four on their way at a time
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (i + j * R < pieces) v[j] = ((const uint4v *)x)[i + j * R];
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (i + j * R < pieces) ((uint4v *)lds)[i + j * R] = v[j];
    }
    for (int i = pieces * N + threadIdx.x; i < n; i += R) row[i] = x[(i / V) * p.row + i % V];
    __syncthreads();
    float term = 0.0f;
    if ((int)threadIdx.x < rows) {
        T *y = row + threadIdx.x * V;
        // each column once
        auto columns = [&](auto f) {
            if (TURN) {
                for (int i = 0, j = (int)threadIdx.x % V; i < V; i++, j = j + 1 == V ? 0 : j + 1) f(j);
            } else {
#pragma unroll 1
                for (int j = 0; j < V; j++) f(j);
            }
        };
        if (of.weight == 0.0f) {
            p.logp[t] = 0.0f;
            columns([&](int j) { y[j] = (T)0.0f; });
        } else {
            const Scale k = p.scale;
            float m = neg_inf(), sum = 0.0f, logp;
            columns([&](int j) { m = fmaxf(m, (float)y[j]); });
            const float m0 = m == neg_inf() ? 0.0f : m;
            columns([&](int j) { sum += k.exp((float)y[j] - m0); });
            const int64_t a = of.action;
            const float xa = a >= 0 && a < V ? (float)y[a] : __builtin_nanf("");
            const RowGrad g = finish_row<T>(p, of, xa, m0, sum, term, logp);
            p.logp[t] = logp;
            if (p.dlogits)
                columns([&](int j) {
                    y[j] = (T)((j == a ? g.g : 0.0f) + g.gs * k.exp_nearest((float)y[j] - m0));
                });
        }
    }
    double s = term;
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = red[0];
        for (int i = 1; i < R / 64; i++) s += red[i];
        terms[blockIdx.x] = s;
    }
    if (!p.dlogits) return;
    T *dx = (T *)p.dlogits + t0 * p.drow;
    for (int i = threadIdx.x; i < pieces; i += R) ((uint4v *)dx)[i] = ((const uint4v *)lds)[i];
    for (int i = pieces * N + threadIdx.x; i < n; i += R) dx[(i / V) * p.drow + i % V] = row[i];
}

// the blocks' terms in one fixed order, in 64 bits
__global__ __launch_bounds__(1024) void policy_sum(const double *terms, int64_t n, float *loss) {
    __shared__ double red[16];
    double s = 0.0;
#pragma unroll 8
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

// Rows of a policy_symbols block: 256 while they fit 32 KB of LDS, fewer
// beyond; 0: too long a row, whose kernel has a wave or more to it (65,536 rows in
// bf16 of 64 symbols: 21 against 64 us, of 256: 46 against 62 us; of 512 it would
// take 152 against 62 us).
int symbol_rows(const SeqPolicyLoss &p) {
    const int64_t bytes = p.vocab * (p.dtype == SEQ_FP32 ? 4 : 2);
    return bytes <= 128 ? 256 : (bytes <= 256 ? 128 : (bytes <= 512 ? 64 : 0));
}

int check_policy(const SeqPolicyLoss *p) {
    if (!p || p->struct_size != (int32_t)sizeof(SeqPolicyLoss)) return CO_ERR_NULLARG;
    if (p->tokens < 0 || p->vocab < 1) return CO_ERR_NULLARG;
    if (p->tokens > SEQ_MAX_ROWS || p->vocab > SEQ_MAX_ROWS) return CO_ERR_BOUNDS;
    if (p->dtype < SEQ_FP32 || p->dtype > SEQ_FP16) return CO_ERR_DATA;
    return CO_OK;
}

template <typename T, int R>
void launch_symbols(const Policy &p, bool turn, bool joined, dim3 grid, size_t lds,
                    double *terms, hipStream_t s) {
    if (turn) policy_symbols<T, R, true><<<grid, R, lds, s>>>(p, joined, terms);
    else policy_symbols<T, R, false><<<grid, R, lds, s>>>(p, joined, terms);
}

template <typename T, int THREADS, int NV>
void launch_row(const Policy &p, double *terms, hipStream_t s) {
    policy_row<T, THREADS, NV><<<grid_of(p.tokens, THREADS), THREADS, 0, s>>>(p, terms);
}

// Launches the rows' kernel; returns the number of terms it leaves.
template <typename T>
int64_t launch_policy(const Policy &p, double *terms, hipStream_t s) {
    constexpr int N = Vec<T>::n;
    const int rows = symbol_rows(p);
    if (rows) {
        const int64_t blocks = (p.tokens + rows - 1) / rows;
        const dim3 grid((unsigned)blocks);
        const bool joined = p.row == p.vocab && !((uintptr_t)p.logits & 15) &&
                            (!p.dlogits || (p.drow == p.vocab && !((uintptr_t)p.dlogits & 15)));
        const size_t lds = (size_t)rows * p.vocab * sizeof(T);
        // five waves a compute unit, for rows beyond 256 bytes, wait longer for reads one
        // by one than the turns cost (262,144 rows of 252 in bf16: 186 against 157 us)
        const bool turn = p.vocab * sizeof(T) % 16 == 0;
        if (rows == 256) launch_symbols<T, 256>(p, turn, joined, grid, lds, terms, s);
        else if (rows == 128) launch_symbols<T, 128>(p, turn, joined, grid, lds, terms, s);
        else policy_symbols<T, 64, true><<<grid, 64, lds, s>>>(p, joined, terms);
        return blocks;
    }
    // A row stays in registers while it has at most 16 pieces for each of 1024 threads
    // (4,096 rows in bf16 of 1,000: 18 against 33 us streamed, of 32,001: 141 against
    // 178 us, 2,048 of 131,071: 257 against 396 us); the threads are as few as hold it.
    const int64_t n = (p.vocab + N - 1) / N;       // no row has more pieces
    const bool same = p.dlogits && !(((uintptr_t)p.logits ^ (uintptr_t)p.dlogits) & 15) &&
                      (p.row - p.drow) % N == 0;
    if (!same || n > 1024 * 16)
        policy_stream<T><<<grid_of(p.tokens, 1024), 1024, 0, s>>>(p, terms);
    else if (n <= 64 * 2) launch_row<T, 64, 2>(p, terms, s);
    else if (n <= 256 * 1) launch_row<T, 256, 1>(p, terms, s);
    else if (n <= 256 * 2) launch_row<T, 256, 2>(p, terms, s);
    else if (n <= 256 * 4) launch_row<T, 256, 4>(p, terms, s);
    else if (n <= 256 * 8) launch_row<T, 256, 8>(p, terms, s);
    else if (n <= 1024 * 4) launch_row<T, 1024, 4>(p, terms, s);
    else if (n <= 1024 * 6) launch_row<T, 1024, 6>(p, terms, s);
    else if (n <= 1024 * 8) launch_row<T, 1024, 8>(p, terms, s);
    else if (n <= 1024 * 12) launch_row<T, 1024, 12>(p, terms, s);
    else launch_row<T, 1024, 16>(p, terms, s);
    return p.tokens;
}

}  // namespace seq

extern "C" int64_t seq_policy_loss_workspace(const SeqPolicyLoss *p) {
    const int rc = seq::check_policy(p);
    if (rc != CO_OK) return rc > 0 ? -rc : rc;
    return 8 * p->tokens;
}

extern "C" int seq_policy_loss(const SeqPolicyLoss *p, void *stream) {
    int rc = seq::check_policy(p);
    if (rc != CO_OK) return rc;
    if (!p->loss) return CO_ERR_NULLARG;
    if (!(p->temperature >= SEQ_LEAST && p->temperature <= SEQ_MOST) || !(p->clip_lo >= 0.0f) ||
        !(p->clip_hi >= 0.0f) || !(fabsf(p->kl_coef) <= 3.4028235e38f))
        return CO_ERR_DATA;
    hipStream_t s = (hipStream_t)stream;
    double *ws = (double *)p->workspace;
    int64_t terms = 0;
    if (p->tokens) {
        const seq::Policy x = seq::make_policy(p);
        if (!p->logits || !p->actions || !p->logp_old || !p->advantages || !p->weights ||
            !p->logp || !p->workspace)
            return CO_ERR_NULLARG;
        if (p->workspace_bytes < 8 * p->tokens) return CO_ERR_DATA;
        switch (p->dtype) {
            case SEQ_FP32: terms = seq::launch_policy<float>(x, ws, s); break;
            case SEQ_BF16: terms = seq::launch_policy<__bf16>(x, ws, s); break;
            default: terms = seq::launch_policy<_Float16>(x, ws, s); break;
        }
        rc = seq::launch_status();
        if (rc != CO_OK) return rc;
    }
    seq::policy_sum<<<1, 1024, 0, s>>>(ws, terms, p->loss);
    return seq::launch_status();
}
