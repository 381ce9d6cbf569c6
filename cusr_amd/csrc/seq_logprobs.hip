// seq_logprobs.hip -- log-probabilities of given tokens, with the entropy and the largest
// alternatives of their rows, and the gradient of the first two (include/cusr_seq.h,
// seq_logprobs, seq_logprobs_grad).
//
// With m the largest logit, t = x - m and e = exp(t / temperature), a row needs
// S = sum e and U = sum t e: logp = t_id / temperature - log S, and the entropy is
// log S - U / (S temperature), a sum of two terms of one sign. The bound is memory: a
// forward pass reads a row once, or twice where its largest value has nearly all the weight
// and a block has the row (logprob_rows), the gradient reads and writes it once.
#include "seq_rows.h"

namespace seq {

// exp(t / temperature) for t <= 0 as a power of two, and t / temperature, with both
// factors in two parts: what 32 bits round away of them would be the same relative
// error in every exponent of every row.
struct Warmth {
    float high, low;                             // log2(e) / temperature
    float inverse, inverse_low;                  // 1 / temperature
    __device__ float power(float t) const { return __builtin_fmaf(t, high, t * low); }
    __device__ float exp(float t) const { return exp2_fast(power(t)); }
    __device__ float times(float t) const { return __builtin_fmaf(t, inverse, t * inverse_low); }
};
// both parts positive, so that t = -inf stays itself
void two_parts(double x, float &high, float &low) {
    high = (float)x;
    if ((double)high > x) high = nextafterf(high, 0.0f);
    low = fmaxf((float)(x - (double)high), 1e-37f);
}
Warmth make_warmth(float temperature) {
    Warmth w;
    two_parts(1.4426950408889634 / (double)temperature, w.high, w.low);
    two_parts(1.0 / (double)temperature, w.inverse, w.inverse_low);
    return w;
}

// x y, but 0 where x is 0, whatever y
__device__ inline float times_or_0(float x, float y) { return x == 0.0f ? 0.0f : x * y; }

// t, or the lowest number for -inf, whose e is 0: no 0 * inf. A NaN shows in the sum of e.
__device__ inline float finite(float t) { return max2(t, -3.4028235e38f); }

// 16 bytes of a row
template <typename T> struct Sixteen {
    static constexpr int n = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(n)));
};

// The largest value so far, m, sum of e and sum of t e of a thread's values.
struct Sums {
    float m = neg_inf(), s = 0.0f, u = 0.0f;
    template <int N> __device__ void add(const float *x, const Warmth &w) {
        float c = x[0];
#pragma unroll
        for (int j = 1; j < N; j++) c = fmaxf(c, x[j]);
        const float mn = fmaxf(m, c), m0 = mn == neg_inf() ? 0.0f : mn;
        lower(m0, w);
        m = mn;
#pragma unroll
        for (int j = 0; j < N; j++) {
            const float t = x[j] - m0, e = w.exp(t);
            s += e;
            u = __builtin_fmaf(e, finite(t), u);
        }
    }
    // the sums for a larger value m0: t falls by its distance
    __device__ void lower(float m0, const Warmth &w) {
        const float d = m - m0, f = w.exp(d);    // m = -inf: f = 0, and s = u = 0
        u = times_or_0(f, u + times_or_0(s, d)); // s d may pass the largest float
        s *= f;
    }
};

// A block's sums: every thread gets the largest value and both sums, formed in one order.
template <int WAVES> __device__ inline Sums over_block(Sums a, const Warmth &w, float *red) {
    Sums r;
    r.m = over_lanes<Larger, 64>(a.m);
    const int wave = threadIdx.x >> 6;
    const bool first = (threadIdx.x & 63) == 0;
    if constexpr (WAVES > 1) {
        if (first) red[wave] = r.m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WAVES; i++) r.m = fmaxf(r.m, red[i]);
    }
    const float m0 = r.m == neg_inf() ? 0.0f : r.m;
    if (a.m != neg_inf()) a.lower(m0, w);        // else s = u = 0, or NaN
    r.s = over_lanes<Add, 64>(a.s);
    r.u = over_lanes<Add, 64>(a.u);
    if constexpr (WAVES > 1) {
        if (first) {
            red[WAVES + wave] = r.s;
            red[2 * WAVES + wave] = r.u;
        }
        __syncthreads();
        r.s = red[WAVES];
        r.u = red[2 * WAVES];
#pragma unroll
        for (int i = 1; i < WAVES; i++) {
            r.s += red[WAVES + i];
            r.u += red[2 * WAVES + i];
        }
    }
    return r;
}

// Below this much beside the largest value (a weight above 98.5 %), 1 + the rest has lost too
// much of the rest: the rest is summed again without it, from a second reading of the row.
constexpr float kPeak = 0x1p-6f;

struct Row { float m, rest, log_sum, entropy; }; // S = 1 + rest
__device__ inline Row row_of(float m, float rest, float u, const Warmth &w) {
    Row r;
    r.m = m;
    r.rest = rest;
    r.log_sum = log1pf(rest);
    r.entropy = r.log_sum - w.times(u / (1.0f + rest));
    return r;
}
__device__ inline Row empty_row() { return {0.0f, 0.0f, 0.0f, 0.0f}; }

__device__ inline void put_row(const SeqLogprobs &p, const Warmth &w, int64_t t, const Row &r,
                               bool none, int64_t id, float xa) {
    float logp = w.times(xa - r.m) - r.log_sum;
    if (none) logp = neg_inf();
    if (id < 0 || id >= p.vocab) logp = __builtin_nanf("");
    p.logp[t] = logp;
    p.entropy[t] = r.entropy;
    if (p.stats) {
        p.stats[2 * t] = r.m;
        p.stats[2 * t + 1] = r.rest;
    }
}

// Alternatives are ordered by keys: a value's place among floats, NaN the largest, then
// the lower column before the higher. 0 is below every key and ~0 above: a NaN's place is not
// the last one, so that its key in column 0 is none either.
typedef unsigned long long Key;
constexpr uint32_t kNanPlace = 0xfffffffeu;
__device__ inline Key key_of(float x, uint32_t col) {
    const uint32_t b = __float_as_uint(x + 0.0f);             // -0 as +0
    const uint32_t o = x != x ? kNanPlace : (b >> 31 ? ~b : b | 0x80000000u);
    return ((Key)o << 32) | (uint32_t)~col;
}
__device__ inline uint32_t col_of(Key k) { return ~(uint32_t)k; }
__device__ inline float value_of(Key k) {
    const uint32_t o = (uint32_t)(k >> 32);
    if (o == kNanPlace) return __builtin_nanf("");
    return __uint_as_float(o >> 31 ? o & 0x7fffffffu : ~o);
}
__device__ inline Key larger(Key a, Key b) { return a > b ? a : b; }
// over the wave's lanes, all of them: the value first, then the place among its equals
__device__ inline Key wave_largest(Key k) {
    const uint32_t high = over_lanes<Larger, 64>((uint32_t)(k >> 32));
    const uint32_t low = (uint32_t)(k >> 32) == high ? (uint32_t)k : 0;
    return ((Key)high << 32) | over_lanes<Larger, 64>(low);
}
__device__ inline void put_top(const SeqLogprobs &p, const Warmth &w, int64_t t, int i, Key k,
                               const Row &r, bool none) {
    const float lp = none ? neg_inf() : w.times(value_of(k) - r.m) - r.log_sum;
    p.top_logp[t * p.top + i] = lp;
    p.top_ids[t * p.top + i] = col_of(k);
}

// A row a block of THREADS, in 16-byte pieces between its first and last aligned
// address, the few values before and after them one to a thread. TOP: each thread keeps
// the place of its largest value; the largest of all is taken out `top` times, and the
// wave that owned it looks through that thread's values for the next below it. Memory bounds
// it, with the exponentials close behind: 8,192 rows of 131,071 in bf16 (2.15 GB) take 363
// us, 5.9 TB/s, the vector instructions some 90 in 100 of that time, and 710 us at least where
// the largest value has nearly all the weight of each row; 2,048 of 32,001 in fp32 43 and 77.
// Few rows wait for a row's way to four waves, eight trips one after the other (64 of 32,001 in
// fp32 8.3 us), and for a round an alternative: 9.1 with one, 12.1 with five, 22 with twenty.
template <typename T, int THREADS, bool TOP>
__global__ __launch_bounds__(THREADS) void logprob_rows(SeqLogprobs p, Warmth w) {
    constexpr int N = Sixteen<T>::n, WAVES = THREADS / 64;
    typedef typename Sixteen<T>::vec vec;
    __shared__ float red[4 * WAVES];
    __shared__ Key best[WAVES];
    const int64_t t = block_number();
    if (t >= p.tokens) return;
    const T *x = (const T *)p.logits + t * p.row;
    const int tid = threadIdx.x;
    const int64_t id = get_id(p.ids, p.ids_64, t);
    const float xa = id >= 0 && id < p.vocab ? (float)x[id] : 0.0f;
    int64_t head = (int64_t)((-(uintptr_t)x & 15) / sizeof(T));
    if (head > p.vocab) head = p.vocab;
    const int64_t pieces = (p.vocab - head) / N, edge = p.vocab - pieces * N;
    const int64_t my_edge = tid < head ? tid : pieces * N + tid;      // edge < 2 N <= THREADS
    const vec *x4 = (const vec *)(x + head);
    Sums a;
    int64_t where = -1;                          // piece of the largest value; -1: all -inf
#pragma unroll 4
    for (int64_t i = tid; i < pieces; i += THREADS) {
        const vec v = x4[i];
        float f[N];
#pragma unroll
        for (int j = 0; j < N; j++) f[j] = (float)v[j];
        const float had = a.m;
        a.add<N>(f, w);
        if (TOP && a.m > had) where = i;
    }
    if (tid < edge) {
        const float f = (float)x[my_edge];
        a.add<1>(&f, w);
    }
    const Sums all = over_block<WAVES>(a, w, red);
    const bool none = all.m == neg_inf() && all.s == 0.0f;
    const float m0 = all.m == neg_inf() ? 0.0f : all.m;
    Row r = empty_row();
    if (!none) {
        float rest = all.s - 1.0f;
        if (rest < kPeak) {                      // the block's branch; a NaN does not take it
            float again = 0.0f;
            int tops = 0;                        // values at the largest: all but one count
            auto add = [&](float f) {
                const float d = f - m0;
                if (d == 0.0f) tops++;
                else again += w.exp(d);
            };
            if (tid < edge) add((float)x[my_edge]);
            for (int64_t i = tid; i < pieces; i += THREADS) {
                const vec v = x4[i];
#pragma unroll
                for (int j = 0; j < N; j++) add((float)v[j]);
            }
            __syncthreads();
            again = over_group<Add, THREADS>(again, red);
            rest = again + (over_group<Add, THREADS>((float)tops, red) - 1.0f);
        }
        r = row_of(m0, rest, all.u, w);
    }
    if (tid == 0) put_row(p, w, t, r, none, id, xa);
    if constexpr (TOP) {
        // keys below `last` among the values of thread `who`, by this wave
        const int lane = tid & 63;
        auto next_of = [&](int who, Key last) {
            Key k = 0;
            if (lane == 0 && who < edge) {
                const int64_t at = who < head ? who : pieces * N + who;
                const Key e = key_of((float)x[at], (uint32_t)at);
                if (e < last) k = e;
            }
            for (int64_t i = who + (int64_t)lane * THREADS; i < pieces; i += 64ll * THREADS) {
                const vec v = x4[i];
#pragma unroll
                for (int j = 0; j < N; j++) {
                    const Key e = key_of((float)v[j], (uint32_t)(head + i * N + j));
                    if (e < last) k = larger(k, e);
                }
            }
            return wave_largest(k);
        };
        Key mine = 0;
        const bool odd = all.s != all.s;         // NaN: places of largest values say nothing
        if (!odd) {
            if (tid < edge) mine = key_of((float)x[my_edge], (uint32_t)my_edge);
            if (where >= 0) {
                const vec v = x4[where];
#pragma unroll
                for (int j = 0; j < N; j++)
                    mine = larger(mine, key_of((float)v[j], (uint32_t)(head + where * N + j)));
            } else if (tid < pieces) {
                mine = larger(mine, key_of(neg_inf(), (uint32_t)(head + (int64_t)tid * N)));
            }
        } else {
            for (int64_t i = tid; i < pieces; i += THREADS) {
                const vec v = x4[i];
#pragma unroll
                for (int j = 0; j < N; j++)
                    mine = larger(mine, key_of((float)v[j], (uint32_t)(head + i * N + j)));
            }
            if (tid < edge) mine = larger(mine, key_of((float)x[my_edge], (uint32_t)my_edge));
        }
        Key wave_best = wave_largest(mine);
        for (int i = 0; i < p.top; i++) {
            Key most = wave_best;
            if constexpr (WAVES > 1) {
                if (lane == 0) best[tid >> 6] = wave_best;
                __syncthreads();
#pragma unroll
                for (int o = 0; o < WAVES; o++) most = larger(most, best[o]);
                __syncthreads();
            }
            if (tid == 0) put_top(p, w, t, i, most, r, none);
            const uint64_t owner = __ballot(mine == most);
            if (owner) {                         // this wave's branch
                const int l = __ffsll((unsigned long long)owner) - 1;
                const Key next = next_of((tid & ~63) + l, most);
                if (lane == l) mine = next;
                wave_best = wave_largest(mine);
            }
        }
    }
}

// Few long rows: a row is cut into parts of kPartPieces, a block of 256 each, which keeps its
// values in registers and leaves its sums and its largest alternatives in the workspace;
// a wave a row joins them.
constexpr int kPartPieces = 1024, kMostParts = 64;
struct RowPart { float m, rest, u; int32_t bad; };  // sums over a part; bad: a value was NaN or inf

template <typename T>
__global__ __launch_bounds__(256) void logprob_parts(SeqLogprobs p, Warmth w, int parts, RowPart *sums,
                                                     Key *keys) {
    constexpr int N = Sixteen<T>::n, NV = kPartPieces / 256;
    typedef typename Sixteen<T>::vec vec;
    __shared__ float red[12];
    __shared__ Key best[4];
    const int64_t block = block_number(), t = block / parts;
    if (t >= p.tokens) return;
    const int part = (int)(block % parts), tid = threadIdx.x, lane = tid & 63;
    const T *x = (const T *)p.logits + t * p.row;
    int64_t head = (int64_t)((-(uintptr_t)x & 15) / sizeof(T));
    if (head > p.vocab) head = p.vocab;
    const int64_t pieces = (p.vocab - head) / N, edge = p.vocab - pieces * N;
    const vec *x4 = (const vec *)(x + head);
    // the row's first part takes the values outside the pieces, one to a thread
    const bool has_edge = part == 0 && tid < edge;
    const int64_t at_edge = tid < head ? tid : pieces * N + tid;
    const int64_t piece0 = (int64_t)part * kPartPieces + tid;
    vec v[NV];
    const float on_edge = has_edge ? (float)x[at_edge] : neg_inf();
#pragma unroll
    for (int i = 0; i < NV; i++) {
#pragma unroll
        for (int j = 0; j < N; j++) v[i][j] = (T)neg_inf();
        if (piece0 + i * 256 < pieces) v[i] = x4[piece0 + i * 256];
    }
    float m = on_edge;
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int j = 0; j < N; j++) m = fmaxf(m, (float)v[i][j]);
    m = over_group<Larger, 256>(m, red);
    const float m0 = m == neg_inf() ? 0.0f : m;
    float rest = 0.0f, u = 0.0f, tops = 0.0f;    // values at the largest: all but one count
    auto add = [&](float f) {
        const float d = f - m0, e = w.exp(d);
        if (d == 0.0f) tops += 1.0f;
        else rest += e;
        u = __builtin_fmaf(e, finite(d), u);
    };
    add(on_edge);
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int j = 0; j < N; j++) add((float)v[i][j]);
    rest = over_group<Add, 256>(rest, red);
    u = over_group<Add, 256>(u, red);
    tops = over_group<Add, 256>(tops, red);
    if (tid == 0) {
        // a part of -inf alone adds nothing; a NaN stays one
        RowPart r = {m, m == neg_inf() ? rest : rest + (tops - 1.0f), u, 0};
        r.bad = r.rest != r.rest || m == __builtin_inff();
        sums[t * parts + part] = r;
    }
    if (p.top == 0) return;
    Key last = ~0ull;
    auto next = [&] {                            // the thread's largest below `last`
        Key k = 0;
        if (has_edge) {
            const Key e = key_of(on_edge, (uint32_t)at_edge);
            if (e < last) k = e;
        }
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (piece0 + i * 256 < pieces)
#pragma unroll
                for (int j = 0; j < N; j++) {
                    const Key e = key_of((float)v[i][j], (uint32_t)(head + (piece0 + i * 256) * N + j));
                    if (e < last) k = larger(k, e);
                }
        return k;
    };
    Key mine = next(), wave_best = wave_largest(mine);
    Key *out = keys + (t * parts + part) * p.top;
    for (int i = 0; i < p.top; i++) {
        if (lane == 0) best[tid >> 6] = wave_best;
        __syncthreads();
        last = larger(larger(best[0], best[1]), larger(best[2], best[3]));
        __syncthreads();
        if (tid == 0) out[i] = last;             // 0: the part has no more
        if (last == 0) continue;
        if (__ballot(mine == last)) {            // this wave's branch
            if (mine == last) mine = next();
            wave_best = wave_largest(mine);
        }
    }
}

__global__ __launch_bounds__(64) void logprob_join(SeqLogprobs p, Warmth w, int parts,
                                                   const RowPart *sums, const Key *keys) {
    extern __shared__ __align__(8) Key lists[];  // parts x top
    const int64_t t = block_number();
    if (t >= p.tokens) return;
    const int lane = threadIdx.x;
    const int64_t id = get_id(p.ids, p.ids_64, t);
    const float xa = id >= 0 && id < p.vocab
                         ? get1(p.logits, p.dtype, t * p.row + id) : 0.0f;
    RowPart a = {neg_inf(), 0.0f, 0.0f, 0};
    if (lane < parts) a = sums[t * parts + lane];
    for (int i = lane; i < parts * p.top; i += 64) lists[i] = keys[t * parts * p.top + i];
    __syncthreads();
    const float m = over_lanes<Larger, 64>(a.m);
    const float m0 = m == neg_inf() ? 0.0f : m;
    const bool bad = __ballot(a.bad) != 0;
    // the first part with the largest value gives the one that the others are beside
    const uint64_t with = __ballot(a.m == m);
    const bool owner = with && lane == __ffsll((unsigned long long)with) - 1;
    float rest = 0.0f, u = 0.0f;
    if (a.m != neg_inf()) {
        const float d = a.m - m0, f = w.exp(d), s = 1.0f + a.rest;
        rest = owner ? a.rest : times_or_0(f, s);
        u = times_or_0(f, a.u + times_or_0(s, d));
    }
    rest = over_group<Add, 64>(rest, nullptr);
    u = over_group<Add, 64>(u, nullptr);
    const bool none = m == neg_inf() && !bad;
    Row r = none ? empty_row() : row_of(m0, bad ? __builtin_nanf("") : rest, u, w);
    if (lane == 0) put_row(p, w, t, r, none, id, xa);
    int at = 0;                                  // in the part's list
    Key mine = lane < parts && p.top ? lists[lane * p.top] : 0;
    for (int i = 0; i < p.top; i++) {
        const Key k = wave_largest(mine);
        if (lane == 0) put_top(p, w, t, i, k, r, none);
        if (mine == k) mine = ++at < p.top ? lists[lane * p.top + at] : 0;
    }
}

// Few symbols: a block takes R rows through LDS, in 16-byte pieces when they lie end to
// end (`joined`); a thread owns a row and goes through its columns. A thread starts at a
// column of its own where rows of a multiple of 16 bytes would meet in the banks. Vector
// instructions and LDS bound them: 1.3 M rows of 21 in bf16 (86 MB) take 20 us, 4.3 TB/s, the
// gradient (145 MB) 28, 5.2 TB/s, of operands that the last cache holds in part.
template <typename T, int R> struct Rows {
    __device__ static void fetch(const T *x, int64_t step, int rows, int V, bool joined, T *lds) {
        constexpr int N = Sixteen<T>::n;
        const int n = rows * V, pieces = joined ? n / N : 0;
        for (int i = threadIdx.x; i < pieces; i += R * 4) {
            uint4v v[4];                         // four on their way at a time
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i + j * R < pieces) v[j] = ((const uint4v *)x)[i + j * R];
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i + j * R < pieces) ((uint4v *)lds)[i + j * R] = v[j];
        }
        for (int i = pieces * N + threadIdx.x; i < n; i += R) lds[i] = x[(i / V) * step + i % V];
    }
    template <typename F> __device__ static void columns(int V, bool turn, F f) {
        if (turn) {
            for (int i = 0, j = (int)threadIdx.x % V; i < V; i++, j = j + 1 == V ? 0 : j + 1) f(j);
        } else {
#pragma unroll 1
            for (int j = 0; j < V; j++) f(j);
        }
    }
};

template <typename T, int R>
__global__ __launch_bounds__(R) void logprob_symbols(SeqLogprobs p, Warmth w, bool joined,
                                                     bool turn) {
    extern __shared__ __align__(16) unsigned char lds[];
    const int V = (int)p.vocab;
    const int64_t t0 = (int64_t)blockIdx.x * R;
    const int rows = (int)(p.tokens - t0 < R ? p.tokens - t0 : R);
    const int64_t t = t0 + ((int)threadIdx.x < rows ? threadIdx.x : 0);
    const int64_t id = get_id(p.ids, p.ids_64, t);
    Rows<T, R>::fetch((const T *)p.logits + t0 * p.row, p.row, rows, V, joined, (T *)lds);
    __syncthreads();
    if ((int)threadIdx.x >= rows) return;
    const T *y = (const T *)lds + threadIdx.x * V;
    auto columns = [&](auto f) { Rows<T, R>::columns(V, turn, f); };
    float m = neg_inf(), s = 0.0f, u = 0.0f;
    columns([&](int j) { m = fmaxf(m, (float)y[j]); });
    const float m0 = m == neg_inf() ? 0.0f : m;
    // the largest value is left out, and its equals counted: rows of few symbols have nearly
    // all weight on one often enough that a second pass for them is most waves' (24 us
    // for 1.3 M rows of 21 in bf16)
    float tops = 0.0f;
    columns([&](int j) {
        const float d = (float)y[j] - m0, e = w.exp(d);
        if (d == 0.0f) tops += 1.0f;
        else s += e;
        u = __builtin_fmaf(e, finite(d), u);
    });
    const bool none = m == neg_inf() && s == 0.0f;
    const Row r = none ? empty_row() : row_of(m0, s + (tops - 1.0f), u, w);
    put_row(p, w, t, r, none, id, id >= 0 && id < V ? (float)y[id] : 0.0f);
    Key last = ~0ull;
    for (int i = 0; i < p.top; i++) {
        Key k = 0;
        columns([&](int j) {
            const Key e = key_of((float)y[j], (uint32_t)j);
            if (e < last) k = larger(k, e);
        });
        put_top(p, w, t, i, k, r, none);
        last = k;
    }
}

// ------------------------------------------------------------------- gradient

// A row's gradient: d_j = g [j = id] - p_j (g + h (log p_j + entropy)), with g and h the
// gradients of logp and entropy over the temperature.
struct LogprobGrad {
    float m0, inverse, log_sum, entropy, g, h;
    float own;                                   // the token's own
    bool skip;                                   // both gradients are 0: nothing is read
    __device__ float of(float x, const Warmth &w) const {
        const float t = x - m0, prob = w.exp(t) * inverse;
        // below -256 prob is 0, and lp may be -inf
        const float lp = max2(w.times(t) - log_sum, -256.0f);
        return -prob * __builtin_fmaf(h, lp + entropy, g);
    }
};
__device__ inline LogprobGrad grad_of(const SeqLogprobsGrad &p, const Warmth &w, int64_t t, int64_t id,
                                  bool in, float xa) {
    LogprobGrad r;
    const float dl = p.dlogp ? p.dlogp[t] : 0.0f, dh = p.dentropy ? p.dentropy[t] : 0.0f;
    const float rest = p.stats[2 * t + 1];
    r.skip = dl == 0.0f && dh == 0.0f;
    r.m0 = p.stats[2 * t];
    r.inverse = 1.0f / (1.0f + rest);
    r.log_sum = log1pf(rest);
    r.entropy = p.entropy[t];
    r.g = w.times(dl);
    r.h = w.times(dh);
    if (!in && dl != 0.0f) r.g = __builtin_nanf("");
    if (in && w.times(xa - r.m0) - r.log_sum == neg_inf()) r.g = 0.0f;       // logp is
    r.own = r.of(xa, w) + r.g;
    // at the largest logit 1 - p is what the rest has: formed as such, for p rounds it away
    if (in && xa == r.m0)
        r.own = r.g * (rest * r.inverse) - r.inverse * times_or_0(r.h, r.entropy - r.log_sum);
    return r;
}

// A row is cut among `cuts` blocks, in turns of 256 pieces. Memory bounds it: 8,192 rows of
// 131,071 in bf16 (4.3 GB) take 830 us, 5.2 TB/s, as a copy does.
template <typename T>
__global__ __launch_bounds__(256) void logprob_grad_rows(SeqLogprobsGrad p, Warmth w, bool same,
                                                         int cuts) {
    constexpr int N = Sixteen<T>::n;
    typedef typename Sixteen<T>::vec vec;
    const int64_t t = cuts == 1 ? block_number() : block_number() / cuts;
    const int cut = cuts == 1 ? 0 : block_number() % cuts;
    if (t >= p.tokens) return;
    const T *x = (const T *)p.logits + t * p.row;
    T *dx = (T *)p.dlogits + t * p.drow;
    const int64_t id = get_id(p.ids, p.ids_64, t);
    const bool in = id >= 0 && id < p.vocab;
    const LogprobGrad r = grad_of(p, w, t, id, in, in ? (float)x[id] : 0.0f);
    // Pieces where both rows have them at the same places, from a boundary of 128 bytes of the
    // gradient's row on, so that waves write whole lines; past the caches, which keep the
    // logits: 8,192 rows of 131,071 in bf16 take 840 us (from the first boundary of 16 bytes
    // 938, and by way of the caches 901), 4,000 of 32,001 83 (109 by way of the caches).
    int64_t head = same ? (int64_t)((-(uintptr_t)dx & 127) / sizeof(T)) : 0;
    if (head > p.vocab) head = p.vocab;
    const int64_t pieces = same ? (p.vocab - head) / N : 0, edge = p.vocab - pieces * N;
    const vec *x4 = (const vec *)(x + head);
    vec *d4 = (vec *)(dx + head);
    auto value = [&](float f, int64_t j) {
        return (T)(j == id ? r.own : r.of(f, w));
    };
#pragma unroll 1
    for (int64_t i = cut * 256 + threadIdx.x; i < pieces; i += cuts * 256) {
        vec v = {};
        if (!r.skip) {
            v = x4[i];
#pragma unroll
            for (int j = 0; j < N; j++) v[j] = value((float)v[j], head + i * N + j);
        }
        __builtin_nontemporal_store(v, d4 + i);
    }
    for (int64_t i = cut * 256 + threadIdx.x; i < edge; i += cuts * 256) {
        const int64_t j = i < head ? i : pieces * N + i;
        dx[j] = r.skip ? (T)0.0f : value((float)x[j], j);
    }
}

template <typename T, int R>
__global__ __launch_bounds__(R) void logprob_grad_symbols(SeqLogprobsGrad p, Warmth w, bool joined,
                                                          bool turn) {
    extern __shared__ __align__(16) unsigned char lds[];
    constexpr int N = Sixteen<T>::n;
    const int V = (int)p.vocab;
    const int64_t t0 = (int64_t)blockIdx.x * R;
    const int rows = (int)(p.tokens - t0 < R ? p.tokens - t0 : R);
    const int64_t t = t0 + ((int)threadIdx.x < rows ? threadIdx.x : 0);
    const int64_t id = get_id(p.ids, p.ids_64, t);
    const bool in = id >= 0 && id < V;
    Rows<T, R>::fetch((const T *)p.logits + t0 * p.row, p.row, rows, V, joined, (T *)lds);
    __syncthreads();
    if ((int)threadIdx.x < rows) {
        T *y = (T *)lds + threadIdx.x * V;
        const LogprobGrad r = grad_of(p, w, t, id, in, in ? (float)y[id] : 0.0f);
        Rows<T, R>::columns(V, turn, [&](int j) {
            const float d = j == id ? r.own : r.of((float)y[j], w);
            y[j] = (T)(r.skip ? 0.0f : d);
        });
    }
    __syncthreads();
    T *dx = (T *)p.dlogits + t0 * p.drow;
    const int n = rows * V, pieces = joined ? n / N : 0;
    for (int i = threadIdx.x; i < pieces; i += R) ((uint4v *)dx)[i] = ((const uint4v *)lds)[i];
    for (int i = pieces * N + threadIdx.x; i < n; i += R)
        dx[(i / V) * p.drow + i % V] = ((const T *)lds)[i];
}

// ------------------------------------------------------------------- launches

// Rows of a block of the symbols' kernels, which keep them in 32 KB of LDS; 0: too long.
int symbol_rows_of(int64_t vocab, int dtype) {
    const int64_t bytes = vocab * type_bytes(dtype);
    return bytes <= 128 ? 256 : (bytes <= 256 ? 128 : (bytes <= 512 ? 64 : 0));
}

int check_logprobs(int64_t tokens, int64_t vocab, int dtype, float temperature) {
    if (tokens < 0 || vocab < 1) return CO_ERR_NULLARG;
    if (tokens > SEQ_MAX_ROWS || vocab > SEQ_MAX_ROWS) return CO_ERR_BOUNDS;
    if (!float_type(dtype) || !(temperature >= SEQ_LEAST && temperature <= SEQ_MOST))
        return CO_ERR_DATA;
    return CO_OK;
}
int check_logprobs(const SeqLogprobs *p) {
    if (!p || p->struct_size != (int32_t)sizeof(SeqLogprobs) || p->top < 0) return CO_ERR_NULLARG;
    const int rc = check_logprobs(p->tokens, p->vocab, p->dtype, p->temperature);
    if (rc != CO_OK) return rc;
    return p->top > SEQ_MAX_TOP || p->top > p->vocab ? CO_ERR_BOUNDS : CO_OK;
}

template <typename T, int THREADS>
void launch_rows(const SeqLogprobs &p, const Warmth &w, hipStream_t s) {
    const dim3 grid = grid_of(p.tokens, THREADS);
    if (p.top) logprob_rows<T, THREADS, true><<<grid, THREADS, 0, s>>>(p, w);
    else logprob_rows<T, THREADS, false><<<grid, THREADS, 0, s>>>(p, w);
}
// Parts of a row where rows are few and long; 0: a block a row. A call of 131,071 in fp32
// with five alternatives takes 18 against 26 us for a row, 24 against 30 for 64 and 60
// against 37 for 256; of 32,001, 18 against 14 for a row and for 64, for its second launch.
int parts_of(const SeqLogprobs &p) {
    const int n = 16 / type_bytes(p.dtype);
    const int64_t parts = (p.vocab / n + kPartPieces - 1) / kPartPieces;
    return p.tokens <= 64 && parts > 8 && parts <= kMostParts ? (int)parts : 0;
}
template <typename T> void launch_logprobs(const SeqLogprobs &p, hipStream_t s) {
    const Warmth w = make_warmth(p.temperature);
    const int parts = parts_of(p);
    if (parts) {
        RowPart *sums = (RowPart *)p.workspace;
        Key *keys = (Key *)(sums + p.tokens * parts);
        logprob_parts<T><<<(unsigned)(p.tokens * parts), 256, 0, s>>>(p, w, parts, sums, keys);
        const size_t lds = (size_t)parts * p.top * sizeof(Key);
        logprob_join<<<(unsigned)p.tokens, 64, lds, s>>>(p, w, parts, sums, keys);
        return;
    }
    const int rows = symbol_rows_of(p.vocab, p.dtype);
    if (rows) {
        const dim3 grid((unsigned)((p.tokens + rows - 1) / rows));
        const bool joined = p.row == p.vocab && !((uintptr_t)p.logits & 15);
        const bool turn = p.vocab * sizeof(T) % 16 == 0;
        const size_t lds = (size_t)rows * p.vocab * sizeof(T);
        if (rows == 256) logprob_symbols<T, 256><<<grid, 256, lds, s>>>(p, w, joined, turn);
        else if (rows == 128) logprob_symbols<T, 128><<<grid, 128, lds, s>>>(p, w, joined, turn);
        else logprob_symbols<T, 64><<<grid, 64, lds, s>>>(p, w, joined, turn);
        return;
    }
    const int64_t pieces = p.vocab / Sixteen<T>::n;
    // 1,024 threads took 17 against 14 us for 32,001 in fp32 with five alternatives, and 45
    // against 21 with twenty, whose rounds wait for each other
    if (pieces <= 256) launch_rows<T, 64>(p, w, s);
    else launch_rows<T, 256>(p, w, s);
}

template <typename T> void launch_grad(const SeqLogprobsGrad &p, hipStream_t s) {
    const Warmth w = make_warmth(p.temperature);
    const int rows = symbol_rows_of(p.vocab, p.dtype);
    if (rows) {
        const dim3 grid((unsigned)((p.tokens + rows - 1) / rows));
        const bool joined = p.row == p.vocab && p.drow == p.vocab &&
                            !(((uintptr_t)p.logits | (uintptr_t)p.dlogits) & 15);
        const bool turn = p.vocab * sizeof(T) % 16 == 0;
        const size_t lds = (size_t)rows * p.vocab * sizeof(T);
        if (rows == 256) logprob_grad_symbols<T, 256><<<grid, 256, lds, s>>>(p, w, joined, turn);
        else if (rows == 128)
            logprob_grad_symbols<T, 128><<<grid, 128, lds, s>>>(p, w, joined, turn);
        else logprob_grad_symbols<T, 64><<<grid, 64, lds, s>>>(p, w, joined, turn);
        return;
    }
    const bool same = !(((uintptr_t)p.logits ^ (uintptr_t)p.dlogits) & 15) &&
                      (p.row - p.drow) % Sixteen<T>::n == 0;
    // blocks to fill the chip, with a turn of pieces each at least
    const int64_t turns = (p.vocab / Sixteen<T>::n + 255) / 256;
    int64_t cuts = p.tokens < 2048 ? 2048 / p.tokens : 1;
    if (cuts > turns) cuts = turns;
    if (cuts < 1) cuts = 1;
    logprob_grad_rows<T><<<grid_of(p.tokens * cuts, 256), 256, 0, s>>>(p, w, same, (int)cuts);
}

}  // namespace seq

extern "C" int64_t seq_logprobs_workspace(const SeqLogprobs *p) {
    const int rc = seq::check_logprobs(p);
    if (rc != CO_OK) return rc > 0 ? -rc : rc;
    return p->tokens * seq::parts_of(*p) * (int64_t)(sizeof(seq::RowPart) + p->top * sizeof(seq::Key));
}

extern "C" int seq_logprobs(const SeqLogprobs *p, void *stream) {
    const int rc = seq::check_logprobs(p);
    if (rc != CO_OK) return rc;
    if (p->tokens == 0) return CO_OK;
    if (!p->logits || !p->ids || !p->logp || !p->entropy || (p->top && (!p->top_logp || !p->top_ids)))
        return CO_ERR_NULLARG;
    const int64_t bytes = seq_logprobs_workspace(p);
    if (bytes && !p->workspace) return CO_ERR_NULLARG;
    if (p->workspace_bytes < bytes || ((uintptr_t)p->workspace & 15)) return CO_ERR_DATA;
    hipStream_t s = (hipStream_t)stream;
    switch (p->dtype) {
        case SEQ_FP32: seq::launch_logprobs<float>(*p, s); break;
        case SEQ_BF16: seq::launch_logprobs<__bf16>(*p, s); break;
        default: seq::launch_logprobs<_Float16>(*p, s); break;
    }
    return seq::launch_status();
}

extern "C" int seq_logprobs_grad(const SeqLogprobsGrad *p, void *stream) {
    if (!p || p->struct_size != (int32_t)sizeof(SeqLogprobsGrad)) return CO_ERR_NULLARG;
    const int rc = seq::check_logprobs(p->tokens, p->vocab, p->dtype, p->temperature);
    if (rc != CO_OK) return rc;
    if (p->tokens == 0) return CO_OK;
    if (!p->logits || !p->ids || !p->stats || !p->entropy || !p->dlogits) return CO_ERR_NULLARG;
    hipStream_t s = (hipStream_t)stream;
    switch (p->dtype) {
        case SEQ_FP32: seq::launch_grad<float>(*p, s); break;
        case SEQ_BF16: seq::launch_grad<__bf16>(*p, s); break;
        default: seq::launch_grad<_Float16>(*p, s); break;
    }
    return seq::launch_status();
}
