// seq_attention_grad.hip -- gradient of causal attention over packed sequences
// (include/cusr_seq.h, seq_attention_grad).
//
// With P = exp(S - lse) formed again from q, k and lse, delta = sum(do * o) per
// row and dP = do V^T:  dS = P (dP - delta),  dQ = scale dS K,
// dK = scale dS^T Q,  dV = P^T do. One kernel owns rows and sums over keys
// (dQ, delta), one owns keys and sums over rows (dK, dV, all heads of the
// group): every sum has one owner and one order, so no atomics.
#include "seq_hidden.h"

namespace seq {

struct AttnGrad : Attn {
    SeqAttentionGrad g;
    // lse in powers of two [hq, tq] and +inf, then delta [hq, tq] and 0
    float *stat;
};

template <typename T>
__device__ inline float dot_row(const uint4v *x, const uint4v *y, int n) {
    float s = 0.0f;
    for (int c = 0; c < n; c++)
#pragma unroll
        for (int j = 0; j < 4; j++)
            s += T::lo(x[c][j]) * T::lo(y[c][j]) + T::hi(x[c][j]) * T::hi(y[c][j]);
    return s;
}

// The rows' statistics for the kernel that owns keys; one thread adds the
// values that stand for rows beyond a tile's last.
__device__ inline void put_stat(const AttnGrad &a, int64_t at, float lse2, float delta, bool ok) {
    const int64_t n = a.tq * a.hq;
    if (ok && (threadIdx.x & 63) < 32) {
        a.stat[at] = lse2;
        a.stat[n + 1 + at] = delta;
        if (at == 0) {
            a.stat[n] = __builtin_inff();
            a.stat[2 * n + 1] = 0.0f;
        }
    }
}

__device__ inline uint32_t pinned(int64_t x) {
    uint32_t y = (uint32_t)x;
    asm("" : "+s"(y));
    return y;
}

// A key head's rows and keys, for what seq_hidden.h does with them.
template <typename T> struct HeadRows {
    const AttnGrad &a;
    const Place &p;
    int hk;
    __device__ int64_t t(int row) const { return p.q0 + row / a.G; }
    __device__ int head(int row) const { return hk * a.G + row % a.G; }
    __device__ const uint16_t *q(int row) const {
        return (const uint16_t *)a.q + t(row) * a.q_row + head(row) * a.q_head;
    }
    __device__ const uint16_t *d_o(int row) const {
        return (const uint16_t *)a.g.d_o + t(row) * a.g.do_row + head(row) * a.g.do_head;
    }
    __device__ const uint16_t *k(int key) const {
        return (const uint16_t *)a.k + (p.k0 + key) * a.k_row + hk * a.k_head;
    }
    __device__ const uint16_t *v(int key) const {
        return (const uint16_t *)a.v + (p.k0 + key) * a.v_row + hk * a.v_head;
    }
    __device__ float lse2(int row) const { return a.lse[head(row) * a.tq + t(row)] * kLog2e; }
    // from o and what rounding took from it; short sequences keep only o: within the
    // bounds that follow from its rounding
    __device__ float delta(int row) const {
        const uint16_t *y = d_o(row);
        float s = dot<T>((const uint16_t *)a.o + t(row) * a.o_row + head(row) * a.o_head, y, a.d);
        if (keeps_low(a, p.lq * a.G))
            s += dot<T>((const uint16_t *)a.o_low + (t(row) * a.hq + head(row)) * a.d, y, a.d);
        return s;
    }
    __device__ float probability(int row, int key, float lse2) const {
        return exp2_fast(__builtin_fmaf(dot<T>(q(row), k(key), a.d), a.c, -lse2));
    }
    __device__ float dp(int row, int key) const { return dot<T>(d_o(row), v(key), a.d); }
};

// dq of rows first + r, for the r of `bad`, where a hidden key reached them.
template <typename T>
__device__ inline void mend_rows(const AttnGrad &a, const Place &p, int hk, int first,
                                 uint32_t bad) {
    const HeadRows<T> of{a, p, hk};
    auto k = [&](int key) { return of.k(key); };
    const int rows = p.lq * a.G;
    wait_copies<0>();                // stores on their way come first
    for (; bad && first + __builtin_ctz(bad) < rows; bad &= bad - 1) {
        const int row = first + __builtin_ctz(bad);
        const int end = row / a.G + p.lk - p.lq + 1;             // beyond its last key
        float sum[2] = {0.0f, 0.0f}, lse2 = 0.0f, delta = 0.0f;
        if (end > 0) {
            lse2 = of.lse2(row);
            delta = of.delta(row);
            if (!__all(finite(lse2) && finite(delta))) continue;     // not finite by what it sees
        }
        if (!hidden_cause<T>(k, a.d, max(end, 0), min(end + kReach, p.lk), end > 0 ? end - 1 : -1))
            continue;
        add_seen<T>(k, a.d, 0, end, [&](int key) {
            return rounded<T>(of.probability(row, key, lse2) * (of.dp(row, key) - delta));
        }, sum);
        typename T::elem *to = (typename T::elem *)a.g.dq + of.t(row) * a.g.dq_row +
                               of.head(row) * a.g.dq_head;
        each_column(a.d, [&](int e, int col) { to[col] = (typename T::elem)(sum[e] * a.scale); });
    }
}

// dk and dv of keys first + r, where a row that does not see them reached them. Tiles of
// rows begin less than a tile of keys and a tile of rows before the first that does.
template <typename T>
__device__ inline void mend_keys(const AttnGrad &a, const Place &p, int hk, int first,
                                 uint32_t bad) {
    const HeadRows<T> of{a, p, hk};
    auto q = [&](int row) { return of.q(row); };
    auto d_o = [&](int row) { return of.d_o(row); };
    const int rows = p.lq * a.G;
    if (rows == 0 || !__all(finite(of.lse2(rows - 1)))) return;  // the last sees every key
    wait_copies<0>();
    for (; bad && first + __builtin_ctz(bad) < p.lk; bad &= bad - 1) {
        const int key = first + __builtin_ctz(bad);
        if (key < 0) continue;
        const int start = max(key - p.lk + p.lq, 0) * a.G;       // the first row that sees it
        const int before = max(start - 31 * a.G - 31, 0);
        if (!hidden_cause<T>(q, a.d, before, start, -1) &&
            !hidden_cause<T>(d_o, a.d, before, start, rows - 1))
            continue;
        float dk[2] = {0.0f, 0.0f}, dv[2] = {0.0f, 0.0f};
        add_seen<T>(d_o, a.d, start, rows, [&](int row) {
            return rounded<T>(of.probability(row, key, of.lse2(row)));
        }, dv);
        add_seen<T>(q, a.d, start, rows, [&](int row) {
            return rounded<T>(of.probability(row, key, of.lse2(row)) *
                              (of.dp(row, key) - of.delta(row)));
        }, dk);
        typedef typename T::elem E;
        E *to_k = (E *)a.g.dk + (p.k0 + key) * a.g.dk_row + hk * a.g.dk_head;
        E *to_v = (E *)a.g.dv + (p.k0 + key) * a.g.dv_row + hk * a.g.dv_head;
        each_column(a.d, [&](int e, int col) {
            to_k[col] = (E)(dk[e] * a.scale);
            to_v[col] = (E)dv[e];
        });
    }
}

// Called by the long kernels: of rows, or of keys.
template <typename T, bool KEYS>
__device__ __attribute__((noinline)) void mend_long(Arguments<AttnGrad> args, Place place, int hk,
                                                    int first, uint32_t bad) {
    const AttnGrad &a = *(const AttnGrad *)uniform(args);
    const Place p = uniform(place);
    if (KEYS) mend_keys<T>(a, p, uniform(hk), uniform(first), uniform((int)bad));
    else mend_rows<T>(a, p, uniform(hk), uniform(first), uniform((int)bad));
}
// Called by the short kernel: all of a wave's rows and keys, the wave's number `item`.
template <typename T>
__device__ __attribute__((noinline)) void mend_short(Arguments<AttnGrad> args, int item) {
    const AttnGrad &a = *(const AttnGrad *)uniform(args);
    item = uniform(item);
    const int slot = item / a.hkv, hk = item - slot * a.hkv;
    const Found f = find_sequence(a.cu_q, a.n_seq, a.tq, a.G, kShortRows, slot);
    const Place p = place_of(a, f.b, f.start, f.end);
    const int mine = slot - slot_of(f.start, a.G, kShortRows, f.b);
    const int shares = max((p.lq * a.G + kShortRows - 1) / kShortRows, 1);
    const int s0 = a.cu_k == a.cu_q && a.tk == a.tq ? f.start : offset_at(a.cu_k, f.b, a.tk);
#pragma unroll 1
    for (int tile = mine * 4; tile < mine * 4 + 4; tile++) mend_rows<T>(a, p, hk, tile * 32, ~0u);
#pragma unroll 1
    for (int first = mine * 32 + s0 - p.k0; first < p.lk; first += shares * 32)
        mend_keys<T>(a, p, hk, first, ~0u);
}

// Short sequences: a wave owns up to 128 rows of a sequence and key head, and
// every so many tiles of 32 of its keys; most have a sequence to themselves and
// need no statistics from another kernel. First the rows: delta = sum of P dP,
// which needs no o, then dQ^T = sum over keys of K^T dS^T, from S^T. Then the
// keys: dV^T = dO^T P and dK^T = Q^T dS, from S formed the other way round: the
// same tiles are the left or the right operand. What is read passes through LDS,
// past the registers. What bounds it is the chain of loads from the slot to the
// rows beside vector instructions (half the time) with two waves a SIMD, hence
// the path of its own for up to 64 rows and keys, in which few loads wait for
// others and P and dS are formed once: 8,192 sequences of 3 to 63, 8 heads of 64,
// take 0.47 ms (4.1 TB/s), with P and dS formed twice 0.58, on the general path 0.73.
// Its part of a wave, in LDS: four tiles, and a fifth for P and dS of a pair of tiles,
// for results on their way out, or for rows' statistics: lse, delta, last visible key.
// Returns whether all sums are finite.
template <int DP> constexpr int kShortLds = 4 * 32 * Tile<DP>::stride +
                                            (DP < 64 ? 64 * 32 : 32 * Tile<DP>::stride);
template <typename T, int DP>
__device__ inline bool grad_short(const AttnGrad &a, int slots, uint16_t *lds_wave) {
    constexpr int C = DP / 16, S = Tile<DP>::stride;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, h = lane >> 5;
    uint16_t (*lds)[32 * S] = (uint16_t(*)[32 * S])lds_wave, *fifth = lds[4];
    float odd = 0.0f;
    const uint32_t lds_at = lds_address(lds[0]);
    float *lses = (float *)fifth, *deltas = lses + kShortRows;
    int *lims = (int *)(deltas + kShortRows);
    const int item = block_number() * 4 + wave;
    const int slot = item / a.hkv, hk = item - slot * a.hkv;
    if (slot >= slots) return true;
    const Found f = find_sequence(a.cu_q, a.n_seq, a.tq, a.G, kShortRows, slot);
    const Place p = place_of(a, f.b, f.start, f.end);
    const int rows = p.lq * a.G, tiles = (rows + 31) / 32;
    const int mine = slot - slot_of(f.start, a.G, kShortRows, f.b);
    const int shares = max((rows + kShortRows - 1) / kShortRows, 1);
    if (mine < 0 || mine >= shares) return true;
    // the key rows of the segment, of which p.lk are keys
    const bool same = a.cu_k == a.cu_q && a.tk == a.tq;
    const int s0 = same ? f.start : offset_at(a.cu_k, f.b, a.tk);
    const int s1 = same ? f.end : (f.b >= a.n_seq ? (int)a.tk
                                                  : max(offset_at(a.cu_k, f.b + 1, a.tk), s0));
    const int shift = p.lk - p.lq;
    const float inv = 1.0f / (float)a.G;
    const uint16_t *kp = (const uint16_t *)a.k + p.k0 * a.k_row + hk * a.k_head;
    const uint16_t *vp = (const uint16_t *)a.v + p.k0 * a.v_row + hk * a.v_head;
    const uint16_t *qp = (const uint16_t *)a.q + p.q0 * a.q_row + hk * a.G * a.q_head;
    uint16_t *dqp = (uint16_t *)a.g.dq + p.q0 * a.g.dq_row + hk * a.G * a.g.dq_head;
    const uint16_t *dop = (const uint16_t *)a.g.d_o + p.q0 * a.g.do_row + hk * a.G * a.g.do_head;

    // Strides in 32 bits, each in a register of its own: as parts of the arguments they
    // would be laid by and fetched 16 at a time.
    const uint32_t n_q_row = pinned(a.q_row), n_q_head = pinned(a.q_head), n_k_row = pinned(a.k_row),
                   n_v_row = pinned(a.v_row), n_do_row = pinned(a.g.do_row),
                   n_do_head = pinned(a.g.do_head), n_dq_row = pinned(a.g.dq_row),
                   n_dq_head = pinned(a.g.dq_head), n_dk_row = pinned(a.g.dk_row),
                   n_dv_row = pinned(a.g.dv_row);
    auto step = [](auto as, int64_t wide, uint32_t near) {
        if constexpr (sizeof(as) == 4) return (int64_t)near;
        else return wide;
    };
    // tiles to LDS tiles, past the registers. Beyond the last row or key, the last
    // again: it is masked, by its last visible key -1
    auto row_at = [&](auto as, int i, int64_t step, int64_t head) {
        typedef decltype(as) I;
        const int row = min(i, rows - 1), qi = quotient<I>(row, a.G, inv);
        return times<I>(qi, step) + times<I>(row - qi * a.G, head);
    };
    auto copy_q = [&](auto as, int tile, int to) {
        copy_tile<DP>(qp, a.d, lds_at + to * 64 * S, [&](int i) {
            return row_at(as, tile * 32 + i, step(as, a.q_row, n_q_row), step(as, a.q_head, n_q_head));
        });
    };
    auto copy_do = [&](auto as, int tile, int to) {
        copy_tile<DP>(dop, a.d, lds_at + to * 64 * S, [&](int i) {
            return row_at(as, tile * 32 + i, step(as, a.g.do_row, n_do_row),
                          step(as, a.g.do_head, n_do_head));
        });
    };
    auto copy_keys = [&](auto as, int k0, int end, int tk, int tv) {
        typedef decltype(as) I;
        copy_tile<DP>(kp, a.d, lds_at + tk * 64 * S,
                      [&](int i) { return times<I>(min(k0 + i, end - 1), step(as, a.k_row, n_k_row)); });
        copy_tile<DP>(vp, a.d, lds_at + tv * 64 * S,
                      [&](int i) { return times<I>(min(k0 + i, end - 1), step(as, a.v_row, n_v_row)); });
    };
    // keys that a tile of rows sees
    auto seen_by = [&](int tile) {
        return divide(min(tile * 32 + 31, rows - 1), a.G, inv) + shift + 1;
    };

    // a tile of rows: this lane's, and their sums
    uint4v q[C], dO[C];
    int lim;
    float lse2, delta;
    float16v dq[DP / 32];
    auto begin_rows = [&](int tile, bool load) {
        const int row = tile * 32 + (lane & 31);
        const bool ok = row < rows;
        const int qi = divide(ok ? row : 0, a.G, inv), g = ok ? row - qi * a.G : 0;
        lim = ok ? qi + shift : -1;
        if (load) {
            load_row<DP>(q, qp, qi * a.q_row + g * a.q_head, a.d, ok);
            load_row<DP>(dO, dop, qi * a.g.do_row + g * a.g.do_head, a.d, ok);
        }
        lse2 = ok ? a.lse[(hk * a.G + g) * a.tq + p.q0 + qi] * kLog2e : 0.0f;
        delta = 0.0f;
#pragma unroll
        for (int dt = 0; dt < DP / 32; dt++) dq[dt] = float16v{};
    };
    auto end_rows = [&](auto as, int tile, uint16_t *free) {
        watch<DP>(odd, dq);
        store_tile<T, DP>(dqp, dq, a.scale, a.d, rows - tile * 32, free, [&](int i) {
            return row_at(as, tile * 32 + i, step(as, a.g.dq_row, n_dq_row),
                          step(as, a.g.dq_head, n_dq_head));
        });
    };
    auto products = [&](int k0, int tk, int tv, float16v &s, float16v &dp) {
        s = dp = float16v{};
#pragma unroll
        for (int c = 0; c < C; c++) s = T::mfma(Tile<DP>::row(lds[tk], 0, c), q[c], s);
#pragma unroll
        for (int c = 0; c < C; c++) dp = T::mfma(Tile<DP>::row(lds[tv], 0, c), dO[c], dp);
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int key = k0 + 8 * (i / 4) + 4 * h + i % 4;
            s[i] = key <= lim ? exp2_fast(__builtin_fmaf(s[i], a.c, -lse2)) : 0.0f;
            dp[i] = key <= lim ? s[i] * dp[i] : 0.0f;
        }
    };
    // dS in the type, and dQ's sum
    auto add = [&](int tk, const float16v &s, const float16v &dp, uint4v (&ds)[2]) {
#pragma unroll
        for (int kc = 0; kc < 2; kc++) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int i = 8 * kc + 2 * j;
                ds[kc][j] = T::pack(dp[i] - s[i] * delta, dp[i + 1] - s[i + 1] * delta);
            }
#pragma unroll
            for (int dt = 0; dt < DP / 32; dt++)
                dq[dt] = T::mfma(Tile<DP>::transposed(lds[tk], kc * 16, dt), ds[kc], dq[dt]);
        }
    };

    // a tile of keys: this lane's, and their sums
    uint4v k[C], v[C];
    int key;
    float16v dk[DP / 32], dv[DP / 32];
    auto begin_keys = [&](int kt) {          // with zeros
        key = kt * 32 + s0 - p.k0 + (lane & 31);
#pragma unroll
        for (int dt = 0; dt < DP / 32; dt++) dk[dt] = dv[dt] = float16v{};
    };
    auto load_keys = [&](int kt) {
        const int at = kt * 32 + s0 - p.k0 + (lane & 31);
        const bool live = s0 + kt * 32 + (lane & 31) < s1 && at >= 0 && at < p.lk;
        load_row<DP>(k, kp, at * a.k_row, a.d, live);
        load_row<DP>(v, vp, at * a.v_row, a.d, live);
    };
    // adds the rows in the LDS tiles q and dO, statistics from `at` on
    auto add_rows = [&](const uint16_t *tq, const uint16_t *to, int at) {
        float16v s = {}, dp = {};
#pragma unroll
        for (int c = 0; c < C; c++) s = T::mfma(Tile<DP>::row(tq, 0, c), k[c], s);
#pragma unroll
        for (int c = 0; c < C; c++) dp = T::mfma(Tile<DP>::row(to, 0, c), v[c], dp);
        uint32_t pp[8], pd[8];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float4v l4 = *(const float4v *)(lses + at + 8 * i + 4 * h);
            const float4v e4 = *(const float4v *)(deltas + at + 8 * i + 4 * h);
            const uint4v m4 = *(const uint4v *)(lims + at + 8 * i + 4 * h);
            float pr[4], ds[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const bool see = key <= (int)m4[j];
                pr[j] = see ? exp2_fast(__builtin_fmaf(s[4 * i + j], a.c, -l4[j])) : 0.0f;
                ds[j] = see ? pr[j] * (dp[4 * i + j] - e4[j]) : 0.0f;
            }
            pp[2 * i] = T::pack(pr[0], pr[1]);
            pp[2 * i + 1] = T::pack(pr[2], pr[3]);
            pd[2 * i] = T::pack(ds[0], ds[1]);
            pd[2 * i + 1] = T::pack(ds[2], ds[3]);
        }
#pragma unroll
        for (int kc = 0; kc < 2; kc++) {
            const uint4v pb = {pp[4 * kc], pp[4 * kc + 1], pp[4 * kc + 2], pp[4 * kc + 3]};
            const uint4v db = {pd[4 * kc], pd[4 * kc + 1], pd[4 * kc + 2], pd[4 * kc + 3]};
#pragma unroll
            for (int dt = 0; dt < DP / 32; dt++) {
                dv[dt] = T::mfma(Tile<DP>::transposed(to, kc * 16, dt), pb, dv[dt]);
                dk[dt] = T::mfma(Tile<DP>::transposed(tq, kc * 16, dt), db, dk[dt]);
            }
        }
    };
    uint16_t *dkp = (uint16_t *)a.g.dk + s0 * a.g.dk_row + hk * a.g.dk_head;
    uint16_t *dvp = (uint16_t *)a.g.dv + s0 * a.g.dv_row + hk * a.g.dv_head;
    auto end_keys = [&](auto as, int kt, uint16_t *free) {
        typedef decltype(as) I;
        const int n = s1 - s0 - kt * 32;
        if (n <= (lane & 31) || key < 0 || key >= p.lk)      // a row that is no key's: zeros
#pragma unroll
            for (int dt = 0; dt < DP / 32; dt++) dk[dt] = dv[dt] = float16v{};
        // a row with a value that is not finite has such a dq itself, if it sees a key
        // and is this wave's
        if (shares > 1 || shift < 0) {
            watch<DP>(odd, dk);
            watch<DP>(odd, dv);
        }
        store_tile<T, DP>(dkp, dk, a.scale, a.d, n, free,
                          [&](int i) { return times<I>(kt * 32 + i, step(as, a.g.dk_row, n_dk_row)); });
        store_tile<T, DP>(dvp, dv, 1.0f, a.d, n, free,
                          [&](int i) { return times<I>(kt * 32 + i, step(as, a.g.dv_row, n_dv_row)); });
    };

    // Up to 64 rows and keys, the first 32 rows with up to 32 keys: P and dS are formed
    // once and turned round by way of LDS, and each tile comes from memory once or
    // twice. K is in LDS tiles 0 and 1, V in 2 and 3; then the second rows, and at
    // last the first, in 1 and 3.
    if (a.near && rows > 0 && rows <= 64 && s1 - s0 <= 64 && s0 == p.k0 && seen_by(0) > 0 &&
        seen_by(0) <= 32) {
        const uint32_t as = 0;
        // this lane's row of an LDS tile, zero beyond d, where the tile repeats columns
        auto row_of = [&](uint4v *f, int t) {
#pragma unroll
            for (int c = 0; c < C; c++) {
                f[c] = Tile<DP>::row(lds[t], 0, c);
                if (a.d < DP && c * 16 + h * 8 >= a.d) f[c] = uint4v{0, 0, 0, 0};
            }
        };
        auto pack = [&](const float16v &s, uint4v (&ps)[2]) {
#pragma unroll
            for (int i = 0; i < 8; i++) ps[i / 4][i % 4] = T::pack(s[2 * i], s[2 * i + 1]);
        };
        // dK's and dV's sums, with the rows' tiles in 1 and 3
        auto add_block = [&](const uint4v (&ps)[2], const uint4v (&ds)[2]) {
            typedef Tile<32> Block;
            uint16_t *pt = fifth, *dt_ = fifth + 32 * 32;
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const int at = Block::at(lane & 31, g) + 4 * h;
                const uint2v x = {ps[g / 2][g % 2 * 2], ps[g / 2][g % 2 * 2 + 1]};
                const uint2v y = {ds[g / 2][g % 2 * 2], ds[g / 2][g % 2 * 2 + 1]};
                *(uint2v *)(pt + at) = x;
                *(uint2v *)(dt_ + at) = y;
            }
            wave_sync();
#pragma unroll
            for (int kc = 0; kc < 2; kc++) {
                const uint4v pb = Block::transposed(pt, kc * 16, 0);
                const uint4v db = Block::transposed(dt_, kc * 16, 0);
#pragma unroll
                for (int dt = 0; dt < DP / 32; dt++) {
                    dv[dt] = T::mfma(Tile<DP>::transposed(lds[3], kc * 16, dt), pb, dv[dt]);
                    dk[dt] = T::mfma(Tile<DP>::transposed(lds[1], kc * 16, dt), db, dk[dt]);
                }
            }
            wave_sync();
        };
        const int end = seen_by(tiles - 1);
        const bool second = s1 - s0 > 32;    // a second tile of keys
        float16v s, dp;
        uint4v ps[2], ds[2];
        copy_keys(as, 0, end, 0, 2);
        if (tiles == 2) {
            if (end > 32) copy_keys(as, 32, end, 1, 3);
            begin_rows(1, true);
            wait_copies<0>();
            products(0, 0, 2, s, dp);
            float16v s1, dp1;
            uint4v ps1[2], ds1[2];
            if (end > 32) products(32, 1, 3, s1, dp1);
            else s1 = dp1 = float16v{};
#pragma unroll
            for (int i = 0; i < 16; i++) delta += dp[i] + dp1[i];
            delta = add_halves(delta);
            pack(s, ps);
            pack(s1, ps1);
            add(0, s, dp, ds);
            if (end > 32) add(1, s1, dp1, ds1);
            copy_q(as, 1, 1);
            copy_do(as, 1, 3);
            end_rows(as, 1, fifth);
            wait_copies<0>();
            if (second) {
                begin_keys(1);
                if (end > 32) add_block(ps1, ds1);
                end_keys(as, 1, fifth);
            }
            begin_keys(0);
            add_block(ps, ds);
        } else {
            if (second) {
                begin_keys(1);
                end_keys(as, 1, fifth);
            }
            begin_keys(0);
        }
        copy_q(as, 0, 1);
        copy_do(as, 0, 3);
        begin_rows(0, false);
        wait_copies<0>();
        row_of(q, 1);
        row_of(dO, 3);
        products(0, 0, 2, s, dp);
#pragma unroll
        for (int i = 0; i < 16; i++) delta += dp[i];
        delta = add_halves(delta);
        pack(s, ps);
        add(0, s, dp, ds);
        add_block(ps, ds);
        end_rows(as, 0, fifth);
        end_keys(as, 0, fifth);
        return finite(odd);
    }

    // Any other: the first row tile that sees a key of tile kt; the keys' part, kt by
    // kt and tile by tile, has its next tile on the way while it works on one, and
    // its first from here on
    auto first_tile = [&](int kt) {
        const int key0 = kt * 32 + s0 - p.k0;
        return kt * 32 < s1 - s0 && key0 < p.lk ? max(key0 - shift, 0) * a.G / 32 : tiles;
    };
    const int64_t as = 0;
    int next = first_tile(mine);
    int pair = 2;                            // the LDS tiles that the keys' part reads next
    if (next < tiles) copy_q(as, next, pair), copy_do(as, next, pair + 1);

    for (int tile = mine * 4; tile < mine * 4 + 4 && tile < tiles; tile++) {
        const int end = seen_by(tile);
        if (end > 0) copy_keys(as, 0, end, 0, 1);
        begin_rows(tile, true);
        float16v s, dp;
        for (int k0 = 0; k0 < end; k0 += 32) {
            if (k0) copy_keys(as, k0, end, 0, 1);
            wait_copies<0>();
            products(k0, 0, 1, s, dp);
#pragma unroll
            for (int i = 0; i < 16; i++) delta += dp[i];
        }
        delta = add_halves(delta);
        uint4v ds[2];
        if (end > 0 && end <= 32) {
            add(0, s, dp, ds);
        } else {                             // once more, with delta
            for (int k0 = 0; k0 < end; k0 += 32) {
                copy_keys(as, k0, end, 0, 1);
                wait_copies<0>();
                products(k0, 0, 1, s, dp);
                add(0, s, dp, ds);
            }
        }
        end_rows(as, tile, lds[0]);
        if (h == 0) {
            lses[(tile & 3) * 32 + lane] = lse2;
            deltas[(tile & 3) * 32 + lane] = delta;
            lims[(tile & 3) * 32 + lane] = lim;
        }
    }

    for (int kt = mine; kt * 32 < s1 - s0; kt += shares) {
        begin_keys(kt);
        if (kt * 32 + s0 - p.k0 < p.lk) {
            load_keys(kt);
            for (int tile = next; tile < tiles; tile++) {
                int at = (tile & 3) * 32;
                if (shares > 1) {
                    // the rows may be another wave's: delta from o and what its type
                    // rounded away, which a sequence of so many rows keeps
                    const int row = tile * 32 + (lane & 31);
                    const bool ok = row < rows;
                    const int qi = divide(ok ? row : 0, a.G, inv), g = ok ? row - qi * a.G : 0;
                    const int64_t t = p.q0 + qi, head = hk * a.G + g;
                    uint4v x[C], y[C];
                    load_row<DP>(x, a.o, t * a.o_row + head * a.o_head, a.d, ok);
                    load_row<DP>(y, dop, qi * a.g.do_row + g * a.g.do_head, a.d, ok);
                    float delta = dot_row<T>(x, y, C);
                    if (a.o_low) {
                        load_row<DP>(x, a.o_low, (t * a.hq + head) * a.d, a.d, ok);
                        delta += dot_row<T>(x, y, C);
                    }
                    delta = add_halves(delta);
                    at = 0;
                    wave_sync();
                    if (h == 0) {
                        lses[lane] = ok ? a.lse[head * a.tq + t] * kLog2e : 0.0f;
                        deltas[lane] = delta;
                        lims[lane] = ok ? qi + shift : -1;
                    }
                }
                wait_copies<0>();
                const uint16_t *tq = lds[pair], *to = lds[pair + 1];
                pair ^= 2;
                next = tile + 1 < tiles ? tile + 1 : first_tile(kt + shares);
                if (next < tiles) copy_q(as, next, pair), copy_do(as, next, pair + 1);
                add_rows(tq, to, at);
            }
        }
        end_keys(as, kt, lds[pair ^ 2]);     // the next tile is on its way to the others
    }
    return finite(odd);
}

template <typename T, int DP>
__global__ __launch_bounds__(256, DP <= 64 ? 2 : 1)
void attn_grad_short(AttnGrad a, int slots) {
    __shared__ __align__(256) uint16_t lds[4][kShortLds<DP>];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool plain = grad_short<T, DP>(a, slots, lds[wave]);
    if (__builtin_expect(__any(!plain), 0)) mend_short<T>(arguments<AttnGrad>(), block_number() * 4 + wave);
}

// Long sequences, rows: a block of four waves owns 128 rows of one key head; keys
// and values pass through LDS 64 at a time, as in the forward. No unit is full: the
// matrix cores are busy 51 % of the time, the vector instructions 31 %, and the waves
// wait 47 % of theirs, for tiles and for each other: five sequences of 700 to 4,801, 32
// heads of 128 over 8, 0.50 ms.
template <typename T, int DP, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void attn_grad_q_tiles(AttnGrad a, int slots) {
    typedef KeyTiles<DP, 64, WAVES> Keys;
    constexpr int KB = 64, ROWS = WAVES * 32, STRIDE = Keys::STRIDE;
    __shared__ __align__(256) unsigned char lds[2 * Keys::BYTES];
    const int lane = threadIdx.x & 63, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int item = block_number(), slot = item / a.hkv, hk = item - slot * a.hkv;
    if (slot >= slots) return;
    const Found f = find_sequence(a.cu_q, a.n_seq, a.tq, a.G, ROWS, slot);
    const int b = f.b;
    const Place p = place_of(a, b, f.start, f.end);
    const int rows = p.lq * a.G;
    const int tile = (rows + ROWS - 1) / ROWS - 1 - (slot - slot_of(p.q0, a.G, ROWS, b));
    if (tile < 0 || tile * ROWS >= rows) return;
    const int row = tile * ROWS + wave * 32 + (lane & 31);
    const bool ok = row < rows;
    const int qi = ok ? row / a.G : 0, g = ok ? row % a.G : 0;
    const int head = hk * a.G + g;
    const int lim = ok ? qi + p.lk - p.lq : -1;
    const int64_t t = p.q0 + qi;
    uint4v q[DP / 16], dO[DP / 16];
    float delta, lse2;
    load_row<DP>(dO, a.g.d_o, t * a.g.do_row + head * a.g.do_head, a.d, ok);
    load_row<DP>(q, a.o, t * a.o_row + head * a.o_head, a.d, ok);
    delta = dot_row<T>(q, dO, DP / 16);
    if (a.o_low) {
        load_row<DP>(q, a.o_low, ((int64_t)t * a.hq + head) * a.d, a.d, ok);
        delta += dot_row<T>(q, dO, DP / 16);
    }
    delta = add_halves(delta);
    lse2 = ok ? a.lse[head * a.tq + t] * kLog2e : 0.0f;
    put_stat(a, head * a.tq + t, lse2, delta, ok);
    load_row<DP>(q, a.q, t * a.q_row + head * a.q_head, a.d, ok);
    auto seen_by = [&](int r) {
        return min(r, rows - 1) / a.G + p.lk - p.lq + 1;
    };
    const int keys = seen_by(tile * ROWS + ROWS - 1);
    const int w0 = tile * ROWS + wave * 32;
    const int wave_keys = w0 < rows ? seen_by(w0 + 31) : 0;
    const int all_keys = w0 + 31 < rows ? seen_by(w0) : 0;
    const Keys tiles(a, p, hk, keys);
    landed(q);
    landed(dO);
    const uint32_t lds0 = lds_address(lds);
    const typename Tile<DP>::Rows kr = Tile<DP>::rows(lds0);
    const typename Tile<DP>::Columns kc_ = Tile<DP>::columns(lds0);

    float16v dq[DP / 32] = {};
    auto work = [&](auto buf, int k0) {
        constexpr uint32_t B = decltype(buf)::value * Keys::BYTES, V = B + Keys::BYTES / 2;
        wait_copies<0>();
        block_barrier();
        if (k0 + KB < keys) tiles.copy(k0 + KB, lds0 + (Keys::BYTES - B));
        if (k0 >= wave_keys) return;
        const bool edge = k0 + KB > all_keys;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            float16v s = {}, dp = {};
#pragma unroll
            for (int c = 0; c < DP / 16; c++) {
                s = T::mfma(Tile<DP>::row(kr.c[c], B + u * 32 * STRIDE), q[c], s);
                dp = T::mfma(Tile<DP>::row(kr.c[c], V + u * 32 * STRIDE), dO[c], dp);
            }
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const float pr = exp2_fast(__builtin_fmaf(s[r], a.c, -lse2));
                dp[r] = pr * (dp[r] - delta);
            }
            if (edge)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (k0 + u * 32 + 8 * (r / 4) + 4 * h + r % 4 > lim) dp[r] = 0.0f;
#pragma unroll
            for (int kc = 0; kc < 2; kc++) {
                uint4v pb;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    pb[j] = T::pack(dp[8 * kc + 2 * j], dp[8 * kc + 2 * j + 1]);
#pragma unroll
                for (int dt = 0; dt < DP / 32; dt++)
                    dq[dt] = T::mfma(Tile<DP>::transposed(kc_, dt, B + (u * 32 + kc * 16) * STRIDE),
                                     pb, dq[dt]);
            }
        }
    };
    if (keys > 0) tiles.copy(0, lds0);
    for (int k0 = 0; k0 < keys; k0 += 2 * KB) {
        work(Const<0>{}, k0);
        if (k0 + KB < keys) work(Const<1>{}, k0 + KB);
    }
    const uint32_t bad = not_finite<DP>(dq);
    store_row<T, DP>(a.g.dq, t * a.g.dq_row + head * a.g.dq_head, dq, a.scale, a.d, ok);
    if (__builtin_expect(bad, 0)) mend_long<T, false>(arguments<AttnGrad>(), p, hk, w0, bad);
}

// Long sequences, keys: a block owns KX * 32 keys of one key head, a wave 32 of
// them and every other tile of 32 rows. Both gradients of its keys are in the
// wave's registers; keys and values are in LDS, since with them in registers too
// no operand could be read ahead of its product and each product waited for its
// own. The two waves that share keys add up at the end: with one, a block's
// longest run over the rows would last twice as long, and the longest run is what
// few sequences wait for. Rows pass through LDS 64 at a time, copied there past
// the registers one tile ahead of their use. Rows beyond the last repeat it with
// lse +inf, which makes their P and dS 0. No unit is full: the matrix cores are busy
// 49 % of the time, the vector instructions 28 %, and eight waves wait at one barrier
// for a third of theirs. 32 heads of 128 over 8, five sequences of 700 to 4,801 in 0.74 ms, 0.84 PFLOP/s.
template <typename T, int DP, int KX>
__global__ __launch_bounds__(KX * 128, KX == 4 || DP <= 64 ? 2 : 1) void attn_grad_kv_tiles(AttnGrad a, int slots) {
    constexpr int RB = 64, KEYS = KX * 32, WAVES = KX * 2;
    constexpr int STRIDE = Tile<DP>::stride * 2;        // bytes
    constexpr int PER = RB * STRIDE / 1024;             // copies of 1 KB a tile of q or do
    constexpr int COPIES = 2 * PER / WAVES;                 // of a wave
    constexpr uint32_t TILE = RB * STRIDE, BUF = 2 * TILE + 512;   // q, do, lse and delta
    constexpr uint32_t BYTES = 2 * BUF + 2 * KEYS * STRIDE, SUMS = KX * 2 * 32 * DP * 4;
    __shared__ __align__(256) unsigned char lds[BYTES > SUMS ? BYTES : SUMS];
    const int lane = threadIdx.x & 63, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kx = wave % KX, rx = wave / KX;
    const int item = block_number(), slot = item / a.hkv, hk = item - slot * a.hkv;
    if (slot >= slots) return;
    const Found f = find_sequence(a.cu_k, a.n_seq, a.tk, 1, KEYS, slot);
    const int b = f.b, s0 = f.start, s1 = max(f.end, s0);
    const int tile = slot - slot_of(s0, 1, KEYS, b);
    if (tile < 0 || tile * KEYS >= s1 - s0) return;
    const Place p = b >= a.n_seq ? Place{0, s0, 0, 0} : place_of(a, b);
    const int base = s0 - p.k0;                  // key number of the segment's first row
    const int key0 = tile * KEYS + base;         // of the block
    const int wkey0 = key0 + kx * 32;                   // of the wave
    const int key = wkey0 + (lane & 31);
    const bool live = key >= 0 && key < p.lk;
    float16v dk[DP / 32] = {}, dv[DP / 32] = {};
    // this wave's keys, and 128 rows further their values
    uint16_t *kl = (uint16_t *)(lds + 2 * BUF) + kx * 32 * Tile<DP>::stride;
    {
        uint4v x[DP / 16];               // one of the two waves brings the keys, one the values
        const void *from = rx ? a.v : a.k;
        const int64_t step = rx ? a.v_row : a.k_row, head = rx ? a.v_head : a.k_head;
        load_row<DP>(x, from, (p.k0 + key) * step + hk * head, a.d, live);
#pragma unroll
        for (int c = 0; c < DP / 16; c++)
            *(uint4v *)(kl + rx * KEYS * Tile<DP>::stride + Tile<DP>::at(lane & 31, 2 * c + h)) = x[c];
    }
    const int rows = key0 < p.lk ? p.lq * a.G : 0;
    const int shift = p.lk - p.lq;
    auto first_row = [&](int key) {      // of the tile of 32 with a row that sees the key
        return (int)((int64_t)(key - shift > 0 ? key - shift : 0) * a.G / 32 * 32);
    };
    const int start = first_row(key0);
    const int wave_start = wkey0 < p.lk ? first_row(wkey0) : rows;
    const uint32_t lds0 = lds_address(lds);
    // One tile's copies: this wave's share of q and do, and two waves' statistics.
    // When the group's heads divide 32 rows, and the rows from one copy of the wave to
    // its next (narrow blocks of wide heads: 16), a whole tile's rows lie at the same
    // lane offsets from an address of the wave.
    constexpr int NEXT = PER > WAVES ? WAVES * (1024 / STRIDE) : RB;
    const int row_l = wave % PER * (1024 / STRIDE) + lane * 16 / STRIDE;    // in the tile
    const int ch_l = (lane * 16 % STRIDE / 16) ^ Tile<DP>::swz(row_l);
    const int col_l = ch_l * 8 < a.d ? ch_l * 8 : 0;
    const int64_t q_most = a.q_row * 64 + a.q_head * a.G, o_most = a.g.do_row * 64 + a.g.do_head * a.G;
    const bool plain = 32 % a.G == 0 && NEXT % a.G == 0 && a.q_row >= 0 && a.q_head >= 0 &&
                       a.g.do_row >= 0 && a.g.do_head >= 0 && q_most < 1 << 30 && o_most < 1 << 30;
    const uint32_t q_off = 2 * (uint32_t)(row_l / a.G * a.q_row + row_l % a.G * a.q_head + col_l);
    const uint32_t o_off = 2 * (uint32_t)(row_l / a.G * a.g.do_row + row_l % a.G * a.g.do_head + col_l);
    const uint16_t *q0p = (const uint16_t *)a.q + p.q0 * a.q_row + (int64_t)hk * a.G * a.q_head;
    const uint16_t *o0p = (const uint16_t *)a.g.d_o + p.q0 * a.g.do_row +
                          (int64_t)hk * a.G * a.g.do_head;
    auto copy = [&](int r0, uint32_t buf) {
        if (plain && r0 + RB <= rows) {
#pragma unroll
            for (int x = 0; x < COPIES; x++) {
                const int idx = wave + x * WAVES;
                const int t = (r0 + (idx % PER - wave % PER) * (1024 / STRIDE)) / a.G;
                copy_to_lds16(idx < PER ? q0p + t * a.q_row : o0p + t * a.g.do_row,
                              idx < PER ? q_off : o_off, buf + idx * 1024);
            }
        } else {
#pragma unroll
            for (int x = 0; x < COPIES; x++) {
                const int idx = wave + x * WAVES;
                const int row =
                    min(r0 + (idx % PER - wave % PER) * (1024 / STRIDE) + row_l, rows - 1);
                const int t = row / a.G, g = row % a.G;
                copy_to_lds16((idx < PER ? q0p + t * a.q_row + g * a.q_head
                                         : o0p + t * a.g.do_row + g * a.g.do_head) + col_l,
                              buf + idx * 1024);
            }
        }
        if (kx == 0) {
            const int row = r0 + rx * 32 + (lane & 31);
            const int64_t at = ((int64_t)(hk * a.G) + row % a.G) * a.tq + p.q0 + row / a.G;
            // past the rows: the workspace's +inf and 0
            copy_to_lds4(a.stat + (row < rows ? at : a.tq * a.hq) + h * (a.tq * a.hq + 1),
                         buf + 2 * TILE + rx * 256);
        }
    };
    const typename Tile<DP>::Rows qr = Tile<DP>::rows(lds0 + rx * (TILE / 2));
    const typename Tile<DP>::Columns qc = Tile<DP>::columns(lds0 + rx * (TILE / 2));
    // from a row's address in q to the same row and column of this wave's keys
    const uint32_t to_k = lds_address(kl) - (lds0 + rx * (TILE / 2));
    const uint32_t stat = lds0 + 2 * TILE + rx * 256 + 16 * h;
    auto work = [&](auto buf, int r0) {
        constexpr uint32_t B = decltype(buf)::value * BUF;
        // this tile has landed for every wave, and none reads the one before it
        wait_copies<0>();
        block_barrier();
        if (r0 > start) copy(r0 - RB, lds0 + (BUF - B));
        const int rw = r0 + rx * 32;                     // this wave's rows
        if (rw < wave_start || rw >= rows) return;
        float16v s = {}, dp = {};
        uint32_t kd = to_k;
        asm volatile("" : "+s"(kd));     // the keys' addresses are formed here, not kept
#pragma unroll
        for (int c = 0; c < DP / 16; c++) {
            const uint32_t ka = qr.c[c] + kd;
            s = T::mfma(Tile<DP>::row(qr.c[c], B), Tile<DP>::row(ka, 0), s);
            dp = T::mfma(Tile<DP>::row(qr.c[c], B + TILE), Tile<DP>::row(ka, KEYS * STRIDE), dp);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float4v l4 = __builtin_bit_cast(float4v, Tile<DP>::row(stat, B + 32 * i));
            const float4v e4 = __builtin_bit_cast(float4v, Tile<DP>::row(stat, B + 128 + 32 * i));
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int r = 4 * i + j;
                const float pr = exp2_fast(__builtin_fmaf(s[r], a.c, -l4[j]));
                s[r] = pr;
                dp[r] = pr * (dp[r] - e4[j]);
            }
        }
        // rows before the keys' last do not all see them (and rows that see no
        // key at all have lse -inf)
        if (rw / a.G + shift < wkey0 + 31) {
            const float inv = 1.0f / (float)a.G;
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int lim = divide(rw + 8 * (r / 4) + 4 * h + r % 4, a.G, inv) + shift;
                s[r] = key > lim ? 0.0f : s[r];
                dp[r] = key > lim ? 0.0f : dp[r];
            }
        }
#pragma unroll
        for (int kc = 0; kc < 2; kc++) {
            uint4v pb, db;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                pb[j] = T::pack(s[8 * kc + 2 * j], s[8 * kc + 2 * j + 1]);
                db[j] = T::pack(dp[8 * kc + 2 * j], dp[8 * kc + 2 * j + 1]);
            }
#pragma unroll
            for (int dt = 0; dt < DP / 32; dt++) {
                dv[dt] = T::mfma(Tile<DP>::transposed(qc, dt, B + TILE + kc * 16 * STRIDE), pb, dv[dt]);
                dk[dt] = T::mfma(Tile<DP>::transposed(qc, dt, B + kc * 16 * STRIDE), db, dk[dt]);
            }
        }
    };
    // From the last rows to the first: blocks of one sequence start at rows of
    // their own but end at the same one, so those that run together read the same
    // rows at the same time and find them in the L2.
    const int last = start + (rows - 1 - start) / RB * RB;
    if (start < rows) {
        copy(last, lds0);
        for (int r0 = last; r0 >= start; r0 -= 2 * RB) {
            work(Const<0>{}, r0);
            if (r0 - RB >= start) work(Const<1>{}, r0 - RB);
        }
    }
    // no copy is on its way and no wave reads a tile: the LDS takes the second
    // halves' sums
    wait_copies<0>();
    block_barrier();
    float4v *sums = (float4v *)lds + kx * (2 * DP / 8 * 64) + lane;
    if (rx == 1)
#pragma unroll
        for (int dt = 0; dt < DP / 32; dt++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float4v x = {dk[dt][4 * j], dk[dt][4 * j + 1], dk[dt][4 * j + 2],
                                   dk[dt][4 * j + 3]};
                const float4v y = {dv[dt][4 * j], dv[dt][4 * j + 1], dv[dt][4 * j + 2],
                                   dv[dt][4 * j + 3]};
                sums[(dt * 4 + j) * 64] = x;
                sums[(DP / 8 + dt * 4 + j) * 64] = y;
            }
    __syncthreads();
    if (rx == 1) return;
#pragma unroll
    for (int dt = 0; dt < DP / 32; dt++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float4v x = sums[(dt * 4 + j) * 64], y = sums[(DP / 8 + dt * 4 + j) * 64];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                // a column that is not a key's: zeros
                dk[dt][4 * j + e] = live ? dk[dt][4 * j + e] + x[e] : 0.0f;
                dv[dt][4 * j + e] = live ? dv[dt][4 * j + e] + y[e] : 0.0f;
            }
        }
    const int64_t kr = s0 + tile * KEYS + kx * 32 + (lane & 31);
    const uint32_t bad = not_finite<DP>(dk) | not_finite<DP>(dv);
    store_row<T, DP>(a.g.dk, kr * a.g.dk_row + hk * a.g.dk_head, dk, a.scale, a.d, kr < s1);
    store_row<T, DP>(a.g.dv, kr * a.g.dv_row + hk * a.g.dv_head, dv, 1.0f, a.d, kr < s1);
    if (__builtin_expect(bad, 0)) mend_long<T, true>(arguments<AttnGrad>(), p, hk, wkey0, bad);
}

template <typename T, int DP>
int launch_grad(const AttnGrad &a, hipStream_t s) {
    if (short_sequences(a)) {
        const int slots = slot_of(a.tq, a.G, kShortRows, a.n_seq) + 1;
        const dim3 grid = grid_of((slots * (int64_t)a.hkv + 3) / 4, 256);
        attn_grad_short<T, DP><<<grid, 256, 0, s>>>(a, slots);
        return launch_status();
    }
    if (a.tq) {
        const int slots = slot_of(a.tq, a.G, 128, a.n_seq) + 1;
        const dim3 grid = grid_of((int64_t)slots * a.hkv, 256);
        attn_grad_q_tiles<T, DP, 4><<<grid, 256, 0, s>>>(a, slots);
        if (hipGetLastError() != hipSuccess) return CO_ERR_CUDA;
    }
    // Blocks of 64 keys where 128 would not fill the chip once (one sequence of 2,000,
    // 32 heads of 128 over 8: 263 against 289 us with the rows' part), and for heads up
    // to 64, whose registers and LDS leave room for three a compute unit (16 sequences
    // of 300, 8 heads: 32 against 39 us); wider heads have room for one and need all
    // eight waves (two of 6,000: 2.0 against 2.5 ms).
    const int slots = slot_of(a.tk, 1, 128, a.n_seq) + 1;
    if constexpr (DP > 64) {
        if (slots * a.hkv > 256) {
            const dim3 grid = grid_of((int64_t)slots * a.hkv, 512);
            attn_grad_kv_tiles<T, DP, 4><<<grid, 512, 0, s>>>(a, slots);
            return launch_status();
        }
    }
    const int more = slot_of(a.tk, 1, 64, a.n_seq) + 1;
    const dim3 grid = grid_of((int64_t)more * a.hkv, 256);
    attn_grad_kv_tiles<T, DP, 2><<<grid, 256, 0, s>>>(a, more);
    return launch_status();
}

template <typename T>
int launch_grad_head(const AttnGrad &a, hipStream_t s) {
    switch (padded_head(a.d)) {
        case 32: return launch_grad<T, 32>(a, s);
        case 64: return launch_grad<T, 64>(a, s);
        case 96: return launch_grad<T, 96>(a, s);
        default: return launch_grad<T, 128>(a, s);
    }
}

int check_attention_data(const SeqAttention *a);

}  // namespace seq

extern "C" int64_t seq_attention_grad_workspace(const SeqAttention *a) {
    const int rc = seq::check_attention(a);
    return rc == CO_OK ? 8 * (a->hq * a->tq + 1) : (rc > 0 ? -rc : rc);
}

extern "C" int seq_attention_grad(const SeqAttention *sa, const SeqAttentionGrad *g,
                                  void *stream) {
    int rc = seq::check_attention(sa);
    if (rc != CO_OK) return rc;
    if (!g || g->struct_size != (int32_t)sizeof(SeqAttentionGrad)) return CO_ERR_NULLARG;
    if (sa->tq == 0 && sa->tk == 0) return CO_OK;
    rc = seq::check_attention_data(sa);
    if (rc != CO_OK) return rc;
    if ((sa->tq && (!sa->lse || !g->d_o || !g->dq || !sa->workspace)) ||
        (sa->tk && (!g->dk || !g->dv)))
        return CO_ERR_NULLARG;
    if ((uintptr_t)sa->o_low & 15) return CO_ERR_DATA;
    if (((uintptr_t)g->d_o | (uintptr_t)g->dq | (uintptr_t)g->dk | (uintptr_t)g->dv) & 15)
        return CO_ERR_DATA;
    if ((g->do_row | g->do_head | g->dq_row | g->dq_head | g->dk_row | g->dk_head | g->dv_row |
         g->dv_head) & 7)
        return CO_ERR_DATA;
    if (sa->workspace_bytes < 8 * (sa->hq * sa->tq + 1)) return CO_ERR_DATA;
    seq::AttnGrad a;
    static_cast<seq::Attn &>(a) = seq::make_attn(sa);
    a.g = *g;
    a.near = a.near && seq::near_strides(g->do_row, g->do_head, g->dq_row, g->dq_head) &&
             seq::near_strides(g->dk_row, g->dk_head, g->dv_row, g->dv_head);
    a.stat = (float *)sa->workspace;
    hipStream_t s = (hipStream_t)stream;
    return a.dtype == SEQ_BF16 ? seq::launch_grad_head<seq::Bf16>(a, s)
                               : seq::launch_grad_head<seq::Fp16>(a, s);
}
