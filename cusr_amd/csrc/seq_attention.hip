// seq_attention.hip -- causal attention over packed sequences
// (include/cusr_seq.h, seq_attention).
#include "seq_hidden.h"

namespace seq {

// A row's output from its unscaled sum, and its lse. No visible key: l is 0.
__device__ inline void store_lse(const Attn &a, int t, int head, float m, float l, bool ok) {
    if (a.lse && ok && (threadIdx.x & 63) < 32)
        a.lse[head * a.tq + t] = l == 0.0f ? neg_inf() : m * a.scale + logf(l);
}

template <typename T, int DP>
__device__ inline void store_out(const Attn &a, int t, int head, const float16v *o, float m,
                                 float l, bool ok, bool low) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    store_row<T, DP>(a.o, t * a.o_row + head * a.o_head, o, inv, a.d, ok);
    if (low)
        store_row<T, DP, true>(a.o_low, ((int64_t)t * a.hq + head) * a.d, o, inv, a.d, ok);
    store_lse(a, t, head, m, l, ok);
}

// Outputs of rows first + r of a sequence, for the r of `bad`, and so on every `step` rows
// before `last`, where hidden keys among key0 .. key1-1 reached them; of a chunk of keys,
// its unscaled sums, to sums + row * width, for the maximum and sum at stat + 2 row.
template <typename T>
__device__ __attribute__((noinline)) void mend_out(Arguments<Attn> args, Place place, int hk,
                                                   int first, int last, int step, uint32_t bad,
                                                   int key0, int key1, float *sums,
                                                   const float *stat, int width) {
    const Attn &a = *(const Attn *)uniform(args);
    const Place p = uniform(place);
    hk = uniform(hk), first = uniform(first), last = uniform(last), step = uniform(step);
    bad = uniform((int)bad);
    key0 = uniform(key0), key1 = uniform(key1), width = uniform(width);
    sums = uniform(sums), stat = uniform(stat);
    const int lane = threadIdx.x & 63, rows = p.lq * a.G;
    last = min(last, rows);
    auto k = [&](int j) {
        return (const uint16_t *)a.k + (p.k0 + j) * a.k_row + hk * a.k_head;
    };
    auto v = [&](int j) {
        return (const uint16_t *)a.v + (p.k0 + j) * a.v_row + hk * a.v_head;
    };
    wait_copies<0>();                // stores on their way come first
    uint32_t left = bad;
    for (;; left &= left - 1) {
        while (first < last && !left) first += step, left = bad;
        if (first >= last) return;
        const int row = first + __builtin_ctz(left);
        if (row >= last) return;
        const int qi = row / a.G, head = hk * a.G + row % a.G;
        const int end = min(qi + p.lk - p.lq + 1, key1);         // beyond its last key
        if (!hidden_cause<T>(v, a.d, max(end, key0), min(end + kReach, key1),
                             end > key0 ? end - 1 : -1))
            continue;
        const int64_t t = p.q0 + qi;
        const uint16_t *q = (const uint16_t *)a.q + t * a.q_row + head * a.q_head;
        auto score = [&](int j) { return dot<T>(q, k(j), a.d); };
        float m = neg_inf(), l = 0.0f;
        if (stat) {
            m = stat[2 * row];
            l = stat[2 * row + 1];
        } else {
            for (int j = key0 + lane; j < end; j += 64) m = fmaxf(m, score(j));
            for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
            for (int j = key0 + lane; j < end; j += 64) l += exp2_fast((score(j) - m) * a.c);
            for (int o = 32; o; o >>= 1) l += __shfl_xor(l, o);
        }
        if (!__all(finite(l))) continue;         // not finite by what it sees
        float sum[2] = {0.0f, 0.0f};
        add_seen<T>(v, a.d, key0, end, [&](int j) {
            return rounded<T>(exp2_fast((score(j) - m) * a.c));
        }, sum);
        typedef typename T::elem E;
        each_column(a.d, [&](int e, int col) {
            if (sums) {
                sums[(int64_t)row * width + col] = sum[e];
                return;
            }
            const float x = l == 0.0f ? 0.0f : sum[e] / l;
            ((E *)a.o)[t * a.o_row + head * a.o_head + col] = (E)x;
            if (keeps_low(a, rows))
                ((E *)a.o_low)[(t * a.hq + head) * a.d + col] = (E)(x - (float)(E)x);
        });
    }
}

// A wave's tile of 32 rows over the keys key0 .. key1-1, 32 at a time with a
// running maximum and sum. AHEAD: K comes straight from memory as the left operand,
// V passes through the wave's LDS tile to be transposed, and the next 32 keys are
// loaded to registers while the present ones are worked on. Without it both go to
// LDS past the registers, which leaves room for more waves.
struct Row { int t, head; bool ok; };
template <typename T, int DP, bool AHEAD, typename I>
__device__ inline Row run_rows(const Attn &a, const Place &p, int hk, int tile, int key0, int key1,
                               uint16_t *kt, uint16_t *vt, float16v *o, float &m, float &l) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
    const int rows = p.lq * a.G, row = tile * 32 + (lane & 31);
    const float inv = 1.0f / (float)a.G;
    const bool ok = row < rows;
    const int qi = divide(ok ? row : 0, a.G, inv);
    const int head = hk * a.G + (ok ? row - qi * a.G : 0);
    const int lim = ok ? qi + p.lk - p.lq : -1;          // last visible key
    const int seen = divide(min(tile * 32 + 31, rows - 1), a.G, inv) + p.lk - p.lq + 1;
    const int end = min(key1, seen);
    const uint16_t *kp = (const uint16_t *)a.k + p.k0 * a.k_row + hk * a.k_head;
    const uint16_t *vp = (const uint16_t *)a.v + p.k0 * a.v_row + hk * a.v_head;
    uint4v q[DP / 16], k[DP / 16], v[DP / 16];
    auto load_q = [&] {
        load_row<DP>(q, a.q, (p.q0 + qi) * a.q_row + head * a.q_head, a.d, ok);
    };
    // keys beyond the last repeat it: their scores are masked
    auto fetch = [&](int k0) {
        if (!AHEAD) {
            copy_tile<DP>(kp, a.d, lds_address(kt),
                          [&](int i) { return times<I>(min(k0 + i, end - 1), a.k_row); });
            if (k0 == key0) load_q();
            copy_tile<DP>(vp, a.d, lds_address(vt),
                          [&](int i) { return times<I>(min(k0 + i, end - 1), a.v_row); });
        } else {
            const int r = min(k0 + (lane & 31), end - 1);
            load_row<DP>(k, kp, r * a.k_row, a.d, true);
            load_row<DP>(v, vp, r * a.v_row, a.d, true);
        }
    };
    if (key0 < end) fetch(key0);
    if (AHEAD) load_q();
#pragma unroll
    for (int dt = 0; dt < DP / 32; dt++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[dt][r] = 0.0f;
    m = neg_inf();
    l = 0.0f;
    for (int k0 = key0; k0 < end; k0 += 32) {
        float16v s = {};
        if (!AHEAD) wait_copies<Tile<DP>::stride / 16>();      // K is there, V on its way
#pragma unroll
        for (int c = 0; c < DP / 16; c++)
            s = T::mfma(AHEAD ? k[c] : Tile<DP>::row(kt, 0, c), q[c], s);
        if (AHEAD) {
            wave_sync();
#pragma unroll
            for (int c = 0; c < DP / 16; c++)
                *(uint4v *)(vt + Tile<DP>::at(lane & 31, 2 * c + h)) = v[c];
        }
        if (AHEAD && k0 + 32 < end) fetch(k0 + 32);
        float mx = neg_inf();
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const int key = k0 + 8 * (r / 4) + 4 * h + r % 4;
            s[r] = key <= lim && key < end ? s[r] : neg_inf();
            mx = fmaxf(mx, s[r]);
        }
        const float mn = fmaxf(m, max_halves(mx));
        const float m0 = mn == neg_inf() ? 0.0f : mn;
        const float alpha = exp2_fast((m - m0) * a.c);
        float sum = 0.0f;
        uint32_t pk[8];
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
            const float p0 = exp2_fast((s[r] - m0) * a.c);
            const float p1 = exp2_fast((s[r + 1] - m0) * a.c);
            sum += p0 + p1;
            pk[r / 2] = T::pack(p0, p1);
        }
        l = l * alpha + sum;
        m = mn;
#pragma unroll
        for (int dt = 0; dt < DP / 32; dt++) o[dt] *= alpha;
        if (AHEAD) wave_sync();
        else wait_copies<0>();
#pragma unroll
        for (int kc = 0; kc < 2; kc++) {
            const uint4v pb = {pk[4 * kc], pk[4 * kc + 1], pk[4 * kc + 2], pk[4 * kc + 3]};
#pragma unroll
            for (int dt = 0; dt < DP / 32; dt++)
                o[dt] = T::mfma(Tile<DP>::transposed(vt, kc * 16, dt), pb, o[dt]);
        }
        if (!AHEAD && k0 + 32 < end) fetch(k0 + 32);
    }
    l = add_halves(l);
    return {p.q0 + qi, head, ok};
}

// Short sequences: a wave owns up to 128 rows of a sequence and key head, in
// tiles of 32: most waves then have a sequence to themselves, and few slots are
// empty. What bounds it is memory, and before that the chain of loads from the
// slot to the rows, with 16 waves a compute unit, and the cache's lines: hence K by
// way of LDS and whole rows stored. 16,384 sequences of 1 to 31, 8 heads of 64 over
// 4, take 191 us (4.2 TB/s); with K to registers 207, with the output stored as 32
// bytes of each row 205.
// Returns whether all sums are finite.
template <typename T, int DP, typename I>
__device__ inline bool wave_tiles(const Attn &a, const Place &p, int hk, int first, uint16_t *kt,
                                  uint16_t *vt) {
    const int rows = p.lq * a.G;
    const bool low = keeps_low(a, rows);
    const float inv = 1.0f / (float)a.G;
    float odd = 0.0f;
    for (int tile = first; tile < first + kShortRows / 32 && tile * 32 < rows; tile++) {
        float16v o[DP / 32];
        float m, l;
        const Row r = run_rows<T, DP, false, I>(a, p, hk, tile, 0, p.lk, kt, vt, o, m, l);
        watch<DP>(odd, o);
        if (low) {
            store_out<T, DP>(a, r.t, r.head, o, m, l, r.ok, true);
            continue;
        }
        uint16_t *op = (uint16_t *)a.o + p.q0 * a.o_row + hk * a.G * a.o_head;
        store_tile<T, DP>(op, o, l == 0.0f ? 0.0f : 1.0f / l, a.d, rows - tile * 32, kt, [&](int i) {
            const int row = min(tile * 32 + i, rows - 1), qi = quotient<I>(row, a.G, inv);
            return times<I>(qi, a.o_row) + times<I>(row - qi * a.G, a.o_head);
        });
        store_lse(a, r.t, r.head, m, l, r.ok);
    }
    return finite(odd);
}
template <typename T, int DP>
__global__ __launch_bounds__(256, DP <= 64 ? 4 : 2) void attn_wave(Attn a, int slots) {
    __shared__ __align__(256) uint16_t lds[4][2][32 * Tile<DP>::stride];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint16_t *kt = lds[wave][0], *vt = lds[wave][1];
    const int item = block_number() * 4 + wave;
    const int slot = item / a.hkv, hk = item - slot * a.hkv;
    if (slot >= slots) return;
    const Found f = find_sequence(a.cu_q, a.n_seq, a.tq, a.G, kShortRows, slot);
    const int b = f.b;
    const Place p = place_of(a, b, f.start, f.end);
    const int first = (slot - slot_of(p.q0, a.G, kShortRows, b)) * (kShortRows / 32);
    if (first < 0) return;
    bool plain;
    if (a.near && p.lq * a.G <= kNear && p.lk <= kNear)
        plain = wave_tiles<T, DP, uint32_t>(a, p, hk, first, kt, vt);
    else
        plain = wave_tiles<T, DP, int64_t>(a, p, hk, first, kt, vt);
    if (__builtin_expect(__any(!plain), 0))
        mend_out<T>(arguments<Attn>(), p, hk, first * 32, first * 32 + kShortRows, 32, ~0u, 0, p.lk,
                    nullptr, nullptr, 0);
}

// Long sequences: a block of WAVES waves owns WAVES * 32 rows of one key head;
// 64 keys at a time pass through LDS for all of them, the next 64 on their way
// there meanwhile. Two waves a SIMD, so that one's softmax runs beside the
// other's matrix instructions; the vector instructions of the softmax and the
// matrix instructions take about as long, so addresses are kept out of the loop.
// Four waves a block, two blocks a compute unit, which do not wait for each other:
// two sequences of 6,000, 32 heads of 128 over 8, take 583 us, with eight waves
// 627; ten of 1 to 8,191 1.09 and 1.07 ms (1 PFLOP/s, matrix cores busy 53 %, vector
// instructions 41 %).
// The sums are rescaled only when some row's maximum has grown by more than 2^8:
// a lower reference is as exact, since numerator and denominator share it, and
// 2^8 is far from any overflow.
template <typename T, int DP, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void attn_tiles(Attn a, int slots) {
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
    // the last tiles, which see most keys, go first
    const int tile = (rows + ROWS - 1) / ROWS - 1 - (slot - slot_of(p.q0, a.G, ROWS, b));
    if (tile < 0 || tile * ROWS >= rows) return;
    const int row = tile * ROWS + wave * 32 + (lane & 31);
    const bool ok = row < rows;
    const int qi = ok ? row / a.G : 0, g = ok ? row % a.G : 0;
    const int head = hk * a.G + g;
    const int lim = ok ? qi + p.lk - p.lq : -1;
    uint4v q[DP / 16];
    load_row<DP>(q, a.q, (p.q0 + qi) * a.q_row + head * a.q_head, a.d, ok);
    // keys that the block's rows see, that this wave's see, and that each of
    // this wave's rows sees
    auto seen_by = [&](int r) {
        return min(r, rows - 1) / a.G + p.lk - p.lq + 1;
    };
    const int keys = seen_by(tile * ROWS + ROWS - 1);
    const int w0 = tile * ROWS + wave * 32;
    const int wave_keys = w0 < rows ? seen_by(w0 + 31) : 0;
    const int all_keys = w0 + 31 < rows ? seen_by(w0) : 0;
    const Keys tiles(a, p, hk, keys);
    landed(q);
    const uint32_t lds0 = lds_address(lds);
    const typename Tile<DP>::Rows kr = Tile<DP>::rows(lds0);
    const typename Tile<DP>::Columns vc = Tile<DP>::columns(lds0 + Keys::BYTES / 2);

    float16v o[DP / 32] = {};
    float m = neg_inf(), l = 0.0f;
    // 64 keys from k0, in buffer `buf`
    auto work = [&](auto buf, int k0) {
        constexpr uint32_t B = decltype(buf)::value * Keys::BYTES;
        wait_copies<0>();
        block_barrier();
        if (k0 + KB < keys) tiles.copy(k0 + KB, lds0 + (Keys::BYTES - B));
        if (k0 >= wave_keys) return;
        float16v s[2] = {};
#pragma unroll
        for (int c = 0; c < DP / 16; c++)
#pragma unroll
            for (int u = 0; u < 2; u++)
                s[u] = T::mfma(Tile<DP>::row(kr.c[c], B + u * 32 * STRIDE), q[c], s[u]);
        if (k0 + KB > all_keys)
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (k0 + u * 32 + 8 * (r / 4) + 4 * h + r % 4 > lim) s[u][r] = neg_inf();
        float top[4] = {s[0][0], s[0][8], s[1][0], s[1][8]};     // four chains of eight
#pragma unroll
        for (int r = 1; r < 8; r++)
#pragma unroll
            for (int i = 0; i < 4; i++) top[i] = max2(top[i], s[i / 2][i % 2 * 8 + r]);
        float mx = max2(max2(top[0], top[1]), max2(top[2], top[3]));
        mx = max_halves(mx);
        if (__any((mx - m) * a.c > 8.0f)) {
            const float mn = fmaxf(m, mx), m0 = mn == neg_inf() ? 0.0f : mn;
            const float alpha = exp2_fast((m - m0) * a.c);
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < DP / 32; dt++) o[dt] *= alpha;
            m = mn;
        }
        const float mc = m == neg_inf() ? 0.0f : m * a.c;
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int kc = 0; kc < 2; kc++) {
                uint4v pb;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float p0 = exp2_fast(__builtin_fmaf(s[u][8 * kc + 2 * j], a.c, -mc));
                    const float p1 = exp2_fast(__builtin_fmaf(s[u][8 * kc + 2 * j + 1], a.c, -mc));
                    sum[0] += p0;
                    sum[1] += p1;
                    pb[j] = T::pack(p0, p1);
                }
#pragma unroll
                for (int dt = 0; dt < DP / 32; dt++)
                    o[dt] = T::mfma(Tile<DP>::transposed(vc, dt, B + (u * 32 + kc * 16) * STRIDE), pb,
                                    o[dt]);
            }
        l += sum[0] + sum[1];
    };
    if (keys > 0) tiles.copy(0, lds0);
    for (int k0 = 0; k0 < keys; k0 += 2 * KB) {
        work(Const<0>{}, k0);
        if (k0 + KB < keys) work(Const<1>{}, k0 + KB);
    }
    l = add_halves(l);
    const uint32_t bad = not_finite<DP>(o) & row_bits(finite(l));
    store_out<T, DP>(a, p.q0 + qi, head, o, m, l, ok, keeps_low(a, rows));
    if (__builtin_expect(bad, 0))
        mend_out<T>(arguments<Attn>(), p, hk, w0, w0 + 32, 32, bad, 0, p.lk, nullptr, nullptr, 0);
}

// Few rows over many keys (single tokens over a cache). A sequence's keys are
// cut into chunks, one wave to a chunk, key head and tile of 32 rows; each
// leaves its maximum, sum and unscaled output, and attn_join adds them up. With
// the next 32 keys always on their way, eight waves a compute unit keep 128 KB
// in flight: memory bounds it, 24 tokens over 940,000 keys (3.85 GB), 32 heads of 128
// over 8, take 0.72 ms, 5.3 TB/s. Chunks are slots over the key rows, as tiles are
// over the query rows.
struct Step {
    int chunk;          // keys of a chunk, a multiple of 32
    int tiles;          // row tiles of a slot
    int rows;           // rows of a slot that have room in the partials
    int slots;
    float *o, *ml;      // [slot][hkv][rows][DP], [slot][hkv][rows][2]
};

template <typename T, int DP>
__global__ __launch_bounds__(256, 2) void attn_step(Attn a, Step st) {
    __shared__ __align__(16) uint16_t lds[4][32 * Tile<DP>::stride];
    uint16_t *vt = lds[threadIdx.x >> 6];
    const int lane = threadIdx.x & 63, h = lane >> 5;
    const int item = block_number() * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int slot = item / a.hkv, hk = item - slot * a.hkv;
    if (slot >= st.slots) return;
    const Found f = find_sequence(a.cu_k, a.n_seq, a.tk, 1, st.chunk, slot);
    const int b = f.b;
    // the rows after the last sequence see no key: entry n_seq, chunk 0
    const Place p = place_of(a, b);
    const int chunk = slot - slot_of(f.start, 1, st.chunk, b);
    const int rows = p.lq * a.G;
    if (chunk < 0 || rows == 0) return;
    const int chunks = (p.lk + st.chunk - 1) / st.chunk;
    const bool split = chunks > 1 && rows <= st.rows;
    if (chunk >= (split ? chunks : 1)) return;
    const int key0 = split ? chunk * st.chunk : 0;
    const int key1 = split && key0 + st.chunk < p.lk ? key0 + st.chunk : p.lk;
    const int64_t first = ((int64_t)slot * a.hkv + hk) * st.rows;
    bool bad = false;
    // a sequence with more rows than the partials have room for is not split
    for (int tile = blockIdx.y; tile * 32 < rows; tile += st.tiles) {
        float16v o[DP / 32];
        float m, l;
        const Row r = run_rows<T, DP, true, int64_t>(a, p, hk, tile, key0, key1, vt, vt, o, m, l);
        bad |= (not_finite<DP>(o) & row_bits(finite(l))) != 0;
        if (!split) {
            store_out<T, DP>(a, r.t, r.head, o, m, l, r.ok, keeps_low(a, rows));
            continue;
        }
        const int64_t pr = first + tile * 32 + (lane & 31);
        if (!r.ok) continue;
#pragma unroll
        for (int dt = 0; dt < DP / 32; dt++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float4v f = {o[dt][4 * j], o[dt][4 * j + 1], o[dt][4 * j + 2],
                                   o[dt][4 * j + 3]};
                *(float4v *)(st.o + pr * DP + dt * 32 + 8 * j + 4 * h) = f;
            }
        if (h == 0) {
            st.ml[2 * pr] = m;
            st.ml[2 * pr + 1] = l;
        }
    }
    if (__builtin_expect(bad, 0))
        mend_out<T>(arguments<Attn>(), p, hk, blockIdx.y * 32, rows, st.tiles * 32, ~0u, key0, key1,
                    split ? st.o + first * DP : nullptr, split ? st.ml + 2 * first : nullptr, DP);
}

// Joins the chunks of a split sequence: a wave to a row of the output, which
// has one owner and one order of summation.
template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_join(Attn a, Step st) {
    const int lane = threadIdx.x & 63;
    const int item = block_number() * 4 + (int)(threadIdx.x >> 6);
    if (item >= a.tq * a.hq) return;
    const int t = item / a.hq, head = item - t * a.hq, hk = head / a.G;
    const int b = sequence_of_row(a.cu_q, a.n_seq, a.tq, t);
    const Place p = place_of(a, b);
    const int chunks = (p.lk + st.chunk - 1) / st.chunk;
    const int rows = p.lq * a.G;
    if (chunks <= 1 || rows > st.rows || t < p.q0 || t >= p.q0 + p.lq) return;
    const int row = (t - p.q0) * a.G + head % a.G;
    const int64_t slot0 = slot_of(offset_at(a.cu_k, b, a.tk), 1, st.chunk, b);
    const int64_t stride = (int64_t)a.hkv * st.rows;
    const int64_t pr = slot0 * stride + (int64_t)hk * st.rows + row;
    float m = neg_inf();
    for (int c = lane; c < chunks; c += 64) m = fmaxf(m, st.ml[2 * (pr + c * stride)]);
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    const float m0 = m == neg_inf() ? 0.0f : m;
    float l = 0.0f;
    for (int c = lane; c < chunks; c += 64) {
        const float *x = st.ml + 2 * (pr + c * stride);
        l += x[1] * exp2_fast((x[0] - m0) * a.c);
    }
    for (int o = 32; o; o >>= 1) l += __shfl_xor(l, o);
    float acc[2] = {0.0f, 0.0f};
#pragma unroll 8
    for (int c = 0; c < chunks; c++) {
        const float w = exp2_fast((st.ml[2 * (pr + c * stride)] - m0) * a.c);
        const float *x = st.o + (pr + c * stride) * DP;
        for (int e = 0; e < (DP + 63) / 64; e++)
            if (lane + 64 * e < DP) acc[e] += w * x[lane + 64 * e];
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    typename T::elem *out = (typename T::elem *)a.o + t * a.o_row + head * a.o_head;
    typename T::elem *low = (typename T::elem *)a.o_low + (int64_t)item * a.d;
    for (int e = 0; e < (DP + 63) / 64; e++)
        if (lane + 64 * e < a.d) {
            const float x = acc[e] * inv;
            out[lane + 64 * e] = (typename T::elem)x;
            if (keeps_low(a, rows)) low[lane + 64 * e] = (typename T::elem)(x - (float)(typename T::elem)x);
        }
    if (a.lse && lane == 0)
        a.lse[head * a.tq + t] = l == 0.0f ? neg_inf() : m * a.scale + logf(l);
}

// Whether a call is few rows over many keys, and its chunks. At most 256 rows a
// sequence on average, and at least four keys a query: then the keys decide. Fewer
// than 512 keys are as soon read by the waves that the rows have (256 sequences of
// 200 keys, 32 heads over 8: 36 against 63 us; 64 of 4,000: 250 against 222 us; one
// of 4,000: 195 against 24 us), unless there are hardly any waves. Chunks of 512
// keys, or as few as 128 as long as that leaves less than a wave per compute unit
// (8 sequences of 4,000: 512 40 us, 256 45 us; one: 38 and 24 us).
bool plan_step(const Attn &a, Step &st) {
    if (a.n_seq == 0 || a.tq * a.G > 256ll * a.n_seq || a.tk < 4 * a.tq) return false;
    st.tiles = (int)((a.tq * a.G + 32ll * a.n_seq - 1) / (32ll * a.n_seq));
    const int64_t waves = (int64_t)a.n_seq * a.hkv * st.tiles;
    if (a.tk < (waves < 256 ? 256ll : 512ll) * a.n_seq) return false;
    st.chunk = 512;
    while (st.chunk > 128 && a.tk * a.hkv * st.tiles / st.chunk < 256) st.chunk /= 2;
    st.slots = slot_of(a.tk, 1, st.chunk, a.n_seq) + 1;
    // room for twice the average: a sequence of more rows is not split
    const int64_t twice = (2 * a.tq * a.G + a.n_seq - 1) / a.n_seq;
    st.rows = (int)(twice < 32ll * st.tiles ? (twice + 3) / 4 * 4 : 32ll * st.tiles);
    return true;
}
int64_t step_rows(const Attn &a, const Step &st) {
    return (int64_t)st.slots * a.hkv * st.rows;
}
int64_t step_bytes(const Attn &a, const Step &st) {
    return a.tk <= st.chunk ? 0 : step_rows(a, st) * (padded_head(a.d) + 2) * 4;
}

template <typename T, int DP>
int launch_step(const Attn &a, Step st, hipStream_t s) {
    st.o = (float *)a.workspace;
    st.ml = st.o + step_rows(a, st) * DP;
    const dim3 grid = grid_of((st.slots * (int64_t)a.hkv + 3) / 4, 256, st.tiles);
    attn_step<T, DP><<<grid, 256, 0, s>>>(a, st);
    if (a.tk > st.chunk) {
        if (hipGetLastError() != hipSuccess) return CO_ERR_CUDA;
        attn_join<T, DP><<<grid_of((a.tq * a.hq + 3) / 4, 256), 256, 0, s>>>(a, st);
    }
    return launch_status();
}

template <typename T, int DP, int WAVES>
int launch_tiles(const Attn &a, hipStream_t s) {
    const int slots = slot_of(a.tq, a.G, WAVES * 32, a.n_seq) + 1;
    const dim3 grid = grid_of((int64_t)slots * a.hkv, WAVES * 64);
    attn_tiles<T, DP, WAVES><<<grid, WAVES * 64, 0, s>>>(a, slots);
    return launch_status();
}

template <typename T, int DP>
int launch_head(const Attn &a, hipStream_t s) {
    Step st;
    if (plan_step(a, st)) return launch_step<T, DP>(a, st, s);
    const int64_t rows = a.n_seq ? a.tq * a.G / a.n_seq : 0;      // of a sequence, on average
    // Tiles shared by four waves from 96 rows on; below, two of the waves would idle
    // (4 heads of 64, sequences of 32: 45 against 85 us, 64: alike, 96: 74 against 69 us).
    if (rows >= 96) return launch_tiles<T, DP, 4>(a, s);
    const int slots = slot_of(a.tq, a.G, kShortRows, a.n_seq) + 1;
    const int64_t blocks = (slots * (int64_t)a.hkv + 3) / 4;
    attn_wave<T, DP><<<grid_of(blocks, 256), 256, 0, s>>>(a, slots);
    return launch_status();
}

template <typename T>
int launch_forward(const Attn &a, hipStream_t s) {
    switch (padded_head(a.d)) {
        case 32: return launch_head<T, 32>(a, s);
        case 64: return launch_head<T, 64>(a, s);
        case 96: return launch_head<T, 96>(a, s);
        default: return launch_head<T, 128>(a, s);
    }
}

static bool misaligned(const void *p, int64_t row, int64_t head) {
    return ((uintptr_t)p & 15) || row % 8 || head % 8;
}

int check_attention(const SeqAttention *a) {
    if (!a || a->struct_size != (int32_t)sizeof(SeqAttention)) return CO_ERR_NULLARG;
    if (a->n_seq < 0 || a->tq < 0 || a->tk < 0 || a->hkv < 1 || a->hq < 1 || a->d < 1)
        return CO_ERR_NULLARG;
    if (a->d % 8 || a->d > SEQ_MAX_HEAD || a->hq % a->hkv || a->n_seq > 1 << 28 ||
        a->tq > SEQ_MAX_ROWS / a->hq || a->tk > SEQ_MAX_ROWS || a->hq > 1 << 15 ||
        // the most waves that a launch has: a slot for 32 rows of either kind
        (a->tq / 32 * (a->hq / a->hkv) + a->tk / 32 + a->n_seq + 2) * a->hkv > SEQ_MAX_ROWS)
        return CO_ERR_BOUNDS;
    if ((a->dtype != SEQ_BF16 && a->dtype != SEQ_FP16) || !(a->scale >= SEQ_LEAST) ||
        a->scale > SEQ_MOST)
        return CO_ERR_DATA;
    return CO_OK;
}

// the rest of the checks, for a call with pointers
int check_attention_data(const SeqAttention *a) {
    if (!a->cu_q || !a->cu_k || !a->q || !a->o || (a->tk && (!a->k || !a->v)))
        return CO_ERR_NULLARG;
    if (misaligned(a->q, a->q_row, a->q_head) || misaligned(a->k, a->k_row, a->k_head) ||
        misaligned(a->v, a->v_row, a->v_head) || misaligned(a->o, a->o_row, a->o_head) ||
        ((uintptr_t)a->o_low & 15))
        return CO_ERR_DATA;
    return CO_OK;
}

}  // namespace seq

extern "C" int64_t seq_attention_workspace(const SeqAttention *a) {
    const int rc = seq::check_attention(a);
    if (rc != CO_OK) return rc > 0 ? -rc : rc;
    const seq::Attn x = seq::make_attn(a);
    seq::Step st;
    return seq::plan_step(x, st) ? seq::step_bytes(x, st) : 0;
}

extern "C" int seq_attention(const SeqAttention *sa, void *stream) {
    int rc = seq::check_attention(sa);
    if (rc != CO_OK) return rc;
    if (sa->tq == 0) return CO_OK;
    rc = seq::check_attention_data(sa);
    if (rc != CO_OK) return rc;
    const seq::Attn a = seq::make_attn(sa);
    const int64_t need = seq_attention_workspace(sa);
    if (need && !a.workspace) return CO_ERR_NULLARG;
    if (need > a.workspace_bytes || ((uintptr_t)a.workspace & 15)) return CO_ERR_DATA;
    hipStream_t s = (hipStream_t)stream;
    return a.dtype == SEQ_BF16 ? seq::launch_forward<seq::Bf16>(a, s)
                               : seq::launch_forward<seq::Fp16>(a, s);
}
