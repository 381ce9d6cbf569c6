// seq_attn.h -- pieces of the attention kernels (forward, gradient, steps).
//
// Rows. A sequence's lq queries and the G heads that share a key head fold
// into lq * G rows, row r = query r / G, head r % G: the heads of a group read
// the same keys, so they share tiles, and short sequences fill them better.
//
// Products. Scores are formed transposed, S^T = K Q^T, so that a lane of the
// 32x32 product holds 16 keys of one query: the softmax runs along registers,
// with one exchange between the wave's halves. The same registers, packed to
// 16 bits, are the right operand of O^T = V^T P^T: a contraction may take its
// index in any order, so V's rows are read in the order the lane's keys have
// (4h..4h+3, 8+4h..8+4h+3 of every 16, h the half). P never passes through LDS.
#ifndef CUSR_SEQ_ATTN_H
#define CUSR_SEQ_ATTN_H

#include "seq_common.h"

namespace seq {

struct Attn : SeqAttention {
    int32_t G;       // query heads per key head
    float c;         // scale * log2(e): scores in powers of two
    int32_t near;    // every stride is below 2^16 elements
    int32_t low_all; // the gradient reads o_low of every row
};
inline bool near_strides(int64_t a, int64_t b, int64_t c, int64_t d) {
    const int64_t most = 1 << 16;
    return a >= 0 && b >= 0 && c >= 0 && d >= 0 && a < most && b < most && c < most && d < most;
}

// Rows that a wave owns where a sequence is mostly one wave's.
constexpr int kShortRows = 128;

// Whether the gradient of a call is that of short sequences. Below these keys a
// sequence, on average, blocks of the long kernels mostly wait for themselves; above, a
// wave alone takes longer (4 heads of 64: sequences of 96 199 against 282 us, of 128 300
// against 297 us; heads of 128, with half the waves: of 64 157 against 311 us, of 100
// 607 against 464 us).
inline int padded_head(int d) { return (d + 31) / 32 * 32; }   // 32, 64, 96 or 128
inline bool short_sequences(const SeqAttention &a) {
    return a.tk < (padded_head(a.d) <= 64 ? 128ll : 80ll) * a.n_seq || a.n_seq == 0;
}

// Whether a sequence's rows leave in o_low what rounding took from o. The gradient needs
// delta = sum(o * do) of a row wherever another wave than the row's uses it: everywhere in
// the long kernels, and in the short one for a sequence of more rows than a wave has.
// Elsewhere delta is summed anew from P and dP.
__device__ inline bool keeps_low(const Attn &a, int rows) {
    return a.o_low && (a.low_all || rows > kShortRows);
}

__device__ inline int clamp_to(int x, int lo, int64_t hi) {
    return x < lo ? lo : (x > hi ? (int)hi : x);
}

// x / n for 0 <= x < 2^31, n >= 1, without a branch: the quotient by a float
// reciprocal `inv` is off by at most a few hundred for large x, so the remainder,
// taken exactly, corrects it once by its own quotient and once by one.
__device__ inline int divide(int x, int n, float inv) {
    int q = (int)((float)x * inv);
    q += (int)((float)(x - q * n) * inv);
    const int r = x - q * n;
    return q + (r >= n) - (r < 0);
}

// Offsets inside a sequence as int64_t, or as uint32_t where the strides are near and
// rows, queries and keys at most kNear: then they, in bytes too, have 32 bits, their
// factors 24, and the quotient of a row needs no correction.
constexpr int kNear = 1 << 14;
template <typename I> __device__ inline I times(int i, int64_t step) {
    if constexpr (sizeof(I) == 4) return __umul24(i, (uint32_t)step);
    else return i * step;
}
template <typename I> __device__ inline int quotient(int x, int n, float inv) {
    if constexpr (sizeof(I) == 4) return (int)(((float)x + 0.5f) * inv);
    else return divide(x, n, inv);
}

// Rows, query rows times heads among them, number less than 2^31 (the entry
// checks it), so places and tiles have 32 bits; only addresses have 64.

// A sequence's place: first query and key row, number of queries and keys.
struct Place { int q0, k0, lq, lk; };

__device__ inline int offset_at(const int32_t *cu, int b, int64_t t) {
    return b <= 0 ? 0 : clamp_to(cu[b], 0, t);
}

// Work is handed out in tiles of `rows` rows without a list of tiles: tile
// slots of sequence b start at floor(cu[b] * fold / rows) + b, which leaves
// each at least as many as it has tiles and numbers them without gaps for a
// search. Entry n_seq stands for the rows after the last sequence.
__device__ __host__ inline int slot_of(int64_t at, int fold, int rows, int b) {
    return (int)((uint32_t)at * (uint32_t)fold / (uint32_t)rows) + b;
}

// A slot's sequence: the last b of 0..n_seq with slot_of(b) <= slot, and the
// offsets of it and the next (the tensor's end after n_seq). 64 probes at a time,
// one per lane: first around the place that the slot would have if all sequences
// were of one length, then, when that does not enclose it, over all of them. Each
// round waits for a load, so the last one also brings the offsets. Every lane of a
// wave calls it with the same arguments.
struct Found { int b, start, end; };
__device__ inline Found find_sequence(const int32_t *cu, int n_seq, int64_t t, int fold, int rows,
                                      int slot) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = n_seq + 1, step = (n + 63) / 64;
    const int slots = slot_of(t, fold, rows, n_seq) + 1;
    if (step > 1) {
        // sequences of like lengths lie within a fraction of n of the guess
        const int narrow = (n + 2047) / 2048;
        const int guess = (int)((float)slot / (float)slots * (float)n) - 32 * narrow;
        const int i = min(max(guess, 0), n - 64 * narrow) + lane * narrow;
        const uint64_t ok = __ballot(slot_of(offset_at(cu, i, t), fold, rows, i) <= slot);
        // the first holds and the last does not, or there is none after it
        const int last = __popcll(ok) - 1;
        const int first = __builtin_amdgcn_readfirstlane(i);
        if (last >= 0 && (last < 63 || first + 64 * narrow >= n)) {
            lo = first + last * narrow;
            n = min(narrow, n - lo);
            step = (n + 63) / 64;
        }
    }
    for (;;) {
        const int i = lane * step;
        const int at = offset_at(cu, min(lo + i, n_seq), t);
        const bool ok = i < n && slot_of(at, fold, rows, lo + i) <= slot;
        const int last = max(__popcll(__ballot(ok)) - 1, 0);   // offsets out of order: the first
        if (step == 1) {
            Found f;
            f.b = __builtin_amdgcn_readfirstlane(lo + last);
            f.start = __builtin_amdgcn_readlane(at, last);
            // the next offset is the next lane's, unless this is the last lane
            f.end = f.b >= n_seq ? (int)t
                                 : (last < 63 ? __builtin_amdgcn_readlane(at, last + 1)
                                              : offset_at(cu, f.b + 1, t));
            return f;
        }
        lo += last * step;
        n = min(n - last * step, step);
        step = (n + 63) / 64;
    }
}

__device__ inline Place place_of(const Attn &a, int b, int q0, int q1) {
    Place p;
    p.q0 = q0;
    p.lq = q1 > q0 ? q1 - q0 : 0;
    p.k0 = p.lk = 0;
    if (b >= a.n_seq) return p;          // the rows after the last sequence: no keys
    int k1 = q1;
    if (a.cu_k == a.cu_q && a.tk == a.tq) {
        p.k0 = q0;
    } else {
        p.k0 = clamp_to(a.cu_k[b], 0, a.tk);
        k1 = clamp_to(a.cu_k[b + 1], p.k0, a.tk);
    }
    p.lk = max(k1 - p.k0, 0);
    if (a.k_lens) p.lk = clamp_to(a.k_lens[b], 0, p.lk);
    return p;
}

// The sequence of query row t (n_seq: none): the last whose offset is not
// beyond it. Empty sequences share their offset with the next.
__device__ inline int sequence_of_row(const int32_t *cu, int n_seq, int64_t tq, int t) {
    int lo = 0, hi = n_seq;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (offset_at(cu, mid, tq) <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
__device__ inline Place place_of(const Attn &a, int b) {
    return place_of(a, b, offset_at(a.cu_q, b, a.tq),
                    b >= a.n_seq ? (int)a.tq : offset_at(a.cu_q, b + 1, a.tq));
}

// Waits here for loads of operands that a loop uses. At their first use the
// compiler would wait in the loop, each time round, for every copy under way.
template <int N> __device__ inline void landed(uint4v (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) asm volatile("" : "+v"(x[i]));
}

// Barrier of the block that no memory access of the program moves across.
__device__ inline void block_barrier() { asm volatile("s_barrier" ::: "memory"); }

// 16-bit tile rows in LDS: DP elements a row (96 padded to 128), the row's 16-byte
// pieces permuted by the row's place among 16.
template <int DP> struct Tile {
    static constexpr int stride = DP == 96 ? 128 : DP;      // elements
    static constexpr int chunks = stride / 8;
    // The LDS serves 256 bytes at a time. A transposed read of half a wave takes 64
    // bytes of each of four rows in turn: they have to lie in different quarters. A row
    // read takes one piece of 16 rows: they have to lie in different pieces.
    static __device__ int swz(int row) {
        return DP == 32   ? row >> 2 & 3
               : DP == 64 ? (row >> 1 & 1) << 2 | (row >> 2 & 3)
                          : (row & 3) << 2 | (row >> 2 & 3);
    }
    static __device__ int at(int row, int chunk) {          // element offset
        return row * stride + ((chunk ^ swz(row)) << 3);
    }
    // left operand of a product over the tile's rows: column dt * 32 + lane % 32,
    // rows k0 + {4h..4h+3, 8+4h..8+4h+3}
    static __device__ uint4v transposed(const uint16_t *t, int k0, int dt) {
        const int lane = threadIdx.x & 63, h = lane >> 5, i = lane & 15;
        const int col = dt * 32 + (lane & 16) + (i & 3) * 4;
        const int r0 = k0 + 4 * h + (i >> 2), r1 = r0 + 8;
        const uint2v lo = read_transposed(t + at(r0, col >> 3) + (col & 7));
        const uint2v hi = read_transposed(t + at(r1, col >> 3) + (col & 7));
        uint4v v = {lo[0], lo[1], hi[0], hi[1]};
        return v;
    }
    // The same two reads by LDS byte address, for the inner loops. A lane keeps
    // one address for each column (rows) or 32 columns (transposed); rows and
    // buffers are constants in the instruction, so a read costs no arithmetic.
    // `at` is a multiple of 16 rows in bytes, and a tile starts on 256 bytes.
    struct Rows { uint32_t c[DP / 16]; };
    static __device__ Rows rows(uint32_t tile) {
        const int lane = threadIdx.x & 63;
        Rows r;
#pragma unroll
        for (int c = 0; c < DP / 16; c++) r.c[c] = tile + 2 * at(lane & 31, 2 * c + (lane >> 5));
        return r;
    }
    static __device__ uint4v row(uint32_t address, uint32_t at) {
        return *(lds_ptr4)(uintptr_t)(address + at);
    }
    struct Columns { uint32_t lo[DP / 32], hi[DP / 32]; };
    static __device__ Columns columns(uint32_t tile) {
        const int lane = threadIdx.x & 63, h = lane >> 5, i = lane & 15;
        Columns x;
#pragma unroll
        for (int dt = 0; dt < DP / 32; dt++) {
            const int col = dt * 32 + (lane & 16) + (i & 3) * 4, r = 4 * h + (i >> 2);
            x.lo[dt] = tile + 2 * (at(r, col >> 3) + (col & 7));
            x.hi[dt] = tile + 2 * (at(r + 8, col >> 3) + (col & 7));
        }
        return x;
    }
    static __device__ uint4v transposed(const Columns &x, int dt, uint32_t at) {
        const uint2v a = read_transposed((lds_ptr)(uintptr_t)(x.lo[dt] + at));
        const uint2v b = read_transposed((lds_ptr)(uintptr_t)(x.hi[dt] + at));
        uint4v v = {a[0], a[1], b[0], b[1]};
        return v;
    }
    // left operand over the columns: row r0 + lane % 32, columns 16 c + 8h..+7
    static __device__ uint4v row(const uint16_t *t, int r0, int c) {
        const int lane = threadIdx.x & 63;
        return *(const uint4v *)(t + at(r0 + (lane & 31), 2 * c + (lane >> 5)));
    }
};

// Tiles of KB keys and their values on their way to LDS, for a block of WAVES
// waves. Whole tiles take their addresses from the wave's registers alone; the
// last one repeats its last key.
template <int DP, int KB, int WAVES> struct KeyTiles {
    static constexpr int STRIDE = Tile<DP>::stride * 2;          // bytes of a row in LDS
    static constexpr int PER = KB * STRIDE / 1024;               // copies of k, and of v
    static constexpr int ROWS = 1024 / STRIDE;                   // rows of a copy
    static constexpr int COPIES = 2 * PER / WAVES;               // of a wave
    static_assert(COPIES >= 1 && 2 * PER % WAVES == 0 && (PER % WAVES == 0 || PER * 2 == WAVES), "");
    static constexpr uint32_t BYTES = 2 * KB * STRIDE;           // k, then v
    const char *k, *v;
    int64_t k_step, v_step;
    int keys, wave, row, col;                                    // this lane's first row, column
    uint32_t k_off, v_off;
    bool plain;

    __device__ KeyTiles(const Attn &a, const Place &p, int hk, int keys_) {
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int lane = threadIdx.x & 63;
        k = (const char *)a.k + 2 * (p.k0 * a.k_row + hk * a.k_head);
        v = (const char *)a.v + 2 * (p.k0 * a.v_row + hk * a.v_head);
        k_step = 2 * a.k_row;
        v_step = 2 * a.v_row;
        keys = keys_;
        row = wave % PER * ROWS + lane * 16 / STRIDE;
        const int ch = (lane * 16 % STRIDE / 16) ^ Tile<DP>::swz(row);
        col = ch * 8 < a.d ? ch * 16 : 0;
        // a lane's offset within a tile has 32 bits
        plain = k_step >= 0 && k_step < 1 << 25 && v_step >= 0 && v_step < 1 << 25;
        k_off = (uint32_t)(row * k_step) + col;
        v_off = (uint32_t)(row * v_step) + col;
    }
    __device__ void copy(int k0, uint32_t to) const {
        const bool whole = plain && k0 + KB <= keys;
        if (whole) {
#pragma unroll
            for (int x = 0; x < COPIES; x++) {
                const int idx = wave + x * WAVES, r = k0 + (idx % PER - wave % PER) * ROWS;
                copy_to_lds16(idx < PER ? k + r * k_step : v + r * v_step,
                              idx < PER ? k_off : v_off, to + idx * 1024);
            }
            return;
        }
#pragma unroll
        for (int x = 0; x < COPIES; x++) {
            const int idx = wave + x * WAVES, r = k0 + (idx % PER - wave % PER) * ROWS + row;
            const int mine = r < keys ? r : keys - 1;
            copy_to_lds16((idx < PER ? k + mine * k_step : v + mine * v_step) + col,
                          to + idx * 1024);
        }
    }
};

// Row `r` of a [rows, heads, d] tensor as operand fragments: columns
// 16 c + 8h .. + 7 for c < DP/16; zero beyond d, and altogether when !ok.
template <int DP>
__device__ inline void load_row(uint4v *f, const void *base, int64_t off, int d, bool ok) {
    const int h = (threadIdx.x & 63) >> 5;
    const uint16_t *p = (const uint16_t *)base + off;
    const uint4v z = {0, 0, 0, 0};
    if (d == DP) {                       // the same for all: no test for each piece
#pragma unroll
        for (int c = 0; c < DP / 16; c++) f[c] = z;
        if (ok)
#pragma unroll
            for (int c = 0; c < DP / 16; c++) f[c] = *(const uint4v *)(p + c * 16 + h * 8);
        return;
    }
#pragma unroll
    for (int c = 0; c < DP / 16; c++)
        f[c] = ok && c * 16 + h * 8 < d ? *(const uint4v *)(p + c * 16 + h * 8) : z;
}

// A column of a transposed accumulator (DP values of this lane's row, split
// between the halves) scaled and packed to 16-byte pieces for sink(piece, value).
// LOW: what the packing rounds away instead.
template <typename T, int DP, bool LOW, typename F>
__device__ inline void pack_row(const float16v *acc, float scale, F sink) {
    const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int dt = 0; dt < DP / 32; dt++)
#pragma unroll
        for (int g = 0; g < 2; g++) {
            uint32_t x[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float u = acc[dt][8 * g + 2 * j] * scale;
                const float w = acc[dt][8 * g + 2 * j + 1] * scale;
                x[j] = T::pack(u, w);
                if (LOW) x[j] = T::pack(u - T::lo(x[j]), w - T::hi(x[j]));
            }
            // halves hold columns 0-3, 8-11 and 4-7, 12-15: after the exchange
            // 0-7 and 8-15
            auto s0 = __builtin_amdgcn_permlane32_swap(x[0], x[2], false, false);
            auto s1 = __builtin_amdgcn_permlane32_swap(x[1], x[3], false, false);
            uint4v v = {s0[0], s1[0], s0[1], s1[1]};
            sink(dt * 4 + g * 2 + h, v);
        }
}
// ... stored: row `off` of this lane.
template <typename T, int DP, bool LOW = false>
__device__ inline void store_row(void *base, int64_t off, const float16v *acc, float scale, int d,
                                 bool ok) {
    uint16_t *p = (uint16_t *)base + off;
    pack_row<T, DP, LOW>(acc, scale, [&](int piece, uint4v v) {
        if (d == DP ? ok : ok && piece * 8 < d) *(uint4v *)(p + piece * 8) = v;
    });
}
// ... stored for the wave's 32 rows, of which n exist, by way of an LDS tile: a
// store then covers whole rows instead of 32 bytes of each. row_offset(i) is row
// i's element offset.
template <typename T, int DP, typename F>
__device__ inline void store_tile(void *base, const float16v *acc, float scale, int d, int n,
                                  uint16_t *t, F row_offset) {
    constexpr int CHUNKS = Tile<DP>::chunks, ROWS = 64 / CHUNKS;
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));           // addresses are formed here, not held from before
    pack_row<T, DP, false>(acc, scale, [&](int piece, uint4v v) {
        *(uint4v *)(t + Tile<DP>::at(lane & 31, piece)) = v;
    });
    wave_sync();
#pragma unroll
    for (int x = 0; x < 32 / ROWS; x++) {
        const int r = x * ROWS + lane / CHUNKS, piece = lane % CHUNKS ^ Tile<DP>::swz(r);
        const uint4v v = *(const uint4v *)(t + (x * 64 + lane) * 8);
        const auto at = row_offset(r) + piece * 8;
        if (r < n && piece * 8 < d) *(uint4v *)((char *)base + 2 * at) = v;
    }
}

// 32 rows of a tensor to a wave's LDS tile, past the registers: row_offset(i)
// is row i's element offset from `base`, which is the wave's. Columns beyond d repeat the first.
template <int DP, typename F>
__device__ inline void copy_tile(const void *base, int d, uint32_t to, F row_offset) {
    constexpr int STRIDE = Tile<DP>::stride * 2, ROWS = 1024 / STRIDE;
    const int lane = threadIdx.x & 63;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // the tile's last reads are done
#pragma unroll
    for (int x = 0; x < 32 / ROWS; x++) {
        const int r = x * ROWS + lane * 16 / STRIDE;
        const int ch = (lane * 16 % STRIDE / 16) ^ Tile<DP>::swz(r);
        const auto at = row_offset(r) + (ch * 8 < d ? ch * 8 : 0);
        if constexpr (sizeof(at) == 4) copy_to_lds16(base, 2 * at, to + x * 1024);
        else copy_to_lds16((const uint16_t *)base + at, to + x * 1024);
    }
}

inline Attn make_attn(const SeqAttention *s) {
    Attn a;
    static_cast<SeqAttention &>(a) = *s;
    a.G = a.hq / a.hkv;
    a.c = a.scale * kLog2e;
    a.near = near_strides(a.q_row, a.q_head, a.k_row, a.k_head) &&
             near_strides(a.v_row, a.v_head, a.o_row, a.o_head);
    a.low_all = !short_sequences(*s);
    return a;
}

int check_attention(const SeqAttention *a);

}  // namespace seq
#endif
