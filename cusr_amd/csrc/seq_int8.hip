// seq_int8.hip -- product of 8-bit integers with a scale for each row of both sides
// (include/cusr_seq.h, seq_int8_product).
//
// o[i, j] = a_scale[i] w_scale[j] sum_l a[i, l] w[j, l]. Both sides lie along l, which is
// what the matrix instructions take: a lane of either operand of the 32x32x32 product
// holds 16 values of row lane % 32, and of the 16x16x64 product of row lane % 16. The sum
// is exact in 32 bits up to 131,071 terms, so it may be cut and joined in any order.
#include "seq_rows.h"

namespace seq {

typedef int int4v __attribute__((ext_vector_type(4)));
typedef int int16v __attribute__((ext_vector_type(16)));

// what a piece past the end of a row is read from
__device__ const uint4v kZeros[1] = {{0, 0, 0, 0}};

// 16 values of a row from l on, zeros beyond its end. Any alignment: the memory takes
// wide loads at any byte.
__device__ inline uint4v row_piece(const int8_t *row, int64_t l, int64_t inner) {
    uint4v v = {0, 0, 0, 0};
    if (l + 16 <= inner) {
        __builtin_memcpy(&v, row + l, 16);
    } else {
        for (int j = 0; j < 16; j++)
            if (l + j < inner) v[j / 4] |= (uint32_t)(uint8_t)row[l + j] << (8 * (j % 4));
    }
    return v;
}

// Outputs j .. j + 7 of row i from their sums; `whole`: all of them are inside and lie on
// a boundary of 16 bytes.
__device__ inline void put_sums(const SeqInt8Product &p, int64_t i, int64_t j, const int4v &lo,
                                const int4v &hi, const float *sw, bool whole) {
    const float sa = p.a_scale[i];
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; e++) f[e] = (float)(e < 4 ? lo[e] : hi[e - 4]) * sa * sw[e];
    if (whole) {
        put8(p.o, p.out_dtype, i * p.o_row + j, f);
    } else {
        for (int e = 0; e < 8; e++)
            if (j + e < p.n) put1(p.o, p.out_dtype, i * p.o_row + j + e, f[e]);
    }
}

// A wave's TW columns of 32 rows from its accumulators to memory: turned round through the
// wave's own LDS, so that a lane has 8 columns of a row.
template <int TW>
__device__ inline void put_slab(const SeqInt8Product &p, int64_t i0, int64_t j0,
                                const int16v *acc, int *lds, const float *sw, bool wide) {
    constexpr int PITCH = TW + 8;      // halves of a wave, 4 rows apart, in other banks
    const int lane = threadIdx.x & 63;
    wave_sync();
#pragma unroll
    for (int y = 0; y < TW / 32; y++)
#pragma unroll
        for (int r = 0; r < 16; r++)
            lds[(8 * (r / 4) + 4 * (lane / 32) + r % 4) * PITCH + y * 32 + lane % 32] = acc[y][r];
    wave_sync();
    constexpr int LANES = TW / 8, ROWS = 64 / LANES;       // of a row; at a time
    const int col = lane % LANES * 8;
    const int64_t j = j0 + col;
    if (j >= p.n) return;
    const bool whole = wide && j + 8 <= p.n;
#pragma unroll
    for (int r = 0; r < 32; r += ROWS) {
        const int row = r + lane / LANES;
        const int4v lo = *(const int4v *)(lds + row * PITCH + col);
        const int4v hi = *(const int4v *)(lds + row * PITCH + col + 4);
        if (i0 + row < p.m) put_sums(p, i0 + row, j, lo, hi, sw, whole);
    }
}
template <int TW>
__device__ inline void column_scales(const SeqInt8Product &p, int64_t j0, float *sw) {
    const int64_t j = j0 + (int)(threadIdx.x & 63) % (TW / 8) * 8;
#pragma unroll
    for (int e = 0; e < 8; e++) sw[e] = j + e < p.n ? p.w_scale[j + e] : 0.0f;
}

// A block's tile. Blocks go to the eight dies in turn, so each die takes a run of tiles of
// its own, eight rows of them by columns, whose operands its cache holds.
__device__ inline bool tile_of(int64_t block, int64_t rows, int64_t columns, int64_t &ti,
                               int64_t &tj) {
    const int64_t tiles = rows * columns, each = (tiles + 7) / 8;
    const int64_t t = block % 8 * each + block / 8;
    if (block / 8 >= each || t >= tiles) return false;
    const int64_t band = t / (8 * columns), in = t % (8 * columns);
    const int64_t high = rows - band * 8 < 8 ? rows - band * 8 : 8;
    ti = band * 8 + in % high;
    tj = in / high;
    return true;
}

// T x T outputs a block of four waves, T / 2 x T / 2 a wave, 64 terms a step. Operands come
// to LDS past the registers, three steps ahead in four buffers; a step's second half and
// the next one's first are read from LDS while the half before is multiplied. Row r of a
// buffer holds its four pieces of 16 bytes turned by r / 4, so that 16 lanes' reads meet
// every bank once.
constexpr int kStep = 64, kStages = 4;
template <int T> constexpr int tile_bytes() { return 2 * T * kStep; }

template <int T>
__global__ __launch_bounds__(256, T == 256 ? 1 : 2) void int8_tiles(SeqInt8Product p, bool wide) {
    constexpr int W = T / 2, F = W / 32;         // a wave's side, in products
    constexpr int COPIES = tile_bytes<T>() / 4096;           // a wave's copies of a step
    extern __shared__ __align__(16) unsigned char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int64_t ti, tj;
    if (!tile_of(block_number(), (p.m + T - 1) / T, (p.n + T - 1) / T, ti, tj)) return;
    const int64_t i0 = ti * T, j0 = tj * T;
    const uint32_t base = lds_address(lds);
    // copy x of the wave fills 16 rows: this lane row lane / 4, place lane % 4
    const int8_t *from[COPIES];
    int piece[COPIES];
#pragma unroll
    for (int x = 0; x < COPIES; x++) {
        const int row = (wave * COPIES + x) * 16 + lane / 4;           // of a, then of w
        const bool is_a = row < T;
        const int64_t r = is_a ? i0 + row : j0 + row - T, most = (is_a ? p.m : p.n) - 1;
        piece[x] = (lane % 4 - row / 4 % 4 + 4) % 4 * 16;
        from[x] = (is_a ? p.a : p.w) + (r < most ? r : most) * (is_a ? p.a_row : p.w_row) + piece[x];
    }
    auto fetch = [&](int64_t step) {
        const uint32_t to = base + (uint32_t)(step % kStages) * tile_bytes<T>() +
                            wave * COPIES * 1024;
#pragma unroll
        for (int x = 0; x < COPIES; x++) {
            const int64_t l = step * kStep;
            const void *at = l + piece[x] < p.inner ? (const void *)(from[x] + l) : kZeros;
            copy_to_lds16(at, to + x * 1024);
        }
    };
    const int row = lane % 32;
    auto read = [&](int64_t step, int half, int4v *a, int4v *w) {
        const uint32_t at = base + (uint32_t)(step % kStages) * tile_bytes<T>() +
                            (half * 2 + lane / 32 + row / 4) % 4 * 16 + row * kStep;
#pragma unroll
        for (int x = 0; x < F; x++) {
            a[x] = __builtin_bit_cast(int4v, *(lds_ptr4)(uintptr_t)(at + (wave / 2 * W + x * 32) * kStep));
            w[x] = __builtin_bit_cast(int4v, *(lds_ptr4)(uintptr_t)(at + (T + wave % 2 * W + x * 32) * kStep));
        }
    };
    int16v acc[F][F];
#pragma unroll
    for (int x = 0; x < F; x++)
#pragma unroll
        for (int y = 0; y < F; y++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[x][y][r] = 0;
    auto multiply = [&](const int4v *a, const int4v *w) {
#pragma unroll
        for (int x = 0; x < F; x++)
#pragma unroll
            for (int y = 0; y < F; y++)
                acc[x][y] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[x], w[y], acc[x][y], 0, 0, 0);
    };
    auto all_here = [] { asm volatile("s_barrier" ::: "memory"); };
    int4v a0[F], w0[F], a1[F], w1[F];
    fetch(0);
    fetch(1);
    fetch(2);
    wait_copies<COPIES>();
    all_here();
    read(0, 0, a0, w0);
    const int64_t steps = (p.inner + kStep - 1) / kStep;
    for (int64_t s = 0; s < steps; s++) {
        fetch(s + 3);                            // where step s - 1 was: all have read it
        read(s, 1, a1, w1);
        multiply(a0, w0);
        read(s + 1, 0, a0, w0);
        multiply(a1, w1);
        wait_copies<COPIES>();                   // step s + 2 is here
        all_here();
    }
    wait_copies<0>();
    all_here();
    float sw[8];
    const int64_t j = j0 + wave % 2 * W;
    column_scales<W>(p, j, sw);
#pragma unroll
    for (int x = 0; x < F; x++)
        put_slab<W>(p, i0 + wave / 2 * W + x * 32, j, acc[x], (int *)lds + wave * 32 * (W + 8), sw,
                    wide);
}

// The same for operands off 16-byte boundaries or rows that no whole number of pieces
// fills: 128 x 128 outputs, operands by way of registers.
constexpr int kPitch = kStep + 16;
__global__ __launch_bounds__(256) void int8_any(SeqInt8Product p, bool wide) {
    constexpr int T = 128, W = 64;
    __shared__ __align__(16) int8_t lds[4 * 32 * (W + 8) * 4];         // 2 T kPitch, or the sums
    int8_t *as = lds, *ws = lds + T * kPitch;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int64_t ti, tj;
    if (!tile_of(block_number(), (p.m + T - 1) / T, (p.n + T - 1) / T, ti, tj)) return;
    const int64_t i0 = ti * T, j0 = tj * T;
    const int wi = wave / 2 * W, wj = wave % 2 * W;
    int16v acc[2][2];
#pragma unroll
    for (int x = 0; x < 2; x++)
#pragma unroll
        for (int y = 0; y < 2; y++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[x][y][r] = 0;
    for (int64_t l = 0; l < p.inner; l += kStep) {
        uint4v va[2], vw[2];
#pragma unroll
        for (int x = 0; x < 2; x++) {
            const int at = x * 256 + tid, row = at / 4, col = at % 4 * 16;
            va[x] = vw[x] = uint4v{0, 0, 0, 0};
            if (i0 + row < p.m) va[x] = row_piece(p.a + (i0 + row) * p.a_row, l + col, p.inner);
            if (j0 + row < p.n) vw[x] = row_piece(p.w + (j0 + row) * p.w_row, l + col, p.inner);
        }
        __syncthreads();
#pragma unroll
        for (int x = 0; x < 2; x++) {
            const int at = x * 256 + tid, row = at / 4, col = at % 4 * 16;
            *(uint4v *)(as + row * kPitch + col) = va[x];
            *(uint4v *)(ws + row * kPitch + col) = vw[x];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kStep; k += 32) {
            int4v a[2], w[2];
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int col = k + lane / 32 * 16;
                a[x] = *(const int4v *)(as + (wi + x * 32 + lane % 32) * kPitch + col);
                w[x] = *(const int4v *)(ws + (wj + x * 32 + lane % 32) * kPitch + col);
            }
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
                for (int y = 0; y < 2; y++)
                    acc[x][y] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[x], w[y], acc[x][y], 0, 0, 0);
        }
    }
    __syncthreads();
    float sw[8];
    column_scales<W>(p, j0 + wj, sw);
#pragma unroll
    for (int x = 0; x < 2; x++)
        put_slab<W>(p, i0 + wi + x * 32, j0 + wj, acc[x], (int *)lds + wave * 32 * (W + 8), sw, wide);
}

// Few tokens: 16 channels a block and up to 16 M tokens, the terms cut among eight waves,
// which read both operands from memory as the 16x16x64 product takes them and join their
// sums in LDS. The weights are read once, which is what bounds it.
template <int M>
__global__ __launch_bounds__(512) void int8_few(SeqInt8Product p) {
    constexpr int WAVES = 8;
    __shared__ int4v sums[WAVES][M][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t j0 = block_number() * 16ll;
    if (j0 >= p.n) return;
    const int row = lane % 16, col = lane / 16 * 16;
    const int64_t j = j0 + row < p.n ? j0 + row : p.n - 1;
    const int8_t *w = p.w + j * p.w_row + col;
    const int8_t *a[M];
#pragma unroll
    for (int x = 0; x < M; x++) {
        const int64_t i = x * 16 + row;
        a[x] = p.a + (i < p.m ? i : p.m - 1) * p.a_row + col;
    }
    int4v acc[M];
#pragma unroll
    for (int x = 0; x < M; x++) acc[x] = int4v{0, 0, 0, 0};
    const int4v zero = {0, 0, 0, 0};
#pragma unroll 4
    for (int64_t l = wave * 64; l < p.inner; l += WAVES * 64) {
        const bool in = l + col < p.inner;       // the weights' zero is enough
        int4v vw = zero, va[M];
        if (in) vw = *(const int4v *)(w + l);
#pragma unroll
        for (int x = 0; x < M; x++) {
            va[x] = zero;
            if (in) va[x] = *(const int4v *)(a[x] + l);
        }
#pragma unroll
        for (int x = 0; x < M; x++)
            acc[x] = __builtin_amdgcn_mfma_i32_16x16x64_i8(va[x], vw, acc[x], 0, 0, 0);
    }
#pragma unroll
    for (int x = 0; x < M; x++) sums[wave][x][lane] = acc[x];
    __syncthreads();
    for (int at = tid; at < M * 64; at += 512) {
        int4v s = sums[0][at / 64][lane];
#pragma unroll
        for (int v = 1; v < WAVES; v++) s += sums[v][at / 64][lane];
        const int64_t jj = j0 + lane % 16;
        if (jj >= p.n) continue;
        const float sw = p.w_scale[jj];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int64_t i = at / 64 * 16 + lane / 16 * 4 + r;
            if (i < p.m) put1(p.o, p.out_dtype, i * p.o_row + jj, (float)s[r] * p.a_scale[i] * sw);
        }
    }
}

int64_t tiles_of(const SeqInt8Product &p, int64_t t) {
    return ((p.m + t - 1) / t) * ((p.n + t - 1) / t);
}

int check_int8(const SeqInt8Product *p) {
    if (!p || p->struct_size != (int32_t)sizeof(SeqInt8Product)) return CO_ERR_NULLARG;
    if (p->m < 0 || p->n < 0 || p->inner < 0) return CO_ERR_NULLARG;
    if (p->m > SEQ_MAX_ROWS || p->n > SEQ_MAX_ROWS || p->inner > SEQ_MAX_INNER) return CO_ERR_BOUNDS;
    if (!float_type(p->out_dtype)) return CO_ERR_DATA;
    return tiles_of(*p, 64) > SEQ_MAX_ROWS ? CO_ERR_BOUNDS : CO_OK;
}

template <int M> void launch_few(const SeqInt8Product &p, hipStream_t s) {
    int8_few<M><<<grid_of((p.n + 15) / 16, 512), 512, 0, s>>>(p);
}
template <int T> void launch_tiles(const SeqInt8Product &p, bool wide, hipStream_t s) {
    const int64_t blocks = (tiles_of(p, T) + 7) / 8 * 8;
    int8_tiles<T><<<grid_of(blocks, 256), 256, kStages * tile_bytes<T>(), s>>>(p, wide);
}

}  // namespace seq

extern "C" int64_t seq_int8_product_workspace(const SeqInt8Product *p) {
    const int rc = seq::check_int8(p);
    return rc == CO_OK ? 0 : (rc > 0 ? -rc : rc);
}

extern "C" int seq_int8_product(const SeqInt8Product *p, void *stream) {
    const int rc = seq::check_int8(p);
    if (rc != CO_OK) return rc;
    if (p->m == 0 || p->n == 0) return CO_OK;
    if (!p->a_scale || !p->w_scale || !p->o || (p->inner && (!p->a || !p->w)))
        return CO_ERR_NULLARG;
    hipStream_t s = (hipStream_t)stream;
    const bool wide = seq::in_eights(p->o, p->o_row);
    const bool pieces = !(((uintptr_t)p->a | (uintptr_t)p->w) & 15) && p->a_row % 16 == 0 &&
                        p->w_row % 16 == 0 && p->inner % 16 == 0;
    if (!pieces) {
        const int64_t blocks = (seq::tiles_of(*p, 128) + 7) / 8 * 8;
        seq::int8_any<<<seq::grid_of(blocks, 256), 256, 0, s>>>(*p, wide);
    } else if (p->m <= 16) {
        seq::launch_few<1>(*p, s);
    } else if (p->m <= 32) {
        seq::launch_few<2>(*p, s);
    } else if (p->m <= 64) {
        seq::launch_few<4>(*p, s);
    } else if (seq::tiles_of(*p, 256) >= 256) {
        seq::launch_tiles<256>(*p, wide, s);
    } else if (seq::tiles_of(*p, 128) >= 128) {
        seq::launch_tiles<128>(*p, wide, s);
    } else {
        seq::launch_tiles<64>(*p, wide, s);
    }
    return seq::launch_status();
}
