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

// (sum sa) sw. The first product passes float32's largest number only where |sa| is 2^96 or
// more (a sum is below 2^31): sa is taken 2^-64 times as large there, and sw as much larger,
// which changes no bit of the product. Where sw so passes the largest number, the product
// does too, but for a sum of 0.
__device__ inline bool large_scale(float sa) { return fabsf(sa) >= 0x1p96f; }
__device__ inline float lowered(float sa) { return large_scale(sa) ? sa * 0x1p-64f : sa; }
__device__ inline float raised(float sw) {
    const float up = sw * 0x1p64f;
    return fabsf(up) < __builtin_inff() || fabsf(sw) == __builtin_inff() || sw != sw
               ? up : copysignf(3.4028235e38f, sw);
}
__device__ inline float scaled(int sum, float sa, float sw) {
    return (float)sum * lowered(sa) * (large_scale(sa) ? raised(sw) : sw);
}

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

// A wave's F x F products of 32 channels by 32 tokens to memory; scales: the wave's, in
// LDS. A lane of a product has one token's channels 8 g + 4 h .. + 3, h its half of the
// wave; two groups g change halves, and it has 8 channels side by side. 32 tokens' go
// through LDS to leave as whole rows: stores of 32 bytes a row took 156 us for 8,192 x
// 16,384 outputs of 128 terms. Those of large tiles pass the caches by, which hold operands
// that are read again: 8,192 x 4,096 x 16,384 took 9 in 100 less time. WIDE: every 8
// channels lie on a boundary of 16 bytes and are all inside or all outside. RAW: the sums as
// they are, in a float's place. w_scale holds the N channels' scales and, a tile's side
// behind, the `raised` ones for tokens with a large scale: a lane's address says which (a branch
// around another product took 97.3 us rather than 90.7 for 8,192 x 16,384 outputs of 128 terms).
template <typename O, int F> constexpr int slab_pitch() { return F * 32 + 16 / (int)sizeof(O); }
template <typename O, bool WIDE, int F, bool RAW>
__device__ inline void put_sums(const SeqInt8Product &p, int64_t i0, int64_t j0,
                                const int16v (&acc)[F][F], const float *a_scale,
                                const float *w_scale, O *slab) {
    constexpr int N = F * 32, PITCH = slab_pitch<O, F>();
    const int lane = threadIdx.x & 63;
    float scales[F];                             // here before the first address needs one
#pragma unroll
    for (int x = 0; x < F; x++) scales[x] = a_scale[x * 32 + lane % 32];
#pragma unroll
    for (int x = 0; x < F; x++) {
        const float *ws = w_scale + (large_scale(scales[x]) ? 2 * N : 0);
        const float sa = lowered(scales[x]);
        wave_sync();
#pragma unroll
        for (int y = 0; y < F; y++)
#pragma unroll
            for (int g = 0; g < 2; g++) {
                __builtin_amdgcn_sched_barrier(0);           // few sums in registers at a time
                const int col = y * 32 + g * 16 + lane / 32 * 8;
                const float4v lo = *(const float4v *)(ws + col);
                const float4v hi = *(const float4v *)(ws + col + 4);
                float f[8];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const auto s = __builtin_amdgcn_permlane32_swap(
                        (uint32_t)acc[x][y][g * 8 + e], (uint32_t)acc[x][y][g * 8 + 4 + e], false, false);
                    if constexpr (RAW) {
                        f[e] = __uint_as_float(s[0]);
                        f[4 + e] = __uint_as_float(s[1]);
                    } else {
                        f[e] = (float)(int)s[0] * sa * lo[e];
                        f[4 + e] = (float)(int)s[1] * sa * hi[e];
                    }
                }
                Eight<O>::put(slab + lane % 32 * PITCH + col, f);
            }
        wave_sync();
        const int64_t i = i0 + x * 32;
        if constexpr (WIDE) {
            constexpr int PER = 16 / sizeof(O), LANES = N / PER, ROWS = LANES < 64 ? 64 / LANES : 1;
            const int col = lane % LANES * PER;
            O *to = (O *)p.o + (i + lane / LANES) * p.o_row + j0 + col;
            const bool in = j0 + col < p.n;
#pragma unroll
            for (int r = lane / LANES; r < 32; r += ROWS) {
                const uint4v v = *(const uint4v *)(slab + r * PITCH + col);
                if (in && i + r < p.m) {
                    if constexpr (F == 4) __builtin_nontemporal_store(v, (uint4v *)to);
                    else *(uint4v *)to = v;
                }
                to += ROWS * p.o_row;
            }
        } else {
            for (int r = 0; r < 32 && i + r < p.m; r++)
#pragma unroll
                for (int c = lane; c < N; c += 64)
                    if (j0 + c < p.n) ((O *)p.o)[(i + r) * p.o_row + j0 + c] = slab[r * PITCH + c];
        }
    }
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
// to LDS past the registers into five buffers, so that a copy has two and a half steps to
// arrive: a step of 256 x 256 is a microsecond's half, an operand's way from beyond the
// die's cache more than one. A step's second half is read from LDS while its first is
// multiplied, and the next one's first with its second. Row r of a buffer holds its four
// pieces of 16 bytes turned by r / 4, so that 16 lanes' reads meet every bank once. At 8,192
// x 8,192 x 16,384 the products alone take 578 us (3.8 POP/s at the clock that the card
// falls to), with the reads from LDS 718, with the copies into it 718, with both 941. LDS has
// time for both (some 770 clocks a step, the products 1,024): what is lost is their overlap, with
// one wave a SIMD, a barrier a step and the matrix unit busy 58 in 100 of the time. 8,192 x 4,096
// x 16,384 take 490 to 690 us by the clock that the card is at, 530 to 570 from a cool start.
constexpr int kStep = 64, kStages = 5, kMostCuts = 32;
template <int T> constexpr int tile_bytes() { return 2 * T * kStep; }

// RAW: a tile's terms are cut among `cuts` blocks, `terms` each, which leave their sums in
// `parts` [cuts, m, n rounded up to 8] for int8_join.
template <typename O, bool WIDE, int T, bool RAW>
__global__ __launch_bounds__(256, T == 256 ? 1 : 2) void int8_tiles(SeqInt8Product p, int cuts,
                                                                    int terms, float *parts) {
    constexpr int W = T / 2, F = W / 32;         // a wave's side, in products
    constexpr int COPIES = tile_bytes<T>() / 4096;           // a wave's copies of a step
    constexpr uint32_t BYTES = tile_bytes<T>(), ALL = kStages * BYTES;
    extern __shared__ __align__(16) unsigned char lds[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int64_t ti, tj;
    int64_t block = block_number(), cut = 0;
    if constexpr (RAW) {                         // a cut's blocks are a multiple of eight
        const int64_t each = (((p.m + T - 1) / T) * ((p.n + T - 1) / T) + 7) / 8 * 8;
        cut = block / each;
        block %= each;
        if (cut >= cuts) return;                 // the launch's last numbers
    }
    if (!tile_of(block, (p.m + T - 1) / T, (p.n + T - 1) / T, ti, tj)) return;
    const int64_t i0 = ti * T, j0 = tj * T;
    float a_scale = 0.0f, w_scale = 0.0f;        // of row and column tid
    if (!RAW && tid < T && i0 + tid < p.m) a_scale = p.a_scale[i0 + tid];
    if (!RAW && tid < T && j0 + tid < p.n) w_scale = p.w_scale[j0 + tid];
    const uint32_t base = lds_address(lds);
    // Waves 0 and 1 bring a, waves 2 and 3 w. Copy x fills 16 rows, this lane row lane / 4,
    // place lane % 4; rows past the last are the last.
    const bool is_a = wave < 2;
    const int64_t row_bytes = is_a ? p.a_row : p.w_row, first = is_a ? i0 : j0;
    const int64_t left = (is_a ? p.m : p.n) - 1 - first;
    const int8_t *from = (is_a ? p.a : p.w) + first * row_bytes;
    int inner = (int)p.inner;
    if constexpr (RAW) {
        from += cut * terms;
        inner -= (int)cut * terms;
        if (inner > terms) inner = terms;
    }
    uint32_t offset[COPIES];                     // below 2^32: the launch sees to it
    int piece[COPIES];
#pragma unroll
    for (int x = 0; x < COPIES; x++) {
        const int row = (wave % 2 * COPIES + x) * 16 + lane / 4;
        piece[x] = (lane % 4 - row / 4 % 4 + 4) % 4 * 16;
        offset[x] = (uint32_t)((row < left ? row : (int)left) * row_bytes) + piece[x];
    }
    // Copy x of the step at l to the buffer at `to`. CUT: of a step that passes the rows' end,
    // whose pieces there are zeros; steps past the last are, so that every step counts alike.
    auto copy = [&](int l, uint32_t to, int x, auto cut) {
        to += base + wave * COPIES * 1024 + x * 1024;
        if constexpr (cut.value) {
            uint32_t o = offset[x];
            asm volatile("" : "+v"(o));          // no addresses kept over steps
            copy_to_lds16(piece[x] < inner - l ? (const void *)(from + l + o) : kZeros, to);
        } else {
            copy_to_lds16(from + l, offset[x], to);
        }
    };
    const int row = lane % 32;
    auto read = [&](uint32_t at, int half, int4v *a, int4v *w) {
        at += base + (half * 2 + lane / 32 + row / 4) % 4 * 16 + row * kStep;
#pragma unroll
        for (int x = 0; x < F; x++) {
            const uint32_t ra = at + (wave / 2 * W + x * 32) * kStep;
            const uint32_t rw = at + (T + wave % 2 * W + x * 32) * kStep;
            a[x] = __builtin_bit_cast(int4v, *(lds_ptr4)(uintptr_t)ra);
            w[x] = __builtin_bit_cast(int4v, *(lds_ptr4)(uintptr_t)rw);
        }
    };
    int16v acc[F][F];
#pragma unroll
    for (int x = 0; x < F; x++)
#pragma unroll
        for (int y = 0; y < F; y++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[x][y][r] = 0;
    int4v a0[F], w0[F], a1[F], w1[F];
    // until at most the newest N steps' copies are on their way, everyone's
    auto wait = [&](auto steps) {
        wait_copies<steps.value * COPIES>();
        asm volatile("s_barrier" ::: "memory");
    };
    uint32_t here = 0, ahead = (kStages - 1) * BYTES;        // buffers of this step and of the copies
    int l = 0;
    // Copies go between products: issued together they would leave the matrix unit idle.
    constexpr int EVERY = F * F / COPIES ? F * F / COPIES : 1;
    auto step = [&](auto cut) {
        read(here, 1, a1, w1);
#pragma unroll
        for (int x = 0; x < F; x++)
#pragma unroll
            for (int y = 0; y < F; y++) {
                const int at = x * F + y;
                if (at % EVERY == 0)             // to where the step before was: all have read it
#pragma unroll
                    for (int c = at / EVERY; c < COPIES; c += F * F)
                        copy(l + (kStages - 1) * kStep, ahead, c, cut);
                __builtin_amdgcn_sched_barrier(0);
                acc[x][y] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w0[y], a0[x], acc[x][y], 0, 0, 0);
            }
        __builtin_amdgcn_sched_barrier(0);
        wait(Const<kStages - 2>());              // the next step is here
        ahead = here;
        here = here + BYTES == ALL ? 0 : here + BYTES;
        // a1 and w1 are too, which the compiler is told: it would wait for the newer reads
#pragma unroll
        for (int x = 0; x < F; x++) asm volatile("" : "+v"(a1[x]), "+v"(w1[x]));
        read(here, 0, a0, w0);
#pragma unroll
        for (int x = 0; x < F; x++)
#pragma unroll
            for (int y = 0; y < F; y++)
                acc[x][y] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w1[y], a1[x], acc[x][y], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        l += kStep;
    };
#pragma unroll
    for (int x = 0; x < (kStages - 1) * COPIES; x++)
        copy(x / COPIES * kStep, x / COPIES * BYTES, x % COPIES, Const<1>());
    wait(Const<kStages - 2>());
    read(here, 0, a0, w0);
    const int whole = inner - kStages * kStep;
    while (l <= whole) step(Const<0>());
    while (l < inner) step(Const<1>());
    wait(Const<0>());                            // the last step's reads are done
    float *scales = (float *)lds;
    static_assert(12 * T + 4 * 32 * slab_pitch<O, F>() * sizeof(O) <= ALL, "");
    if (tid < T) {
        scales[tid] = a_scale;
        scales[T + tid] = w_scale;
        scales[2 * T + tid] = raised(w_scale);
    }
    __syncthreads();
    if constexpr (RAW) {                         // whole eights of columns, those past n too
        const int64_t pitch = (p.n + 7) / 8 * 8;
        p.o = parts + cut * p.m * pitch;
        p.o_row = p.n = pitch;
    }
    put_sums<O, WIDE, F, RAW>(p, i0 + wave / 2 * W, j0 + wave % 2 * W, acc, scales + wave / 2 * W,
                              scales + T + wave % 2 * W,
                              (O *)(scales + 3 * T) + wave * 32 * slab_pitch<O, F>());
}

// Adds up the cuts' sums, which are exact in any order: eight columns a thread. A launch more
// and the way of the sums through the last cache: 5 us with 16 cuts of 24 x 1,024, 8 with
// four of 64 x 4,096.
__global__ __launch_bounds__(256) void int8_join(SeqInt8Product p, int cuts, const int *parts) {
    const int64_t eights = (p.n + 7) / 8, at = (int64_t)block_number() * 256 + threadIdx.x;
    const int64_t i = at / eights, j = at % eights * 8;
    if (i >= p.m) return;
    const int4v *from = (const int4v *)(parts + at * 8);
    const int64_t step = p.m * eights * 2;
    int4v lo = {0, 0, 0, 0}, hi = lo;
#pragma unroll 8
    for (int c = 0; c < cuts; c++) {
        lo += from[c * step];
        hi += from[c * step + 1];
    }
    const int n = cells_of<true>(p.n, (int)(j / 8));
    const float sa = p.a_scale[i];
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; e++)
        f[e] = e < n ? scaled(e < 4 ? lo[e % 4] : hi[e % 4], sa, p.w_scale[j + e]) : 0.0f;
    put_cells<true>(p.o, p.out_dtype, i * p.o_row + j, f, n);
}

// Rows off 16-byte boundaries, or that no whole number of pieces fills, are laid out anew
// first, padded with zeros: 2^g threads a row, a piece each at a time. Products that read
// such rows as they lie took 280 us rather than 158 for 8,192 x 4,095 x 4,096, and 48 rather
// than 29 for 24 x 4,095 x 6,144.
__global__ __launch_bounds__(256) void int8_pack(const int8_t *from, int64_t row, int64_t rows,
                                                 int64_t inner, int g, int8_t *to, int64_t to_row) {
    const int64_t r = (int64_t)block_number() * (256 >> g) + (threadIdx.x >> g);
    if (r >= rows) return;
#pragma unroll 4
    for (int64_t l = (threadIdx.x & ((1 << g) - 1)) * 16; l < to_row; l += 16 << g)
        *(uint4v *)(to + r * to_row + l) = row_piece(from + r * row, l, inner);
}

// Few tokens: 16 channels a block and up to 16 M tokens, the terms cut among eight waves,
// which read both operands from memory as the 16x16x64 product takes them and join their
// sums in LDS. The weights are read once. 1 x 4,096 x 4,096 takes 4.4 us, 3.8 TB/s of what the
// caches hold, 24 x 4,096 x 4,096 7.5: the steps of a wave wait for the way to memory.
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
            if (i < p.m) put1(p.o, p.out_dtype, i * p.o_row + jj, scaled(s[r], p.a_scale[i], sw));
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

// Whether rows are laid out anew: whole pieces on their boundaries, and 256 rows and a step
// within 2^32 bytes
bool needs_pack(const SeqInt8Product &p, const int8_t *x, int64_t row) {
    return p.inner % 16 || ((uintptr_t)x & 15) || row % 16 || row < 0 || row >= 1 << 23;
}
int64_t packed_row(const SeqInt8Product &p) { return (p.inner + 15) / 16 * 16; }
int64_t packed_bytes(int64_t rows, const SeqInt8Product &p) {
    return (rows * packed_row(p) + 255) / 256 * 256;
}

// How a product is made: by int8_few<few>, or tiles of `side`, their terms in `cuts`.
struct Int8Plan { int few, side, cuts, terms; };

// Tiles first, those that take the least time: 256 of them, one to a compute unit, take 9, 21
// and 46 us for 4,096 terms (sides of 64, 128 and 256), and more take as many times as long
// (512 x 4,096 x 4,096: 19, 19, 48 us; 1,024: 36, 24, 52; 3,000: 97, 61, 58; 4,096: 122, 80,
// 66). Then the same with the terms cut, whose sums are written and joined, and few tokens'
// own kernel, by the times in ns that these come to. Tiles, their terms in 2, 4, 8 and 16,
// few tokens' kernel, in us:
//   24 x 4,096 x 4,096    10.0  10.5   9.6   9.7  12.5    7.6
//   24 x 4,096 x 6,144    10.1  10.8  10.9  12.3  15.2   12.1
//   24 x 16,384 x 1,024   31.0  21.1  14.4  10.7  10.1   20.5
//   16 x 16,384 x 4,096   31.4  22.3  16.7  16.9  17.9   16.9
//   64 x 4,096 x 4,096    10.1  11.2  10.8  13.3  18.6
//   64 x 16,384 x 4,096   34.0  24.1  18.3  19.6  21.8
//   512 x 16,384 x 4,096  58.0  48.8  55.1  61.9  77.0
// What is taken is the least of a row, or within 1 in 20 of it.
Int8Plan int8_plan(const SeqInt8Product &p) {
    const int64_t inner = packed_row(p);
    auto rounds = [](int64_t blocks) { return (blocks + 255) / 256; };
    const int64_t t64 = rounds(tiles_of(p, 64)), t128 = rounds(tiles_of(p, 128)),
                  t256 = rounds(tiles_of(p, 256));
    Int8Plan r = {0, 256, 1, 0};
    if (9 * t64 <= 21 * t128 && 9 * t64 <= 46 * t256) r.side = 64;
    else if (21 * t128 <= 46 * t256) r.side = 128;
    int64_t best = r.side == 64 ? 2600 + t64 * 7500 * inner / 4096
                 : r.side == 128 ? 3000 + t128 * 18000 * inner / 4096
                                 : 4000 + t256 * 42000 * inner / 4096;
    auto cut = [&](int side, int64_t base, int64_t each, int cuts) {
        const int64_t time = base + rounds(tiles_of(p, side) * cuts) * each * (inner / cuts) / 4096 +
                             4500 + p.m * p.n / 600 * cuts;
        if (time < best) {
            best = time;
            r.side = side;
            r.cuts = cuts;
        }
    };
    const int64_t tiles = tiles_of(p, 64);       // enough of them leave nothing to cut for
    for (int cuts = 2; cuts <= kMostCuts && inner / cuts >= 512 && tiles * cuts <= 2048; cuts++) {
        cut(64, 2600, 7500, cuts);
        cut(128, 3000, 18000, cuts);
    }
    const int64_t channels = rounds((p.n + 15) / 16);
    if (p.m <= 16 && 2500 + channels * 3500 * inner / 4096 < best) r = {1, 0, 1, 0};
    else if (p.m > 16 && p.m <= 32 && 2700 + channels * 4500 * inner / 4096 < best) r = {2, 0, 1, 0};
    if (r.cuts > 1) {
        r.terms = (int)((inner + r.cuts - 1) / r.cuts + kStep - 1) / kStep * kStep;
        r.cuts = (int)((inner + r.terms - 1) / r.terms);
    }
    return r;
}
int64_t parts_bytes(const SeqInt8Product &p, const Int8Plan &r) {
    return r.cuts > 1 ? 4 * r.cuts * p.m * ((p.n + 7) / 8 * 8) : 0;
}
int64_t int8_bytes(const SeqInt8Product &p) {
    if (p.m == 0 || p.n == 0 || p.inner == 0) return 0;
    return (needs_pack(p, p.a, p.a_row) ? packed_bytes(p.m, p) : 0) +
           (needs_pack(p, p.w, p.w_row) ? packed_bytes(p.n, p) : 0) + parts_bytes(p, int8_plan(p));
}
void pack(const int8_t *&x, int64_t &row, int64_t rows, const SeqInt8Product &p, char *&ws,
          hipStream_t s) {
    if (!needs_pack(p, x, row)) return;
    const int64_t to_row = packed_row(p);
    int g = 0;
    while (g < 8 && (16 << g) < to_row) g++;
    const int64_t each = 256 >> g;
    int8_pack<<<grid_of((rows + each - 1) / each, 256), 256, 0, s>>>(x, row, rows, p.inner, g,
                                                                     (int8_t *)ws, to_row);
    x = (const int8_t *)ws;
    row = to_row;
    ws += packed_bytes(rows, p);
}

template <int M> void launch_few(const SeqInt8Product &p, hipStream_t s) {
    int8_few<M><<<grid_of((p.n + 15) / 16, 512), 512, 0, s>>>(p);
}
template <typename O, bool WIDE, int T> void launch_tiles(const SeqInt8Product &p, hipStream_t s) {
    const int64_t blocks = (tiles_of(p, T) + 7) / 8 * 8;
    int8_tiles<O, WIDE, T, false><<<grid_of(blocks, 256), 256, kStages * tile_bytes<T>(), s>>>(
        p, 1, 0, nullptr);
}
template <int T> void launch_cuts(const SeqInt8Product &p, const Int8Plan &r, void *parts,
                                  hipStream_t s) {
    const int64_t blocks = (tiles_of(p, T) + 7) / 8 * 8 * r.cuts;
    int8_tiles<float, true, T, true><<<grid_of(blocks, 256), 256, kStages * tile_bytes<T>(), s>>>(
        p, r.cuts, r.terms, (float *)parts);
    const int64_t threads = p.m * ((p.n + 7) / 8);
    int8_join<<<grid_of((threads + 255) / 256, 256), 256, 0, s>>>(p, r.cuts, (const int *)parts);
}
template <typename O, bool WIDE>
void launch_tiles(const SeqInt8Product &p, const Int8Plan &r, hipStream_t s) {
    if (r.side == 64) launch_tiles<O, WIDE, 64>(p, s);
    else if (r.side == 128) launch_tiles<O, WIDE, 128>(p, s);
    else launch_tiles<O, WIDE, 256>(p, s);
}
template <typename O> void launch_tiles(const SeqInt8Product &p, const Int8Plan &r, hipStream_t s) {
    if (in_eights(p.o, p.o_row) && p.n % 8 == 0) launch_tiles<O, true>(p, r, s);
    else launch_tiles<O, false>(p, r, s);
}

}  // namespace seq

extern "C" int64_t seq_int8_product_workspace(const SeqInt8Product *p) {
    const int rc = seq::check_int8(p);
    if (rc != CO_OK) return rc > 0 ? -rc : rc;
    return seq::int8_bytes(*p);
}

extern "C" int seq_int8_product(const SeqInt8Product *p, void *stream) {
    const int rc = seq::check_int8(p);
    if (rc != CO_OK) return rc;
    if (p->m == 0 || p->n == 0) return CO_OK;
    if (!p->a_scale || !p->w_scale || !p->o || (p->inner && (!p->a || !p->w)))
        return CO_ERR_NULLARG;
    const int64_t bytes = seq::int8_bytes(*p);
    if (bytes && !p->workspace) return CO_ERR_NULLARG;
    if (p->workspace_bytes < bytes || (bytes && ((uintptr_t)p->workspace & 255))) return CO_ERR_DATA;
    hipStream_t s = (hipStream_t)stream;
    SeqInt8Product q = *p;
    const seq::Int8Plan plan = seq::int8_plan(q);
    char *ws = (char *)q.workspace;
    if (q.inner) {
        seq::pack(q.a, q.a_row, q.m, *p, ws, s);
        seq::pack(q.w, q.w_row, q.n, *p, ws, s);
        q.inner = seq::packed_row(*p);           // zeros beyond it, or nothing
    } else {
        q.a_row = q.w_row = 0;                   // no row is read
    }
    if (plan.few == 1) {
        seq::launch_few<1>(q, s);
    } else if (plan.few) {
        seq::launch_few<2>(q, s);
    } else if (plan.cuts > 1) {
        if (plan.side == 64) seq::launch_cuts<64>(q, plan, ws, s);
        else seq::launch_cuts<128>(q, plan, ws, s);
    } else {
        switch (q.out_dtype) {
            case SEQ_FP32: seq::launch_tiles<float>(q, plan, s); break;
            case SEQ_BF16: seq::launch_tiles<__bf16>(q, plan, s); break;
            default: seq::launch_tiles<_Float16>(q, plan, s); break;
        }
    }
    return seq::launch_status();
}
