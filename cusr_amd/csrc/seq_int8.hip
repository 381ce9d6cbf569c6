// seq_int8.hip -- product of 8-bit integers with a scale for each row of both sides
// (include/cusr_seq.h, seq_int8_product).
//
// o[i, j] = a_scale[i] w_scale[j] sum_l a[i, l] w[j, l]. Both sides lie along l, which is
// what the matrix instruction takes: lane l of either operand of the 32x32x32 product
// holds 16 values of row l % 32 at l / 32 * 16. The sum is exact in 32 bits up to 131,071
// terms.
#include "seq_rows.h"

namespace seq {

typedef int int4v __attribute__((ext_vector_type(4)));
typedef int int16v __attribute__((ext_vector_type(16)));

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

// 128 x 128 outputs a block of four waves, 64 x 64 a wave, 64 terms at a time.
constexpr int kTile = 128, kStep = 64, kPitch = kStep + 16;
__global__ __launch_bounds__(256) void int8_tiles(SeqInt8Product p) {
    __shared__ __align__(16) int8_t as[kTile * kPitch], ws[kTile * kPitch];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t columns = (p.n + kTile - 1) / kTile;
    const int64_t block = block_number();
    const int64_t i0 = block / columns * kTile, j0 = block % columns * kTile;
    if (i0 >= p.m) return;
    const int wi = wave / 2 * 64, wj = wave % 2 * 64;
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
#pragma unroll
    for (int y = 0; y < 2; y++) {
        const int64_t j = j0 + wj + y * 32 + lane % 32;
        if (j >= p.n) continue;
        const float sw = p.w_scale[j];
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int64_t i = i0 + wi + x * 32 + 8 * (r / 4) + 4 * (lane / 32) + r % 4;
                if (i < p.m)
                    put1(p.o, p.out_dtype, i * p.o_row + j, (float)acc[x][y][r] * p.a_scale[i] * sw);
            }
    }
}

int check_int8(const SeqInt8Product *p) {
    if (!p || p->struct_size != (int32_t)sizeof(SeqInt8Product)) return CO_ERR_NULLARG;
    if (p->m < 0 || p->n < 0 || p->inner < 0) return CO_ERR_NULLARG;
    if (p->m > SEQ_MAX_ROWS || p->n > SEQ_MAX_ROWS || p->inner > SEQ_MAX_INNER) return CO_ERR_BOUNDS;
    if (!float_type(p->out_dtype)) return CO_ERR_DATA;
    const int64_t blocks = ((p->m + kTile - 1) / kTile) * ((p->n + kTile - 1) / kTile);
    return blocks > SEQ_MAX_ROWS ? CO_ERR_BOUNDS : CO_OK;
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
    const int64_t blocks = ((p->m + seq::kTile - 1) / seq::kTile) *
                           ((p->n + seq::kTile - 1) / seq::kTile);
    seq::int8_tiles<<<seq::grid_of(blocks, 256), 256, 0, s>>>(*p);
    return seq::launch_status();
}
