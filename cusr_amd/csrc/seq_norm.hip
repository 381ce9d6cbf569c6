// seq_norm.hip -- root-mean-square norm of rows with the residual's addition, to a type
// or to 8-bit integers, and its gradient (include/cusr_seq.h, seq_norm, seq_norm_grad).
//
// A row needs one sum before its first output value: rho = (mean h^2 + eps)^-1/2, and
// for 8 bits its largest magnitude too. The bound is memory: a row stays in registers
// between its one reading and its one writing.
#include "seq_rows.h"

namespace seq {

// x + residual as the stream holds it
template <typename H> __device__ inline float stream_sum(float x, float r) {
    return (float)(H)(x + r);
}

__device__ inline float rms_factor(float sum, int64_t width, float eps) {
    return 1.0f / sqrtf(sum / (float)width + eps);
}

// 8-bit integers of a row whose largest magnitude is `most`. The quotient by the scale is
// rounded as a division is. A product with the scale's reciprocal is off by 2^-16 at most;
// where that leaves the integer open, next to a half, the division is made: 8,192 rows of
// 4,096 in bf16 take 21 us, and some 5 more with a division for each value.
struct Bits8 {
    float scale, inverse;
    __device__ explicit Bits8(float most) {
        scale = most < __builtin_inff() ? most * (1.0f / 127.0f) : __builtin_nanf("");
        // no number, which leaves every integer open, where the scale has not all its bits
        inverse = scale >= 0x1p-126f ? 1.0f / scale : __builtin_nanf("");
    }
    __device__ int of(float y) const {
        const float near = y * inverse;
        float q = rintf(near);
        if (!(fabsf(near - q) <= 0.4995f))
            q = scale > 0.0f ? fminf(fmaxf(rintf(y / scale), -127.0f), 127.0f) : 0.0f;
        return (int)q;
    }
};

// A row per group of G threads, NV parts of 8 values a thread: every load of a row is on its
// way before the first sum, and the row is read once. Memory bounds it: 1.3 M rows of 128 in
// bf16 into a stream in fp32 (2.0 GB) take 336 us at best, 5.9 TB/s, 16,383 of 4,096 into one
// in bf16 (537 MB) 87, 6.2 TB/s, 24 of 4,096 3.4 us, which are three trips to memory and two
// barriers. The gain is asked for before the first sum is joined.
template <typename X, typename H, bool RES, bool ANY, int G, int NV>
__global__ __launch_bounds__(G < 256 ? 256 : G) void norm_rows(SeqNorm p) {
    constexpr int THREADS = G < 256 ? 256 : G, ROWS = THREADS / G;
    __shared__ float red[16];
    const int64_t t = (int64_t)block_number() * ROWS + threadIdx.x / G;
    if (t >= p.tokens) return;                   // the whole group, and a block of one group
    const int lane = threadIdx.x % G;
    constexpr int W = 8;
    const int parts = (int)((p.width + 7) / 8);
    auto n_of = [&](int at) { return cells_of<ANY>(p.width, at); };
    const X *x = (const X *)p.x + t * p.x_row;
    Cells<X, ANY> xs[NV];
    Cells<H, ANY> rs[RES ? NV : 1];
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int at = i * G + lane;
        xs[i].zero();
        if (at < parts) xs[i].load(x + at * W, n_of(at));
    }
    if constexpr (RES) {
        const H *r = (const H *)p.residual + t * p.residual_row;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int at = i * G + lane;
            rs[i].zero();
            if (at < parts) rs[i].load(r + at * W, n_of(at));
        }
    }
    float f[NV][W], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        xs[i].get(f[i]);
        if constexpr (RES) {
            float r[W];
            rs[i].get(r);
#pragma unroll
            for (int j = 0; j < W; j++) f[i][j] = stream_sum<H>(f[i][j], r[j]);
            const int at = i * G + lane;
            if (at < parts) Cells<H, ANY>::put((H *)p.h + t * p.h_row + at * W, f[i], n_of(at));
        }
#pragma unroll
        for (int j = 0; j < W; j++) sum += f[i][j] * f[i][j];
    }
    if (!p.identity) {
        float g[NV][W];
        if (p.gain) {
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int at = i * G + lane;
                if (at < parts) get_cells<ANY>(p.gain, p.gain_dtype, at * W, g[i], n_of(at));
            }
        }
        const float rho = rms_factor(over_group<Add, G>(sum, red), p.width, p.eps);
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int j = 0; j < W; j++) f[i][j] *= rho;
        if (p.gain) {
#pragma unroll
            for (int i = 0; i < NV; i++)
#pragma unroll
                for (int j = 0; j < W; j++) f[i][j] *= g[i][j];
        }
    }
    if (p.y_dtype != SEQ_INT8) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int at = i * G + lane;
            if (at < parts) put_cells<ANY>(p.y, p.y_dtype, t * p.y_row + at * W, f[i], n_of(at));
        }
        return;
    }
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; i++)
        if (i * G + lane < parts)
#pragma unroll
            for (int j = 0; j < W; j++) most = Most::of(most, fabsf(f[i][j]));
    const Bits8 bits(over_group<Most, G>(most, red));
    if (lane == 0) p.y_scale[t] = bits.scale;
    int8_t *y = (int8_t *)p.y + t * p.y_row;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int at = i * G + lane;
        if (at >= parts) continue;
        uint2v v = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; j++)
            v[j / 4] |= (uint32_t)(bits.of(f[i][j]) & 0xff) << (8 * (j % 4));
        if (!ANY) {
            *(uint2v *)(y + at * 8) = v;
        } else if (n_of(at) == 8) {
            __builtin_memcpy(y + at * 8, &v, 8);
        } else {
            for (int j = 0; j < n_of(at); j++)
                y[at * 8 + j] = (int8_t)(v[j / 4] >> (8 * (j % 4)));
        }
    }
}

// Rows longer than registers hold, in any layout: a block per row reads it once for
// each of its sums and once more to write, a value a thread at a time. 8,192 rows of 28,672 in
// bf16 take 615 us, to 8 bits without a norm 580 (of 16,384: 91 and 77).
__global__ __launch_bounds__(1024) void norm_long(SeqNorm p) {
    __shared__ float red[16];
    const int64_t t = block_number();
    if (t >= p.tokens) return;
    auto h_at = [&](int64_t j) {
        const float x = get1(p.x, p.x_dtype, t * p.x_row + j);
        if (!p.residual) return x;
        const float r = get1(p.residual, p.h_dtype, t * p.residual_row + j);
        if (p.h_dtype == SEQ_FP32) return x + r;
        return p.h_dtype == SEQ_BF16 ? stream_sum<__bf16>(x, r) : stream_sum<_Float16>(x, r);
    };
    float rho = 1.0f;
    if (!p.identity) {
        float sum = 0.0f;
        for (int64_t j = threadIdx.x; j < p.width; j += 1024) {
            const float h = h_at(j);
            if (p.residual) put1(p.h, p.h_dtype, t * p.h_row + j, h);
            sum += h * h;
        }
        rho = rms_factor(over_group<Add, 1024>(sum, red), p.width, p.eps);
    }
    auto y_at = [&](int64_t j) {
        const float y = p.identity ? h_at(j) : h_at(j) * rho;
        return p.gain ? y * get1(p.gain, p.gain_dtype, j) : y;
    };
    if (p.y_dtype != SEQ_INT8) {
        for (int64_t j = threadIdx.x; j < p.width; j += 1024)
            put1(p.y, p.y_dtype, t * p.y_row + j, y_at(j));
        return;
    }
    float most = 0.0f;
    for (int64_t j = threadIdx.x; j < p.width; j += 1024) most = Most::of(most, fabsf(y_at(j)));
    const Bits8 bits(over_group<Most, 1024>(most, red));
    if (threadIdx.x == 0) p.y_scale[t] = bits.scale;
    for (int64_t j = threadIdx.x; j < p.width; j += 1024)
        ((int8_t *)p.y)[t * p.y_row + j] = (int8_t)bits.of(y_at(j));
}

// ------------------------------------------------------------------- gradient

// A group's rows one after the other; the gain's gradient stays in registers and is
// left as one row of partial sums a block. Memory bounds it: 16,383 rows of 4,096 in bf16
// with the stream's gradient (537 MB) take 115 us, 4.7 TB/s, the next row's loads waiting for
// this one's sums; four such blocks a compute unit cover for each other.
template <typename Y, typename H, bool ANY, int G, int NV>
__global__ __launch_bounds__(G < 256 ? 256 : G) void norm_grad_rows(SeqNormGrad p,
                                                                    float *partial) {
    constexpr int THREADS = G < 256 ? 256 : G, ROWS = THREADS / G, W = 8;
    __shared__ float red[16];
    __shared__ float columns[ROWS > 1 ? ROWS * G * NV * W : 1];
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    const int parts = (int)((p.width + 7) / 8);
    auto n_of = [&](int at) { return cells_of<ANY>(p.width, at); };
    float dgain[NV][W], gain[NV][W];             // the gain is read once
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int j = 0; j < W; j++) {
            dgain[i][j] = 0.0f;
            gain[i][j] = 1.0f;
        }
    if (p.gain)
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int at = i * G + lane;
            if (at < parts) get_cells<ANY>(p.gain, p.gain_dtype, at * W, gain[i], n_of(at));
        }
    const int64_t step = (int64_t)gridDim.x * gridDim.z * ROWS;
    for (int64_t t = (int64_t)block_number() * ROWS + group; t < p.tokens; t += step) {
        Cells<Y, ANY> ys[NV];
        Cells<H, ANY> hs[NV], es[NV];
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int at = i * G + lane;
            ys[i].zero();
            hs[i].zero();
            if (at < parts) {
                ys[i].load((const Y *)p.dy + t * p.dy_row + at * W, n_of(at));
                hs[i].load((const H *)p.h + t * p.h_row + at * W, n_of(at));
            }
        }
        if (p.dh) {
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int at = i * G + lane;
                if (at < parts) es[i].load((const H *)p.dh + t * p.dh_row + at * W, n_of(at));
            }
        }
        float sum = 0.0f, dot = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            float h[W], u[W];
            hs[i].get(h);
            ys[i].get(u);
#pragma unroll
            for (int j = 0; j < W; j++) u[j] *= gain[i][j];
#pragma unroll
            for (int j = 0; j < W; j++) { sum += h[j] * h[j]; dot += u[j] * h[j]; }
        }
        sum = over_group<Add, G>(sum, red);
        dot = over_group<Add, G>(dot, red);
        const float rho = rms_factor(sum, p.width, p.eps);
        const float pull = dot / (float)p.width * rho * rho;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int at = i * G + lane;
            float h[W], u[W], d[W];
            hs[i].get(h);
            ys[i].get(u);
#pragma unroll
            for (int j = 0; j < W; j++) dgain[i][j] += u[j] * (h[j] * rho);
            if (at >= parts) continue;
#pragma unroll
            for (int j = 0; j < W; j++) u[j] *= gain[i][j];
#pragma unroll
            for (int j = 0; j < W; j++) d[j] = (u[j] - h[j] * pull) * rho;
            if (p.dh) {
                float e[W];
                es[i].get(e);
#pragma unroll
                for (int j = 0; j < W; j++) d[j] += e[j];
            }
            Cells<H, ANY>::put((H *)p.d + t * p.d_row + at * W, d, n_of(at));
            if (p.dx) put_cells<ANY>(p.dx, p.x_dtype, t * p.dx_row + at * W, d, n_of(at));
        }
    }
    if (!partial) return;
    float *out = partial + block_number() * p.width;
    if constexpr (ROWS == 1) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int at = i * G + lane;
            if (at < parts) Cells<float, ANY>::put(out + at * W, dgain[i], n_of(at));
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int j = 0; j < W; j++)
                columns[group * (G * NV * W) + (i * G + lane) * W + j] = dgain[i][j];
        __syncthreads();
        for (int c = threadIdx.x; c < p.width; c += THREADS) {
            float s = 0.0f;
#pragma unroll
            for (int r = 0; r < ROWS; r++) s += columns[r * (G * NV * W) + c];
            out[c] = s;
        }
    }
}

// Any layout and length; leaves each row's factor for the gain's gradient. 8,192 rows of
// 28,672 in bf16 take 1,695 us with the gain's (of 16,384: 118).
__global__ __launch_bounds__(1024) void norm_grad_long(SeqNormGrad p, float *rhos) {
    __shared__ float red[16];
    const int64_t t = block_number();
    if (t >= p.tokens) return;
    auto u_at = [&](int64_t j) {
        const float u = get1(p.dy, p.dy_dtype, t * p.dy_row + j);
        return p.gain ? u * get1(p.gain, p.gain_dtype, j) : u;
    };
    float sum = 0.0f, dot = 0.0f;
    for (int64_t j = threadIdx.x; j < p.width; j += 1024) {
        const float h = get1(p.h, p.h_dtype, t * p.h_row + j);
        sum += h * h;
        dot += u_at(j) * h;
    }
    sum = over_group<Add, 1024>(sum, red);
    dot = over_group<Add, 1024>(dot, red);
    const float rho = rms_factor(sum, p.width, p.eps);
    const float pull = dot / (float)p.width * rho * rho;
    if (rhos && threadIdx.x == 0) rhos[t] = rho;
    for (int64_t j = threadIdx.x; j < p.width; j += 1024) {
        float d = (u_at(j) - get1(p.h, p.h_dtype, t * p.h_row + j) * pull) * rho;
        if (p.dh) d += get1(p.dh, p.h_dtype, t * p.dh_row + j);
        put1(p.d, p.h_dtype, t * p.d_row + j, d);
        if (p.dx) put1(p.dx, p.x_dtype, t * p.dx_row + j, d);
    }
}
__global__ __launch_bounds__(256) void norm_gain_long(SeqNormGrad p, const float *rhos,
                                                      int64_t chunk, float *partial) {
    const int64_t j = blockIdx.x * 256ll + threadIdx.x;
    if (j >= p.width) return;
    const int64_t a = blockIdx.y * chunk, b = a + chunk < p.tokens ? a + chunk : p.tokens;
    double s = 0.0;                              // a chunk may have any number of rows
    for (int64_t t = a; t < b; t++)
        s += get1(p.dy, p.dy_dtype, t * p.dy_row + j) *
             (get1(p.h, p.h_dtype, t * p.h_row + j) * rhos[t]);
    partial[blockIdx.y * p.width + j] = (float)s;
}

// The blocks' partial sums, column by column in one order: 32 columns a block, each the
// sum of 32 threads' sums. 1,024 rows of 4,096 take 5.0 us. S: float up to those, else double.
template <typename S>
__global__ __launch_bounds__(1024) void norm_columns(const float *partial, int rows,
                                                     int64_t width, float *dgain) {
    __shared__ S part[32][33];
    const int c = threadIdx.x % 32, g = threadIdx.x / 32;
    const int64_t j = blockIdx.x * 32ll + c;
    S s = 0;
    if (j < width)
#pragma unroll 4
        for (int r = g; r < rows; r += 32) s += partial[r * width + j];
    part[g][c] = s;
    __syncthreads();
    if (g == 0 && j < width) {
        s = part[0][c];
#pragma unroll
        for (int i = 1; i < 32; i++) s += part[i][c];
        dgain[j] = (float)s;
    }
}

// ------------------------------------------------------------------- launches

// Calls f(Const<G>, Const<NV>) with the threads of a row of `parts` parts and the parts of
// each; false where registers do not hold it. Up to 128 parts a row is a wave's at most, which
// needs no barrier; beyond, a wave's registers would hold so much of a row that few waves
// find room (the gradient of 16,383 rows of 4,096 in bf16: 147 us with a wave a row, 92 with
// four).
template <typename F> bool row_shape(int64_t parts, F f) {
    if (parts <= 16) f(Const<16>(), Const<1>());
    else if (parts <= 32) f(Const<32>(), Const<1>());
    else if (parts <= 64) f(Const<64>(), Const<1>());
    else if (parts <= 128) f(Const<64>(), Const<2>());
    else if (parts <= 256) f(Const<256>(), Const<1>());
    else if (parts <= 512) f(Const<256>(), Const<2>());
    else if (parts <= 1024) f(Const<256>(), Const<4>());
    else if (parts <= 2048) f(Const<1024>(), Const<2>());
    else return false;
    return true;
}

template <typename X, typename H, bool RES, bool ANY>
bool launch_norm(const SeqNorm &p, hipStream_t s) {
    return row_shape((p.width + 7) / 8, [&](auto g, auto nv) {
        constexpr int G = g.value, NV = nv.value, THREADS = G < 256 ? 256 : G;
        constexpr int ROWS = THREADS / G;
        norm_rows<X, H, RES, ANY, G, NV>
            <<<grid_of((p.tokens + ROWS - 1) / ROWS, THREADS), THREADS, 0, s>>>(p);
    });
}
template <typename X, typename H, bool RES> bool launch_norm(const SeqNorm &p, hipStream_t s) {
    const bool eights = p.width % 8 == 0 && in_eights(p.x, p.x_row) &&
                        in_eights(p.residual, p.residual_row) && in_eights(p.h, p.h_row) &&
                        in_eights(p.gain, 0) && in_eights(p.y, p.y_row);
    return eights ? launch_norm<X, H, RES, false>(p, s) : launch_norm<X, H, RES, true>(p, s);
}
template <typename X> bool launch_norm(const SeqNorm &p, hipStream_t s) {
    if (!p.residual) return launch_norm<X, X, false>(p, s);
    if (p.h_dtype == p.x_dtype) return launch_norm<X, X, true>(p, s);
    if constexpr (sizeof(X) == 2) return launch_norm<X, float, true>(p, s);
    return false;
}

int check_norm(const SeqNorm *p) {
    if (!p || p->struct_size != (int32_t)sizeof(SeqNorm)) return CO_ERR_NULLARG;
    if (p->tokens < 0 || p->width < 1) return CO_ERR_NULLARG;
    if (p->tokens > SEQ_MAX_ROWS || p->width > SEQ_MAX_WIDTH) return CO_ERR_BOUNDS;
    if (!float_type(p->x_dtype) || !(float_type(p->y_dtype) || p->y_dtype == SEQ_INT8) ||
        (p->gain && !float_type(p->gain_dtype)) || !(p->eps >= 0.0f && p->eps <= 3.4028235e38f))
        return CO_ERR_DATA;
    if (p->residual && p->h_dtype != p->x_dtype && p->h_dtype != SEQ_FP32) return CO_ERR_DATA;
    if (p->identity && (p->residual || p->gain)) return CO_ERR_DATA;
    return CO_OK;
}

// Blocks of the gain's partial sums: enough to fill the chip, few enough that the sums
// are small beside the rows (16,383 rows of 4,096 in bf16: 94 us with 1,024, with 512 105,
// with 2,048 98; h in dh's place too). A group adds 2,048 rows at most one after the other in
// 32 bits, so that the error of many rows does not grow with them: beyond, there are as many
// blocks more.
constexpr int kGradBlocks = 1024, kGradRows = 2048;
constexpr int64_t kLongChunks = 64;
bool grad_is_long(const SeqNormGrad &p) { return p.width > 16384; }

int check_norm_grad(const SeqNormGrad *p) {
    if (!p || p->struct_size != (int32_t)sizeof(SeqNormGrad)) return CO_ERR_NULLARG;
    if (p->tokens < 0 || p->width < 1) return CO_ERR_NULLARG;
    if (p->tokens > SEQ_MAX_ROWS || p->width > SEQ_MAX_WIDTH) return CO_ERR_BOUNDS;
    if (!float_type(p->dy_dtype) || !float_type(p->h_dtype) ||
        (p->gain && !float_type(p->gain_dtype)) || (p->dx && !float_type(p->x_dtype)) ||
        !(p->eps >= 0.0f && p->eps <= 3.4028235e38f))
        return CO_ERR_DATA;
    return CO_OK;
}
// blocks of `threads` threads and `rows` rows each at a time that leave partial sums
int64_t grad_blocks(int64_t tokens, int threads, int rows) {
    const int64_t blocks = (tokens + rows - 1) / rows, most = kGradBlocks * 256 / threads;
    const int64_t turn = most * rows * kGradRows, all = most * ((tokens + turn - 1) / turn);
    return blocks < all ? blocks : all;
}
int64_t norm_grad_bytes(const SeqNormGrad &p) {
    if (!p.dgain || p.tokens == 0) return 0;
    if (grad_is_long(p)) return 4 * (p.tokens + kLongChunks * p.width);
    int64_t blocks = 0;
    row_shape((p.width + 7) / 8, [&](auto g, auto) {
        constexpr int G = g.value, THREADS = G < 256 ? 256 : G;
        blocks = grad_blocks(p.tokens, THREADS, THREADS / G);
    });
    return 4 * blocks * p.width;
}

// Launches the rows' kernel; returns the rows of partial sums that it leaves.
template <typename Y, typename H, bool ANY>
int launch_norm_grad(const SeqNormGrad &p, float *partial, hipStream_t s) {
    int rows = 0;
    row_shape((p.width + 7) / 8, [&](auto g, auto nv) {
        constexpr int G = g.value, NV = nv.value, THREADS = G < 256 ? 256 : G;
        constexpr int ROWS = THREADS / G;
        const int64_t blocks = partial ? grad_blocks(p.tokens, THREADS, ROWS)
                                       : (p.tokens + ROWS - 1) / ROWS;
        rows = partial ? (int)blocks : 0;
        norm_grad_rows<Y, H, ANY, G, NV><<<grid_of(blocks, THREADS), THREADS, 0, s>>>(p, partial);
    });
    return rows;
}
template <typename Y, typename H>
int launch_norm_grad(const SeqNormGrad &p, float *partial, hipStream_t s) {
    const bool eights = p.width % 8 == 0 && in_eights(p.dy, p.dy_row) &&
                        in_eights(p.h, p.h_row) && in_eights(p.gain, 0) &&
                        in_eights(p.dh, p.dh_row) && in_eights(p.d, p.d_row) &&
                        in_eights(p.dx, p.dx_row);
    return eights ? launch_norm_grad<Y, H, false>(p, partial, s)
                  : launch_norm_grad<Y, H, true>(p, partial, s);
}
template <typename Y> int launch_norm_grad(const SeqNormGrad &p, float *partial, hipStream_t s) {
    switch (p.h_dtype) {
        case SEQ_FP32: return launch_norm_grad<Y, float>(p, partial, s);
        case SEQ_BF16: return launch_norm_grad<Y, __bf16>(p, partial, s);
        default: return launch_norm_grad<Y, _Float16>(p, partial, s);
    }
}

}  // namespace seq

extern "C" int seq_norm(const SeqNorm *p, void *stream) {
    const int rc = seq::check_norm(p);
    if (rc != CO_OK) return rc;
    if (p->tokens == 0) return CO_OK;
    if (!p->x || !p->y || (p->residual && !p->h) || (p->y_dtype == SEQ_INT8 && !p->y_scale))
        return CO_ERR_NULLARG;
    hipStream_t s = (hipStream_t)stream;
    bool held;
    switch (p->x_dtype) {
        case SEQ_FP32: held = seq::launch_norm<float>(*p, s); break;
        case SEQ_BF16: held = seq::launch_norm<__bf16>(*p, s); break;
        default: held = seq::launch_norm<_Float16>(*p, s); break;
    }
    if (!held) seq::norm_long<<<seq::grid_of(p->tokens, 1024), 1024, 0, s>>>(*p);
    return seq::launch_status();
}

extern "C" int64_t seq_norm_grad_workspace(const SeqNormGrad *p) {
    const int rc = seq::check_norm_grad(p);
    if (rc != CO_OK) return rc > 0 ? -rc : rc;
    return seq::norm_grad_bytes(*p);
}

extern "C" int seq_norm_grad(const SeqNormGrad *p, void *stream) {
    int rc = seq::check_norm_grad(p);
    if (rc != CO_OK) return rc;
    hipStream_t s = (hipStream_t)stream;
    const unsigned blocks = (unsigned)((p->width + 31) / 32);
    if (p->tokens == 0) {
        if (!p->dgain) return CO_OK;
        seq::norm_columns<float><<<blocks, 1024, 0, s>>>(nullptr, 0, p->width, p->dgain);
        return seq::launch_status();
    }
    if (!p->dy || !p->h || !p->d) return CO_ERR_NULLARG;
    const int64_t bytes = seq::norm_grad_bytes(*p);
    if (bytes && !p->workspace) return CO_ERR_NULLARG;
    if (p->workspace_bytes < bytes || ((uintptr_t)p->workspace & 15)) return CO_ERR_DATA;
    float *ws = p->dgain ? (float *)p->workspace : nullptr;
    int rows = 0;
    if (seq::grad_is_long(*p)) {
        float *partial = ws ? ws + p->tokens : nullptr;
        seq::norm_grad_long<<<seq::grid_of(p->tokens, 1024), 1024, 0, s>>>(*p, ws);
        if (ws) {
            const int64_t chunk = (p->tokens + seq::kLongChunks - 1) / seq::kLongChunks;
            rows = (int)((p->tokens + chunk - 1) / chunk);
            seq::norm_gain_long<<<dim3((unsigned)((p->width + 255) / 256), (unsigned)rows), 256, 0,
                                  s>>>(*p, ws, chunk, partial);
            ws = partial;
        }
    } else {
        switch (p->dy_dtype) {
            case SEQ_FP32: rows = seq::launch_norm_grad<float>(*p, ws, s); break;
            case SEQ_BF16: rows = seq::launch_norm_grad<__bf16>(*p, ws, s); break;
            default: rows = seq::launch_norm_grad<_Float16>(*p, ws, s); break;
        }
    }
    rc = seq::launch_status();
    if (rc != CO_OK || !p->dgain) return rc;
    if (rows <= seq::kGradBlocks)
        seq::norm_columns<float><<<blocks, 1024, 0, s>>>(ws, rows, p->width, p->dgain);
    else
        seq::norm_columns<double><<<blocks, 1024, 0, s>>>(ws, rows, p->width, p->dgain);
    return seq::launch_status();
}
