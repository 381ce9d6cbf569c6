// seq_rotary.hip -- rotary positions (include/cusr_seq.h, seq_rotary).
//
// A pair (a, b) of a head turns by its token's angle: a' = a c - b s,
// b' = b c + a s, in fp32, rounded once to the tensor's type. (c, s) come from
// a table made in fp64, so that far positions lose nothing to the angle's
// rounding. The bound is memory: q and k are read once and written once.
#include "seq_common.h"

namespace seq {

template <typename T> __device__ inline float load1(const T *p) { return (float)*p; }
__device__ inline int64_t position(const SeqRotary &r, int64_t t) {
    return r.positions_64 ? ((const int64_t *)r.positions)[t] : ((const int32_t *)r.positions)[t];
}

// Any size, stride and alignment: a thread per pair or copied element. 32,768
// tokens of 40 heads of 128 in bf16 would take 331 us, 2.0 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void rotary_kernel(SeqRotary r) {
    const int heads = r.hq + r.hkv, half = r.rot / 2;
    const int per_head = half + (r.d - r.rot);   // pairs, then copied elements
    const int64_t n = r.tokens * heads * per_head;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
        const int e = (int)(i % per_head);
        const int64_t th = i / per_head;
        const int h = (int)(th % heads);
        const int64_t t = th / heads;
        const bool is_q = h < r.hq;
        const T *x = is_q ? (const T *)r.q + t * r.q_row + h * r.q_head
                          : (const T *)r.k + t * r.k_row + (h - r.hq) * r.k_head;
        T *y = is_q ? (T *)r.q_out + t * r.qo_row + h * r.qo_head
                    : (T *)r.k_out + t * r.ko_row + (h - r.hq) * r.ko_head;
        if (e >= half) {
            y[r.rot + e - half] = x[r.rot + e - half];
            continue;
        }
        const int ia = r.interleaved ? 2 * e : e, ib = r.interleaved ? 2 * e + 1 : e + half;
        const int64_t p = position(r, t);
        float c = __builtin_nanf(""), s = c;
        if (p >= 0 && p < r.table_len) {
            c = r.table[(p * half + e) * 2];
            s = r.table[(p * half + e) * 2 + 1];
        }
        if (r.inverse) s = -s;
        const float a = load1(x + ia), b = load1(x + ib);
        y[ia] = (T)(a * c - b * s);
        y[ib] = (T)(b * c + a * s);
    }
}

// 16-byte pieces: N values of T
template <typename T> struct Piece {
    static constexpr int n = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(n)));
};

// A thread owns one piece's place in the head (in the half layout, the piece
// and its partner half a turn further) of one token and runs over `per` heads
// of q and k with the same cosines and sines: 146 us, 4.6 TB/s, for the same. Needs
// 16-byte rows and heads and pairs that fill pieces.
template <typename T, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_pieces(SeqRotary r, int items, int per) {
    constexpr int N = Piece<T>::n, P = INTERLEAVED ? N / 2 : N;    // pairs of a thread
    typedef typename Piece<T>::vec vec;
    const int tokens = 256 / items;
    const int slot = (int)threadIdx.x / items, e = (int)threadIdx.x % items;
    const int64_t t = (int64_t)block_number() * tokens + slot;
    if (slot >= tokens || t >= r.tokens) return;
    const int half = r.rot / 2, turning = half / P;      // pieces that turn
    const int h0 = (int)blockIdx.y * per, h1 = min(h0 + per, r.hq + r.hkv);
    const bool turn = e < turning;
    float c[P], s[P];
    if (turn) {
        const int64_t pos = position(r, t);
        const bool in = pos >= 0 && pos < r.table_len;
        const float4v *cs = (const float4v *)(r.table + ((in ? pos : 0) * half + e * P) * 2);
#pragma unroll
        for (int j = 0; j < P; j += 2) {
            const float nan = __builtin_nanf("");
            float4v v = {nan, nan, nan, nan};
            if (in) v = cs[j / 2];
            c[j] = v[0]; c[j + 1] = v[2];
            s[j] = r.inverse ? -v[1] : v[1];
            s[j + 1] = r.inverse ? -v[3] : v[3];
        }
    }
    // first element of the piece, and of its partner
    const int ia = turn ? e * (INTERLEAVED ? N : P) : r.rot + (e - turning) * N;
    const int ib = ia + half;
#pragma unroll 4
    for (int h = h0; h < h1; h++) {
        const bool is_q = h < r.hq;
        const T *x = is_q ? (const T *)r.q + t * r.q_row + h * r.q_head
                          : (const T *)r.k + t * r.k_row + (h - r.hq) * r.k_head;
        T *y = is_q ? (T *)r.q_out + t * r.qo_row + h * r.qo_head
                    : (T *)r.k_out + t * r.ko_row + (h - r.hq) * r.ko_head;
        vec a = *(const vec *)(x + ia);
        if (!turn) {
            *(vec *)(y + ia) = a;
        } else if (INTERLEAVED) {
            vec o;
#pragma unroll
            for (int j = 0; j < P; j++) {
                const float u = (float)a[2 * j], w = (float)a[2 * j + 1];
                o[2 * j] = (T)(u * c[j] - w * s[j]);
                o[2 * j + 1] = (T)(w * c[j] + u * s[j]);
            }
            *(vec *)(y + ia) = o;
        } else {
            const vec b = *(const vec *)(x + ib);
            vec oa, ob;
#pragma unroll
            for (int j = 0; j < P; j++) {
                const float u = (float)a[j], w = (float)b[j];
                oa[j] = (T)(u * c[j] - w * s[j]);
                ob[j] = (T)(w * c[j] + u * s[j]);
            }
            *(vec *)(y + ia) = oa;
            *(vec *)(y + ib) = ob;
        }
    }
}

bool off(const void *p, int64_t row, int64_t head, int n) {
    return ((uintptr_t)p & 15) || row % n || head % n;
}

// Whether every piece lies on a 16-byte boundary, and pairs fill pieces.
bool in_pieces(const SeqRotary &r, int n) {
    const int turned = r.interleaved ? r.rot : r.rot / 2;
    if (turned % n || r.d % n || r.d / n > 256 || ((uintptr_t)r.table & 15)) return false;
    if (r.hq && (off(r.q, r.q_row, r.q_head, n) || off(r.q_out, r.qo_row, r.qo_head, n)))
        return false;
    return !(r.hkv && (off(r.k, r.k_row, r.k_head, n) || off(r.k_out, r.ko_row, r.ko_head, n)));
}

template <typename T>
int launch_rotary(const SeqRotary &r, hipStream_t s) {
    constexpr int N = Piece<T>::n;
    if (in_pieces(r, N)) {
        const int items = (r.interleaved ? r.rot : r.rot / 2) / N + (r.d - r.rot) / N;
        const int heads = r.hq + r.hkv, tokens = 256 / items;
        const int64_t blocks = (r.tokens + tokens - 1) / tokens;
        // A thread takes up to 8 heads, as many as leave 4 blocks per compute unit:
        // the table is read once for them, few tokens spread over heads instead. 32,768
        // tokens of 40 heads of 128: 1 head 236 us, 4 182 us, 8 146 us, 16 178 us, 40 164 us.
        int per = 1;
        while (per < 8 && blocks * ((heads + 2 * per - 1) / (2 * per)) >= 1024) per *= 2;
        const dim3 grid = grid_of(blocks, 256, (heads + per - 1) / per);
        if (r.interleaved) rotary_pieces<T, true><<<grid, 256, 0, s>>>(r, items, per);
        else rotary_pieces<T, false><<<grid, 256, 0, s>>>(r, items, per);
        return launch_status();
    }
    const int64_t n = r.tokens * (r.hq + r.hkv) * (r.d - r.rot / 2);
    int64_t blocks = (n + 255) / 256;
    if (blocks > 65536) blocks = 65536;
    rotary_kernel<T><<<dim3((unsigned)blocks), 256, 0, s>>>(r);
    return launch_status();
}

}  // namespace seq

extern "C" int seq_rotary(const SeqRotary *r, void *stream) {
    if (!r || r->struct_size != (int32_t)sizeof(SeqRotary)) return CO_ERR_NULLARG;
    if (r->tokens < 0 || r->hq < 0 || r->hkv < 0 || r->d < 1 || r->table_len < 0)
        return CO_ERR_NULLARG;
    if (r->rot < 0 || r->rot > r->d || r->rot % 2 || r->tokens > SEQ_MAX_ROWS ||
        r->hq > 32767 || r->hkv > 32767 || r->d > 65535)
        return CO_ERR_BOUNDS;
    if (r->dtype < SEQ_FP32 || r->dtype > SEQ_FP16) return CO_ERR_DATA;
    if (r->tokens == 0 || r->hq + r->hkv == 0) return CO_OK;
    if ((r->hq && (!r->q || !r->q_out)) || (r->hkv && (!r->k || !r->k_out)) || !r->positions ||
        (!r->table && r->rot && r->table_len))
        return CO_ERR_NULLARG;
    hipStream_t s = (hipStream_t)stream;
    switch (r->dtype) {
        case SEQ_FP32: return seq::launch_rotary<float>(*r, s);
        case SEQ_BF16: return seq::launch_rotary<__bf16>(*r, s);
        default: return seq::launch_rotary<_Float16>(*r, s);
    }
}
