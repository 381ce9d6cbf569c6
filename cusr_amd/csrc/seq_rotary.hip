// seq_rotary.hip -- rotary positions (include/cusr_seq.h, seq_rotary).
//
// A pair (a, b) of a head turns by its token's angle: a' = a c - b s,
// b' = b c + a s, in fp32, rounded once to the tensor's type. (c, s) come from
// a table made in fp64, so that far positions lose nothing to the angle's
// rounding. The bound is memory: q and k are read once and written once.
#include "seq_common.h"

namespace seq {

template <typename T> __device__ inline float load1(const T *p) { return (float)*p; }

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
        const int64_t p = r.positions[t];
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

template <typename T>
int launch_rotary(const SeqRotary &r, hipStream_t s) {
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
        r->hq > 65535 || r->hkv > 65535 || r->d > 65535)
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
