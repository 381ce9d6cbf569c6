// seq_attention.hip -- causal attention over packed sequences
// (include/cusr_seq.h, seq_attention).
#include "seq_attn.h"

namespace seq {

// One wave owns a tile of 32 rows of one key head and runs over the keys 32 at
// a time with a running maximum and sum. K comes straight from memory as the
// left operand; V passes through the wave's own LDS tile to be transposed.
template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_wave(Attn a, int64_t slots) {
    __shared__ __align__(16) uint16_t lds[4][32 * Tile<DP>::stride];
    uint16_t *vt = lds[threadIdx.x >> 6];
    const int lane = threadIdx.x & 63, h = lane >> 5;
    const int64_t item = blockIdx.x * 4ll + (threadIdx.x >> 6);
    const int64_t slot = item / a.hkv;
    const int hk = (int)(item % a.hkv);
    if (slot >= slots) return;
    const int b = find_sequence(a.cu_q, a.n_seq, a.tq, a.G, 32, slot);
    const Place p = place_of(a, b);
    const int64_t tile = slot - slot_of(p.q0, a.G, 32, b);
    const int64_t rows = (int64_t)p.lq * a.G;
    if (tile < 0 || tile * 32 >= rows) return;
    const int64_t row = tile * 32 + (lane & 31);
    const bool ok = row < rows;
    const int qi = ok ? (int)(row / a.G) : 0, g = ok ? (int)(row % a.G) : 0;
    const int head = hk * a.G + g;
    const int lim = ok ? qi + p.lk - p.lq : -1;      // last visible key
    uint4v q[DP / 16];
    load_row<DP>(q, a.q, (p.q0 + qi) * a.q_row + head * a.q_head, a.d, ok);

    const int64_t last_row = tile * 32 + 31 < rows ? tile * 32 + 31 : rows - 1;
    const int keys = (int)(last_row / a.G) + p.lk - p.lq + 1;   // visible to the tile
    float16v o[DP / 32] = {};
    float m = neg_inf(), l = 0.0f;
    for (int k0 = 0; k0 < keys; k0 += 32) {
        // V: 32 rows to LDS, rows beyond the keys as zeros
        wave_sync();
        for (int i = lane; i < 32 * (DP / 8); i += 64) {
            const int r = i / (DP / 8), ch = i % (DP / 8);
            uint4v z = {0, 0, 0, 0};
            if (k0 + r < keys && ch * 8 < a.d)
                z = *(const uint4v *)((const uint16_t *)a.v + (p.k0 + k0 + r) * a.v_row +
                                      hk * a.v_head + ch * 8);
            *(uint4v *)(vt + Tile<DP>::at(r, ch)) = z;
        }
        uint4v k[DP / 16];
        const int kr = k0 + (lane & 31);
        load_row<DP>(k, a.k, (p.k0 + kr) * a.k_row + hk * a.k_head, a.d, kr < keys);
        float16v s = {};
#pragma unroll
        for (int c = 0; c < DP / 16; c++) s = T::mfma(k[c], q[c], s);
        float mx = neg_inf();
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const int key = k0 + 8 * (r / 4) + 4 * h + r % 4;
            s[r] = key <= lim ? s[r] : neg_inf();
            mx = fmaxf(mx, s[r]);
        }
        const float mn = fmaxf(m, max_halves(mx));
        const float m0 = mn == neg_inf() ? 0.0f : mn;
        const float alpha = exp2_fast((m - m0) * a.c);
        float sum = 0.0f;
        uint32_t pk[8];
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
            const float p0 = exp2_fast((s[r] - m0) * a.c), p1 = exp2_fast((s[r + 1] - m0) * a.c);
            sum += p0 + p1;
            pk[r / 2] = T::pack(p0, p1);
        }
        l = l * alpha + sum;
        m = mn;
#pragma unroll
        for (int dt = 0; dt < DP / 32; dt++) o[dt] *= alpha;
        wave_sync();
#pragma unroll
        for (int kc = 0; kc < 2; kc++) {
            const uint4v pb = {pk[4 * kc], pk[4 * kc + 1], pk[4 * kc + 2], pk[4 * kc + 3]};
#pragma unroll
            for (int dt = 0; dt < DP / 32; dt++)
                o[dt] = T::mfma(Tile<DP>::transposed(vt, kc * 16, dt), pb, o[dt]);
        }
    }
    l = add_halves(l);
    store_row<T, DP>(a.o, (p.q0 + qi) * a.o_row + head * a.o_head, o, l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l), a.d, ok);
    if (a.lse && ok && h == 0)
        a.lse[head * a.tq + p.q0 + qi] = l == 0.0f ? neg_inf() : m * a.scale + logf(l);
}

template <typename T, int DP>
int launch_wave(const Attn &a, hipStream_t s) {
    const int64_t slots = slot_of(a.tq, a.G, 32, a.n_seq) + 1;
    const int64_t blocks = (slots * a.hkv + 3) / 4;
    attn_wave<T, DP><<<dim3((unsigned)blocks), 256, 0, s>>>(a, slots);
    return launch_status();
}

template <typename T>
int launch_forward(const Attn &a, hipStream_t s) {
    switch (padded_head(a.d)) {
        case 32: return launch_wave<T, 32>(a, s);
        case 64: return launch_wave<T, 64>(a, s);
        case 96: return launch_wave<T, 96>(a, s);
        default: return launch_wave<T, 128>(a, s);
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
        a->tq * a->hq > SEQ_MAX_ROWS || a->tk > SEQ_MAX_ROWS || a->hq > 1 << 15)
        return CO_ERR_BOUNDS;
    if (a->dtype != SEQ_BF16 && a->dtype != SEQ_FP16) return CO_ERR_DATA;
    return CO_OK;
}

// the rest of the checks, for a call with pointers
int check_attention_data(const SeqAttention *a) {
    if (!a->cu_q || !a->cu_k || !a->q || !a->o || (a->tk && (!a->k || !a->v)))
        return CO_ERR_NULLARG;
    if (misaligned(a->q, a->q_row, a->q_head) || misaligned(a->k, a->k_row, a->k_head) ||
        misaligned(a->v, a->v_row, a->v_head) || misaligned(a->o, a->o_row, a->o_head))
        return CO_ERR_DATA;
    return CO_OK;
}

}  // namespace seq

extern "C" int64_t seq_attention_workspace(const SeqAttention *a) {
    const int rc = seq::check_attention(a);
    return rc == CO_OK ? 0 : (rc > 0 ? -rc : rc);
}

extern "C" int seq_attention(const SeqAttention *sa, void *stream) {
    int rc = seq::check_attention(sa);
    if (rc != CO_OK) return rc;
    if (sa->tq == 0) return CO_OK;
    rc = seq::check_attention_data(sa);
    if (rc != CO_OK) return rc;
    seq::Attn a;
    static_cast<SeqAttention &>(a) = *sa;
    a.G = a.hq / a.hkv;
    a.c = a.scale * seq::kLog2e;
    hipStream_t s = (hipStream_t)stream;
    return a.dtype == SEQ_BF16 ? seq::launch_forward<seq::Bf16>(a, s)
                               : seq::launch_forward<seq::Fp16>(a, s);
}
