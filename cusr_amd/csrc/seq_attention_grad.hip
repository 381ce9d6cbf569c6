// seq_attention_grad.hip -- gradient of causal attention over packed sequences
// (include/cusr_seq.h, seq_attention_grad).
//
// With P = exp(S - lse) formed again from q, k and lse, delta = sum(do * o) per
// row and dP = do V^T:  dS = P (dP - delta),  dQ = scale dS K,
// dK = scale dS^T Q,  dV = P^T do. One kernel owns rows and sums over keys
// (dQ, delta), one owns keys and sums over rows (dK, dV, all heads of the
// group): every sum has one owner and one order, so no atomics.
#include "seq_attn.h"

namespace seq {

struct AttnGrad : Attn {
    SeqAttentionGrad g;
    float *delta;            // [hq, tq]
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

// A wave owns 32 rows: delta, then dQ^T = sum over keys of K^T dS^T.
template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_grad_q(AttnGrad a, int64_t slots) {
    __shared__ __align__(16) uint16_t lds[4][32 * Tile<DP>::stride];
    uint16_t *kt = lds[threadIdx.x >> 6];
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
    const int lim = ok ? qi + p.lk - p.lq : -1;
    const int64_t t = p.q0 + qi;
    uint4v q[DP / 16], dO[DP / 16];
    float delta, lse2;
    {
        uint4v o[DP / 16];
        load_row<DP>(o, a.o, t * a.o_row + head * a.o_head, a.d, ok);
        load_row<DP>(dO, a.g.d_o, t * a.g.do_row + head * a.g.do_head, a.d, ok);
        delta = add_halves(dot_row<T>(o, dO, DP / 16));
        lse2 = ok ? a.lse[head * a.tq + t] * kLog2e : 0.0f;
        if (ok && h == 0) a.delta[head * a.tq + t] = delta;
    }
    load_row<DP>(q, a.q, t * a.q_row + head * a.q_head, a.d, ok);
    const int64_t last_row = tile * 32 + 31 < rows ? tile * 32 + 31 : rows - 1;
    const int keys = (int)(last_row / a.G) + p.lk - p.lq + 1;
    float16v dq[DP / 32] = {};
    for (int k0 = 0; k0 < keys; k0 += 32) {
        const int kr = k0 + (lane & 31);
        uint4v k[DP / 16], v[DP / 16];
        load_row<DP>(k, a.k, (p.k0 + kr) * a.k_row + hk * a.k_head, a.d, kr < keys);
        load_row<DP>(v, a.v, (p.k0 + kr) * a.v_row + hk * a.v_head, a.d, kr < keys);
        wave_sync();
#pragma unroll
        for (int c = 0; c < DP / 16; c++)
            *(uint4v *)(kt + Tile<DP>::at(lane & 31, 2 * c + h)) = k[c];
        float16v s = {}, dp = {};
#pragma unroll
        for (int c = 0; c < DP / 16; c++) s = T::mfma(k[c], q[c], s);
#pragma unroll
        for (int c = 0; c < DP / 16; c++) dp = T::mfma(v[c], dO[c], dp);
        uint32_t pk[8];
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
            float ds[2];
            for (int j = 0; j < 2; j++) {
                const int key = k0 + 8 * (r / 4) + 4 * h + (r + j) % 4;
                const float pr = exp2_fast(s[r + j] * a.c - lse2);
                ds[j] = key <= lim ? pr * (dp[r + j] - delta) : 0.0f;
            }
            pk[r / 2] = T::pack(ds[0], ds[1]);
        }
        wave_sync();
#pragma unroll
        for (int kc = 0; kc < 2; kc++) {
            const uint4v pb = {pk[4 * kc], pk[4 * kc + 1], pk[4 * kc + 2], pk[4 * kc + 3]};
#pragma unroll
            for (int dt = 0; dt < DP / 32; dt++)
                dq[dt] = T::mfma(Tile<DP>::transposed(kt, kc * 16, dt), pb, dq[dt]);
        }
    }
    store_row<T, DP>(a.g.dq, t * a.g.dq_row + head * a.g.dq_head, dq, a.scale, a.d, ok);
}

// A wave owns 32 keys of one key head and sums over the rows that see them.
// Slots are tiles of the key rows 0..tk-1, whatever sequence they belong to:
// entry n_seq covers the rows after the last sequence.
template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_grad_kv(AttnGrad a, int64_t slots) {
    __shared__ __align__(16) uint16_t lds[4][2 * 32 * Tile<DP>::stride + 192];
    uint16_t *qt = lds[threadIdx.x >> 6], *ot = qt + 32 * Tile<DP>::stride;
    float *stat = (float *)(ot + 32 * Tile<DP>::stride);     // lse, delta, limit of 32 rows
    const int lane = threadIdx.x & 63, h = lane >> 5;
    const int64_t item = blockIdx.x * 4ll + (threadIdx.x >> 6);
    const int64_t slot = item / a.hkv;
    const int hk = (int)(item % a.hkv);
    if (slot >= slots) return;
    const int b = find_sequence(a.cu_k, a.n_seq, a.tk, 1, 32, slot);
    const int64_t s0 = offset_at(a.cu_k, b, a.tk);
    const int64_t s1 = b >= a.n_seq ? a.tk : clamp64(a.cu_k[b + 1], s0, a.tk);
    const int64_t tile = slot - slot_of(s0, 1, 32, b);
    if (tile < 0 || tile * 32 >= s1 - s0) return;
    // rows of segment 0 before its start belong to no sequence
    const Place p = b >= a.n_seq ? Place{0, s0, 0, 0} : place_of(a, b);
    const int key = (int)(tile * 32 + (s0 - p.k0)) + (lane & 31);   // in the sequence
    const bool ok = tile * 32 + (lane & 31) < s1 - s0;
    const bool live = ok && key >= 0 && key < p.lk;
    const int64_t kr = s0 + tile * 32 + (lane & 31);
    uint4v k[DP / 16], v[DP / 16];
    load_row<DP>(k, a.k, kr * a.k_row + hk * a.k_head, a.d, live);
    load_row<DP>(v, a.v, kr * a.v_row + hk * a.v_head, a.d, live);
    float16v dk[DP / 32] = {}, dv[DP / 32] = {};
    const int64_t rows = (int64_t)p.lq * a.G;
    const int key0 = (int)(tile * 32 + (s0 - p.k0));
    // the first query that sees a key of the tile
    int64_t r0 = (int64_t)(key0 - (p.lk - p.lq) > 0 ? key0 - (p.lk - p.lq) : 0) * a.G / 32 * 32;
    if (key0 >= p.lk) r0 = rows;
    for (; r0 < rows; r0 += 32) {
        const int64_t row = r0 + (lane & 31);
        const bool rok = row < rows;
        const int qi = rok ? (int)(row / a.G) : 0, g = rok ? (int)(row % a.G) : 0;
        const int head = hk * a.G + g;
        const int64_t t = p.q0 + qi;
        uint4v q[DP / 16], dO[DP / 16];
        load_row<DP>(q, a.q, t * a.q_row + head * a.q_head, a.d, rok);
        load_row<DP>(dO, a.g.d_o, t * a.g.do_row + head * a.g.do_head, a.d, rok);
        wave_sync();
#pragma unroll
        for (int c = 0; c < DP / 16; c++) {
            *(uint4v *)(qt + Tile<DP>::at(lane & 31, 2 * c + h)) = q[c];
            *(uint4v *)(ot + Tile<DP>::at(lane & 31, 2 * c + h)) = dO[c];
        }
        if (h == 0) {
            stat[lane] = rok ? a.lse[head * a.tq + t] * kLog2e : 0.0f;
            stat[32 + lane] = rok ? a.delta[head * a.tq + t] : 0.0f;
            ((int *)stat)[64 + lane] = rok ? qi + p.lk - p.lq : -1;
        }
        float16v s = {}, dp = {};
#pragma unroll
        for (int c = 0; c < DP / 16; c++) s = T::mfma(q[c], k[c], s);
#pragma unroll
        for (int c = 0; c < DP / 16; c++) dp = T::mfma(dO[c], v[c], dp);
        wave_sync();
        uint32_t pp[8], pd[8];
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
            float pr[2], ds[2];
            for (int j = 0; j < 2; j++) {
                const int i = 8 * (r / 4) + 4 * h + (r + j) % 4;
                const bool see = live && key <= ((const int *)stat)[64 + i];
                pr[j] = see ? exp2_fast(s[r + j] * a.c - stat[i]) : 0.0f;
                ds[j] = see ? pr[j] * (dp[r + j] - stat[32 + i]) : 0.0f;
            }
            pp[r / 2] = T::pack(pr[0], pr[1]);
            pd[r / 2] = T::pack(ds[0], ds[1]);
        }
#pragma unroll
        for (int kc = 0; kc < 2; kc++) {
            const uint4v pb = {pp[4 * kc], pp[4 * kc + 1], pp[4 * kc + 2], pp[4 * kc + 3]};
            const uint4v db = {pd[4 * kc], pd[4 * kc + 1], pd[4 * kc + 2], pd[4 * kc + 3]};
#pragma unroll
            for (int dt = 0; dt < DP / 32; dt++) {
                dv[dt] = T::mfma(Tile<DP>::transposed(ot, kc * 16, dt), pb, dv[dt]);
                dk[dt] = T::mfma(Tile<DP>::transposed(qt, kc * 16, dt), db, dk[dt]);
            }
        }
    }
    store_row<T, DP>(a.g.dk, kr * a.g.dk_row + hk * a.g.dk_head, dk, a.scale, a.d, ok);
    store_row<T, DP>(a.g.dv, kr * a.g.dv_row + hk * a.g.dv_head, dv, 1.0f, a.d, ok);
}

template <typename T, int DP>
int launch_grad(const AttnGrad &a, hipStream_t s) {
    if (a.tq) {
        const int64_t slots = slot_of(a.tq, a.G, 32, a.n_seq) + 1;
        attn_grad_q<T, DP><<<dim3((unsigned)((slots * a.hkv + 3) / 4)), 256, 0, s>>>(a, slots);
        if (hipGetLastError() != hipSuccess) return CO_ERR_CUDA;
    }
    if (a.tk) {
        const int64_t slots = slot_of(a.tk, 1, 32, a.n_seq) + 1;
        attn_grad_kv<T, DP><<<dim3((unsigned)((slots * a.hkv + 3) / 4)), 256, 0, s>>>(a, slots);
    }
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
    return rc == CO_OK ? 4 * a->hq * a->tq : (rc > 0 ? -rc : rc);
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
    if (((uintptr_t)g->d_o | (uintptr_t)g->dq | (uintptr_t)g->dk | (uintptr_t)g->dv) & 15)
        return CO_ERR_DATA;
    if ((g->do_row | g->do_head | g->dq_row | g->dq_head | g->dk_row | g->dk_head | g->dv_row |
         g->dv_head) & 7)
        return CO_ERR_DATA;
    if (sa->workspace_bytes < 4 * sa->hq * sa->tq) return CO_ERR_DATA;
    seq::AttnGrad a;
    static_cast<SeqAttention &>(a) = *sa;
    a.G = a.hq / a.hkv;
    a.c = a.scale * seq::kLog2e;
    a.g = *g;
    a.delta = (float *)sa->workspace;
    hipStream_t s = (hipStream_t)stream;
    return a.dtype == SEQ_BF16 ? seq::launch_grad_head<seq::Bf16>(a, s)
                               : seq::launch_grad_head<seq::Fp16>(a, s);
}
