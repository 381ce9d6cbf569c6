// seq_embedding.hip -- rows of a table by token, and the table's gradient
// (include/cusr_seq.h, seq_embedding, seq_embedding_grad).
//
// The bound is memory. The lookup reads a row and writes it. The gradient adds the rows
// of each token: tokens are sorted first (stably, by counting digits), so that a row of
// the table is one run of places, added in the order of the tokens, with nothing
// left to atomics. Runs are cut into chunks of equal length, however many tokens a row
// has: what a run leaves in a chunk that it only passes through goes to a slot, and
// slots are joined in order at the end.
#include "seq_rows.h"

namespace seq {

// log2 of the threads of a row of `parts` parts
inline int group_log(int64_t parts) {
    int g = 0;
    while (g < 8 && (1 << g) < parts) g++;
    return g;
}

// 2^g threads a token, a part of its row each at a time, four on their way. 24 rows of 4,096
// in bf16 take 3.0 us: the token, its row, the output, one after the other. Many are bound by
// memory: 16,383 rows of 4,096 in bf16 (134 MB written, words from 32,001) take 31.4 us, 1.3 M of
// 128 in fp32 from 22 (676 MB) 166 to 178, 4 TB/s, of 64 in bf16 from 131,071 (194 MB) 36, 5.4.
template <typename T, bool ANY>
__global__ __launch_bounds__(256) void embed_rows(SeqEmbedding p, int g) {
    const int64_t t = (int64_t)block_number() * (256 >> g) + (threadIdx.x >> g);
    if (t >= p.tokens) return;
    const int parts = (int)((p.width + 7) / 8), lane = threadIdx.x & ((1 << g) - 1);
    const int64_t id = get_id(p.ids, p.ids_64, t);
    const bool in = id >= 0 && id < p.rows;
    const T *row = (const T *)p.table + (in ? id : 0) * p.table_row;
    const float scale = in ? p.scale : __builtin_nanf("");
#pragma unroll 4
    for (int at = lane; at < parts; at += 1 << g) {
        const int n = cells_of<ANY>(p.width, at);
        Cells<T, ANY> v;
        v.zero();
        if (in) v.load(row + at * 8, n);         // a table may have no row at all
        float f[8];
        v.get(f);
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] *= scale;
        put_cells<ANY>(p.out, p.out_dtype, t * p.out_row + at * 8, f, n);
    }
}

// ------------------------------------------------------------- few rows: symbols

// A table of up to kSymbolRows rows: a wave keeps the sums of its tokens, 128 columns of
// every row, in LDS and reads its tokens' gradients one after the other, so no order of
// tokens is needed. A lane adds to columns of its own, in the tokens' order, four tokens at a
// time: where two of them have one row the later takes the earlier's sum. (LDS adds
// floats by itself, but hardly a lane at a time: 839 us for 1.3 M tokens of 128 in fp32
// and 22 rows.) Against sorting, that takes 126 against 229 us, with 30 rows 128 against
// 227, with 40 rows of 1,024 columns 1,320 against 1,183 and with 80 rows 321 against 229:
// fewer blocks find room in LDS.
constexpr int kSymbolRows = 32, kSymbolCols = 128, kSymbolWaves = 4;

template <typename T, bool PAIR>
__global__ __launch_bounds__(256) void embed_symbols(SeqEmbeddingGrad p, int slabs, int64_t chunk,
                                                     float *partial) {
    constexpr int AHEAD = 8;                     // rows on their way
    extern __shared__ __align__(16) float sums[];            // of each wave: rows + 1 by 128
    constexpr int waves = kSymbolWaves;
    const int V = (int)p.rows, lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int slab = (int)(blockIdx.x % slabs);
    const int64_t c = blockIdx.x / slabs;
    for (int i = threadIdx.x; i < waves * (V + 1) * kSymbolCols; i += 256) sums[i] = 0.0f;
    __syncthreads();
    // PAIR: columns 2 lane and 2 lane + 1, else lane and lane + 64
    const int64_t col0 = (int64_t)slab * kSymbolCols + (PAIR ? 2 * lane : lane);
    const int64_t col1 = PAIR ? col0 + 1 : col0 + 64;
    const bool in0 = col0 < p.width, in1 = col1 < p.width;
    // the lane's two places of a row; tokens outside the table have one behind the rows
    float *mine = sums + wave * (V + 1) * kSymbolCols + (PAIR ? 2 * lane : lane);
    auto at = [&](int id) -> float2v {
        const float *q = mine + id * kSymbolCols;
        if constexpr (PAIR) return *(const float2v *)q;
        else return float2v{q[0], q[64]};
    };
    auto put = [&](int id, float2v v) {
        float *q = mine + id * kSymbolCols;
        if constexpr (PAIR) {
            *(float2v *)q = v;
        } else {
            q[0] = v[0];
            q[64] = v[1];
        }
    };
    // the wave's tokens
    const int64_t first = c * chunk, end = first + chunk < p.tokens ? first + chunk : p.tokens;
    const int64_t each = (chunk + waves - 1) / waves;
    const int64_t a = first + wave * each, b = a + each < end ? a + each : end;
    typedef T pair __attribute__((ext_vector_type(2)));
    // the rows of 64 tokens from t on, a lane each; V: none
    auto rows_of = [&](int64_t t) {
        const int64_t id = t + lane < b ? get_id(p.ids, p.ids_64, t + lane) : -1;
        return id >= 0 && id < V ? (int)id : V;
    };
    struct Batch { int id[AHEAD]; T x0[AHEAD], x1[AHEAD]; };
    auto load = [&](Batch &r, int ids, int k, int64_t t0) {
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            r.id[u] = __builtin_amdgcn_readlane(ids, k + u);
            r.x0[u] = r.x1[u] = (T)0.0f;
            if (r.id[u] == V) continue;          // behind the last token too
            const T *row = (const T *)p.d_out + (t0 + k + u) * p.dout_row;
            if constexpr (PAIR) {
                if (in0) {
                    const pair v = *(const pair *)(row + col0);
                    r.x0[u] = v[0];
                    r.x1[u] = v[1];
                }
            } else {
                if (in0) r.x0[u] = row[col0];
                if (in1) r.x1[u] = row[col1];
            }
        }
    };
    auto add = [&](const Batch &r) {
#pragma unroll
        for (int u = 0; u < AHEAD; u += 4) {
            float2v sum[4];
#pragma unroll
            for (int v = 0; v < 4; v++) sum[v] = at(r.id[u + v]);
#pragma unroll
            for (int v = 0; v < 4; v++) {
#pragma unroll
                for (int o = 0; o < v; o++)
                    if (r.id[u + o] == r.id[u + v]) sum[v] = sum[o];
                sum[v][0] += (float)r.x0[u + v];
                sum[v][1] += (float)r.x1[u + v];
            }
#pragma unroll
            for (int v = 0; v < 4; v++) put(r.id[u + v], sum[v]);
        }
    };
    // a batch is added while the next one is on its way
    int ids = rows_of(a);
    Batch even, odd;
    load(even, ids, 0, a);
    for (int64_t t0 = a; t0 < b; t0 += 64) {
        const int next = rows_of(t0 + 64);
        for (int k = 0; k < 64; k += 2 * AHEAD) {
            load(odd, ids, k + AHEAD, t0);
            add(even);
            if (k + 2 * AHEAD < 64) load(even, ids, k + 2 * AHEAD, t0);
            else load(even, next, 0, t0 + 64);
            add(odd);
        }
        ids = next;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < V * kSymbolCols; i += 256) {
        const int64_t col = (int64_t)slab * kSymbolCols + i % kSymbolCols;
        if (col >= p.width) continue;
        float s = sums[i];
        for (int w = 1; w < waves; w++) s += sums[w * (V + 1) * kSymbolCols + i];
        partial[(c * V + i / kSymbolCols) * p.width + col] = s;
    }
}

// The chunks' sums in their order: 32 places of the table a block, each by 32 threads (4.3 us
// for 768 chunks of 22 rows of 128). S: float where 1,024 chunks make 32 of a thread's at most,
// else double (which takes 2 us more for 12 rows of 4,096).
template <typename S>
__global__ __launch_bounds__(1024) void embed_chunks(SeqEmbeddingGrad p, int64_t chunks,
                                                     const float *partial) {
    __shared__ S part[32][33];
    const int x = threadIdx.x % 32, g = threadIdx.x / 32;
    const int64_t all = p.rows * p.width, at = blockIdx.x * 32ll + x;
    S s = 0;
    if (at < all)
#pragma unroll 8
        for (int64_t c = g; c < chunks; c += 32) s += partial[c * all + at];
    part[g][x] = s;
    __syncthreads();
    if (g == 0 && at < all) {
        s = part[0][x];
#pragma unroll
        for (int i = 1; i < 32; i++) s += part[i][x];
        put1(p.dtable, p.out_dtype, at / p.width * p.dtable_row + at % p.width, (float)s * p.scale);
    }
}

// ----------------------------------------------------------------------- sort

// Tokens are sorted by digits of at most 9 bits, the lowest first, each time in two
// launches: the digits of each tile are counted; then every tile's block adds up the
// counts of the tiles before it and of the lower digits, and moves its keys to their
// places. Tokens outside the table become the key `rows`, behind all others. Launches and the
// way to memory bound it: 16,383 tokens of 32,001 rows take 26 us in two rounds, 3.6 a count
// and 8 a move.
constexpr int kSortThreads = 512, kSortWaves = kSortThreads / 64;
constexpr int kSortSub = kSortThreads * 4;       // keys of a block at a time
constexpr int kSortTiles = 256, kDigits = 512;

struct Sort {
    const void *ids;                             // first time round; then keys and places
    const uint32_t *keys, *places;
    uint32_t *keys_to, *places_to, *counts;
    uint32_t rows, tile;                         // tile: keys of a block
    uint32_t tokens;
    int ids_64, shift, bits, tiles;
    __device__ uint32_t key(uint32_t t) const {
        if (!ids) return keys[t];
        const int64_t id = get_id(ids, ids_64, t);
        return id >= 0 && id < (int64_t)rows ? (uint32_t)id : rows;
    }
    __device__ int digit(uint32_t key) const { return (key >> shift) & ((1u << bits) - 1); }
};

__global__ __launch_bounds__(kSortThreads) void sort_count(Sort s) {
    __shared__ uint32_t n[kDigits];
    n[threadIdx.x] = 0;
    __syncthreads();
    const uint64_t a = (uint64_t)blockIdx.x * s.tile;
    const uint64_t b = a + s.tile < s.tokens ? a + s.tile : s.tokens;
    for (uint64_t t = a + threadIdx.x; t < b; t += kSortThreads)
        atomicAdd(&n[s.digit(s.key((uint32_t)t))], 1u);     // a count: any order
    __syncthreads();
    if ((int)threadIdx.x < 1 << s.bits) s.counts[(blockIdx.x << s.bits) + threadIdx.x] = n[threadIdx.x];
}

__global__ __launch_bounds__(kSortThreads) void sort_move(Sort s) {
    __shared__ uint32_t wave_n[kSortWaves][kDigits];
    __shared__ uint32_t base[kDigits], total[kSortThreads], before[kSortThreads];
    const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64;
    const int digits = 1 << s.bits, d = tid & (digits - 1);
    // counts of digit d in all tiles and in those before this one
    uint32_t all = 0, prior = 0;
#pragma unroll 8
    for (int t = tid >> s.bits; t < s.tiles; t += kSortThreads >> s.bits) {
        const uint32_t c = s.counts[(t << s.bits) + d];
        all += c;
        prior += t < (int)blockIdx.x ? c : 0;
    }
    total[tid] = all;
    before[tid] = prior;
    __syncthreads();
    if (tid < digits)
        for (int t = tid + digits; t < kSortThreads; t += digits) {
            all += total[t];
            prior += before[t];
        }
    // counts of lower digits: running sums in waves, then over them
    if (tid >= digits) all = 0;
    uint32_t sum = all;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const uint32_t add = __shfl_up(sum, o);
        sum += lane >= o ? add : 0;
    }
    if (lane == 63) base[wave] = sum;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSortWaves - 1; w++) sum += w < wave ? base[w] : 0;
    __syncthreads();
    if (tid < digits) base[tid] = sum - all + prior;
    const uint64_t first = (uint64_t)blockIdx.x * s.tile;
    const uint64_t end = first + s.tile < s.tokens ? first + s.tile : s.tokens;
    for (uint64_t at = first; at < end; at += kSortSub) {
        for (int i = tid; i < kSortWaves * kDigits; i += kSortThreads) (&wave_n[0][0])[i] = 0;
        __syncthreads();
        uint32_t key[4], rank[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {            // a wave's 256 keys in order, 64 at a time
            const uint64_t t = at + wave * 256 + r * 64 + lane;
            const bool is = t < end;
            key[r] = is ? s.key((uint32_t)t) : 0;
            const int x = s.digit(key[r]);
            uint64_t same = __ballot(is);
            for (int b = 0; b < s.bits; b++) {
                const uint64_t set = __ballot((x >> b) & 1);
                same &= (x >> b) & 1 ? set : ~set;
            }
            const uint32_t lower = __popcll(same & ((1ull << lane) - 1));
            const uint32_t have = wave_n[wave][x];
            wave_sync();
            if (is && lower == 0) wave_n[wave][x] = have + __popcll(same);
            wave_sync();
            rank[r] = have + lower;
        }
        __syncthreads();
        if (tid < digits) {
            uint32_t run = base[tid];
#pragma unroll
            for (int w = 0; w < kSortWaves; w++) {
                const uint32_t n = wave_n[w][tid];
                wave_n[w][tid] = run;
                run += n;
            }
            base[tid] = run;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const uint64_t t = at + wave * 256 + r * 64 + lane;
            if (t >= end) continue;
            const uint32_t to = wave_n[wave][s.digit(key[r])] + rank[r];
            s.keys_to[to] = key[r];
            s.places_to[to] = s.ids ? (uint32_t)t : s.places[t];
        }
        __syncthreads();
    }
}

// ----------------------------------------------------------------------- sums

struct Runs {
    const uint32_t *keys, *places;               // sorted
    float *slots;                                // two rows of `pitch` a chunk
    int64_t chunks, pitch, sum_blocks;
    int chunk, g, slabs, zero_rows;
};

// Whether row v has a token: the first key not below v
__device__ inline bool has_token(const uint32_t *keys, uint32_t n, uint32_t v) {
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (keys[mid] < v) lo = mid + 1;
        else hi = mid;
    }
    return lo < n && keys[lo] == v;
}

// Zeros in those of `rows` rows from v0 on that are not present: 16 bytes a thread, several
// rows at a time where they are narrow, past the caches, which hold what is added
template <bool ANY>
__device__ inline void zero_absent(const SeqEmbeddingGrad &p, int64_t v0, int rows,
                                   const bool *present) {
    const int e = p.out_dtype == SEQ_FP32 ? 4 : 2, bytes = (int)p.width * e;
    const int parts = (bytes + 15) / 16;
    int g = 0;
    while (g < 8 && (1 << g) < parts) g++;
    for (int row = threadIdx.x >> g; row < rows; row += 256 >> g) {
        if (present[row]) continue;
        char *to = (char *)p.dtable + (v0 + row) * p.dtable_row * e;
        for (int i = threadIdx.x & ((1 << g) - 1); i < parts; i += 1 << g) {
            const uint4v zero = {0, 0, 0, 0};
            if (!ANY) {
                __builtin_nontemporal_store(zero, (uint4v *)to + i);
            } else if (i * 16 + 16 <= bytes) {
                __builtin_memcpy(to + i * 16, &zero, 16);
            } else {
                for (int b = i * 16; b < bytes; b += 2) *(uint16_t *)(to + b) = 0;
            }
        }
    }
}

// The first blocks: 2^g threads add a chunk's rows, a slab of columns at a time. The
// others write zeros where a row of the table has no token: they need no sums, and fill the
// memory's time while the first wait for rows. 16,383 tokens of 4,096 in bf16 and 32,001 rows
// in fp32 (134 MB in, 524 out) take 91 us, 7.2 TB/s.
template <typename T, bool ANY>
__global__ __launch_bounds__(256) void embed_sum(SeqEmbeddingGrad p, Runs r) {
    constexpr int AHEAD = 8, W = 8;              // rows on their way
    __shared__ bool present[256];
    const uint32_t n = (uint32_t)p.tokens, V = (uint32_t)p.rows;
    const int64_t block = block_number();
    if (block >= r.sum_blocks) {
        const int64_t v0 = (block - r.sum_blocks) * r.zero_rows;
        if (v0 >= p.rows) return;                // the launch's last numbers
        const int rows = (int)(p.rows - v0 < r.zero_rows ? p.rows - v0 : r.zero_rows);
        if ((int)threadIdx.x < rows)
            present[threadIdx.x] = has_token(r.keys, n, (uint32_t)(v0 + threadIdx.x));
        __syncthreads();
        zero_absent<ANY>(p, v0, rows, present);
        return;
    }
    const int groups = 256 >> r.g, lane = threadIdx.x & ((1 << r.g) - 1);
    const int slab = (int)(block % r.slabs);
    const int64_t c = block / r.slabs * groups + (threadIdx.x >> r.g);
    const int64_t col = ((int64_t)slab * (1 << r.g) + lane) * W;
    if (c >= r.chunks || col >= p.width) return;
    const int cells = ANY && p.width - col < 8 ? (int)(p.width - col) : 8;
    const uint32_t a = (uint32_t)(c * r.chunk);
    const uint32_t b = n - a < (uint32_t)r.chunk ? n : a + r.chunk;
    const uint32_t last = a ? r.keys[a - 1] : 0xffffffffu, next = b < n ? r.keys[b] : 0xffffffffu;
    const T *x = (const T *)p.d_out + col;
    float sum[W] = {};
    uint32_t run = r.keys[a];
    bool from_before = run == last;
    auto flush = [&](bool goes_on) {
        if (run >= V) return;
        if (from_before || goes_on) {
            Eight<float>::put(r.slots + (2 * c + !from_before) * r.pitch + col, sum);
        } else {
            float f[W];
#pragma unroll
            for (int j = 0; j < W; j++) f[j] = sum[j] * p.scale;
            put_cells<ANY>(p.dtable, p.out_dtype, run * p.dtable_row + col, f, cells);
        }
    };
    for (uint32_t at = a; at < b; at += AHEAD) {
        uint32_t key[AHEAD];
        Cells<T, ANY> v[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            key[i] = at + i < b ? r.keys[at + i] : V;
            v[i].zero();
            if (key[i] < V) v[i].load(x + r.places[at + i] * p.dout_row, cells);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            if (at + i >= b) break;
            if (key[i] != run) {
                flush(false);
                run = key[i];
                from_before = false;
#pragma unroll
                for (int j = 0; j < W; j++) sum[j] = 0.0f;
            }
            float f[W];
            v[i].get(f);
#pragma unroll
            for (int j = 0; j < W; j++) sum[j] += f[j];
        }
    }
    flush(run == next);
}

// Joins the slots of a run that begins in a chunk and goes on, 128 columns at a time, 4 to a
// thread. A block looks at eight chunks, 32 threads each, and those join a run of up to
// eight more chunks by themselves; a longer one is the whole block's, in eight parts, each
// added in 64 bits, for it may have any number of chunks. 512 chunks of 32 words of 4,096 take
// 11 us, most of them the search for runs.
typedef double double4v __attribute__((ext_vector_type(4)));
__global__ __launch_bounds__(256) void embed_join(SeqEmbeddingGrad p, Runs r) {
    __shared__ float4v part[8][33];
    __shared__ bool longer[8];
    constexpr int FEW = 8;
    const int x = threadIdx.x % 32, g = threadIdx.x / 32;
    const int64_t c0 = block_number() * 8ll, c = c0 + g;
    uint32_t run = 0;
    bool begins = false;
    if (c < r.chunks - 1) {
        const uint32_t a = (uint32_t)(c * r.chunk), b = a + r.chunk;
        run = r.keys[b - 1];
        begins = run < (uint32_t)p.rows && r.keys[b] == run &&
                 !(a && r.keys[a] == run && r.keys[a - 1] == run);    // began before
    }
    // how many of the next 32 chunks begin with it
    const int64_t k = c + 1 + x;
    const uint64_t with = __ballot(begins && k < r.chunks && r.keys[k * r.chunk] == run);
    const int more = __popc((uint32_t)(with >> (threadIdx.x & 32)));
    if (x == 0) longer[g] = more > FEW;
    __syncthreads();
    auto put = [&](uint32_t row, int64_t col, const float4v &s) {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (col + e < p.width)
                put1(p.dtable, p.out_dtype, (int64_t)row * p.dtable_row + col + e, s[e] * p.scale);
    };
    auto slot = [&](int64_t at, int64_t col) {               // slots are whole eights of columns
        return *(const float4v *)(r.slots + at * r.pitch + col);
    };
    if (begins && more <= FEW)
        for (int64_t col = blockIdx.y * 128ll + x * 4; col < p.width; col += gridDim.y * 128ll) {
            float4v s = slot(2 * c + 1, col), v[FEW];
#pragma unroll
            for (int o = 0; o < FEW; o++)
                if (o < more) v[o] = slot(2 * (c + 1 + o), col);
#pragma unroll
            for (int o = 0; o < FEW; o++)
                if (o < more) s += v[o];
            put(run, col, s);
        }
    for (int i = 0; i < 8; i++) {
        if (!longer[i]) continue;                // the block's branch
        const int64_t from = c0 + i;
        const uint32_t row = r.keys[(from + 1) * r.chunk - 1];
        // the first chunk that does not begin with it, 256 looked at at a time
        int64_t end = from + 1;
        for (int n = 256; n == 256; end += n) {
            const int64_t at = end + threadIdx.x;
            n = __syncthreads_count(at < r.chunks && r.keys[at * r.chunk] == row);
        }
        for (int64_t col0 = blockIdx.y * 128ll; col0 < p.width; col0 += gridDim.y * 128ll) {
            const int64_t col = col0 + x * 4;
            double4v sum = {0, 0, 0, 0};
            if (col < p.width) {
                if (g == 0) sum = __builtin_convertvector(slot(2 * from + 1, col), double4v);
#pragma unroll 8
                for (int64_t at = from + 1 + g; at < end; at += 8)
                    sum += __builtin_convertvector(slot(2 * at, col), double4v);
            }
            __syncthreads();
            part[g][x] = __builtin_convertvector(sum, float4v);
            __syncthreads();
            if (g == 0 && col < p.width) {
                float4v s = part[0][x];
#pragma unroll
                for (int o = 1; o < 8; o++) s += part[o][x];
                put(row, col, s);
            }
        }
    }
}

// Up to 256 tokens, in one launch: a block a token and slab of columns, which adds the rows of
// all tokens like it if it is the first of them, and blocks for the rows without one. A
// call of 256 tokens and 32,001 rows of 1,024 in fp32 takes 23 us, sorted 41, of one token and
// 131,071 rows of 64 9 and 23.
constexpr int kFewTokens = 256;
template <typename T, bool ANY>
__global__ __launch_bounds__(256) void embed_few(SeqEmbeddingGrad p, int slabs, int zero_rows) {
    constexpr int AHEAD = 8, W = 8;              // rows on their way
    __shared__ __align__(16) uint32_t keys[kFewTokens];
    __shared__ uint64_t like[kFewTokens / 64];
    const int tid = threadIdx.x, n = (int)p.tokens;
    const int64_t block = block_number(), sums = (int64_t)n * slabs;
    const int64_t id = tid < n ? get_id(p.ids, p.ids_64, tid) : -1;
    const uint32_t key = id >= 0 && id < p.rows ? (uint32_t)id : 0xffffffffu;
    if (block >= sums) {
        const int64_t v0 = (block - sums) * zero_rows;
        if (v0 >= p.rows) return;                // the launch's last numbers
        __shared__ bool present[256];
        const int rows = (int)(p.rows - v0 < zero_rows ? p.rows - v0 : zero_rows);
        keys[tid] = key;
        __syncthreads();
        if (tid < rows) {                        // four tokens at a time, none behind the last
            bool is = false;
#pragma unroll 4
            for (int u = 0; u < n; u += 4) {
                const uint4v k = *(const uint4v *)(keys + u);
#pragma unroll
                for (int j = 0; j < 4; j++) is |= k[j] == (uint32_t)(v0 + tid);
            }
            present[tid] = is;
        }
        __syncthreads();
        zero_absent<ANY>(p, v0, rows, present);
        return;
    }
    const int t = (int)(block / slabs);
    keys[tid] = key;
    __syncthreads();
    const uint32_t mine = keys[t];
    if (mine == 0xffffffffu || __syncthreads_or(tid < t && key == mine)) return;
    const uint64_t with = __ballot(key == mine);
    if ((tid & 63) == 0) like[tid >> 6] = with;
    __syncthreads();
    const int64_t col = ((int64_t)(block % slabs) * 256 + tid) * W;
    if (col >= p.width) return;
    const int cells = ANY && p.width - col < 8 ? (int)(p.width - col) : 8;
    const T *x = (const T *)p.d_out + col;
    float sum[W] = {};
    for (int w = 0; w < (n + 63) / 64; w++) {
        uint64_t left = like[w];
        while (left) {
            Cells<T, ANY> v[AHEAD];
            bool is[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                is[i] = left != 0;
                v[i].zero();
                if (!is[i]) continue;
                const int u = w * 64 + __ffsll((unsigned long long)left) - 1;
                left &= left - 1;
                v[i].load(x + u * p.dout_row, cells);
            }
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                if (!is[i]) continue;
                float f[W];
                v[i].get(f);
#pragma unroll
                for (int j = 0; j < W; j++) sum[j] += f[j];
            }
        }
    }
#pragma unroll
    for (int j = 0; j < W; j++) sum[j] *= p.scale;
    put_cells<ANY>(p.dtable, p.out_dtype, (int64_t)mine * p.dtable_row + col, sum, cells);
}

__global__ __launch_bounds__(256) void embed_zero(SeqEmbeddingGrad p) {
    const int64_t v = block_number();
    if (v >= p.rows) return;
    for (int64_t j = threadIdx.x; j < p.width; j += 256)
        put1(p.dtable, p.out_dtype, v * p.dtable_row + j, 0.0f);
}

// ------------------------------------------------------------------- launches

int check_embedding(const SeqEmbedding *p) {
    if (!p || p->struct_size != (int32_t)sizeof(SeqEmbedding)) return CO_ERR_NULLARG;
    if (p->tokens < 0 || p->rows < 0 || p->width < 1) return CO_ERR_NULLARG;
    if (p->tokens > SEQ_MAX_ROWS || p->rows > SEQ_MAX_ROWS || p->width > SEQ_MAX_WIDTH)
        return CO_ERR_BOUNDS;
    if (!float_type(p->dtype) || !float_type(p->out_dtype) || !(fabsf(p->scale) <= 3.4028235e38f))
        return CO_ERR_DATA;
    return CO_OK;
}
int check_embedding_grad(const SeqEmbeddingGrad *p) {
    if (!p || p->struct_size != (int32_t)sizeof(SeqEmbeddingGrad)) return CO_ERR_NULLARG;
    if (p->tokens < 0 || p->rows < 0 || p->width < 1) return CO_ERR_NULLARG;
    if (p->tokens > SEQ_MAX_ROWS || p->rows > SEQ_MAX_ROWS || p->width > SEQ_MAX_WIDTH)
        return CO_ERR_BOUNDS;
    if (!float_type(p->dtype) || !float_type(p->out_dtype) || !(fabsf(p->scale) <= 3.4028235e38f))
        return CO_ERR_DATA;
    return CO_OK;
}

// Places of a chunk: few tokens fill the chip with short ones (4,096 words of 4,096 in bf16:
// 137 us with 16, 143 with 32; 16,384: 187, 185, with 64 214; 60,000 of 1,024: 101, 88, 98;
// 500,000 of 128 with 64 99, with 128 131)
int64_t chunk_of(int64_t tokens) {
    return tokens <= 1 << 13 ? 16 : (tokens <= 1 << 16 ? 32 : (tokens <= 1 << 22 ? 64 : 256));
}
int64_t aligned256(int64_t n) { return (n + 255) / 256 * 256; }

// Slabs of columns and chunks of tokens of the symbols' kernel; chunks fill the chip and
// have 16 tokens a wave at least, and 4,096 at most: those are added one after the other in
// 32 bits, so that a sum's error does not grow with the tokens. (1,024 at most cost 3 to 5 in
// 100 of the time, in more blocks.) The chunks' sums are some rows / 8,192 of a gradient in
// 16 bits; where more rows than memory holds lie on each other, chunks are as long as a
// workspace of 4 GiB makes them.
constexpr int64_t kSymbolChunk = 4096 * kSymbolWaves, kSymbolBytes = 1ll << 32;
struct SymbolPlan { int slabs; int64_t chunk, chunks; };
bool few_symbols(const SeqEmbeddingGrad &p) { return p.rows <= kSymbolRows; }
int64_t symbol_lds(const SeqEmbeddingGrad &p) { return kSymbolWaves * (p.rows + 1) * kSymbolCols * 4; }
SymbolPlan symbol_plan(const SeqEmbeddingGrad &p) {
    SymbolPlan r;
    r.slabs = (int)((p.width + kSymbolCols - 1) / kSymbolCols);
    const int64_t fit = (160 << 10) / symbol_lds(p), least = 16 * kSymbolWaves;
    int64_t chunks = 256 * (fit < 8 ? fit : 8) / r.slabs;
    const int64_t most = (p.tokens + least - 1) / least;
    if (chunks < 1) chunks = 1;
    // as many times over as chunks of that length need, so that the chip stays full to the end
    const int64_t turn = chunks * kSymbolChunk;
    const int64_t turns = (p.tokens + turn - 1) / turn;
    const int64_t room = kSymbolBytes / (4 * p.rows * p.width * chunks);
    chunks *= turns < room ? turns : room;       // room: 400 turns at least
    if (chunks > most) chunks = most;
    r.chunk = (p.tokens + chunks - 1) / chunks;
    r.chunks = (p.tokens + r.chunk - 1) / r.chunk;
    return r;
}
template <typename T> void launch_symbols(const SeqEmbeddingGrad &p, float *partial, hipStream_t s) {
    const SymbolPlan r = symbol_plan(p);
    const unsigned grid = (unsigned)(r.chunks * r.slabs);
    const size_t lds = (size_t)symbol_lds(p);
    const bool pairs = !((uintptr_t)p.d_out % (2 * sizeof(T))) && p.dout_row % 2 == 0 && p.width % 2 == 0;
    if (pairs) embed_symbols<T, true><<<grid, 256, lds, s>>>(p, r.slabs, r.chunk, partial);
    else embed_symbols<T, false><<<grid, 256, lds, s>>>(p, r.slabs, r.chunk, partial);
    const unsigned places = (unsigned)((p.rows * p.width + 31) / 32);
    if (r.chunks <= 1024) embed_chunks<float><<<places, 1024, 0, s>>>(p, r.chunks, partial);
    else embed_chunks<double><<<places, 1024, 0, s>>>(p, r.chunks, partial);
}

struct GradPlan {
    int passes, bits;
    int64_t tile, tiles, chunk, chunks, pitch;
    int64_t keys, counts, slots, total;          // bytes of one list, of the rest; offsets
};
GradPlan grad_plan(const SeqEmbeddingGrad &p) {
    GradPlan r = {};
    if (p.tokens <= kFewTokens) return r;
    if (few_symbols(p)) {
        r.total = 4 * symbol_plan(p).chunks * p.rows * p.width;
        return r;
    }
    int bits = 1;
    while (bits < 31 && (1ll << bits) <= p.rows) bits++;              // holds `rows` itself
    r.passes = (bits + 8) / 9;
    r.bits = (bits + r.passes - 1) / r.passes;
    const int64_t subs = (p.tokens + kSortSub - 1) / kSortSub;
    r.tile = (subs + kSortTiles - 1) / kSortTiles * kSortSub;
    r.tiles = (p.tokens + r.tile - 1) / r.tile;
    r.chunk = chunk_of(p.tokens);
    r.chunks = (p.tokens + r.chunk - 1) / r.chunk;
    r.pitch = (p.width + 7) / 8 * 8;
    r.keys = aligned256(4 * p.tokens);
    r.counts = 4 * r.keys;                       // two lists of keys and two of places
    r.slots = r.counts + 4ll * kSortTiles * kDigits;
    r.total = r.slots + 8 * r.chunks * r.pitch;
    return r;
}

template <typename T, bool ANY>
void launch_sum(const SeqEmbeddingGrad &p, Runs r, hipStream_t s) {
    const int64_t parts = (p.width + 7) / 8;
    r.g = group_log(parts);
    r.slabs = (int)((parts + (1 << r.g) - 1) >> r.g);
    const int groups = 256 >> r.g;
    r.sum_blocks = (r.chunks + groups - 1) / groups * r.slabs;
    const int64_t zero = 65536 / p.width;        // rows that make a block's worth of zeros
    r.zero_rows = (int)(zero < 4 ? 4 : (zero > 256 ? 256 : zero));
    const int64_t blocks = r.sum_blocks + (p.rows + r.zero_rows - 1) / r.zero_rows;
    embed_sum<T, ANY><<<grid_of(blocks, 256), 256, 0, s>>>(p, r);
}
template <typename T> void launch_sum(const SeqEmbeddingGrad &p, const Runs &r, hipStream_t s) {
    const bool eights = p.width % 8 == 0 && in_eights(p.d_out, p.dout_row) &&
                        in_eights(p.dtable, p.dtable_row);
    if (eights) launch_sum<T, false>(p, r, s);
    else launch_sum<T, true>(p, r, s);
}

template <typename T, bool ANY> void launch_few(const SeqEmbeddingGrad &p, hipStream_t s) {
    const int slabs = (int)((p.width + 2047) / 2048);
    const int64_t zero = 65536 / p.width;
    const int zero_rows = (int)(zero < 4 ? 4 : (zero > 256 ? 256 : zero));
    const int64_t blocks = p.tokens * slabs + (p.rows + zero_rows - 1) / zero_rows;
    embed_few<T, ANY><<<grid_of(blocks, 256), 256, 0, s>>>(p, slabs, zero_rows);
}
template <typename T> void launch_few(const SeqEmbeddingGrad &p, hipStream_t s) {
    const bool eights = p.width % 8 == 0 && in_eights(p.d_out, p.dout_row) &&
                        in_eights(p.dtable, p.dtable_row);
    if (eights) launch_few<T, false>(p, s);
    else launch_few<T, true>(p, s);
}

template <typename T> void launch_embed(const SeqEmbedding &p, hipStream_t s) {
    const bool eights = p.width % 8 == 0 && in_eights(p.table, p.table_row) &&
                        in_eights(p.out, p.out_row);
    const int g = group_log((p.width + 7) / 8);
    const int rows = 256 >> g;
    const dim3 grid = grid_of((p.tokens + rows - 1) / rows, 256);
    if (eights) embed_rows<T, false><<<grid, 256, 0, s>>>(p, g);
    else embed_rows<T, true><<<grid, 256, 0, s>>>(p, g);
}

}  // namespace seq

extern "C" int seq_embedding(const SeqEmbedding *p, void *stream) {
    const int rc = seq::check_embedding(p);
    if (rc != CO_OK) return rc;
    if (p->tokens == 0) return CO_OK;
    if (!p->ids || (!p->table && p->rows) || !p->out) return CO_ERR_NULLARG;
    hipStream_t s = (hipStream_t)stream;
    switch (p->dtype) {
        case SEQ_FP32: seq::launch_embed<float>(*p, s); break;
        case SEQ_BF16: seq::launch_embed<__bf16>(*p, s); break;
        default: seq::launch_embed<_Float16>(*p, s); break;
    }
    return seq::launch_status();
}

extern "C" int64_t seq_embedding_grad_workspace(const SeqEmbeddingGrad *p) {
    const int rc = seq::check_embedding_grad(p);
    if (rc != CO_OK) return rc > 0 ? -rc : rc;
    return p->tokens && p->rows ? seq::grad_plan(*p).total : 0;
}

extern "C" int seq_embedding_grad(const SeqEmbeddingGrad *p, void *stream) {
    const int rc = seq::check_embedding_grad(p);
    if (rc != CO_OK) return rc;
    if (p->rows == 0) return CO_OK;
    if (!p->dtable) return CO_ERR_NULLARG;
    hipStream_t s = (hipStream_t)stream;
    if (p->tokens == 0) {
        seq::embed_zero<<<seq::grid_of(p->rows, 256), 256, 0, s>>>(*p);
        return seq::launch_status();
    }
    if (!p->ids || !p->d_out) return CO_ERR_NULLARG;
    if (p->tokens <= seq::kFewTokens) {
        switch (p->dtype) {
            case SEQ_FP32: seq::launch_few<float>(*p, s); break;
            case SEQ_BF16: seq::launch_few<__bf16>(*p, s); break;
            default: seq::launch_few<_Float16>(*p, s); break;
        }
        return seq::launch_status();
    }
    if (!p->workspace) return CO_ERR_NULLARG;
    const seq::GradPlan plan = seq::grad_plan(*p);
    if (p->workspace_bytes < plan.total || ((uintptr_t)p->workspace & 255)) return CO_ERR_DATA;
    char *ws = (char *)p->workspace;
    if (seq::few_symbols(*p)) {
        switch (p->dtype) {
            case SEQ_FP32: seq::launch_symbols<float>(*p, (float *)ws, s); break;
            case SEQ_BF16: seq::launch_symbols<__bf16>(*p, (float *)ws, s); break;
            default: seq::launch_symbols<_Float16>(*p, (float *)ws, s); break;
        }
        return seq::launch_status();
    }
    uint32_t *keys[2] = {(uint32_t *)ws, (uint32_t *)(ws + plan.keys)};
    uint32_t *places[2] = {(uint32_t *)(ws + 2 * plan.keys), (uint32_t *)(ws + 3 * plan.keys)};
    seq::Sort sort = {};
    sort.counts = (uint32_t *)(ws + plan.counts);
    sort.rows = (uint32_t)p->rows;
    sort.tokens = (uint32_t)p->tokens;
    sort.tile = (uint32_t)plan.tile;
    sort.tiles = (int)plan.tiles;
    sort.ids_64 = p->ids_64;
    sort.bits = plan.bits;
    int at = 0;
    for (int i = 0; i < plan.passes; i++, at ^= 1) {
        sort.ids = i ? nullptr : p->ids;
        sort.keys = keys[at ^ 1];
        sort.places = places[at ^ 1];
        sort.keys_to = keys[at];
        sort.places_to = places[at];
        sort.shift = i * plan.bits;
        seq::sort_count<<<sort.tiles, seq::kSortThreads, 0, s>>>(sort);
        seq::sort_move<<<sort.tiles, seq::kSortThreads, 0, s>>>(sort);
    }
    seq::Runs r = {};
    r.keys = keys[at ^ 1];
    r.places = places[at ^ 1];
    r.slots = (float *)(ws + plan.slots);
    r.chunks = plan.chunks;
    r.chunk = (int)plan.chunk;
    r.pitch = plan.pitch;
    switch (p->dtype) {
        case SEQ_FP32: seq::launch_sum<float>(*p, r, s); break;
        case SEQ_BF16: seq::launch_sum<__bf16>(*p, r, s); break;
        default: seq::launch_sum<_Float16>(*p, r, s); break;
    }
    if (r.chunks > 1) {
        // columns of a run go to several blocks while chunks are too few to fill the chip
        const int64_t slabs = (p->width + 127) / 128, blocks = (r.chunks + 6) / 8;
        int64_t y = 4096 / blocks + 1;
        if (y > slabs) y = slabs;
        seq::embed_join<<<seq::grid_of(blocks, 256, (unsigned)y), 256, 0, s>>>(*p, r);
    }
    return seq::launch_status();
}
