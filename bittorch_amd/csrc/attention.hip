// Attention of new tokens over the paged cache (bt_cached_attention): o = softmax(scale q K^T) V over a prefix that all sequences share and
// over the sequence's own pages, causal among the new tokens.
//
// The G query heads of a key head and the new tokens of a sequence are the rows of one product: row i G + h of the sequence.  Its keys are
// cut into chunks, a workgroup each, which keep the softmax running over 16-byte groups of keys: maximum m, sum l and o in registers, all in
// 32 bits.  Workgroups that do not see all keys of their rows leave (m, l, o) in the workspace, and attend_join_kernel joins them in the
// order of the keys.  The rows of every sequence together are the rows of the prefix, whose keys are thus read once for all.
//
// At few rows the launch is bound by the cache's bytes, at many by the matrix cores and the exponentials.
#include "paged_cache.h"

namespace bt {

struct AttendParams {
    const void *q, *k_cache, *v_cache;
    const int32_t *table, *lengths, *starts, *prefix_table;
    int64_t q_token, q_head, tokens;
    void* out;
    float* lse;          // may be null
    float* part_o;       // [row][part][dim], row = token * heads + head; null: a workgroup sees all keys of its rows
    float2* part_ml;     // [row][part]
    int heads, kv_heads, group, dim, dp, n_seq, width, page_shift, pages, prefix;
    int chunk, prefix_chunk, chunks, prefix_chunks;  // places of a chunk; chunks of the longest sequence and of the prefix
    int units, prefix_units;                         // row tiles
    int seq_tiles;                                   // of a sequence's one token
    int longest, wide_q;
    float scale2;                                    // scale / ln 2
};

template <int DT>
struct Half8;  // an operand of 16-bit elements
template <>
struct Half8<BT_F16> { using type = v8h; };
template <>
struct Half8<BT_BF16> { using type = v8bf; };

// Four lanes' groups of E elements of the contraction: a (16 rows) times b (16 columns)
template <int DT>
__device__ __forceinline__ v4f step(u32x4 a, u32x4 b, v4f c) {
    if constexpr (DT == BT_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
    else if constexpr (DT == BT_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    else {
#pragma unroll
        for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(v4f, a)[e], __builtin_bit_cast(v4f, b)[e], c, 0, 0, 0);
        return c;
    }
}
// E weights as an operand; what rounding took from them in `rest`
template <int DT>
__device__ __forceinline__ u32x4 operand(const float (&p)[CacheOrder<DT>::E], u32x4* rest) {
    if constexpr (DT == BT_F32) {
        u32x4 a;
#pragma unroll
        for (int e = 0; e < 4; e++) a[e] = __builtin_bit_cast(uint32_t, p[e]);
        return a;
    } else {
        typename Half8<DT>::type a, r;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            a[e] = (std::remove_reference_t<decltype(a[0])>)p[e];
            r[e] = (std::remove_reference_t<decltype(a[0])>)(p[e] - (float)a[e]);
        }
        if (rest) *rest = __builtin_bit_cast(u32x4, r);
        return __builtin_bit_cast(u32x4, a);
    }
}
// Of a group of E places the first `live` (any number), the others zero
template <int DT>
__device__ __forceinline__ u32x4 first_places(u32x4 v, int live) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (DT == BT_F32) v[i] = i < live ? v[i] : 0u;
        else v[i] = 2 * i + 1 < live ? v[i] : 2 * i < live ? v[i] & 0xffffu : 0u;
    }
    return v;
}
template <int DT>
__device__ __forceinline__ bool any_special(u32x4 v) {  // infinite or not a number
    bool s = false;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (DT == BT_F32) s |= (v[i] & 0x7f800000u) == 0x7f800000u;
        else {
            constexpr uint32_t e = DT == BT_F16 ? 0x7c00u : 0x7f80u;
            s |= (v[i] & e) == e || (v[i] >> 16 & e) == e;
        }
    }
    return s;
}
__device__ __forceinline__ float over_groups_max(float x) {  // over the four lanes of a row
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float over_groups_sum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// What a workgroup works on: up to R rows of one key head and a chunk of their keys.
struct Job {
    const int32_t* table;
    int rows;            // of the tile
    int64_t token0;      // row r is token token0 + (row0 + r) / G, head kv * G + (row0 + r) % G
    int64_t row0;
    int limit0;          // row r sees the places below limit0 + (row0 + r) / G (own) or limit0 (prefix)
    bool causal, bad;    // bad: the length is beyond the table
    int begin, end;      // the chunk's places
    int part;
};
__device__ __forceinline__ int limit_of(const AttendParams& p, const Job& j, int r) { return j.causal ? j.limit0 + (int)((j.row0 + r) / p.group) : j.limit0; }

// A sequence's tokens [t0, t0 + n) and its length, as far as the table goes; whether it goes beyond
__device__ __forceinline__ bool sequence_of(const AttendParams& p, int s, int64_t* t0, int* n, int* length) {
    *t0 = p.starts ? std::max(p.starts[s], 0) : s;
    *n = p.starts ? (int)(std::min<int64_t>(p.starts[s + 1], p.tokens) - *t0) : 1;
    const int got = p.lengths[s];
    *length = std::min(got, p.longest);
    return got > p.longest;
}

// False: nothing to do.
__device__ __forceinline__ bool job_of(const AttendParams& p, int R, int64_t block, Job* j, int* kv) {
    const int64_t prefix_blocks = (int64_t)p.prefix_units * p.kv_heads * p.prefix_chunks;
    if (block < prefix_blocks) {
        const int c = (int)(block % p.prefix_chunks);
        *kv = (int)(block / p.prefix_chunks % p.kv_heads);
        j->row0 = block / p.prefix_chunks / p.kv_heads * R;
        j->token0 = 0;
        j->rows = (int)std::min<int64_t>(R, p.tokens * p.group - j->row0);
        j->table = p.prefix_table;
        j->limit0 = p.prefix;
        j->causal = j->bad = false;
        j->begin = c * p.prefix_chunk;
        j->end = std::min(j->begin + p.prefix_chunk, p.prefix);
        j->part = c;
        return j->rows > 0 && j->begin < j->end;
    }
    block -= prefix_blocks;
    const int c = (int)(block % p.chunks);
    *kv = (int)(block / p.chunks % p.kv_heads);
    const int64_t unit = block / p.chunks / p.kv_heads;
    int s = (int)(unit / p.seq_tiles);
    int64_t tile = unit % p.seq_tiles;
    if (p.starts) {
        // sequence s has the tiles floor(starts[s] G / R) + s and on: n tokens have n G / R + 1 tiles at most
        const int lane = threadIdx.x & 63;
        int found = 0;
        for (int s0 = 0; s0 < p.n_seq; s0 += 64) {
            const int i = s0 + lane;
            const uint64_t hit = __ballot(i < p.n_seq && (int64_t)std::max(p.starts[i < p.n_seq ? i : 0], 0) * p.group / R + i <= unit);
            found += __popcll(hit);
            if (hit != ~0ull) break;
        }
        s = found - 1;
        if (s < 0) return false;
        tile = unit - ((int64_t)std::max(p.starts[s], 0) * p.group / R + s);
    }
    int n, length;
    j->bad = sequence_of(p, s, &j->token0, &n, &length);
    j->row0 = tile * R;
    if (n <= 0 || j->row0 >= (int64_t)n * p.group) return false;
    j->rows = (int)std::min<int64_t>(R, (int64_t)n * p.group - j->row0);
    j->table = p.table + (int64_t)s * p.width;
    j->limit0 = length - n + 1;
    j->causal = true;
    j->begin = c * p.chunk;
    j->end = std::min(j->begin + p.chunk, limit_of(p, *j, j->rows - 1));
    j->part = p.prefix_chunks + c;
    return j->begin < j->end || (!p.part_o && c == 0);
}

// o += V^T P where values among the masked places are infinite or not a number: row by row, with the places that the row does not see set to
// zero (0 times such a value is not zero).
template <int DT, int B>
__device__ __forceinline__ void add_row_by_row(v4f (&o)[2 * B], const u32x4 (&v)[2 * B], u32x4 hi, u32x4 lo, int my_limit, int place) {
    const int lane = threadIdx.x & 63;
#pragma unroll 1
    for (int r = 0; r < 16; r++) {
        const int live = __shfl(my_limit, r) - (place + lane / 16 * CacheOrder<DT>::E);
#pragma unroll
        for (int b = 0; b < 2 * B; b++) {
            const u32x4 seen = first_places<DT>(v[b], live);
            v4f x = step<DT>(seen, hi, o[b]);  // (the same sums as without it: the row's bits do not depend on what it does not see)
            if constexpr (DT != BT_F32) x = step<DT>(seen, lo, x);
            if (lane % 16 == r) o[b] = x;
        }
    }
}

// B: blocks of 32 features that a head has at most.  Four waves take the chunk's tiles of TK places in turn, each with all rows.
template <int DT, int B>
__global__ __launch_bounds__(256) void attend_rows_kernel(AttendParams p) {
    using Order = CacheOrder<DT>;
    constexpr int E = Order::E, TK = Order::TK, C = 32 * B / TK, V = 2 * B, R = 16;
    constexpr int JB = B < 4 ? B : 4, LD = 32 * JB + 4;  // blocks that are joined at a time (LDS)
    __shared__ __attribute__((aligned(16))) float o_all[4][R * LD];
    __shared__ float m_all[4][R], l_all[4][R];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int64_t job_blocks = ((int64_t)p.prefix_units * p.prefix_chunks + (int64_t)p.units * p.chunks) * p.kv_heads;
    if ((int64_t)blockIdx.x >= job_blocks) {  // the rows behind the last sequence, where no other kernel sees to them
        const int64_t n = (int64_t)p.heads * p.dim, behind = std::max<int64_t>(0, std::min<int64_t>(p.starts[p.n_seq], p.tokens));
        for (int64_t i = behind * n + threadIdx.x; i < p.tokens * n; i += 256) store_elem<DT>(p.out, i, 0.0f);
        for (int64_t i = behind * p.heads + threadIdx.x; p.lse && i < p.tokens * p.heads; i += 256) p.lse[i] = -__builtin_inff();
        return;
    }
    Job j;
    int kv;
    if (!job_of(p, R, blockIdx.x, &j, &kv)) return;

    // the chunk's pages, one a lane (at most 64)
    const int page0 = j.begin >> p.page_shift, tiles = j.end > j.begin ? (j.end - j.begin + TK - 1) / TK : 0;
    const int n_pages = j.end > j.begin ? ((j.end - 1) >> p.page_shift) - page0 + 1 : 0;
    int page = lane < n_pages ? j.table[page0 + lane] : 0;
    const bool bad_page = (uint32_t)page >= (uint32_t)p.pages;
    const bool bad = __ballot(bad_page) != 0 || j.bad;
    if (bad_page) page = 0;

    // this lane's row as an operand
    const int64_t row = j.row0 + r;
    const int64_t token = j.token0 + row / p.group;
    const int head = kv * p.group + (int)(row % p.group);
    const int limit = r < j.rows ? limit_of(p, j, r) : 0, lowest = limit_of(p, j, 0);
    u32x4 q[C];
#pragma unroll
    for (int c = 0; c < C; c++) {
        q[c] = u32x4{0, 0, 0, 0};
        const int f = c * TK + g * E;
        if (r < j.rows && f < p.dim) {
            const int64_t at = token * p.q_token + head * p.q_head + f;
            if (p.wide_q) q[c] = *(const u32x4*)((const char*)p.q + at * Order::SIZE);
            else {
                for (int e = 0; e < E; e++) {
                    if (f + e >= p.dim) break;
                    if constexpr (DT == BT_F32) q[c][e] = ((const uint32_t*)p.q)[at + e];
                    else q[c][e / 2] |= (uint32_t)((const uint16_t*)p.q)[at + e] << (e % 2 * 16);
                }
            }
        }
    }

    float m = -__builtin_inff(), l = 0.0f;  // of the row; l: of this lane's places
    v4f o[V];
#pragma unroll
    for (int b = 0; b < V; b++) o[b] = v4f{0, 0, 0, 0};
    const int64_t page_elements = (int64_t)p.dp << p.page_shift;
    for (int tile = wave; tile < tiles; tile += 4) {
        const int place = j.begin + tile * TK;
        const int64_t pg = __builtin_amdgcn_readlane(page, (place >> p.page_shift) - page0);
        const int64_t at = (pg * p.kv_heads + kv) * page_elements + (int64_t)(place & ((1 << p.page_shift) - 1)) * p.dp + lane * E;
        const char* kp = (const char*)p.k_cache + at * Order::SIZE;
        const char* vp = (const char*)p.v_cache + at * Order::SIZE;
        u32x4 k[C][E / 4], v[V];
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int t = 0; t < E / 4; t++) {
                k[c][t] = u32x4{0, 0, 0, 0};
                if (c * TK + g * E < p.dim) k[c][t] = *(const u32x4*)(kp + (c * (E / 4) + t) * 1024);
            }
#pragma unroll
        for (int b = 0; b < V; b++) {
            v[b] = u32x4{0, 0, 0, 0};
            if (b * 16 < p.dim) v[b] = *(const u32x4*)(vp + b * 1024);
        }
        float x[E];
#pragma unroll
        for (int t = 0; t < E / 4; t++) {
            v4f s = {0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < C; c++) s = step<DT>(k[c][t], q[c], s);
#pragma unroll
            for (int i = 0; i < 4; i++) x[4 * t + i] = s[i] * p.scale2;
        }
        const bool masked = place + TK > lowest;  // some row does not see all of the tile
        if (masked) {
#pragma unroll
            for (int e = 0; e < E; e++) x[e] = place + g * E + e < limit ? x[e] : -__builtin_inff();
            const int live = j.end - (place + g * E);  // no row sees what lies behind: whatever it is
#pragma unroll
            for (int b = 0; b < V; b++) v[b] = first_places<DT>(v[b], live);
        }
        float top = x[0];
#pragma unroll
        for (int e = 1; e < E; e++) top = fmaxf(top, x[e]);
        if (__any(top > m)) {
            const float next = fmaxf(m, over_groups_max(top));
            const float shrink = __builtin_amdgcn_exp2f(m == next ? 0.0f : m - next);
            m = next;
            l *= shrink;
#pragma unroll
            for (int b = 0; b < V; b++) o[b] *= shrink;
        }
        const float base = m == -__builtin_inff() ? 0.0f : m;
        float w[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
            w[e] = __builtin_amdgcn_exp2f(x[e] - base);
            l += w[e];
        }
        u32x4 lo;
        const u32x4 hi = operand<DT>(w, &lo);
        bool special = false;
        if (masked) {
#pragma unroll
            for (int b = 0; b < V; b++) special |= any_special<DT>(v[b]);
        }
        if (masked && __any(special)) {
            add_row_by_row<DT, B>(o, v, hi, lo, limit, place);
        } else {
#pragma unroll
            for (int b = 0; b < V; b++) {
                o[b] = step<DT>(v[b], hi, o[b]);
                if constexpr (DT != BT_F32) o[b] = step<DT>(v[b], lo, o[b]);
            }
        }
    }
    l = over_groups_sum(l);

    // the four waves' shares of every row
    if (g == 0) m_all[wave][r] = m, l_all[wave][r] = l;
    const int64_t parts = p.prefix_chunks + p.chunks;
#pragma unroll
    for (int b0 = 0; b0 < B; b0 += JB) {
        if (b0) __syncthreads();
#pragma unroll
        for (int b = 0; b < 2 * JB; b++)
            if (2 * b0 + b < V) *(v4f*)&o_all[wave][r * LD + b * 16 + g * 4] = o[(2 * b0 + b) % V];
        __syncthreads();
        for (int idx = threadIdx.x; idx < j.rows * 8 * JB; idx += 256) {
            const int row_at = idx / (8 * JB), at = idx % (8 * JB) * 4, f = b0 * 32 + at;
            if (f >= p.dim) continue;
            float top = m_all[0][row_at];
#pragma unroll
            for (int w = 1; w < 4; w++) top = fmaxf(top, m_all[w][row_at]);
            const float base = top == -__builtin_inff() ? 0.0f : top;
            float sum = 0.0f;
            v4f acc = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float share = __builtin_amdgcn_exp2f(m_all[w][row_at] - base);
                sum += share * l_all[w][row_at];
                const v4f ow = *(const v4f*)&o_all[w][row_at * LD + at];
                acc += ow * share;
            }
            if (bad) sum = __builtin_nanf("");
            const int64_t rw = j.row0 + row_at, t = j.token0 + rw / p.group;
            const int64_t out_row = t * p.heads + kv * p.group + rw % p.group;
            if (p.part_o) {
                if (f == 0) p.part_ml[out_row * parts + j.part] = make_float2(top, sum);
                float* to = p.part_o + (out_row * parts + j.part) * p.dim;
                for (int i = 0; i < 4; i++)
                    if (f + i < p.dim) to[f + i] = acc[i];
            } else {
                const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
                for (int i = 0; i < 4; i++)
                    if (f + i < p.dim) store_elem<DT>(p.out, out_row * p.dim + f + i, acc[i] * inverse);
                if (f == 0 && p.lse) p.lse[out_row] = sum == 0.0f ? -__builtin_inff() : top * 0.69314718055994530942f + __logf(sum);
            }
        }
    }
}

// A wave to a row: the parts' weights, a lane each, then the sum of the parts in the order of their keys.
template <int DT>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendParams p) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= p.tokens * p.heads) return;
    const int64_t token = row / p.heads;
    const int s = p.starts ? owner_of(p.starts, p.n_seq, token) : (int)token;
    int own = 0;
    bool bad = false;
    if (s >= 0) {
        int64_t t0;
        int n, length;
        bad = sequence_of(p, s, &t0, &n, &length);
        const int64_t limit = length - n + 1 + (token - t0);
        own = limit > 0 ? (int)((limit + p.chunk - 1) / p.chunk) : 0;
    }
    const int64_t parts = p.prefix_chunks + p.chunks;
    const int count = s < 0 ? 0 : p.prefix_chunks + own;
    const float2* ml = p.part_ml + row * parts;
    float top = -__builtin_inff(), sum = 0.0f;
    for (int i = lane; i < count; i += 64) top = fmaxf(top, ml[i].x);
    for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
    const float base = top == -__builtin_inff() ? 0.0f : top;
    for (int i = lane; i < count; i += 64) sum += __builtin_amdgcn_exp2f(ml[i].x - base) * ml[i].y;
    for (int x = 32; x; x >>= 1) sum += __shfl_xor(sum, x);
    if (bad) sum = __builtin_nanf("");
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    for (int f = lane; f < p.dim; f += 64) {
        const float* o = p.part_o + row * parts * p.dim + f;
        float acc = 0.0f;
        for (int i = 0; i < count; i++) acc = __builtin_fmaf(__builtin_amdgcn_exp2f(ml[i].x - base), o[(int64_t)i * p.dim], acc);
        store_elem<DT>(p.out, row * p.dim + f, acc * inverse);
    }
    if (lane == 0 && p.lse) p.lse[row] = sum == 0.0f ? -__builtin_inff() : top * 0.69314718055994530942f + __logf(sum);
}

// ---- host --------------------------------------------------------------------------------------------------------------

struct AttendPlan {
    int64_t chunk, chunks, prefix_chunk, prefix_chunks, units, prefix_units;
    bool parts;  // rows are joined from parts
    size_t ml_bytes, bytes;
};
static int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }
// Chunks of `places` for `tiles` of rows: workgroups for every compute unit, no more than 64 pages each
static int64_t chunk_of(int64_t places, int64_t tiles, int64_t page) {
    const int64_t want = std::max<int64_t>(1, 1024 / std::max<int64_t>(1, tiles));
    int64_t c = round_up(ceil_div(std::max<int64_t>(places, 1), want), 128);
    return std::max<int64_t>(128, std::min<int64_t>({c, 2048, 64 * page / 128 * 128}));
}
static AttendPlan attend_plan(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim, int64_t page, int64_t longest, bool starts, int64_t sequences, int64_t prefix) {
    AttendPlan a;
    const int64_t group = heads / kv_heads, R = 16;
    a.units = starts ? tokens * group / R + sequences : sequences * ceil_div(group, R);
    a.prefix_units = prefix ? ceil_div(tokens * group, R) : 0;
    a.chunk = chunk_of(longest, a.units * kv_heads, page);
    a.chunks = std::max<int64_t>(1, ceil_div(longest, a.chunk));
    a.prefix_chunk = prefix ? chunk_of(prefix, a.prefix_units * kv_heads, page) : 128;
    a.prefix_chunks = prefix ? ceil_div(prefix, a.prefix_chunk) : 0;
    a.parts = a.chunks + a.prefix_chunks > 1;
    const int64_t parts = a.chunks + a.prefix_chunks;
    a.ml_bytes = a.parts ? (size_t)round_up(tokens * heads * parts * 8, 256) : 0;
    a.bytes = a.parts ? a.ml_bytes + (size_t)(tokens * heads * parts * dim * 4) : 0;
    return a;
}

template <int DT>
static void launch_attend(const AttendParams& p, int64_t blocks, hipStream_t st) {
    const dim3 grid((unsigned)blocks), block(256);
    switch (ceil_div(p.dim, 32)) {
        case 1: hipLaunchKernelGGL((attend_rows_kernel<DT, 1>), grid, block, 0, st, p); break;
        case 2: hipLaunchKernelGGL((attend_rows_kernel<DT, 2>), grid, block, 0, st, p); break;
        case 3: hipLaunchKernelGGL((attend_rows_kernel<DT, 3>), grid, block, 0, st, p); break;
        case 4: hipLaunchKernelGGL((attend_rows_kernel<DT, 4>), grid, block, 0, st, p); break;
        case 5: case 6: hipLaunchKernelGGL((attend_rows_kernel<DT, 6>), grid, block, 0, st, p); break;
        default: hipLaunchKernelGGL((attend_rows_kernel<DT, 8>), grid, block, 0, st, p); break;
    }
    if (p.part_o) hipLaunchKernelGGL((attend_join_kernel<DT>), dim3((unsigned)ceil_div(p.tokens * p.heads, 4)), block, 0, st, p);
}

static bool shape_ok(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim, int64_t page, int64_t width, int64_t longest, bool starts, int64_t sequences,
                     int64_t prefix) {
    return tokens > 0 && tokens <= 0x7fffffff && kv_heads > 0 && heads > 0 && heads <= 16384 && heads % kv_heads == 0 && dim > 0 && dim <= 256 && page >= 32 &&
           page <= 65536 && (page & (page - 1)) == 0 && width > 0 && width * page <= 0x7fffff00 && longest >= 0 && longest <= width * page && sequences > 0 &&
           sequences <= (1 << 24) && (starts || sequences == tokens) && prefix >= 0 && prefix <= 0x7fffff00;
}

}  // namespace bt

using namespace bt;

extern "C" size_t bt_cached_attention_workspace_bytes(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t page_size, int64_t table_width,
                                                      int64_t max_length, int has_starts, int64_t sequences, int64_t prefix_length) {
    if (!shape_ok(tokens, heads, kv_heads, head_dim, page_size, table_width, max_length, has_starts != 0, sequences, prefix_length)) return 0;
    return attend_plan(tokens, heads, kv_heads, head_dim, page_size, max_length, has_starts != 0, sequences, prefix_length).bytes;
}

extern "C" int bt_cached_attention(const void* q, int64_t q_token, int64_t q_head, int dtype, const void* k_cache, const void* v_cache, int64_t pages,
                                   int64_t page_size, const int32_t* block_table, int64_t table_width, int64_t max_length, const int32_t* lengths,
                                   const int32_t* q_starts, int64_t sequences, const int32_t* prefix_table, int64_t prefix_length, float scale, int64_t tokens,
                                   int64_t heads, int64_t kv_heads, int64_t head_dim, void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "bt_cached_attention";
    if (!q || !k_cache || !v_cache || !block_table || !lengths || !out || (prefix_length > 0 && !prefix_table) || dtype < BT_F32 || dtype > BT_BF16) {
        set_error("%s: null pointer or bad dtype", who);
        return BT_ERR_INVALID;
    }
    if (!shape_ok(tokens, heads, kv_heads, head_dim, page_size, table_width, max_length, q_starts != nullptr, sequences, prefix_length) || pages <= 0 ||
        pages > 0x7fffffff) {
        set_error("%s: head_dim at most 256, heads a multiple of kv_heads, page_size a power of two from 32 on, places of a sequence below 2^31, one token a "
                  "sequence without q_starts (head_dim=%lld heads=%lld/%lld page_size=%lld width=%lld sequences=%lld tokens=%lld)",
                  who, (long long)head_dim, (long long)heads, (long long)kv_heads, (long long)page_size, (long long)table_width, (long long)sequences,
                  (long long)tokens);
        return BT_ERR_INVALID;
    }
    if (!(scale > 0.0f) || scale > 3.0e38f) {
        set_error("%s: scale must be a positive number", who);
        return BT_ERR_INVALID;
    }
    if (((uintptr_t)k_cache) % 16 != 0 || ((uintptr_t)v_cache) % 16 != 0) {
        set_error("%s: the cache has to be 16-byte aligned", who);
        return BT_ERR_INVALID;
    }
    const AttendPlan a = attend_plan(tokens, heads, kv_heads, head_dim, page_size, max_length, q_starts != nullptr, sequences, prefix_length);
    if (a.bytes && (!workspace || workspace_bytes < a.bytes || ((uintptr_t)workspace) % 256 != 0)) {
        set_error("%s: workspace of %zu bytes (256-byte aligned) needed, %zu given", who, a.bytes, workspace_bytes);
        return BT_ERR_WORKSPACE;
    }
    AttendParams p = {};
    p.q = q, p.k_cache = k_cache, p.v_cache = v_cache, p.table = block_table, p.lengths = lengths, p.starts = q_starts, p.prefix_table = prefix_table;
    p.q_token = q_token, p.q_head = q_head, p.tokens = tokens, p.out = out, p.lse = lse;
    p.part_ml = a.parts ? (float2*)workspace : nullptr;
    p.part_o = a.parts ? (float*)((char*)workspace + a.ml_bytes) : nullptr;
    p.heads = (int)heads, p.kv_heads = (int)kv_heads, p.group = (int)(heads / kv_heads), p.dim = (int)head_dim, p.dp = cache_head_dim(dtype, head_dim);
    p.n_seq = (int)sequences, p.width = (int)table_width, p.page_shift = __builtin_ctzll((unsigned long long)page_size), p.pages = (int)pages;
    p.prefix = (int)prefix_length;
    p.chunk = (int)a.chunk, p.prefix_chunk = (int)a.prefix_chunk, p.chunks = (int)a.chunks, p.prefix_chunks = (int)a.prefix_chunks;
    p.units = (int)a.units, p.prefix_units = (int)a.prefix_units, p.seq_tiles = (int)ceil_div(p.group, 16), p.longest = (int)max_length;
    const int e = 16 / dtype_size(dtype);
    p.wide_q = head_dim % e == 0 && q_token % e == 0 && q_head % e == 0 && ((uintptr_t)q) % 16 == 0;
    p.scale2 = (float)((double)scale * 1.4426950408889634074);
    const int64_t blocks = (a.units * a.chunks + a.prefix_units * a.prefix_chunks) * kv_heads + (q_starts && !a.parts ? 1 : 0);
    if (blocks >= (1 << 24) || a.units > 0x7fffffff || a.prefix_units > 0x7fffffff) {
        set_error("%s: %lld workgroups are beyond one launch", who, (long long)blocks);
        return BT_ERR_INVALID;
    }
    hipStream_t st = (hipStream_t)stream;
    if (dtype == BT_F32) launch_attend<BT_F32>(p, blocks, st);
    else if (dtype == BT_F16) launch_attend<BT_F16>(p, blocks, st);
    else launch_attend<BT_BF16>(p, blocks, st);
    return check_launch(who);
}
