// Attention of new tokens over the paged cache (bt_cached_attention): o = softmax(scale q K^T) V over a prefix that all sequences share and
// over the sequence's own pages, causal among the new tokens.
//
// The G query heads of a key head and the new tokens of a sequence are the rows of one product: row i G + h of the sequence.  Its keys are
// cut into chunks, a workgroup each, which keep the softmax running over 16-byte groups of keys: maximum m, sum l and o in registers, all in
// 32 bits.  Workgroups that do not see all keys of their rows leave (m, l, o) in the workspace, and attend_join_kernel joins them in the
// order of the keys.  The rows of every sequence together are the rows of the prefix, whose keys are thus read once for all.
//
// At few rows the launch is bound by the cache's bytes, at many by the matrix cores and the exponentials.
#include "lds_dma.h"
#include "paged_cache.h"

#include <utility>

namespace bt {

// What workgroups leave for attend_join_kernel: [row][chunk], rows by (sequence, key head, row of it) of attend_rows_kernel's sequences and by
// (token, head) otherwise.
struct Parts {
    float* o;    // part_stride(dim) floats each
    float2* ml;
};
struct AttendParams {
    const void *q, *k_cache, *v_cache;
    const int32_t *table, *lengths, *starts, *prefix_table;
    int64_t q_token, q_head;
    void* out;
    float* lse;          // may be null
    int tokens, heads, kv_heads, group, dim, q_dim, dp, n_seq, width, page_shift, pages, prefix;  // q_dim: features that q's rows have in memory
    int longest;
    int few_rows;        // sequences of up to so many rows are attend_rows_kernel's, others attend_tiles_kernel's
    // of the two kernels: places of a chunk of a sequence, chunks of the longest, and row tiles of each sequence of few rows
    int chunk, chunks, tiles, units, wide_chunk, wide_chunks;
    int all_few;         // every sequence is attend_rows_kernel's, their tiles in units as attend_tiles_kernel's are
    int prefix_chunk, prefix_chunks, prefix_tiles, prefix_wide;  // the prefix, whose rows are tiled by one of them
    Parts few_parts, wide_parts, prefix_parts;       // without: the workgroup sees all keys of its rows
    int few_slots;       // rows of a sequence and key head in few_parts
    int join_few;        // attend_join_kernel goes over few_parts' rows alone
    float scale2;                                    // scale / ln 2
};

__host__ __device__ __forceinline__ int part_stride(int dim) { return (dim + 3) / 4 * 4; }

typedef float v16f __attribute__((ext_vector_type(16)));
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
// Two lanes' groups of 8: 32 rows, 32 columns
template <int DT>
__device__ __forceinline__ v16f step(u32x4 a, u32x4 b, v16f c) {
    if constexpr (DT == BT_F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
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
// fp16 weights are kept times 2^LIFT until they are summed up: as they are, those below 2^-14 of a row's largest would lose bits to fp16's
// exponent and those below 2^-25 everything, and 65536 of them have a share of 2 / 1000.  SLACK: a weight is 2^SLACK at most before.
template <int DT, int SLACK>
struct Lift {
    static constexpr int LIFT = DT == BT_F16 ? 15 - SLACK : 0;
    static constexpr float DOWN = 1.0f / (1 << LIFT);
};
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
// Values that are infinite or not a number, where some rows' weights are zero because they do not see them (zero times such a value is not
// zero): `v` without them, and ones in their places.  A row that sees one is not a number; the others' sums are what they are without them.
template <int DT>
__device__ __forceinline__ bool take_specials(u32x4& v, u32x4& where) {
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (DT == BT_F32) {
            const bool s = (v[i] & 0x7f800000u) == 0x7f800000u;
            where[i] = s ? 0x3f800000u : 0u;
            v[i] = s ? 0u : v[i];
            any |= s;
        } else {
            constexpr uint32_t e = DT == BT_F16 ? 0x7c00u : 0x7f80u, one = DT == BT_F16 ? 0x3c00u : 0x3f80u;
            const bool lo = (v[i] & e) == e, hi = (v[i] >> 16 & e) == e;
            where[i] = (lo ? one : 0u) | (hi ? one << 16 : 0u);
            v[i] = (lo ? 0u : v[i] & 0xffffu) | (hi ? 0u : v[i] & 0xffff0000u);
            any |= lo || hi;
        }
    }
    return any;
}
__device__ __forceinline__ float over_groups_max(float x) {  // over the four lanes of a row
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float over_groups_sum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

template <int ROWS, typename F>
__device__ __forceinline__ float over_rows_lanes(float x, F join) {  // over the lanes of a row, of which there are 64 / ROWS
    if (ROWS == 16) x = join(x, __shfl_xor(x, 16));
    return join(x, __shfl_xor(x, 32));
}

// What a workgroup works on: up to R rows of one key head and a chunk of their keys.
struct Job {
    const int32_t* table;
    int rows, row0;       // row r of the tile is token token0 + (row0 + r) / G, head kv * G + (row0 + r) % G
    int token0, kv;
    int limit0;           // row r sees the places below limit0 + (row0 + r) / G (own) or limit0 (prefix)
    bool causal, bad;     // bad: the length is beyond the table
    int begin, end;       // the chunk's places
    int part, slots;      // slots: parts of a row
    int64_t few_slot;     // >= 0: of row 0 in few_parts
    Parts parts;
};
__device__ __forceinline__ int group_row(const AttendParams& p, const Job& j, int r) { return (int)((uint32_t)(j.row0 + r) / (uint32_t)p.group); }
__device__ __forceinline__ int limit_of(const AttendParams& p, const Job& j, int r) { return j.limit0 + (j.causal ? group_row(p, j, r) : 0); }

// A sequence's tokens [t0, t0 + n) and its length, as far as the table goes; whether it goes beyond
__device__ __forceinline__ bool sequence_of(const AttendParams& p, int s, int* t0, int* n, int* length) {
    const int64_t first = p.starts ? std::max(p.starts[s], 0) : s;
    *n = p.starts ? (int)std::max<int64_t>(0, std::min<int64_t>(p.starts[s + 1], p.tokens) - first) : 1;  // (0 <= t0, t0 + n <= tokens where n > 0)
    *t0 = (int)first;
    const int got = p.lengths[s];
    *length = std::max(0, std::min(got, p.longest));
    return got > p.longest;
}

// Block `block` of the prefix: row tile, key head, chunk.
__device__ __forceinline__ bool prefix_job(const AttendParams& p, int R, uint32_t block, Job* j) {
    const uint32_t at = block / (uint32_t)p.prefix_chunks, c = block - at * p.prefix_chunks, tile = at / (uint32_t)p.kv_heads;
    j->kv = (int)(at - tile * p.kv_heads);
    j->row0 = (int)tile * R;
    j->token0 = 0;
    j->rows = std::min(R, p.tokens * p.group - j->row0);
    j->table = p.prefix_table;
    j->limit0 = p.prefix;
    j->causal = j->bad = false;
    j->begin = (int)c * p.prefix_chunk;
    j->end = std::min(j->begin + p.prefix_chunk, p.prefix);
    j->part = (int)c;
    j->slots = p.prefix_chunks;
    j->few_slot = -1;
    j->parts = p.prefix_parts;
    return j->rows > 0;
}
// The tile of rows [tile * R, ...) of sequence s and chunk c of its places.  False: nothing to do.
__device__ __forceinline__ bool own_job(const AttendParams& p, int R, int s, int tile, int c, int chunk, bool wide, Job* j) {
    int n, length;
    j->bad = sequence_of(p, s, &j->token0, &n, &length);
    j->row0 = tile * R;
    const int rows = n * p.group;
    if (n <= 0 || j->row0 >= rows || (rows > p.few_rows) != wide) return false;
    j->rows = std::min(R, rows - j->row0);
    j->table = p.table + (int64_t)s * p.width;
    j->limit0 = length - n + 1;
    j->causal = true;
    j->begin = c * chunk;
    j->end = std::min(j->begin + chunk, limit_of(p, *j, j->rows - 1));
    j->part = c;
    j->slots = wide ? p.wide_chunks : p.chunks;
    j->few_slot = wide || p.all_few ? -1 : ((int64_t)s * p.kv_heads + j->kv) * p.few_slots + j->row0;
    j->parts = wide ? p.wide_parts : p.few_parts;
    return j->begin < j->end || (!j->parts.o && c == 0);
}
// Sequence and tile of R rows of unit `unit`: sequence s has the units floor(starts[s] G / R) + s and on (n tokens have n G / R + 1 tiles at most).
__device__ __forceinline__ bool tile_of(const AttendParams& p, uint32_t R, uint32_t unit, int* s, int* tile) {
    const int lane = threadIdx.x & 63;
    auto first_of = [&](int i) { return (uint32_t)((uint64_t)(uint32_t)std::max(p.starts[i], 0) * (uint32_t)p.group / R) + (uint32_t)i; };
    int found = 0;
    for (int s0 = 0; s0 < p.n_seq; s0 += 64) {
        const int i = s0 + lane;
        const uint64_t hit = __ballot(i < p.n_seq && first_of(i < p.n_seq ? i : 0) <= unit);
        found += __popcll(hit);
        if (hit != ~0ull) break;
    }
    *s = found - 1;
    if (*s < 0) return false;
    const uint32_t first = first_of(*s);
    *tile = (int)(unit - first);
    return first <= unit;  // (starts that do not ascend)
}
// The chunk's pages, one a lane, 64 at a time.  The first ones are asked for before the length is known.
struct PageWindow {
    int first, last, page;  // numbers of the window's first page and of the chunk's last
    bool bad;
    static __device__ __forceinline__ int ask(const int32_t* table, int width, int from) {
        const int at = from + (int)(threadIdx.x & 63);
        return at < width ? table[at] : 0;
    }
    __device__ __forceinline__ PageWindow(const AttendParams& p, const Job& j, int asked) : bad(j.bad) {
        last = j.end > j.begin ? (j.end - 1) >> p.page_shift : -1;
        take(p, j.begin >> p.page_shift, asked);
    }
    __device__ __forceinline__ void take(const AttendParams& p, int from, int asked) {
        const int at = from + (int)(threadIdx.x & 63);
        first = from;
        const bool wrong = (uint32_t)asked >= (uint32_t)p.pages;
        bad |= __ballot(wrong && at <= last) != 0;
        page = wrong ? 0 : asked;
    }
    __device__ __forceinline__ int64_t of(const AttendParams& p, const Job& j, int place) {  // place: not below those asked for before
        const int number = place >> p.page_shift;
        if (number >= first + 64) {
            const int from = first + (number - first) / 64 * 64;
            take(p, from, ask(j.table, last + 1, from));
        }
        return __builtin_amdgcn_readlane(page, number - first);
    }
};
// The rows behind the last sequence, where no job sees to them: the share of workgroup `block` of `blocks`
template <int DT>
__device__ __forceinline__ void clear_rows_behind(const AttendParams& p, uint32_t block, uint32_t blocks) {
    const int64_t n = (int64_t)p.heads * p.dim, behind = std::max(0, std::min(p.starts[p.n_seq], p.tokens)), at = (int64_t)block * blockDim.x + threadIdx.x,
                  step = (int64_t)blocks * blockDim.x;
    for (int64_t i = behind * n + at; i < p.tokens * n; i += step) store_elem<DT>(p.out, i, 0.0f);
    for (int64_t i = behind * p.heads + at; p.lse && i < (int64_t)p.tokens * p.heads; i += step) p.lse[i] = -__builtin_inff();
}
// Of the row with group_row `in_group`: where its q starts, and E features of it from f on (zero behind the head)
__device__ __forceinline__ int64_t q_row(const AttendParams& p, const Job& j, int r, int in_group) {
    return (int64_t)(j.token0 + in_group) * p.q_token + (int64_t)(j.kv * p.group + j.row0 + r - in_group * p.group) * p.q_head;
}
template <int DT>
__device__ __forceinline__ u32x4 q_piece(const AttendParams& p, int64_t row_at, int f, bool there) {
    return there && f < p.q_dim ? *(const u32x4*)((const char*)p.q + (row_at + f) * CacheOrder<DT>::SIZE) : u32x4{0, 0, 0, 0};
}
// q in rows of dp features, zero behind the head, where its own do not start or end on 16 bytes
template <int DT>
__global__ __launch_bounds__(256) void attend_copy_kernel(AttendParams p, void* to) {
    const int64_t n = (int64_t)p.tokens * p.heads * p.dp;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / p.dp, token = row / p.heads;
        const int f = (int)(i - row * p.dp);
        if constexpr (DT == BT_F32) ((uint32_t*)to)[i] = f < p.dim ? ((const uint32_t*)p.q)[token * p.q_token + (row - token * p.heads) * p.q_head + f] : 0u;
        else ((uint16_t*)to)[i] = f < p.dim ? ((const uint16_t*)p.q)[token * p.q_token + (row - token * p.heads) * p.q_head + f] : (uint16_t)0;
    }
}
// Four features of a row, as they are returned
template <int DT>
__device__ __forceinline__ void put_features(const AttendParams& p, int64_t out_row, int f, v4f acc) {
    if (p.dim % 4 == 0) {
        if constexpr (DT == BT_F32) *(v4f*)((float*)p.out + out_row * p.dim + f) = acc;
        else {
            u32x2 w;
#pragma unroll
            for (int i = 0; i < 2; i++)
                w[i] = DT == BT_F16 ? f32_to_f16_bits(acc[2 * i]) | (uint32_t)f32_to_f16_bits(acc[2 * i + 1]) << 16
                                    : f32_to_bf16_bits(acc[2 * i]) | (uint32_t)f32_to_bf16_bits(acc[2 * i + 1]) << 16;
            *(u32x2*)((uint16_t*)p.out + out_row * p.dim + f) = w;
        }
        return;
    }
#pragma unroll 1
    for (int i = 0; i < 4; i++)
        if (f + i < p.dim) store_elem<DT>(p.out, out_row * p.dim + f + i, i == 0 ? acc[0] : i == 1 ? acc[1] : i == 2 ? acc[2] : acc[3]);
}
__device__ __forceinline__ float lse_of(float top, float sum) { return sum == 0.0f ? -__builtin_inff() : top * 0.69314718055994530942f + __logf(sum); }
// Four features of row r of the job, finished or for attend_join_kernel; top: the row's maximum, in powers of two
template <int DT>
__device__ __forceinline__ void put_row(const AttendParams& p, const Job& j, int r, int f, v4f acc, float top, float sum) {
    const int in_group = group_row(p, j, r);
    const int64_t out_row = (int64_t)(j.token0 + in_group) * p.heads + j.kv * p.group + j.row0 + r - in_group * p.group;
    if (j.parts.o) {
        const int64_t at = (j.few_slot >= 0 ? j.few_slot + r : out_row) * j.slots + j.part;
        if (f == 0) j.parts.ml[at] = make_float2(top, sum);
        *(v4f*)(j.parts.o + at * part_stride(p.dim) + f) = acc;  // (what lies behind the head is not read)
        return;
    }
    put_features<DT>(p, out_row, f, acc * (sum == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(sum)));
    if (f == 0 && p.lse) p.lse[out_row] = lse_of(top, sum);
}

// B: blocks of 32 features, the last one maybe in part (the first FULL groups of TK features are whole).  Four waves take the chunk's tiles of TK places in turn, each with all rows.
//
// Bound by the cache's bytes: keys and values go straight to registers, past the caches (no other workgroup wants them), the next tile's while this
// one is worked on, three workgroups to a compute unit (64 sequences of 1046 to 4022 places, 32 heads on 8, 118 us, 5.7 TB/s; without the two 133; one
// of 100000 places 64 us, 6.4 TB/s).  At little work it is the chain of loads, products and joins: 500 places of one sequence 8.2 us, 120 places 5.5
// (eight waves: 7.6, 5.6).  fp32 heads of 97 to 128 features keep 7 of their registers in scratch memory.
template <int DT, int B>
__global__ __launch_bounds__(256, B <= 4 ? 3 : 1) void attend_rows_kernel(AttendParams p) {
    using Order = CacheOrder<DT>;
    constexpr int E = Order::E, TK = Order::TK, C = 32 * B / TK, V = 2 * B, FULL = 32 * (B - 1) / TK, R = 16;
    constexpr int JB = B < 4 ? B : 4, LD = 32 * JB + 4;  // blocks that are joined at a time (LDS)
    __shared__ __attribute__((aligned(16))) float o_all[4][R * LD];
    __shared__ float m_all[4][R], l_all[4][R];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    Job j;
    int asked;
    {
        uint32_t block = blockIdx.x;
        const uint32_t prefix_blocks = p.prefix_wide ? 0 : p.prefix_tiles * p.kv_heads * p.prefix_chunks;
        if (block < prefix_blocks) {
            if (!prefix_job(p, R, block, &j)) return;
            asked = PageWindow::ask(j.table, ((j.end - 1) >> p.page_shift) + 1, j.begin >> p.page_shift);
        } else {
            block -= prefix_blocks;
            const uint32_t at = block / (uint32_t)p.chunks, unit = at / (uint32_t)p.kv_heads;
            const int c = (int)(block - at * p.chunks);
            j.kv = (int)(at - unit * p.kv_heads);
            if ((int)unit >= p.units) {
                const uint32_t jobs = prefix_blocks + (uint32_t)p.units * p.kv_heads * p.chunks;
                return clear_rows_behind<DT>(p, blockIdx.x - jobs, gridDim.x - jobs);
            }
            int s = (int)(unit / (uint32_t)p.tiles), tile = (int)unit - s * p.tiles;
            if (p.all_few && !tile_of(p, R, unit, &s, &tile)) return;
            asked = PageWindow::ask(p.table + (int64_t)s * p.width, p.width, (c * p.chunk) >> p.page_shift);
            if (!own_job(p, R, s, tile, c, p.chunk, false, &j)) return;
        }
    }
    const int kv = j.kv;

    PageWindow pages(p, j, asked);
    const int tiles = j.end > j.begin ? (j.end - j.begin + TK - 1) / TK : 0;

    // this lane's row as an operand
    const bool there = r < j.rows;
    const int in_group = group_row(p, j, r), limit = there ? j.limit0 + (j.causal ? in_group : 0) : 0, lowest = limit_of(p, j, 0);
    const int64_t q_at = q_row(p, j, r, in_group);
    u32x4 q[C];
#pragma unroll
    for (int c = 0; c < C; c++) q[c] = q_piece<DT>(p, q_at, c * TK + g * E, there);

    float m = -__builtin_inff(), l = 0.0f;  // of the row; l: of this lane's places
    v4f o[V];
    std::conditional_t<(V > 8), uint64_t, uint32_t> nan = 0;  // features 16 b + 4 g + e, bit 4 b + e, that saw a value that is no number
#pragma unroll
    for (int b = 0; b < V; b++) o[b] = v4f{0, 0, 0, 0};
    const int64_t page_elements = (int64_t)p.dp << p.page_shift;
    auto start_of = [&](int tile) {  // in bytes, this lane's first piece
        const int place = j.begin + tile * TK;
        return (((pages.of(p, j, place) * p.kv_heads + kv) * page_elements + (int64_t)(place & ((1 << p.page_shift) - 1)) * p.dp) + lane * E) * Order::SIZE;
    };
    u32x4 k[C][E / 4], v[V];
    auto load_keys = [&](int64_t at) {
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int t = 0; t < E / 4; t++) {
                if (c >= FULL) k[c][t] = u32x4{0, 0, 0, 0};
                if (c < FULL || c * TK + g * E < p.dim) k[c][t] = __builtin_nontemporal_load((const u32x4*)((const char*)p.k_cache + at + (c * (E / 4) + t) * 1024));
            }
    };
    auto value_piece = [&](int64_t at, int b) { return __builtin_nontemporal_load((const u32x4*)((const char*)p.v_cache + at + b * 1024)); };
    auto load_values = [&](int64_t at) {
#pragma unroll
        for (int b = 0; b < V; b++) {
            if (b == V - 1) v[b] = u32x4{0, 0, 0, 0};
            if (b < V - 1 || b * 16 < p.dim) v[b] = value_piece(at, b);
        }
    };
    int64_t at = 0;
    if (wave < tiles) {
        at = start_of(wave);
        load_keys(at);
        load_values(at);
    }
    for (int tile = wave; tile < tiles; tile += 4) {
        const int place = j.begin + tile * TK;
        const bool more = tile + 4 < tiles;
        float x[E];
#pragma unroll
        for (int t = 0; t < E / 4; t++) {
            v4f s = {0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < C; c++) s = step<DT>(k[c][t], q[c], s);
#pragma unroll
            for (int i = 0; i < 4; i++) x[4 * t + i] = s[i] * p.scale2;
        }
        int64_t next = at;
        if (more) {  // (the keys' registers are free)
            next = start_of(tile + 4);
            load_keys(next);
        }
        const bool masked = place + TK > lowest;  // some row does not see all of the tile
        bool special = false;
        if (masked) {
#pragma unroll
            for (int e = 0; e < E; e++) x[e] = place + g * E + e < limit ? x[e] : -__builtin_inff();
#pragma unroll
            for (int b = 0; b < V; b++) special |= any_special<DT>(v[b]);
            special = __any(special);
        }
        float top = x[0];
#pragma unroll
        for (int e = 1; e < E; e++) top = fmaxf(top, x[e]);
        if (__any(top > m)) {
            const float next_m = fmaxf(m, over_groups_max(top));
            const float shrink = __builtin_amdgcn_exp2f(m == next_m ? 0.0f : m - next_m);
            m = next_m;
            l *= shrink;
#pragma unroll
            for (int b = 0; b < V; b++) o[b] *= shrink;
        }
        const float base = m == -__builtin_inff() ? 0.0f : m;
        float w[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
            float exponent = x[e] - base;  // (the difference first: it is exact where logits are large)
            if constexpr (Lift<DT, 0>::LIFT != 0) exponent += (float)Lift<DT, 0>::LIFT;
            w[e] = __builtin_amdgcn_exp2f(exponent);
            l += w[e];
        }
        u32x4 lo;
        const u32x4 hi = operand<DT>(w, &lo);
        if (special) {  // (seldom: what is no number, behind the end or where some row does not look, would make all rows such)
            const int live = j.end - (place + g * E);  // no row sees what lies behind
#pragma unroll 1
            for (int b = 0; b < V && b * 16 < p.dim; b++) {
                u32x4 piece = first_places<DT>(value_piece(at, b), live), where;
                take_specials<DT>(piece, where);
                const v4f seen = step<DT>(where, hi, v4f{0, 0, 0, 0});
#pragma unroll
                for (int e = 0; e < 4; e++) nan |= (decltype(nan + 0))(seen[e] > 0.0f) << (4 * b + e);
            }
#pragma unroll
            for (int b = 0; b < V; b++) {
                u32x4 where;
                v[b] = first_places<DT>(v[b], live);
                take_specials<DT>(v[b], where);
            }
        }
#pragma unroll
        for (int b = 0; b < V; b++) {
            o[b] = step<DT>(v[b], hi, o[b]);
            if constexpr (DT != BT_F32) o[b] = step<DT>(v[b], lo, o[b]);
        }
        if (more) load_values(next);
        at = next;
    }
    if (__any(nan != 0)) {
#pragma unroll
        for (int b = 0; b < V; b++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[b][e] = nan >> (4 * b + e) & 1 ? __builtin_nanf("") : o[b][e];
    }
    l = over_groups_sum(l);
    if (pages.bad) l = __builtin_nanf("");  // (a wave knows of the pages that it had a tile on: the sum over the waves tells all)

    // the four waves' shares of every row
    if (g == 0) m_all[wave][r] = m, l_all[wave][r] = l;
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
                const float share = __builtin_amdgcn_exp2f(m_all[w][row_at] - base) * Lift<DT, 0>::DOWN;
                sum += share * l_all[w][row_at];
                const v4f ow = *(const v4f*)&o_all[w][row_at * LD + at];
                acc += ow * share;
            }
            put_row<DT>(p, j, row_at, f, acc, top, sum);
        }
    }
}

// RT row tiles of 16 a wave and four waves: 128 rows (64 of more than 128 features, whose sums take twice the registers), whose keys and
// values pass through LDS once for all of them, a tile of TK places at a time.  Tiles are read from memory straight into LDS, in the order in
// which they lie there, up to NR tiles ahead.
//
// What bounds it.  One block of instructions works on three tiles, the products of tile i + 1, the weights of tile i and the sums over the values of
// tile i - 1, none of which waits for another (one thing after the other took 1.6 times as long).  A tile costs a wave (128 features, 16 bits) 16 matrix
// instructions of 32 cycles, and about 95 others: 16 exponentials, three or four instructions around each, the rows' maxima.  The matrix unit is busy for 48%
// of a long call's cycles and the vector unit for 47%, at the 1.9 GHz that such a load leaves; 2 x 1024 tokens of 32 heads see 4096 places
// more in 126 us, 1.09 PFLOP/s where a large matrix product of a library reaches 1.22.  Matrix instructions of 16 rows take as many cycles and leave the
// vector instructions less of them (4 x 512 tokens on 2048 places 79 -> 76 us).  LDS is not the bound (its fragments take a fifth of the cycles, and without
// their reads a tile takes as long); one wait and barrier for two tiles was slower (280 us where this takes 263: half as far ahead), and more
// fragments ahead make no difference.  64 rows a wave and one wave a SIMD took twice as long: the sums live in accumulation registers then.
//
// The maximum is that of the products before they are scaled, and one multiply-add and the exponential make a weight.  It is raised only where a
// weight would pass 2^8: it needs to be near the true maximum, not to be it.  16-bit weights are rounded once (the rows kernel's two halves
// would be half as many matrix instructions again): results are 1.4 times as far from 64 bits as by their own rounding, and fp16 ones by up to
// 2^-32 of the row's largest value a place besides (struct Lift; the rows kernel 2^-40).  Their sum is that of the weights before they are
// rounded, as lse wants it.
// The tile of the unit'th workgroup of a key head: sequences by their length, their last rows first, and of the first 2 x CUs workgroups, two of
// which share a compute unit and its LDS, the second ones from the light end (4 x 512 tokens on 1600 to 4000 places 138 -> 120 us).
__device__ __forceinline__ bool heaviest_first(const AttendParams& p, int R, uint32_t unit, int* s, int* tile) {
    const int lane = threadIdx.x & 63;
    int t0, n = 0, length = 0;
    if (lane < p.n_seq) sequence_of(p, lane, &t0, &n, &length);
    const int rows = n * p.group, mine = rows > p.few_rows ? (rows + R - 1) / R : 0;
    int before = 0, total = 0;  // tiles of heavier sequences, and of all
    for (int i = 0; i < p.n_seq; i++) {
        const int tiles = __builtin_amdgcn_readlane(mine, i), its = __builtin_amdgcn_readlane(length, i);
        if (its > length || (its == length && i < lane)) before += tiles;
        total += tiles;
    }
    if ((int)unit >= total) return false;
    const int first = std::max(1, 256 / p.kv_heads), at = (int)unit;
    const int rank = at < first || total <= first ? at : at < 2 * first && at < total ? total - 1 - (at - first) : at - first;
    const uint64_t hit = __ballot(before <= rank && rank < before + mine);
    if (!hit) return false;
    *s = __builtin_ctzll(hit);
    *tile = __builtin_amdgcn_readlane(mine, *s) - 1 - (rank - __builtin_amdgcn_readlane(before, *s));
    return true;
}
template <typename Body, int... I>
__device__ __forceinline__ void unrolled(std::integer_sequence<int, I...>, Body body) {  // body(0), body(1) ..., each with its number as a constant
    (body(std::integral_constant<int, I>()), ...);
}
// N KiB of consecutive memory to LDS, 16 bytes a lane
template <int N>
__device__ __forceinline__ void dma_run(uint32_t lds_off, uint32_t voff, const void* sbase) {
    static_assert(N >= 1 && N <= 4);
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds_off);
    if constexpr (N == 1) dma16(to, voff, sbase);
    if constexpr (N == 2)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\tglobal_load_lds_dwordx4 %1, %2 offset:1024" ::"s"(to), "v"(voff), "s"(sbase) : "memory");
    if constexpr (N == 3)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\tglobal_load_lds_dwordx4 %1, %2 offset:1024\n\t"
                     "global_load_lds_dwordx4 %1, %2 offset:2048" ::"s"(to), "v"(voff), "s"(sbase) : "memory");
    if constexpr (N == 4)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\tglobal_load_lds_dwordx4 %1, %2 offset:1024\n\t"
                     "global_load_lds_dwordx4 %1, %2 offset:2048\n\tglobal_load_lds_dwordx4 %1, %2 offset:3072" ::"s"(to), "v"(voff), "s"(sbase) : "memory");
}
template <int B>
struct WideTile {
    static constexpr int RT = B <= 4 ? 2 : 1, R = 64 * RT;
};
template <int DT, int B>
__global__ __launch_bounds__(256, 2) void attend_tiles_kernel(AttendParams p) {
    using Order = CacheOrder<DT>;
    constexpr int E = Order::E, TK = Order::TK, C = 32 * B / TK, H = E / 4, V = 2 * B, RT = WideTile<B>::RT, R = WideTile<B>::R;
    // 16-bit types with up to 128 features: 32 rows to a matrix instruction; others 16.  A lane has sums of T rows: EL products of each, in SA
    // accumulators of AE, that make W operands of weights, and OA accumulators of sums; KF and V fragments of keys and values make a tile.
    constexpr bool BIG = DT != BT_F32 && B <= 4;
    constexpr int ROWS = BIG ? 32 : 16, T = RT * 16 / ROWS, AE = BIG ? 16 : 4, SA = BIG ? 1 : H, EL = SA * AE, W = EL / E, OA = BIG ? B : V, QC = BIG ? V : C, KF = QC * SA;
    using Acc = std::conditional_t<BIG, v16f, v4f>;
    constexpr int TILE = 2048 * B;                                        // bytes of a tile's keys or values
    constexpr int NR = 32768 / TILE < 4 ? 32768 / TILE : 4;               // of each in LDS (loads into LDS reach 64 KiB)
    constexpr int LOADS = 2 * ((2 * B + 3) / 4);                          // of a wave for a tile
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * NR * TILE];
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane % ROWS, g = lane / ROWS;
    Job j;
    {
        uint32_t block = blockIdx.x;
        const uint32_t prefix_blocks = p.prefix_wide ? p.prefix_tiles * p.kv_heads * p.prefix_chunks : 0;
        if (block < prefix_blocks) {
            if (!prefix_job(p, R, block, &j)) return;
        } else {
            block -= prefix_blocks;
            const uint32_t at = block / (uint32_t)p.wide_chunks, unit = at / (uint32_t)p.kv_heads;
            j.kv = (int)(at - unit * p.kv_heads);
            int s, tile;
            if (p.starts && p.n_seq <= 64) {
                if (!heaviest_first(p, R, unit, &s, &tile)) return;
            } else if (p.starts) {
                if (!tile_of(p, R, unit, &s, &tile)) return;
            } else {
                const uint32_t each = (uint32_t)(p.group + R - 1) / R;
                s = (int)(unit / each);
                tile = (int)(unit - s * each);
            }
            if (!own_job(p, R, s, tile, (int)(block - at * p.wide_chunks), p.wide_chunk, true, &j)) return;
        }
    }
    const int tiles = j.end > j.begin ? (j.end - j.begin + TK - 1) / TK : 0;
    const int mine = wave * RT * 16;  // this wave's first row
    u32x4 q[T][QC];
    int limit[T];
#pragma unroll
    for (int t = 0; t < T; t++) {
        const int at = mine + t * ROWS + r, in_group = group_row(p, j, at);
        const int64_t q_at = q_row(p, j, at, in_group);
        limit[t] = at < j.rows ? j.limit0 + (j.causal ? in_group : 0) : 0;
#pragma unroll
        for (int c = 0; c < QC; c++) q[t][c] = q_piece<DT>(p, q_at, (c * (64 / ROWS) + g) * E, at < j.rows);
    }
    // the places that some row of the wave sees, and those that all see; the wave's tiles
    const int reach = mine < j.rows ? std::min(limit_of(p, j, std::min(mine + 16 * RT, j.rows) - 1), j.end) : 0;
    const int lowest = mine < j.rows ? std::min(limit_of(p, j, mine), j.end) : 0;
    const int my_tiles = reach > j.begin ? (reach - j.begin + TK - 1) / TK : 0;

    // Fragments: where a lane's piece of them is in the tile, and the places of the tile that a lane's products and pieces of values have.  The rows
    // of a fragment of keys are such places that a lane's products are the weights it brings to the values.
    const int key_lane = BIG ? (r >> 3 & 1) * 1024 + g * 256 + ((r >> 4) * 2 + (r >> 2 & 1)) * 64 + (r & 3) * 16 : lane * 16;
    const int value_lane = BIG ? (r >> 4) * 1024 + g * 256 + (r & 15) * 16 : lane * 16;
    auto key_piece = [](int f) { return BIG ? f / 2 * 2048 + f % 2 * 512 : (f % QC * SA + f / QC) * 1024; };
    auto value_piece = [](int f) { return BIG ? f % OA * 2048 + f / OA * 512 : f * 1024; };
    auto place_of = [](int g, int e) { return e / E * (E * (64 / ROWS)) + g * E + e % E; };

    // A tile's KiB are split over the waves, as many to each (some twice where they are not a multiple of four: the loads are counted)
    const int piece = std::min(LOADS / 2 * wave, p.dp * TK * Order::SIZE / 1024 - LOADS / 2);
    auto load = [&](uint32_t to, const char* from) { dma_run<LOADS / 2>(to + piece * 1024, piece * 1024 + lane * 16, from); };
    // The chunk's pages, 64 at a time, one a lane (a scalar load for each would be waited for together with the first fragments), and the tile whose keys
    // are loaded next: behind the last one that one again, for the count of loads.
    const int64_t head_bytes = ((int64_t)p.dp << p.page_shift) * Order::SIZE;
    const int page_bytes = (int)std::min<int64_t>(head_bytes, 0x7fffffff), tile_bytes = TK * p.dp * Order::SIZE;  // (at most 2^26)
    int numbers = 0, first_number = 0, number = j.begin >> p.page_shift, offset = (j.begin & ((1 << p.page_shift) - 1)) * p.dp * Order::SIZE, left = tiles;
    int64_t page_at = 0, at1 = 0, at2 = 0, at3 = 0;  // at: where the last three tiles of keys came from; their values follow
    bool bad = j.bad;
    auto find_page = [&]() {
        if (number >= first_number + 64 || left == tiles) {
            first_number = number;
            numbers = j.table[std::min(number + lane, (j.end - 1) >> p.page_shift)];
            asm volatile("" : "+v"(numbers));  // (waited for here, not at every tile)
        }
        int page = __builtin_amdgcn_readlane(numbers, number - first_number);
        if ((uint32_t)page >= (uint32_t)p.pages) page = 0, bad = true;
        page_at = ((int64_t)page * p.kv_heads + j.kv) * head_bytes;
    };
    auto load_keys = [&](int tile) {
        at3 = at2, at2 = at1, at1 = page_at + offset;
        load(lds0 + (uint32_t)(tile % NR) * TILE, (const char*)p.k_cache + at1);
        left--;
        offset += left > 0 ? tile_bytes : 0;
    };
    auto next_page = [&]() {
        if (offset == page_bytes) offset = 0, number++, find_page();
    };
    // (at: where the tile's keys came from)
    auto load_values = [&](int tile, int64_t at) { load(lds0 + (uint32_t)(NR + tile % NR) * TILE, (const char*)p.v_cache + at); };

    Acc o[T][OA], s[T][SA];     // s: products of the tile whose weights come next
    float m[T], l[T], top[T];   // the rows' maxima (of the products before they are scaled), sums and s's maxima (of this lane's places)
    u32x4 w[T][W];              // weights of the tile before
    std::conditional_t<(BIG || V > 8), uint64_t, uint32_t> nan[T];  // elements e of accumulator b of the sums, bit AE b + e, that saw a value that is no number
    constexpr int SLACK = 8;
    using Lifted = Lift<DT, SLACK>;
    const float slack = std::min((float)SLACK / p.scale2, 3.4e38f);  // (infinite, the maximum would never leave minus infinity)
    // The multiply-add rounds once, the base alone too: logits of a size at which that is more than a part of one are rounded alike first.
    bool large = false;
#pragma unroll
    for (int t = 0; t < T; t++) {
        m[t] = -__builtin_inff(), l[t] = 0.0f, top[t] = 0.0f, nan[t] = 0;
#pragma unroll
        for (int i = 0; i < W; i++) w[t][i] = u32x4{0, 0, 0, 0};
#pragma unroll
        for (int b = 0; b < OA; b++) o[t][b] = Acc{};
#pragma unroll
        for (int h = 0; h < SA; h++) s[t][h] = Acc{};
    }
    auto keys_at = [&](int tile) { return lds + tile % NR * TILE + key_lane; };
    auto values_at = [&](int tile) { return lds + (NR + tile % NR) * TILE + value_lane; };
    // fragment f of keys with the queries; of values with the weights
    auto multiply_keys = [&](auto number, u32x4 k, Acc (&s)[T][SA]) {
        constexpr int f = decltype(number)::value, h = f / QC, c = f % QC;
        if (DT == BT_F32 && c == QC - 1 && c * TK >= p.dp) k = u32x4{0, 0, 0, 0};  // (a tile has one group of features less)
#pragma unroll
        for (int t = 0; t < T; t++) s[t][h] = step<DT>(k, q[t][c], c ? s[t][h] : Acc{});
    };
    auto multiply_values = [&](auto number, u32x4 v) {
        constexpr int f = decltype(number)::value;
#pragma unroll
        for (int t = 0; t < T; t++) o[t][f % OA] = step<DT>(v, w[t][f / OA], o[t][f % OA]);
    };
    auto products = [&](const uint8_t* kf, Acc (&s)[T][SA]) {
        unrolled(std::make_integer_sequence<int, KF>(), [&](auto number) { multiply_keys(number, *(const u32x4*)(kf + key_piece(decltype(number)::value)), s); });
    };
    auto maxima = [&]() {
#pragma unroll
        for (int t = 0; t < T; t++) {
            top[t] = s[t][0][0];
#pragma unroll
            for (int e = 1; e < EL; e++) top[t] = fmaxf(top[t], s[t][e / AE][e % AE]);
        }
    };
    auto weights = [&](float scale, auto base_of) {
#pragma unroll
        for (int t = 0; t < T; t++) {
            const float base = base_of(t);
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < W; i++) {
                float x[E];
#pragma unroll
                for (int e = 0; e < E; e++) x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][(i * E + e) / AE][(i * E + e) % AE], scale, base));
                w[t][i] = operand<DT>(x, nullptr);
#pragma unroll
                for (int e = 0; e < E; e++) sum = i || e ? sum + x[e] : x[0];
            }
            l[t] += sum;
        }
    };
    // of the row's weights as exponents; all its logits may be minus infinity, of infinite keys
    auto base_of = [&](int t) {
        if constexpr (Lifted::LIFT) return __builtin_fmaf(m[t] == -__builtin_inff() ? 0.0f : -m[t], p.scale2, (float)Lifted::LIFT);
        else return m[t] == -__builtin_inff() ? 0.0f : -m[t] * p.scale2;
    };
    auto over = [&](float by) {
        bool any = false;
#pragma unroll
        for (int t = 0; t < T; t++) any |= top[t] > m[t] + by;
        return __any(any);
    };
    float shrink[T];
    bool raised = false;  // m and l are, the sums are not yet
    auto raise = [&]() {  // m and l; the sums over values follow once those of the tile before are in
#pragma unroll
        for (int t = 0; t < T; t++) {
            const float next = fmaxf(m[t], over_rows_lanes<ROWS>(top[t], [](float a, float b) { return fmaxf(a, b); }));
            shrink[t] = __builtin_amdgcn_exp2f(m[t] == next ? 0.0f : (m[t] - next) * p.scale2);
            m[t] = next;
            l[t] *= shrink[t];
            large |= __any(next != -__builtin_inff() && fabsf(next) * p.scale2 > 65536.0f);
        }
    };
    auto shrink_sums = [&]() {
#pragma unroll
        for (int t = 0; t < T; t++)
#pragma unroll
            for (int b = 0; b < OA; b++) o[t][b] *= shrink[t];
    };
    // Iteration i loads the keys of tile i + NR and the values of tile i - 2 + NR into the places that iteration i - 1 read last, and reads
    // what iteration i + 1 - NR loaded: what the last NR - 2 iterations loaded may still be on its way.
    auto turn = [&]() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NR - 2) * LOADS) : "memory"); };
    if (tiles) {
        find_page();
        load_keys(0);
#pragma unroll
        for (int i = 1 - NR; i < 0; i++) {
            next_page();
            load_keys(i + NR);
            load_values(std::max(i + NR - 2, 0), i + NR >= 2 ? at3 : at2);
        }
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NR - 1) * LOADS) : "memory");
        if (my_tiles) products(keys_at(0), s);
    }
    // tiles that all rows of the wave see as a whole
    const int whole = lowest > j.begin ? (lowest - j.begin) / TK : 0;
    for (int i = 0; i <= tiles && tiles;) {
        if (i > 0 && i < whole && !large) {
            maxima();
            for (; i < whole; i++) {
                raised = over(slack);
                if (raised) raise();
                if (large) break;  // (before this tile's weights)
                turn();
                // F fragments, each with its matrix instructions and a share of the other pipe's work; loads run AHEAD fragments in front
                constexpr int F = KF + V, N = T * EL, AHEAD = 3;
                const uint8_t *kf = keys_at(i + 1), *vf = values_at(i - 1);
                u32x4 frag[F], w2[T][W];
                Acc s2[T][SA];
                float x[T][W][E], sum[T], next_top[T], base[T];
                auto fetch = [&](int f) { frag[f] = *(const u32x4*)(f < KF ? kf + key_piece(f) : vf + value_piece(f - KF)); };
#pragma unroll
                for (int f = 0; f < AHEAD; f++) fetch(f);
                __builtin_amdgcn_sched_barrier(0);
                next_page();
#pragma unroll
                for (int t = 0; t < T; t++) base[t] = base_of(t);
                unrolled(std::make_integer_sequence<int, F>(), [&](auto number) {
                    constexpr int f = decltype(number)::value;
                    __builtin_amdgcn_sched_barrier(0);
                    if constexpr (f + AHEAD < F) fetch(f + AHEAD);
                    if constexpr (f < KF) multiply_keys(number, frag[f], s2);
                    else multiply_values(std::integral_constant<int, f - KF>(), frag[f]);
#pragma unroll
                    for (int n = f * N / F; n < (f + 1) * N / F; n++) {  // weights
                        const int t = n / EL, e = n % EL;
                        float& weight = x[t][e / E][e % E];
                        weight = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e / AE][e % AE], p.scale2, base[t]));
                        sum[t] = e ? sum[t] + weight : weight;
                        asm volatile("" : "+v"(sum[t]));
                        if (e % E == E - 1) w2[t][e / E] = operand<DT>(x[t][e / E], nullptr);
                        if (e == EL - 1) l[t] += sum[t];
                    }
                    if constexpr (f == F / 8) load_keys(i + NR);  // (scalar work and loads while the matrix instructions run)
                    if constexpr (f == F / 8 + 1) load_values(i + NR - 2, at3);
                    if constexpr (f >= KF) {  // maxima of the products
#pragma unroll
                        for (int n = (f - KF) * N / V; n < (f + 1 - KF) * N / V; n++) {
                            const int t = n / EL, e = n % EL;
                            next_top[t] = e ? fmaxf(next_top[t], s2[t][e / AE][e % AE]) : s2[t][0][0];
                        }
#pragma unroll
                        for (int t = 0; t < T; t++) if (t <= ((f + 1 - KF) * N / V - 1) / EL) asm volatile("" : "+v"(next_top[t]));  // (here, not behind the last one)
                    }
                });
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int t = 0; t < T; t++) {
                    top[t] = next_top[t];
#pragma unroll
                    for (int h = 0; h < W; h++) {
                        w[t][h] = w2[t][h];
                        asm volatile("" : "+v"(w[t][h]));
                    }
#pragma unroll
                    for (int h = 0; h < SA; h++) {
                        s[t][h] = s2[t][h];
                        asm volatile("" : "+v"(s[t][h]));
                    }
                    asm volatile("" : "+v"(l[t]), "+v"(top[t]));  // (all of it here, not behind the branch)
                }
                if (raised) shrink_sums();
                raised = false;
            }
            if (!large) continue;
        }
        // any other: one thing after the other
        turn();
        if (i < tiles) {
            next_page();
            load_keys(i + NR);
            load_values(i + NR - 2, at3);
        }
        const int place = j.begin + i * TK;
        int here = g;  // (what is made of it and of the limits is made here: kept across the loop above it takes the registers that the loop's loads need)
        asm volatile("" : "+v"(here));
        if (i > 0 && i <= my_tiles) {
            const uint8_t* vf = values_at(i - 1);
            auto values = [&](int f) { return *(const u32x4*)(vf + value_piece(f)); };
            // values that are no numbers, behind the end or where some row does not look, would make all rows such
            bool special = false;
#pragma unroll 1
            for (int f = 0; f < V; f++) {
                u32x4 v = values(f), where;
                special |= take_specials<DT>(v, where);
            }
            special = __any(special);
            auto live = [&](int f) { return j.end - (place - TK) - place_of(here, f / OA * E); };  // no row sees what lies behind
            if (special) {
#pragma unroll 1
                for (int f = 0; f < V; f++) {
                    u32x4 v = first_places<DT>(values(f), live(f)), where;
                    take_specials<DT>(v, where);
#pragma unroll
                    for (int t = 0; t < T; t++) {
                        u32x4 by = w[t][0];
#pragma unroll
                        for (int e = 0; e < 4; e++) by[e] = f < OA ? by[e] : w[t][W - 1][e];
                        const Acc seen = step<DT>(where, by, Acc{});
#pragma unroll
                        for (int e = 0; e < AE; e++) nan[t] |= (decltype(nan[t] + 0))(seen[e] > 0.0f) << (AE * (f % OA) + e);
                    }
                }
            }
            unrolled(std::make_integer_sequence<int, V>(), [&](auto number) {
                __builtin_amdgcn_sched_barrier(0);
                u32x4 v = values(decltype(number)::value);
                if (special) {
                    u32x4 where;
                    v = first_places<DT>(v, live(decltype(number)::value));
                    take_specials<DT>(v, where);
                }
                multiply_values(number, v);
            });
        }
        if (i < my_tiles) {
#pragma unroll
            for (int t = 0; t < T; t++)
#pragma unroll
                for (int e = 0; e < EL; e++) s[t][e / AE][e % AE] = place + place_of(here, e) < limit[t] ? s[t][e / AE][e % AE] : -__builtin_inff();
            maxima();
            float owed[T];
#pragma unroll
            for (int t = 0; t < T; t++) owed[t] = raised ? shrink[t] : 1.0f;
            // (large logits step by more than the slack: a weight one step above it could pass what fp16 holds)
            if (over(large ? 0.0f : slack) || raised) {
                raise();
#pragma unroll
                for (int t = 0; t < T; t++) shrink[t] *= owed[t];
                if (i) shrink_sums();
            }
            raised = false;
            if (large) {
#pragma unroll
                for (int t = 0; t < T; t++)
#pragma unroll
                    for (int e = 0; e < EL; e++) s[t][e / AE][e % AE] = s[t][e / AE][e % AE] * p.scale2 + (m[t] == -__builtin_inff() ? 0.0f : -m[t] * p.scale2);
            }
            weights(large ? 1.0f : p.scale2, [&](int t) { return large ? (float)Lifted::LIFT : base_of(t); });
            products(keys_at(i + 1), s);
        }
        i++;
    }
    // (no load may reach LDS that is used for something else by then)
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    // Some of the wave's rows at a time through its quarter of LDS: whole lines to memory, and a loop where the registers would take a program
    // longer than all the rest, which every workgroup runs once, from memory (1.2 us a KiB: it took 60 us).
    constexpr int LD = 32 * B, TS = std::min(T, (int)(sizeof(lds) / 4 / (ROWS * LD * 4)));
    static_assert(TS >= 1);
    float* mine_lds = (float*)lds + wave * (int)(sizeof(lds) / 16);
#pragma unroll
    for (int t0 = 0; t0 < T; t0 += TS) {
        if (mine + t0 * ROWS >= j.rows) break;
        float sum[TS], most[TS];
#pragma unroll
        for (int t = 0; t < TS; t++) {
            sum[t] = bad ? __builtin_nanf("") : over_rows_lanes<ROWS>(l[t0 + t], [](float a, float b) { return a + b; });
            most[t] = m[t0 + t] == -__builtin_inff() ? m[t0 + t] : m[t0 + t] * p.scale2;
            // (columns of four are turned by the row, so that 16 rows are in 16 places)
#pragma unroll
            for (int b = 0; b < (BIG ? 4 * B : V); b++) {
                const int column = BIG ? b * 2 + g : b * 4 + g, e = BIG ? b % 4 * 4 : 0;
                const Acc& from = o[t0 + t][BIG ? b / 4 : b];
                *(v4f*)&mine_lds[(t * ROWS + r) * LD + (column ^ (r & 7)) * 4] = v4f{from[e], from[e + 1], from[e + 2], from[e + 3]};
            }
        }
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the wave's own
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int i = lane; i < TS * ROWS * 8 * B; i += 64) {
            const int row = i / (8 * B), f = i % (8 * B) * 4, from = row % ROWS;
            v4f acc = *(const v4f*)&mine_lds[row * LD + ((f / 4) ^ (row & 7)) * 4];
            // (the lane and the bits of the row's features f to f + 3)
            const int lane_of = from + f / 4 % (64 / ROWS) * ROWS, bit = BIG ? f / 8 * 4 : f / 16 * 4;
            auto bits = __shfl(nan[t0], lane_of);
            float row_sum = __shfl(sum[0], from), row_most = __shfl(most[0], from);
#pragma unroll
            for (int t = 1; t < TS; t++) {
                const auto b1 = __shfl(nan[t0 + t], lane_of);
                const float s1 = __shfl(sum[t], from), m1 = __shfl(most[t], from);
                if (row >= t * ROWS) bits = b1, row_sum = s1, row_most = m1;
            }
            bits >>= bit;
#pragma unroll
            for (int e = 0; e < 4; e++) acc[e] = bits >> e & 1 ? __builtin_nanf("") : acc[e];
            const int at = mine + t0 * ROWS + row;
            if (at < j.rows && f < p.dim) put_row<DT>(p, j, at, f, acc * Lifted::DOWN, row_most, row_sum * Lifted::DOWN);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// W waves to a row.  Each forms the parts' common maximum and sum; then a lane has four features and every (64 W / lanes of a row)th part,
// and the lanes' sums are added in LDS, in an order that depends on the shape alone.
template <int DT, int W>
__global__ __launch_bounds__(W < 4 ? 256 : 64 * W) void attend_join_kernel(AttendParams p) {
    constexpr int ROWS = W < 4 ? 4 / W : 1;
    __shared__ __attribute__((aligned(16))) float sums[ROWS * 64 * W * 4];
    const int lane = threadIdx.x & 63, in_row = threadIdx.x % (64 * W);
    uint32_t row = blockIdx.x * ROWS + threadIdx.x / (64 * W);
    const int stride = part_stride(p.dim);
    // the row's parts: `shared` of the prefix, then its sequence's
    int shared = 0, count = 0;
    bool there, bad = false;
    const float2 *pml = nullptr, *ml = nullptr;
    const float *po = nullptr, *o = nullptr;
    int s = -1, n = 0, length = 0, t0 = 0, token = 0;
    int64_t few_slot = row;
    if (p.join_few) {
        const uint32_t of = row / (uint32_t)p.few_slots, r = row - of * p.few_slots;
        s = (int)(of / (uint32_t)p.kv_heads);
        there = s < p.n_seq;
        if (there) {
            bad = sequence_of(p, s, &t0, &n, &length);
            there = (int)r < n * p.group && n * p.group <= p.few_rows;
            const uint32_t i = r / (uint32_t)p.group;
            token = t0 + (int)i;
            row = (uint32_t)token * p.heads + (of - s * p.kv_heads) * p.group + r - i * p.group;
        }
    } else {
        there = row < (uint32_t)p.tokens * (uint32_t)p.heads;
        if (there) {
            token = (int)(row / (uint32_t)p.heads);
            s = p.starts ? owner_of(p.starts, p.n_seq, token) : token;
            if (s >= 0) {
                bad = sequence_of(p, s, &t0, &n, &length);
                if (token < t0 || token - t0 >= n) s = -1, bad = false;  // (starts that do not ascend)
                const uint32_t head = row - (uint32_t)token * p.heads, kv = head / (uint32_t)p.group;
                few_slot = ((int64_t)s * p.kv_heads + kv) * p.few_slots + (int64_t)(token - t0) * p.group + head - kv * p.group;
            }
        }
    }
    // What a row can have is asked for before it is known how much of it there is (what no workgroup wrote is not used).
    const int lanes = stride / 4, step = 64 * W / lanes;  // (lanes <= 64)
    const int first = in_row / lanes, f = in_row % lanes * 4;
    int most = 0;
    if (there && s >= 0) {
        const bool wide = n * p.group > p.few_rows;
        const int slots = wide ? p.wide_chunks : p.chunks, chunk = wide ? p.wide_chunk : p.chunk;
        const int64_t at = wide || p.all_few ? (int64_t)row * slots : few_slot * slots;
        const Parts& mine = wide ? p.wide_parts : p.few_parts;
        there = mine.o != nullptr;  // (the other kernel's rows may be finished)
        if (there) {
            ml = mine.ml + at, o = mine.o + at * stride;
            shared = p.prefix_chunks;
            pml = p.prefix_parts.ml + (int64_t)row * shared, po = p.prefix_parts.o + (int64_t)row * shared * stride;
            most = shared + slots;
            const int limit = length - n + 1 + (int)(token - t0);
            count = shared + (limit > 0 ? (limit + chunk - 1) / chunk : 0);
        }
    }
    auto ml_of = [&](int i) { return i < shared ? pml[i] : ml[i - shared]; };
    auto o_of = [&](int i) { return *(const v4f*)((i < shared ? po + (int64_t)i * stride : o + (int64_t)(i - shared) * stride) + f); };
    const float2 own_ml = lane < most ? ml_of(lane) : make_float2(0.0f, 0.0f);
    const bool early = first < step && first < most;
    const float first_m = early ? ml_of(first).x : 0.0f;
    const v4f first_o = early ? o_of(first) : v4f{0, 0, 0, 0};
    float top = lane < count ? own_ml.x : -__builtin_inff(), sum = 0.0f;
    for (int i = lane + 64; i < count; i += 64) top = fmaxf(top, ml_of(i).x);
    for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
    const float base = top == -__builtin_inff() ? 0.0f : top;
    if (lane < count) sum = __builtin_amdgcn_exp2f(own_ml.x - base) * own_ml.y;
    for (int i = lane + 64; i < count; i += 64) sum += __builtin_amdgcn_exp2f(ml_of(i).x - base) * ml_of(i).y;
    for (int x = 32; x; x >>= 1) sum += __shfl_xor(sum, x);
    if (bad) sum = __builtin_nanf("");
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    v4f acc = {0, 0, 0, 0};
    if (first < step) {
        if (first < count) acc = first_o * __builtin_amdgcn_exp2f(first_m - base);
#pragma unroll 2
        for (int i = first + step; i < count; i += step) acc += o_of(i) * __builtin_amdgcn_exp2f(ml_of(i).x - base);
    }
    *(v4f*)&sums[threadIdx.x * 4] = acc;
    __syncthreads();
    if (first != 0 || !there) return;
    for (int i = 1; i < step; i++) acc += *(const v4f*)&sums[(threadIdx.x + i * lanes) * 4];
    put_features<DT>(p, row, f, acc * inverse);
    if (in_row == 0 && p.lse) p.lse[row] = lse_of(top, sum);
}

// ---- host --------------------------------------------------------------------------------------------------------------

struct Region {
    int64_t rows, slots;
    size_t ml, o;  // byte offsets in the workspace
};
struct AttendPlan {
    int64_t chunk, chunks, tiles, few_rows, few_slots, wide_chunk, wide_chunks, wide_tiles, prefix_chunk, prefix_chunks, prefix_tiles;
    bool few, wide, prefix_wide, all_few;     // kernels that have work
    int64_t units;
    bool few_parts, wide_parts, join_few;
    Region few_region, wide_region, prefix_region;
    size_t q_copy;  // byte offset
    size_t bytes;
};
// Which kernel takes what.  A launch of attend_tiles_kernel takes 14 us before its rows pay (a long program, read from memory by every compute
// unit; partly filled tiles) and asks for attend_rows_kernel beside it, which takes the sequences of few rows; then it forms 2.5 times as many
// products a microsecond as attend_rows_kernel, which reads the keys again for every 16 rows.  All of a call, rows / tiles kernel, 32 heads on 8 key heads
// of 128, sequences x tokens at places: 1 x 512 at 512 18 / 44 us, 4 x 64 at 1000 22 / 44, 16 x 40 at 600 34 / 44, 4 x 16 at 4096 35 / 36, 8 x 16
// at 4096 63 / 53, 16 x 16 at 2000 69 / 49, 4 x 64 at 2000 44 / 41; the prefix of 512 rows x 8 key heads x 1000 places 51 / 57, of 128 x 4000
// 31 / 38, of 128 x 16000 70 / 54.
constexpr double TILES_PAY = 3 << 29;  // features of products: rows x places x key heads x dim
constexpr int64_t FEW_ROWS = 32;
static int64_t wide_tile(int64_t dim) { return dim <= 128 ? WideTile<4>::R : WideTile<8>::R; }
static int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }
// Chunks of `places` for `tiles` of rows, so that there are `want` workgroups
static int64_t chunk_of(int64_t places, int64_t tiles, int64_t want, int64_t least, int64_t most) {
    const int64_t n = std::max<int64_t>(1, want / std::max<int64_t>(1, tiles));
    return std::max(least, std::min(most, round_up(ceil_div(std::max<int64_t>(places, 1), n), 128)));
}
static AttendPlan attend_plan(int dt, bool q_in_place, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim, int64_t longest, bool starts, int64_t sequences,
                              int64_t prefix) {
    AttendPlan a = {};
    const int64_t group = heads / kv_heads, most_rows = starts ? tokens * group : group;
    auto pays = [&](int64_t places) { return (double)tokens * heads * places * dim > TILES_PAY; };
    a.all_few = starts && !pays(longest);
    a.few_rows = a.all_few ? 0x7fffffff : FEW_ROWS;
    a.few = starts || group <= a.few_rows;
    a.wide = most_rows > a.few_rows;
    a.few_slots = std::min(most_rows, a.few_rows);
    a.tiles = ceil_div(a.few_slots, 16);
    a.units = a.all_few ? tokens * group / 16 + sequences : sequences * a.tiles;
    a.wide_tiles = starts ? tokens * group / wide_tile(dim) + sequences : sequences * ceil_div(group, wide_tile(dim));
    // Up to 512 places in one workgroup, without parts: a row of 500 places 8.2 us, 5.9 and 5.3 and a launch in parts
    // Three workgroups to a compute unit where the caches are large, else one, with fewer parts to join (37 sequences of up to 7 tokens x 900 places behind 1000
    // 25 / 19 us, 8 x 12 tokens on 1000 22 / 15; 3 x 50000 places 98 / 117)
    const bool little = (double)sequences * kv_heads * longest * dim * 2 * dtype_size(dt) < (64 << 20);
    a.chunk = longest <= 512 && !prefix ? 512
                                        : chunk_of(longest, (a.all_few ? std::max(sequences, ceil_div(tokens * group, 16)) : a.units) * kv_heads, little ? 256 : 768, 128, 4096);
    // (parts of a GiB at most: so many rows fill the chip with longer chunks as well)
    const int64_t few_rows_all = a.all_few ? tokens * heads : sequences * kv_heads * a.few_slots;
    while (a.chunk < longest && (double)few_rows_all * ceil_div(longest, a.chunk) * part_stride((int)dim) * 4 > (1 << 30)) a.chunk *= 2;
    a.chunks = std::max<int64_t>(1, ceil_div(longest, a.chunk));
    a.wide_chunk = chunk_of(longest, a.wide_tiles * kv_heads, 512, 256, 1 << 30);
    a.wide_chunks = std::max<int64_t>(1, ceil_div(longest, a.wide_chunk));
    if (prefix) {
        a.prefix_wide = tokens * group > FEW_ROWS && pays(prefix);
        a.prefix_tiles = ceil_div(tokens * group, a.prefix_wide ? wide_tile(dim) : 16);
        a.prefix_chunk = a.prefix_wide ? chunk_of(prefix, a.prefix_tiles * kv_heads, 512, 256, 1 << 30) : chunk_of(prefix, a.prefix_tiles * kv_heads, 384, 128, 4096);
        a.prefix_chunks = ceil_div(prefix, a.prefix_chunk);
    }
    a.few_parts = a.few && (a.chunks > 1 || prefix);
    a.wide_parts = a.wide && (a.wide_chunks > 1 || prefix);
    a.join_few = a.few_parts && a.wide && !a.wide_parts;
    auto region = [&](bool there, int64_t rows, int64_t slots) {
        Region r = {there ? rows : 0, slots, 0, 0};
        r.ml = a.bytes, a.bytes += (size_t)round_up(r.rows * slots * 8, 256);
        r.o = a.bytes, a.bytes += (size_t)round_up(r.rows * slots * part_stride((int)dim) * 4, 256);
        return r;
    };
    a.few_region = region(a.few_parts, few_rows_all, a.chunks);
    a.wide_region = region(a.wide_parts, tokens * heads, a.wide_chunks);
    a.prefix_region = region(prefix > 0, tokens * heads, a.prefix_chunks);
    a.q_copy = a.bytes;
    if (!q_in_place) a.bytes += (size_t)round_up(tokens * heads * cache_head_dim(dt, dim) * dtype_size(dt), 256);
    return a;
}

template <int DT, int B>
static void launch_attend_cfg(const AttendParams& p, int64_t few_blocks, int64_t wide_blocks, hipStream_t st) {
    if (wide_blocks) hipLaunchKernelGGL((attend_tiles_kernel<DT, B>), dim3((unsigned)wide_blocks), dim3(256), 0, st, p);
    if (few_blocks) hipLaunchKernelGGL((attend_rows_kernel<DT, B>), dim3((unsigned)few_blocks), dim3(256), 0, st, p);
}
template <int DT>
static void launch_attend(AttendParams& p, void* q_copy, int64_t few_blocks, int64_t wide_blocks, int64_t join_rows, hipStream_t st) {
    if (q_copy) {
        hipLaunchKernelGGL((attend_copy_kernel<DT>), dim3((unsigned)std::min<int64_t>(ceil_div((int64_t)p.tokens * p.heads * p.dp, 1024), 4096)), dim3(256), 0, st, p, q_copy);
        p.q = q_copy, p.q_head = p.q_dim = p.dp, p.q_token = (int64_t)p.heads * p.dp;
    }
    switch (ceil_div(p.dim, 32)) {
        case 1: launch_attend_cfg<DT, 1>(p, few_blocks, wide_blocks, st); break;
        case 2: launch_attend_cfg<DT, 2>(p, few_blocks, wide_blocks, st); break;
        case 3: launch_attend_cfg<DT, 3>(p, few_blocks, wide_blocks, st); break;
        case 4: launch_attend_cfg<DT, 4>(p, few_blocks, wide_blocks, st); break;
        case 5: launch_attend_cfg<DT, 5>(p, few_blocks, wide_blocks, st); break;
        case 6: launch_attend_cfg<DT, 6>(p, few_blocks, wide_blocks, st); break;
        case 7: launch_attend_cfg<DT, 7>(p, few_blocks, wide_blocks, st); break;
        default: launch_attend_cfg<DT, 8>(p, few_blocks, wide_blocks, st); break;
    }
    if (!join_rows) return;
    const int64_t parts = p.prefix_chunks + std::max(p.few_parts.o ? p.chunks : 0, p.wide_parts.o ? p.wide_chunks : 0);
    // a wave to a row where there are rows for all of them (4096 rows of 17 parts 9.4 us, with four waves each 14)
    if (parts <= 8 || join_rows >= 2048) hipLaunchKernelGGL((attend_join_kernel<DT, 1>), dim3((unsigned)ceil_div(join_rows, 4)), dim3(256), 0, st, p);
    else if (parts <= 32) hipLaunchKernelGGL((attend_join_kernel<DT, 4>), dim3((unsigned)join_rows), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((attend_join_kernel<DT, 16>), dim3((unsigned)join_rows), dim3(1024), 0, st, p);
}

static bool shape_ok(int dt, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim, int64_t page, int64_t width, int64_t longest, bool starts, int64_t sequences,
                     int64_t prefix) {
    return dt >= BT_F32 && dt <= BT_BF16 && tokens > 0 && tokens <= 0x7fffffff && kv_heads > 0 && heads > 0 && heads <= 16384 && tokens * heads <= 0x7fffffff && heads % kv_heads == 0 && dim > 0 && dim <= 256 && page >= 32 &&
           page <= 65536 && (page & (page - 1)) == 0 && width > 0 && width * page <= (1 << 30) && longest >= 0 && longest <= width * page && sequences > 0 &&
           sequences <= (1 << 24) && (starts || sequences == tokens) && prefix >= 0 && prefix <= (1 << 30);
}

}  // namespace bt

using namespace bt;

extern "C" size_t bt_cached_attention_workspace_bytes(int dtype, int q_in_place, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t page_size, int64_t table_width,
                                                      int64_t max_length, int has_starts, int64_t sequences, int64_t prefix_length) {
    if (!shape_ok(dtype, tokens, heads, kv_heads, head_dim, page_size, table_width, max_length, has_starts != 0, sequences, prefix_length)) return 0;
    return attend_plan(dtype, q_in_place != 0, tokens, heads, kv_heads, head_dim, max_length, has_starts != 0, sequences, prefix_length).bytes;
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
    if (!shape_ok(dtype, tokens, heads, kv_heads, head_dim, page_size, table_width, max_length, q_starts != nullptr, sequences, prefix_length) || pages <= 0 ||
        pages > 0x7fffffff) {
        set_error("%s: head_dim at most 256, heads a multiple of kv_heads, page_size a power of two from 32 on, up to 2^30 places of a sequence, one token a "
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
    const int e = 16 / dtype_size(dtype);
    const bool in_place = head_dim % e == 0 && q_token % e == 0 && q_head % e == 0 && ((uintptr_t)q) % 16 == 0;
    const AttendPlan a = attend_plan(dtype, in_place, tokens, heads, kv_heads, head_dim, max_length, q_starts != nullptr, sequences, prefix_length);
    if (a.bytes && (!workspace || workspace_bytes < a.bytes || ((uintptr_t)workspace) % 256 != 0)) {
        set_error("%s: workspace of %zu bytes (256-byte aligned) needed, %zu given", who, a.bytes, workspace_bytes);
        return BT_ERR_WORKSPACE;
    }
    AttendParams p = {};
    p.q = q, p.k_cache = k_cache, p.v_cache = v_cache, p.table = block_table, p.lengths = lengths, p.starts = q_starts, p.prefix_table = prefix_table;
    p.q_token = q_token, p.q_head = q_head, p.tokens = (int)tokens, p.out = out, p.lse = lse;
    auto parts = [&](const Region& r) { return r.rows ? Parts{(float*)((char*)workspace + r.o), (float2*)((char*)workspace + r.ml)} : Parts{nullptr, nullptr}; };
    p.few_parts = parts(a.few_region), p.wide_parts = parts(a.wide_region), p.prefix_parts = parts(a.prefix_region);
    p.heads = (int)heads, p.kv_heads = (int)kv_heads, p.group = (int)(heads / kv_heads), p.dim = p.q_dim = (int)head_dim, p.dp = cache_head_dim(dtype, head_dim);
    p.n_seq = (int)sequences, p.width = (int)table_width, p.page_shift = __builtin_ctzll((unsigned long long)page_size), p.pages = (int)pages;
    p.prefix = (int)prefix_length;
    p.longest = (int)max_length, p.few_rows = (int)a.few_rows, p.few_slots = (int)a.few_slots, p.join_few = a.join_few;
    p.chunk = (int)a.chunk, p.chunks = (int)a.chunks, p.tiles = (int)a.tiles, p.units = (int)a.units, p.all_few = a.all_few;
    p.wide_chunk = (int)a.wide_chunk, p.wide_chunks = (int)a.wide_chunks;
    p.prefix_chunk = (int)a.prefix_chunk, p.prefix_chunks = (int)a.prefix_chunks, p.prefix_tiles = (int)a.prefix_tiles, p.prefix_wide = a.prefix_wide;
    p.scale2 = (float)((double)scale * 1.4426950408889634074);
    const int64_t prefix_blocks = a.prefix_tiles * a.prefix_chunks * kv_heads;
    const bool clear = q_starts && (a.join_few || (!a.few_parts && !a.wide_parts));  // (attend_join_kernel sees to the rows behind otherwise)
    const int64_t few_blocks = (a.few ? a.units * a.chunks * kv_heads : 0) + (a.prefix_wide ? 0 : prefix_blocks) + (clear ? clearing_blocks(tokens * heads * head_dim) : 0);
    const int64_t wide_blocks = (a.wide ? a.wide_tiles * a.wide_chunks * kv_heads : 0) + (a.prefix_wide ? prefix_blocks : 0);
    const int64_t join_rows = a.join_few ? a.few_region.rows : a.few_parts || a.wide_parts ? tokens * heads : 0;
    if (std::max({few_blocks, wide_blocks, join_rows / 4}) >= (1 << 24) || a.units > 0x7fffffff || a.wide_tiles > 0x7fffffff || a.prefix_tiles > 0x7fffffff) {
        set_error("%s: %lld workgroups are beyond one launch", who, (long long)std::max(few_blocks, wide_blocks));
        return BT_ERR_INVALID;
    }
    hipStream_t st = (hipStream_t)stream;
    if (dtype == BT_F32) launch_attend<BT_F32>(p, in_place ? nullptr : (char*)workspace + a.q_copy, few_blocks, wide_blocks, join_rows, st);
    else if (dtype == BT_F16) launch_attend<BT_F16>(p, in_place ? nullptr : (char*)workspace + a.q_copy, few_blocks, wide_blocks, join_rows, st);
    else launch_attend<BT_BF16>(p, in_place ? nullptr : (char*)workspace + a.q_copy, few_blocks, wide_blocks, join_rows, st);
    return check_launch(who);
}
