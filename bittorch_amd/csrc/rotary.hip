// Rotary positions, alone (bt_rotary) and on the way into the paged cache (bt_cache_append).
//
// A pair (a, b) of a head's first R features at position p is turned by p f_i: a' = A (a cos - b sin), b' = A (b cos + a sin).  The gradient
// is the same with the opposite angle.  The angle is formed in 64 bits in turns, p (f_i / 2 pi), and reduced to [-1/2, 1/2] before it is
// rounded to 32: at position 10^6 a 32-bit product would be off by 0.06.
//
// Both kernels are bound by memory (5 operations an element) if the angles are not formed for every head anew: a workgroup takes a few
// tokens, forms their cosines and sines once in LDS and walks the pieces (16 bytes of either half of the pairs) of all their heads.  bf16: 4096
// tokens x 40 heads of 128 17 to 18 us (4.6 to 4.9 TB/s), the prompts of 8 x 512 tokens, 20 + 20 heads, to the cache 28 us (4.4 TB/s).
#include "paged_cache.h"

namespace bt {

constexpr int TURN_ANGLES = 1024;  // of a workgroup: tokens x pairs
constexpr int TURN_THREADS = 256;
constexpr int64_t APPEND_BLOCKS = 2048;

struct TurnParams {
    const void *q, *k, *v;
    void *q_out, *k_out;         // contiguous; k_out null: k goes to the cache
    int64_t q_token, q_head, k_token, k_head, v_token, v_head;  // strides in elements
    const void *positions, *freq;
    void *k_cache, *v_cache;
    const int32_t *table, *lengths, *starts;
    int64_t first_position, tokens;
    int hq, hk, dim, rot, interleaved, pos64, freq64, group, n_seq, width, page_shift, pages, dp, units;
    float amplitude, sign;
    Divider per_head, slots, by_dim;  // pieces of a head, heads, features
};

template <int DT, int PV>
__device__ __forceinline__ void load_piece(const void* p, int64_t at, float (&v)[PV]) {
    if constexpr (PV == 1) v[0] = load_elem<DT>(p, at);
    else if constexpr (DT == BT_F32) {
        const float4 w = *(const float4*)((const float*)p + at);
        v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
    } else {
        const u32x4 w = *(const u32x4*)((const uint16_t*)p + at);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint16_t h = (uint16_t)(w[i / 2] >> (i % 2 * 16));
            v[i] = DT == BT_F16 ? f16_bits_to_f32(h) : bf16_bits_to_f32(h);
        }
    }
}
template <int DT, int PV>
__device__ __forceinline__ void store_piece(void* p, int64_t at, const float (&v)[PV]) {
    if constexpr (PV == 1) store_elem<DT>(p, at, v[0]);
    else if constexpr (DT == BT_F32) *(float4*)((float*)p + at) = make_float4(v[0], v[1], v[2], v[3]);
    else {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t lo = DT == BT_F16 ? f32_to_f16_bits(v[2 * i]) : f32_to_bf16_bits(v[2 * i]);
            const uint32_t hi = DT == BT_F16 ? f32_to_f16_bits(v[2 * i + 1]) : f32_to_bf16_bits(v[2 * i + 1]);
            w[i] = lo | hi << 16;
        }
        *(u32x4*)((uint16_t*)p + at) = w;
    }
}

// cos and sin of `count` tokens' angles, [token][pair], times the amplitude
template <typename Position>
__device__ __forceinline__ void form_angles(float2* turn, const TurnParams& p, int count, Position position) {
    const int pairs = p.rot / 2;
    for (int idx = threadIdx.x; idx < count * pairs; idx += TURN_THREADS) {
        const int i = idx / pairs, j = idx - i * pairs;
        const double f = p.freq64 ? ((const double*)p.freq)[j] : (double)((const float*)p.freq)[j];
        const double t = (double)position(i) * (f * 0.15915494309189533577);
        float s, c;
        sincospif(2.0f * (float)(t - rint(t)), &s, &c);
        turn[idx] = make_float2(c * p.amplitude, s * p.amplitude * p.sign);
    }
    __syncthreads();
}

// Piece `piece` of one head: pairs PV piece .. + PV - 1, or behind the pairs features that stay as they are.  put(feature, values): PV values from there on.
template <int DT, int PV, typename Put>
__device__ __forceinline__ void turn_piece(const TurnParams& p, const float2* turn, const void* src, int64_t at, int piece, Put put) {
    const int pairs = p.rot / 2, first = piece * PV;
    if (first >= pairs) {
        const int f = p.rot + first - pairs;
        float v[PV] = {};
        if (f < p.dim) load_piece<DT, PV>(src, at + f, v);
        put(f, v);
        return;
    }
    const int fa = p.interleaved ? 2 * first : first, fb = p.interleaved ? fa + PV : first + pairs;
    float lo[PV], hi[PV], a[PV], b[PV];
    load_piece<DT, PV>(src, at + fa, lo);
    load_piece<DT, PV>(src, at + fb, hi);
#pragma unroll
    for (int i = 0; i < PV; i++) {
        // (neighbours are pairs: elements 2 i and 2 i + 1 of the 2 PV)
        const float x = !p.interleaved ? lo[i] : 2 * i < PV ? lo[2 * i % PV] : hi[2 * i % PV];
        const float y = !p.interleaved ? hi[i] : 2 * i + 1 < PV ? lo[(2 * i + 1) % PV] : hi[(2 * i + 1) % PV];
        const float2 cs = turn[first + i];
        a[i] = __builtin_fmaf(x, cs.x, -(y * cs.y));
        b[i] = __builtin_fmaf(y, cs.x, x * cs.y);
    }
    if (p.interleaved) {
#pragma unroll
        for (int i = 0; i < PV; i++) {
            const float x = i % 2 ? b[i / 2] : a[i / 2], y = (PV + i) % 2 ? b[(PV + i) / 2] : a[(PV + i) / 2];
            lo[i] = x, hi[i] = y;
        }
        put(fa, lo);
        put(fb, hi);
    } else {
        put(fa, a);
        put(fb, b);
    }
}

// grid (token groups, shares of a group's pieces)
template <int DT, int PV>
__global__ __launch_bounds__(TURN_THREADS) void rotary_kernel(TurnParams p) {
    __shared__ float2 turn[TURN_ANGLES];
    const int64_t t0 = (int64_t)blockIdx.x * p.group;
    const int count = (int)std::min<int64_t>(p.group, p.tokens - t0);
    form_angles(turn, p, count, [&](int i) { return p.pos64 ? ((const int64_t*)p.positions)[t0 + i] : (int64_t)((const int32_t*)p.positions)[t0 + i]; });
    const uint32_t items = (uint32_t)count * p.slots.d * p.per_head.d;
    for (uint32_t idx = blockIdx.y * TURN_THREADS + threadIdx.x; idx < items; idx += gridDim.y * TURN_THREADS) {
        const uint32_t row = divide(idx, p.per_head), i = divide(row, p.slots);
        const int piece = (int)(idx - row * p.per_head.d), slot = (int)(row - i * p.slots.d);
        const bool is_q = slot < p.hq;
        const int head = is_q ? slot : slot - p.hq, heads = is_q ? p.hq : p.hk;
        const int64_t t = t0 + i, at = is_q ? t * p.q_token + head * p.q_head : t * p.k_token + head * p.k_head;
        void* out = is_q ? p.q_out : p.k_out;
        const int64_t to = (t * heads + head) * p.dim;
        turn_piece<DT, PV>(p, turn + i * (p.rot / 2), is_q ? p.q : p.k, at, piece, [&](int f, const float (&v)[PV]) {
            if (f < p.dim) store_piece<DT, PV>(out, to + f, v);
        });
    }
}

// The new tokens of one sequence whose places share a 16-byte group of the values (E places): their keys and queries are turned, their
// values transposed by the way they are read (a lane owns FV features, the group's tokens are its registers).  grid (units, shares of a
// unit's pieces); units beyond p.units clear the queries behind the last sequence.
template <int DT, int PV, int FV>
__global__ __launch_bounds__(TURN_THREADS) void cache_append_kernel(TurnParams p) {
    using Order = CacheOrder<DT>;
    constexpr int E = Order::E;
    __shared__ float2 turn[TURN_ANGLES];
    if ((int)blockIdx.x >= p.units) {
        const int64_t n = (int64_t)p.hq * p.dim, behind = std::max<int64_t>(0, std::min<int64_t>(p.starts[p.n_seq], p.tokens));
        const int64_t step = (int64_t)(gridDim.x - p.units) * gridDim.y * TURN_THREADS;
        for (int64_t i = behind * n + ((int64_t)(blockIdx.x - p.units) * gridDim.y + blockIdx.y) * TURN_THREADS + threadIdx.x; i < p.tokens * n; i += step)
            store_elem<DT>(p.q_out, i, 0.0f);
        return;
    }
    // the unit: sequence s, its new tokens [t0, t0 + n), the places [low, high) of the group
    int s = blockIdx.x, n = 1;
    int64_t t0 = s, group = 0;
    if (p.starts) {
        // sequence s has the units floor(starts[s] / E) + 2 s and on: n tokens lie in n / E + 2 groups at most
        const int lane = threadIdx.x & 63;
        int found = 0;
        for (int s0 = 0; s0 < p.n_seq; s0 += 64) {
            const int i = s0 + lane;
            const uint64_t hit = __ballot(i < p.n_seq && (int64_t)std::max(p.starts[i < p.n_seq ? i : 0], 0) / E + 2 * (int64_t)i <= (int64_t)blockIdx.x);
            found += __popcll(hit);
            if (hit != ~0ull) break;
        }
        s = found - 1;
        if (s < 0) return;
        t0 = std::max(p.starts[s], 0);
        n = (int)std::max<int64_t>(0, std::min<int64_t>(p.starts[s + 1], p.tokens) - t0);
        group = (int64_t)blockIdx.x - (t0 / E + 2 * (int64_t)s);
    }
    if (n <= 0) return;
    const int64_t length = p.lengths[s], begin = length - n;  // the first new token's place (below zero: it has none)
    const int64_t aligned = (begin >= 0 ? begin / E : -((-begin + E - 1) / E)) + group;
    const int64_t low = std::max(aligned * E, begin), high = std::min(aligned * E + E, length);
    if (low >= high) return;
    const int count = (int)(high - low);
    const int64_t first = t0 + (low - begin);
    if (p.rot) form_angles(turn, p, count, [&](int i) { return p.first_position + low + i; });
    // (places before the first, behind the table's last or on a page that the cache does not have are not written; a group lies on one side
    // of each)
    int64_t page = -1;
    if (aligned >= 0 && aligned * E < (int64_t)p.width << p.page_shift) {
        page = p.table[(int64_t)s * p.width + (aligned * E >> p.page_shift)];
        if (page >= p.pages) page = -1;
    }
    const int inside = (int)(aligned * E & ((1 << p.page_shift) - 1));  // of the page
    const int64_t page_elements = (int64_t)p.dp << p.page_shift;

    // Pieces of a whole group: four tokens side by side, whose 16 bytes are neighbours in the keys' order, then the pieces, then the other four
    // (16 bytes a store each on a line of their own took the prompts of 8 x 512 tokens 41 us)
    const bool whole = count == E;
    const uint32_t turned = (uint32_t)count * p.slots.d * p.per_head.d;                 // slots: the keys' heads, then the queries'
    const uint32_t items = turned + (uint32_t)p.hk * p.by_dim.d;
    for (uint32_t idx = blockIdx.y * TURN_THREADS + threadIdx.x; idx < items; idx += gridDim.y * TURN_THREADS) {
        if (idx < turned) {
            int i, piece, slot;
            if (whole) {
                const uint32_t rest = idx / 4, row = divide(rest, p.per_head);
                piece = (int)(rest - row * p.per_head.d);
                slot = (int)(row / (E / 4));
                i = (int)(idx % 4 + row % (E / 4) * 4);
            } else {
                const uint32_t row = divide(idx, p.per_head), at = divide(row, p.slots);
                piece = (int)(idx - row * p.per_head.d), slot = (int)(row - at * p.slots.d), i = (int)at;
            }
            const int64_t t = first + i;
            if (slot < p.hk) {
                if (page < 0) continue;
                const int place = inside + (int)(low - aligned * E) + i;
                const int64_t base = (page * p.hk + slot) * page_elements;
                turn_piece<DT, PV>(p, turn + i * (p.rot / 2), p.k, t * p.k_token + slot * p.k_head, piece, [&](int f, const float (&v)[PV]) {
                    store_piece<DT, PV>(p.k_cache, base + Order::key(place, f, p.dp), v);
                });
            } else {
                const int64_t to = (t * p.hq + slot - p.hk) * p.dim;
                turn_piece<DT, PV>(p, turn + i * (p.rot / 2), p.q, t * p.q_token + (slot - p.hk) * p.q_head, piece, [&](int f, const float (&v)[PV]) {
                    if (f < p.dim) store_piece<DT, PV>(p.q_out, to + f, v);
                });
            }
            continue;
        }
        if (page < 0) continue;
        const uint32_t head = divide(idx - turned, p.by_dim);
        const int f = (int)(idx - turned - head * p.by_dim.d) * FV;
        const int64_t from = first * p.v_token + head * p.v_head + f;
        const int64_t to = (page * p.hk + head) * page_elements + Order::value(inside, f, p.dp);
        if (FV == 2 && whole) {  // two features a lane: 4 bytes of each token, 16 of each feature
            u32x4 even, odd;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t a = *(const uint32_t*)((const uint16_t*)p.v + from + 2 * i * p.v_token), b = *(const uint32_t*)((const uint16_t*)p.v + from + (2 * i + 1) * p.v_token);
                even[i] = (a & 0xffffu) | b << 16, odd[i] = a >> 16 | (b & 0xffff0000u);
            }
            *(u32x4*)((uint16_t*)p.v_cache + to) = even;
            *(u32x4*)((uint16_t*)p.v_cache + to + E) = odd;
        } else if (FV == 1 && whole) {
            float v[E];
#pragma unroll
            for (int i = 0; i < E; i++) v[i] = load_elem<DT>(p.v, from + i * p.v_token);
            store_piece<DT, E>(p.v_cache, to, v);
        } else {
            const int skip = (int)(low - aligned * E);
#pragma unroll
            for (int e = 0; e < FV; e++) {
                float v[E];  // (all on their way before the first is stored)
#pragma unroll
                for (int i = 0; i < E; i++) v[i] = i < count ? load_elem<DT>(p.v, from + e + i * p.v_token) : 0.0f;
#pragma unroll
                for (int i = 0; i < E; i++)
                    if (i < count) store_elem<DT>(p.v_cache, to + e * E + skip + i, v[i]);
            }
        }
    }
}

static bool known(int dt) { return dt == BT_F32 || dt == BT_F16 || dt == BT_BF16; }
static bool misaligned(const void* p, int to) { return ((uintptr_t)p) % to != 0; }

// Pieces of 16 bytes: everything that is moved starts and ends on one.
static bool whole_pieces(const TurnParams& p, int e) {
    const int64_t strides = p.q_token | p.q_head | p.k_token | p.k_head;
    return p.dim % e == 0 && p.rot / 2 % e == 0 && strides % e == 0 && !misaligned(p.q, 16) && !misaligned(p.k, 16) && !misaligned(p.q_out, 16) &&
           !misaligned(p.k_out, 16);
}
static int turn_checks(const char* who, int dt, int64_t tokens, int64_t hq, int64_t hk, int64_t dim, int64_t rot, int f_dtype_64, const void* freq) {
    if (!known(dt) || tokens <= 0 || hq < 0 || hk < 0 || hq + hk <= 0 || dim <= 0 || (f_dtype_64 != 0 && f_dtype_64 != 1)) {
        set_error("%s: empty shape or bad dtype", who);
        return BT_ERR_INVALID;
    }
    if (rot < 0 || rot % 2 != 0 || rot > dim || (rot && !freq)) {
        set_error("%s: rotary_dim=%lld must be even and at most the head dimension %lld", who, (long long)rot, (long long)dim);
        return BT_ERR_INVALID;
    }
    if (dim > 1024 || hq + hk > 16384 || tokens > 0x7fffffff || (hq + hk) * dim > (1 << 18)) {  // (the divisions of a workgroup's pieces)
        set_error("%s: at most 1024 features a head, 16384 heads and 2^18 features a token (head_dim=%lld, heads=%lld)", who, (long long)dim, (long long)(hq + hk));
        return BT_ERR_INVALID;
    }
    return 0;
}

template <int DT>
static void launch_rotary(TurnParams& p, hipStream_t st) {
    constexpr int E = CacheOrder<DT>::E;
    const bool vec = whole_pieces(p, E);
    const int pv = vec ? E : 1;
    p.per_head = divider((uint32_t)(p.rot / 2 / pv + (p.dim - p.rot) / pv));
    p.slots = divider((uint32_t)(p.hq + p.hk));
    const int64_t per_token = (int64_t)p.slots.d * p.per_head.d;
    p.group = (int)std::max<int64_t>(1, std::min<int64_t>({p.tokens / 1024, 2, p.rot ? TURN_ANGLES / (p.rot / 2) : 2}));
    const int64_t shares = std::min<int64_t>(ceil_div(p.group * per_token, TURN_THREADS), std::max<int64_t>(1, 2048 / ceil_div(p.tokens, p.group)));
    const dim3 grid((unsigned)ceil_div(p.tokens, p.group), (unsigned)std::min<int64_t>(shares, 65535));
    if (vec) hipLaunchKernelGGL((rotary_kernel<DT, E>), grid, dim3(TURN_THREADS), 0, st, p);
    else hipLaunchKernelGGL((rotary_kernel<DT, 1>), grid, dim3(TURN_THREADS), 0, st, p);
}
template <int DT>
static void launch_cache_append(TurnParams& p, hipStream_t st) {
    constexpr int E = CacheOrder<DT>::E;
    const bool vec = whole_pieces(p, E);
    const int pv = vec ? E : 1;
    p.per_head = divider((uint32_t)(p.rot / 2 / pv + (p.dp - p.rot) / pv));  // (keys are written to the end of their pad)
    p.slots = divider((uint32_t)(p.hk + (p.q ? p.hq : 0)));
    // two features of 16 bits a lane where they are 4 bytes together
    const bool two = vec && DT != BT_F32 && (p.v_token | p.v_head) % 2 == 0 && !misaligned(p.v, 4);
    p.by_dim = divider((uint32_t)(two ? p.dim / 2 : p.dim));
    p.units = (int)(p.starts ? p.tokens / E + 2 * (int64_t)p.n_seq : p.n_seq);
    const int64_t per_unit = (p.starts ? std::min<int64_t>(E, ceil_div(p.tokens, p.n_seq)) : 1) * (int64_t)p.slots.d * p.per_head.d + (int64_t)p.hk * p.by_dim.d;
    const int64_t shares = std::min<int64_t>(ceil_div(per_unit, TURN_THREADS), std::max<int64_t>(1, APPEND_BLOCKS / p.units));
    const int64_t clearing = p.starts && p.q ? ceil_div(clearing_blocks(p.tokens * p.hq * p.dim), shares) : 0;
    const dim3 grid((unsigned)(p.units + clearing), (unsigned)std::min<int64_t>(shares, 65535));
    if (two) hipLaunchKernelGGL((cache_append_kernel<DT, E, DT == BT_F32 ? 1 : 2>), grid, dim3(TURN_THREADS), 0, st, p);
    else if (vec) hipLaunchKernelGGL((cache_append_kernel<DT, E, 1>), grid, dim3(TURN_THREADS), 0, st, p);
    else hipLaunchKernelGGL((cache_append_kernel<DT, 1, 1>), grid, dim3(TURN_THREADS), 0, st, p);
}

}  // namespace bt

using namespace bt;

extern "C" int bt_rotary(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token, int64_t k_head, int dtype, const void* positions,
                         int positions_64, const void* inv_freq, int freq_64, int interleaved, float amplitude, int backward, int64_t tokens, int64_t heads,
                         int64_t kv_heads, int64_t head_dim, int64_t rotary_dim, void* q_out, void* k_out, void* stream) {
    const char* who = "bt_rotary";
    if (!k) kv_heads = 0;
    if (!q || !q_out || heads <= 0 || (k && (!k_out || kv_heads <= 0)) || !positions) {
        set_error("%s: null pointer", who);
        return BT_ERR_INVALID;
    }
    if (int rc = turn_checks(who, dtype, tokens, heads, kv_heads, head_dim, rotary_dim, freq_64, inv_freq)) return rc;
    TurnParams p = {};
    p.q = q, p.k = k, p.q_out = q_out, p.k_out = k ? k_out : nullptr;
    p.q_token = q_token, p.q_head = q_head, p.k_token = k ? k_token : 0, p.k_head = k ? k_head : 0;
    p.positions = positions, p.pos64 = positions_64 != 0, p.freq = inv_freq, p.freq64 = freq_64;
    p.tokens = tokens, p.hq = (int)heads, p.hk = (int)kv_heads, p.dim = (int)head_dim, p.rot = (int)rotary_dim, p.interleaved = interleaved != 0;
    p.amplitude = amplitude, p.sign = backward ? -1.0f : 1.0f;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == BT_F32) launch_rotary<BT_F32>(p, st);
    else if (dtype == BT_F16) launch_rotary<BT_F16>(p, st);
    else launch_rotary<BT_BF16>(p, st);
    return check_launch(who);
}

extern "C" int bt_cache_head_dim(int dtype, int64_t head_dim) { return known(dtype) && head_dim > 0 && head_dim <= 256 ? cache_head_dim(dtype, head_dim) : 0; }

extern "C" int bt_cache_append(const void* k, int64_t k_token, int64_t k_head, const void* v, int64_t v_token, int64_t v_head, const void* q, int64_t q_token,
                               int64_t q_head, int dtype, const void* inv_freq, int freq_64, int interleaved, float amplitude, int64_t first_position,
                               int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t rotary_dim, void* k_cache, void* v_cache,
                               int64_t pages, int64_t page_size, const int32_t* block_table, int64_t table_width, const int32_t* lengths,
                               const int32_t* q_starts, int64_t sequences, void* q_out, void* stream) {
    const char* who = "bt_cache_append";
    if (!q) heads = 0;
    if (!k || !v || !k_cache || !v_cache || !block_table || !lengths || kv_heads <= 0 || (q && (!q_out || heads <= 0))) {
        set_error("%s: null pointer or no heads", who);
        return BT_ERR_INVALID;
    }
    if (int rc = turn_checks(who, dtype, tokens, heads, kv_heads, head_dim, rotary_dim, freq_64, inv_freq)) return rc;
    if (head_dim > 256 || page_size < 32 || page_size > 65536 || (page_size & (page_size - 1)) || pages <= 0 || pages > 0x7fffffff || table_width <= 0 ||
        table_width * page_size > (1 << 30) || sequences <= 0 || sequences > (1 << 24) || (!q_starts && sequences != tokens)) {
        set_error("%s: head_dim at most 256, page_size a power of two from 32 on, up to 2^30 places of a sequence, one token a sequence without q_starts "
                  "(head_dim=%lld page_size=%lld width=%lld sequences=%lld tokens=%lld)",
                  who, (long long)head_dim, (long long)page_size, (long long)table_width, (long long)sequences, (long long)tokens);
        return BT_ERR_INVALID;
    }
    if (misaligned(k_cache, 16) || misaligned(v_cache, 16)) {
        set_error("%s: the cache has to be 16-byte aligned", who);
        return BT_ERR_INVALID;
    }
    TurnParams p = {};
    p.q = q, p.k = k, p.v = v, p.q_out = q ? q_out : nullptr;
    p.q_token = q ? q_token : 0, p.q_head = q ? q_head : 0, p.k_token = k_token, p.k_head = k_head, p.v_token = v_token, p.v_head = v_head;
    p.freq = inv_freq, p.freq64 = freq_64, p.k_cache = k_cache, p.v_cache = v_cache, p.table = block_table, p.lengths = lengths, p.starts = q_starts;
    p.first_position = first_position, p.tokens = tokens, p.hq = (int)heads, p.hk = (int)kv_heads, p.dim = (int)head_dim, p.rot = (int)rotary_dim;
    p.interleaved = interleaved != 0, p.n_seq = (int)sequences, p.width = (int)table_width, p.page_shift = __builtin_ctzll((unsigned long long)page_size);
    p.pages = (int)pages, p.dp = cache_head_dim(dtype, head_dim), p.amplitude = amplitude, p.sign = 1.0f;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == BT_F32) launch_cache_append<BT_F32>(p, st);
    else if (dtype == BT_F16) launch_cache_append<BT_F16>(p, st);
    else launch_cache_append<BT_BF16>(p, st);
    return check_launch(who);
}
