// The paged cache of keys and values: its layout in memory and what its kernels share (rotary.hip, attention.hip).
//
// A cache is two arrays [pages][heads][places of a page][Dp]: Dp is the head dimension D rounded up to 64 bytes.  The places of a head's
// page are kept in tiles of TK = 4 E (E elements in 16 bytes: 8 of 16 bits, 4 of 32), each in the order in which a wave hands it to the
// matrix cores, so that every load of the attention is 1 KiB in a row, straight into registers or LDS, and no value is moved again:
//   keys    [Dp / 4E][E / 4][g 4][m 16][E features]:  feature = 4E c + E g + e,  place = E (m / 4) + 4 t + m % 4
//   values  [Dp / 16][g 4][m 16][E places]:           feature = 16 b + m,        place = E g + e
// Features of a key behind D are zero, whatever the array held before.
// The scores of keys in that order leave the matrix cores with lane (m, g) holding places E g .. E g + E - 1 of row m, which is the operand
// that the second product takes beside the values.
#pragma once

#include "bt_common.h"

namespace bt {

template <int DT>
struct CacheOrder {
    static constexpr int SIZE = DT == BT_F32 ? 4 : 2;
    static constexpr int E = 16 / SIZE;
    static constexpr int TK = 4 * E;
    // Elements from the start of a head's page, whose pad is dp features wide
    static __device__ __forceinline__ int key(int place, int feature, int dp) {
        const int r = place % TK, m = r / E * 4 + r % 4, t = r % E / 4;
        const int c = feature / TK, g = feature % TK / E;
        return place / TK * (TK * dp) + (((c * (E / 4) + t) * 4 + g) * 16 + m) * E + feature % E;
    }
    static __device__ __forceinline__ int value(int place, int feature, int dp) {
        const int r = place % TK;
        return place / TK * (TK * dp) + ((feature / 16 * 4 + r / E) * 16 + feature % 16) * E + r % E;
    }
};
static inline int cache_head_dim(int dt, int64_t d) {
    const int unit = 64 / dtype_size(dt);
    return (int)(ceil_div(d, unit) * unit);
}

// Workgroups that clear the rows behind the last sequence, of so many elements if there is no sequence at all (8128 of 8192 tokens of 32 heads of
// 128: the attention takes 67 us, the append 19; with one workgroup for all of them 3.3 and 4.1 ms)
static inline int64_t clearing_blocks(int64_t elements) {
    const int64_t n = ceil_div(elements, 8192);
    return n < 1 ? 1 : n > 256 ? 256 : n;
}

// Which sequence token t belongs to: starts[s] <= t < starts[s + 1], or -1.  All lanes of a wave; one load for 64 sequences.
__device__ __forceinline__ int owner_of(const int32_t* starts, int n_seq, int64_t t) {
    const int lane = threadIdx.x & 63;
    int found = 0;
    for (int s0 = 0; s0 < n_seq; s0 += 64) {
        const int s = s0 + lane;
        const uint64_t hit = __ballot(s < n_seq && starts[s < n_seq ? s : 0] <= t);
        found += __popcll(hit);
        if (hit != ~0ull) break;
    }
    return found - 1 >= 0 && t < starts[found] ? found - 1 : -1;
}

// idx / d for idx < 2^32 / d, with m = ceil(2^32 / d) (0 for d = 1)
struct Divider {
    uint32_t m, d;
};
static inline Divider divider(uint32_t d) { return {d > 1 ? (uint32_t)(((1ull << 32) + d - 1) / d) : 0u, d}; }
__device__ __forceinline__ uint32_t divide(uint32_t idx, const Divider& by) { return by.m ? __umulhi(idx, by.m) : idx; }

}  // namespace bt
