// Eight values of a row at a time, wherever the row starts: what the row kernels of add_norm.hip and gated.hip move.
#pragma once
#include "row_math.h"

namespace bt {

// Eight values as they lie in memory, from any element boundary on (one or two 16-byte loads).  Kept like this until they are used, so
// that a kernel's loads all go out before the first wait.
template <int DT>
struct Raw8 {
    u32x4 d[DT == BT_F32 ? 2 : 1];
};
template <int DT>
__device__ __forceinline__ Raw8<DT> load_raw8(const void* base, int64_t idx) {
    Raw8<DT> r;
    if constexpr (DT == BT_F32) {
        r.d[0] = *(const u32x4_a4*)((const float*)base + idx);
        r.d[1] = *(const u32x4_a4*)((const float*)base + idx + 4);
    } else {
        r.d[0] = *(const u32x4_a2*)((const uint16_t*)base + idx);
    }
    return r;
}
template <int DT>
__device__ __forceinline__ void widen8(const Raw8<DT>& r, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
        if constexpr (DT == BT_F32) {
            const uint32_t u = r.d[e >> 2][e & 3];
            v[e] = __builtin_bit_cast(float, u);
        } else {
            const uint16_t h = (uint16_t)(r.d[0][e >> 1] >> (16 * (e & 1)));
            v[e] = (DT == BT_F16) ? f16_bits_to_f32(h) : bf16_bits_to_f32(h);
        }
    }
}
template <int DT>
__device__ __forceinline__ void store8u(void* base, int64_t idx, const float (&v)[8]) {
    if constexpr (DT == BT_F32) {
        u32x4_a4 a, b;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            a[e] = __builtin_bit_cast(uint32_t, v[e]);
            b[e] = __builtin_bit_cast(uint32_t, v[4 + e]);
        }
        __builtin_nontemporal_store(a, (u32x4_a4*)((float*)base + idx));
        __builtin_nontemporal_store(b, (u32x4_a4*)((float*)base + idx + 4));
    } else {
        u32x4_a2 d;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t lo = (DT == BT_F16) ? f32_to_f16_bits(v[2 * e]) : f32_to_bf16_bits(v[2 * e]);
            const uint32_t hi = (DT == BT_F16) ? f32_to_f16_bits(v[2 * e + 1]) : f32_to_bf16_bits(v[2 * e + 1]);
            d[e] = lo | (hi << 16);
        }
        __builtin_nontemporal_store(d, (u32x4_a2*)((uint16_t*)base + idx));
    }
}

// A row of K >= 8 values in pieces of eight.  The piece from k on is loaded from min(k, K - 8): every load is inside the row and none
// waits for a branch.  widen_piece() puts its values in their places, with zeros where the row has ended.  RAG: K is not a multiple of 8
// (otherwise a piece is whole, or none of it exists).
__device__ __forceinline__ int piece_at(int k, int K) { return k < K - 8 ? k : K - 8; }
template <int DT, bool RAG>
__device__ __forceinline__ void widen_piece(const Raw8<DT>& r, int k, int K, float (&v)[8]) {
    widen8<DT>(r, v);
    const int d = k - piece_at(k, K);  // how far ahead of its place the piece was loaded
    if constexpr (RAG) {
        const bool one = d & 1, two = d & 2, four = d & 4, none = d >= 8;
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = one ? (e + 1 < 8 ? v[e + 1] : 0.0f) : v[e];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = two ? (e + 2 < 8 ? v[e + 2] : 0.0f) : v[e];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = none ? 0.0f : four ? (e + 4 < 8 ? v[e + 4] : 0.0f) : v[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = d == 0 ? v[e] : 0.0f;
    }
}
// Values k .. k + 7 of the row that starts at element `row` of base: those that exist.
template <int DT, bool RAG>
__device__ __forceinline__ void store_piece(void* base, int64_t row, int k, int K, const float (&v)[8]) {
    if (k + 8 <= K) {
        store8u<DT>(base, row + k, v);
    } else if (RAG && k < K) {  // (at most one lane of a row)
#pragma unroll
        for (int e = 0; e < 7; e++)
            if (k + e < K) store_elem<DT>(base, row + k + e, v[e]);
    }
}
__device__ __forceinline__ float wave_sum_f32(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    return v;
}

// out[k] = sum of parts[0 .. n-1][k], in an order of its own that depends on n alone (row_vec.h's users: sums over many rows)
int launch_column_sum(const float* parts, int64_t n, int64_t K, void* out, int out_dtype, hipStream_t st, const char* who);

}  // namespace bt
