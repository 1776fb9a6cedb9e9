// The gated pair of a feed-forward block in training, for gfx950:
//
//   g = a_g (x T_g^T) + b_g,   u = a_u (x T_u^T) + b_u,   h = silu(g) u = g u / (1 + exp(-g))
//
// with T = ternary(W), a = the rows' absolute maxima of two full-precision masters W [F, K] (straight-through gradient, as
// bittorch/nn/ternary_linear_cuda.py:73-111; block structure of the JS runtime, js/src/models/TernaryTransformer.ts:366-423).
// Its gradient, with sig = 1 / (1 + exp(-g)) and incoming dh:
//
//   dg = dh u sig (1 + g (1 - sig)),  du = dh g sig
//   dx = (a_g dg) T_g + (a_u du) T_u,   dW_g = (a_g dg)^T x,  db_g = sum_rows dg,   likewise for up
//
// 16-bit rows: one product forms both projections and h in its output stage (gemm_f16.hip, OUT_GATED) on the tiled copy in pair
// order.  One pass (gated_grad_kernel) makes G = [a_g dg | a_u du] of dh and the kept projections, rounded once to 16 bits as an operand
// of the matrix cores; it serves both products behind it: dx = G [T_g; T_u] on a second tiled copy of the codes, in which the contraction
// runs over the output features, by the forward's kernel, and dW = G^T x by the weight gradient's (grad_w16.hip).  For bf16 a times
// dg, not dg, is what is rounded, so that neither product has a scale for each feature.  fp16 has no range for a (0.01 where dg is 1e-4 would
// leave 4 bits of it), and none for the ratio of two features' a either (one entry of 0.5 among masters of 0.003 is 40 of them): there a is
// taken apart feature by feature (gated_range_kernel), a = m 2^f with m in [1/2, 1), and G = [m_g dg | m_u du] has fp16's full
// precision down to dg of 2^-13.  dW's rows are multiplied by their 2^f in fp32, as they are stored; in dx's product, which sums over the features, 2^f goes with
// the codes as they are decoded, over the power of two above all of them, which is the output's scale.
// fp32 rows: the same steps on the fp32 kernels and the same copies, the projections stored in fp32 and h by the SwiGLU row kernel.  (On the
// packed bytes as rows the fp32 products take longer: 4096 x 4096 x 768 forward 74 us, 68 on the copy, its transpose 89 and 77.)
//
// Features are padded to Fp = F rounded up to 16 where the matrix cores read them: zero codes, scales and biases, zero columns of G.
#include "row_vec.h"

namespace bt {

int launch_gemm_f16_gated(int mode, const void* X, const uint8_t* W_tiled, const Epilogue& epi, void* Y, uint32_t* pre, int64_t H, int64_t M,
                          int64_t N, int64_t K, hipStream_t st);
int launch_gemm_f16_factors(const void* X, const uint8_t* W_tiled, const uint16_t* factors, const float* scale, void* Y, int64_t M, int64_t N, int64_t K,
                            void* workspace, hipStream_t st);
size_t gemm_f16_factors_workspace_bytes(int64_t M, int64_t N, int64_t K);
int launch_pad_rows(const void* X, int64_t B, int64_t K, void* P, hipStream_t st);
float quantize_clamp_min(int w_dtype);
bool gemm_f16_supported(int64_t N, int64_t K, const void* X, const void* W_T, const void* Y, bool tiled);

static int64_t padded(int64_t F) { return ceil_div(F, 16) * 16; }

// ---- the two masters as one operand ---------------------------------------------------------------------------------------

struct GatedWeightsParams {
    const uint8_t* W[2];      // gate, up: packed [ceil(K / 4), F]
    const float* a[2];        // their scales: F entries or one
    const void* b[2];         // biases or null
    int bias_dtype, one_scale;
    int64_t F, Fp, K, Kb;
    uint8_t* pairs;           // forward: tiled copy in pair order of [gate | up], 2 Fp columns
    uint8_t* back;            // backward: tiled copy of the transpose: K columns, contraction over 2 Fp
    float* scale;             // [2 Fp + 1], the last one 1
    float* bias;              // [2 Fp] or null
    uint32_t n_pairs, n_back;          // workgroups of each part, in this order; behind them those of the vectors
    uint32_t steps, back_steps;        // 64-wide steps of the two tiled copies
};

// 16 packed bytes n .. n + 15 of a row of F, zeros past its end
__device__ __forceinline__ u32x4 codes16(const uint8_t* row, int64_t n, int64_t F) {
    if (n + 16 <= F) return *(const u32x4_a1*)(row + n);
    u32x4 d = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < 16; e++)
        if (n + e < F) d[e >> 2] |= (uint32_t)row[n + e] << (8 * (e & 3));
    return d;
}

// the codes at bits 0, 8, 16, 24 as one byte
__device__ __forceinline__ uint32_t byte_of_codes(uint32_t t) {
    const uint32_t x = t & 0x03030303u, y = x | x >> 6;
    return (y | y >> 12) & 0xffu;
}

// From packed bytes.  Bound by them, read once for each copy and written once; all parts in one launch.
__global__ __launch_bounds__(256) void gated_weights_kernel(GatedWeightsParams p) {
    constexpr int PITCH = 256 + 16;
    __shared__ __attribute__((aligned(16))) uint8_t block[16 * PITCH];
    uint32_t wg = blockIdx.x;
    const int tid = threadIdx.x;
    if (wg < p.n_pairs) {
        // 16 packed rows (a step) of 256 features of one half, through LDS: retile_kernel with the order of the pairs
        const uint32_t steps = p.steps, per_half = p.n_pairs / 2;
        const int half = wg >= per_half;
        wg -= half ? per_half : 0u;
        const int64_t s = wg % steps, n0 = (int64_t)(wg / steps) * 256;
        {
            const int r = tid >> 4, c = 16 * (tid & 15);
            const int64_t kb = 16 * s + r;
            u32x4 d = {0u, 0u, 0u, 0u};
            if (kb < p.Kb) d = codes16(p.W[half] + kb * p.F, n0 + c, p.F);
            *(u32x4*)(block + r * PITCH + c) = d;
        }
        __syncthreads();
        const int tile = tid >> 4, g = (tid >> 2) & 3, j = 4 * (tid & 3);
        const int64_t t = (n0 >> 4) + tile;
        if (16 * t >= p.Fp) return;
        uint32_t row[4], out[4];
#pragma unroll
        for (int r = 0; r < 4; r++) row[r] = *(const uint32_t*)(block + (4 * g + r) * PITCH + 16 * tile + j);
        transpose4x4_bytes(row[0], row[1], row[2], row[3], out);
        ((uint4*)p.pairs)[((2 * t + half) * (int64_t)steps + s) * 16 + 4 * g + (j >> 2)] = make_uint4(out[0], out[1], out[2], out[3]);
        return;
    }
    wg -= p.n_pairs;
    if (wg < p.n_back) {
        // A thread takes the codes of 16 features at four k: byte k / 4 of the packed rows, and turns them into four dwords of the copy,
        // column k + c with the codes of feature n + 4 r + i at bits 8 r + 2 i.  A wave: the four bytes of a tile's 16 columns, four
        // groups of 16 features, four steps: 256 consecutive bytes of each of four rows in, 1 KiB out.
        const uint32_t per_tile = (p.back_steps + 15) / 16;
        const int64_t S = p.back_steps, t = wg / per_tile, s = (int64_t)(wg % per_tile) * 16 + (tid >> 4);
        const int g = (tid >> 2) & 3, q = tid & 3;
        if (s >= S) return;
        const int64_t kb = 4 * t + q, n = 64 * s + 16 * g;
        u32x4 d = {0u, 0u, 0u, 0u};
        if (kb < p.Kb && n < 2 * p.Fp) {
            const int half = n >= p.Fp;
            d = codes16(p.W[half] + kb * p.F, n - (half ? p.Fp : 0), p.F);
        }
        uint32_t out[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int c = 0; c < 4; c++) out[c] |= byte_of_codes(d[r] >> (2 * c)) << (8 * r);
        ((uint4*)p.back)[(t * S + s) * 16 + 4 * g + q] = make_uint4(out[0], out[1], out[2], out[3]);
        return;
    }
    const int64_t n = (int64_t)(wg - p.n_back) * 256 + tid;
    if (n < 2 * p.Fp) {
        const int half = n >= p.Fp;
        const int64_t f = n - (half ? p.Fp : 0);
        p.scale[n] = f < p.F ? p.a[half][p.one_scale ? 0 : f] : 0.0f;
        if (p.bias) p.bias[n] = f < p.F && p.b[half] ? load_elem_rt(p.b[half], p.bias_dtype, f) : 0.0f;
    } else if (n == 2 * p.Fp) {
        p.scale[n] = 1.0f;
    }
}

struct GatedQuantizeParams {
    const void* W[2];         // masters gate, up [F, K]
    const void* b[2];
    int bias_dtype;
    float tf, clamp_min;
    int F, K, Fp;             // as above
    int tiles, per_xcd;       // of 16 features, both halves
    uint8_t *pairs, *back;
    float *scale, *bias;
    uint32_t steps, back_steps;
};

// Masters of a DT (BT_F32_AS_F16: fp32, rounded to fp16 as they are read)
constexpr int master_storage(int dt) { return dt == BT_F32_AS_F16 ? BT_F32 : dt; }

// The same from the masters in one pass: a workgroup takes the 16 features of a tile of the copies.  A wave keeps a feature's row in
// registers (ITERS pieces of eight values a lane, K <= 512 ITERS), reduces its absolute maximum, and puts the codes of four k to a byte into
// LDS, from where they leave in each layout: the pairs' tile is one run of memory, its dwords are LDS's; a thread turns the codes of four
// k into 16 bytes of the transpose.  The quantizer's arithmetic is that of quantize_pack.hip, on the same values.  Bound by the masters,
// read once: 2 x 6912 x 2560 bf16 (71 MB) takes 20 us, two passes of the quantizer and the copy of their bytes 34.
template <int DT, int ITERS, bool RAG>
__global__ __launch_bounds__(512) void gated_quantize_kernel(GatedQuantizeParams p) {
    constexpr int ST = master_storage(DT), PITCH = ITERS * 128 + 4, RPW = 2;
    constexpr bool BOTH = ITERS * (ST == BT_F32 ? 2 : 1) <= 10;  // both rows of a wave in registers at once
    __shared__ __attribute__((aligned(16))) uint8_t codes[16 * PITCH];
    const int lin = (int)(blockIdx.x & 7) * p.per_xcd + (int)(blockIdx.x >> 3);
    if (lin >= p.tiles) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per_half = p.tiles / 2, half = lin >= per_half, tile = lin - half * per_half, f0 = 16 * tile;
    const int K = p.K;
    const void* const W = p.W[half];
    Raw8<ST> in[BOTH ? RPW : 1][ITERS];
    auto load = [&](int r, Raw8<ST> (&to)[ITERS]) {
        const int f = f0 + RPW * wave + r;
        const int64_t row = (int64_t)(f < p.F ? f : p.F - 1) * K;  // (a feature past the last one: that row again, its codes are not kept)
#pragma unroll
        for (int i = 0; i < ITERS; i++) to[i] = load_raw8<ST>(W, row + piece_at((i * 64 + lane) * 8, K));
    };
    if constexpr (BOTH) {
#pragma unroll
        for (int r = 0; r < RPW; r++) load(r, in[r]);
    }
#pragma unroll
    for (int r = 0; r < RPW; r++) {
        const int f = f0 + RPW * wave + r;
        const bool there = f < p.F;  // (uniform)
        if constexpr (!BOTH) load(r, in[0]);
        Raw8<ST> (&row)[ITERS] = in[BOTH ? r : 0];
        auto values = [&](int i, float (&v)[8]) {
            widen_piece<ST, RAG>(row[i], (i * 64 + lane) * 8, K, v);
            if constexpr (DT == BT_F32_AS_F16) {
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = round_to_dtype(v[e], BT_F16);
            }
        };
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < ITERS; i++) {
            float v[8];
            values(i, v);
#pragma unroll
            for (int e = 0; e < 8; e++) amax = fmaxf(amax, fabsf(v[e]));
        }
        const float s = fmaxf(wave_max(amax), p.clamp_min);
        const float thr = round_to_dtype(__fmul_rn(p.tf, s), DT == BT_F32_AS_F16 ? BT_F16 : DT);
        // (widened again, not kept in fp32 from above: half the registers)
#pragma unroll
        for (int i = 0; i < ITERS; i++)
#pragma unroll
            for (int q = 0; q < (ST == BT_F32 ? 2 : 1); q++) asm volatile("" : "+v"(row[i].d[q]));
#pragma unroll
        for (int i = 0; i < ITERS; i++) {
            float v[8];
            values(i, v);
            uint32_t c = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) c |= (fabsf(v[e]) > thr ? (v[e] < 0.0f ? 2u : 1u) : 0u) << (2 * e);
            const int k = (i * 64 + lane) * 8;  // (zeros behind the row's end)
            c = !there || k >= K ? 0u : RAG && k + 8 > K ? c & ((1u << (2 * (K - k))) - 1u) : c;
            *(uint16_t*)(codes + (RPW * wave + r) * PITCH + (i * 64 + lane) * 2) = (uint16_t)c;
        }
        if (lane == 0 && f < p.Fp) {
            const int at = half * p.Fp + f;
            p.scale[at] = there ? s : 0.0f;
            if (p.bias) p.bias[at] = there && p.b[half] ? load_elem_rt(p.b[half], p.bias_dtype, f) : 0.0f;
            if (at == 0) p.scale[2 * p.Fp] = 1.0f;
        }
    }
    __syncthreads();
    uint32_t* const pairs = (uint32_t*)p.pairs + (int64_t)(2 * tile + half) * p.steps * 64;
    for (uint32_t i = tid; i < p.steps * 64; i += 512) pairs[i] = *(const uint32_t*)(codes + (i & 15) * PITCH + 16 * (i >> 6) + 4 * ((i >> 4) & 3));
    if (!p.back) return;
    const uint32_t n0 = (uint32_t)(half * p.Fp + f0);
    for (int kb = tid; 4 * kb < K; kb += 512) {  // (the four threads of 16 k read the same dwords)
        uint32_t t[4];  // the bytes kb of features 4 r .. + 3
#pragma unroll
        for (int r = 0; r < 4; r++) {
            uint32_t d[4];
#pragma unroll
            for (int i = 0; i < 4; i++) d[i] = *(const uint32_t*)(codes + (4 * r + i) * PITCH + (kb & ~3)) >> (8 * (kb & 3)) & 0xffu;
            t[r] = d[0] | d[1] << 8 | d[2] << 16 | d[3] << 24;
        }
        uint4* const out = (uint4*)p.back + ((int64_t)(kb >> 2) * p.back_steps + (n0 >> 6)) * 16 + 4 * ((n0 >> 4) & 3) + (kb & 3);
        uint32_t o[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int c = 0; c < 4; c++) o[c] |= byte_of_codes(t[r] >> (2 * c)) << (8 * r);
        *out = make_uint4(o[0], o[1], o[2], o[3]);
    }
    // the bytes of the last column tile behind K
    const uint32_t kbs = (uint32_t)(K + 15) / 16 * 4, kb_end = (uint32_t)(K + 3) / 4;
    if (kb_end + tid < kbs) {
        const uint32_t kb = kb_end + tid;
        ((uint4*)p.back)[((int64_t)(kb >> 2) * p.back_steps + (n0 >> 6)) * 16 + 4 * ((n0 >> 4) & 3) + (kb & 3)] = make_uint4(0u, 0u, 0u, 0u);
    }
    // the features of the last step past both halves, from the workgroup of the last tile
    if (lin == p.tiles - 1) {
        const uint32_t first = (n0 >> 4) + 1, groups = 4 * p.back_steps - first;
        for (uint32_t i = tid; i < kbs * groups; i += 512) {
            const uint32_t kb = i % kbs, g = first + i / kbs;
            ((uint4*)p.back)[((int64_t)(kb >> 2) * p.back_steps + (g >> 2)) * 16 + 4 * (g & 3) + (kb & 3)] = make_uint4(0u, 0u, 0u, 0u);
        }
    }
}

template <int DT>
static void launch_gated_quantize(const GatedQuantizeParams& p, hipStream_t st) {
    const dim3 grid((unsigned)(8 * p.per_xcd)), block(512);
#define BT_GQ(IT)                                                                                          \
    if (p.K <= 512 * IT) {                                                                                 \
        if (p.K % 8 == 0) hipLaunchKernelGGL((gated_quantize_kernel<DT, IT, false>), grid, block, 0, st, p); \
        else hipLaunchKernelGGL((gated_quantize_kernel<DT, IT, true>), grid, block, 0, st, p);              \
        return;                                                                                            \
    }
    BT_GQ(1) BT_GQ(2) BT_GQ(3) BT_GQ(5) BT_GQ(8)
#undef BT_GQ
    hipLaunchKernelGGL((gated_quantize_kernel<DT, 16, false>), grid, block, 0, st, p);
}
// Rows that a wave holds, with a scale each; the others are quantized by bt_quantize_pack and their bytes put in place
static bool gated_quantizes(int64_t K, bool per_channel) { return per_channel && K >= 8 && K <= (K % 8 == 0 ? 8192 : 4096); }

// scale[n] = the least power of two 2^e with scale[i] < 2^e for all i < n, within 2^-24 .. 2^15.  With `split` (bt_gated_split) each scale
// is also taken apart, into a power of two of its own 2^f, scale[i] / 2^f in [1/2, 1), and what is left.  One workgroup: its time is its
// launch.  f stays within 24 below and 15 above e, where 2^(f - e) is an fp16 number (a power of two among the subnormal ones too); beyond
// that what is left is smaller than a half, or not below 1.
__global__ __launch_bounds__(1024) void gated_range_kernel(float* scale, int n, float* split) {
    __shared__ float part[16];
    float m = 0.0f;
#pragma unroll 8
    for (int i = threadIdx.x; i < n; i += 1024) m = fmaxf(m, scale[i]);
    m = wave_max(m);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; i++) m = fmaxf(m, part[i]);
    // the exponent above v's
    auto above = [](float v) { return (int)(__builtin_bit_cast(uint32_t, v) >> 23) - 126; };
    auto power = [](int e) { return __builtin_bit_cast(float, (uint32_t)(127 + e) << 23); };
    const int e = max(-24, min(15, above(m)));
    if (threadIdx.x == 0) scale[n] = power(e);
    if (!split) return;
    float* const rows = split + n + 16;
    uint16_t* const factors = (uint16_t*)(split + 2 * n + 16);
#pragma unroll 8
    for (int i = threadIdx.x; i < n; i += 1024) {
        const int f = max(e - 24, min(e + 15, above(scale[i]))), d = f - e;
        split[i] = scale[i] * power(-f);
        rows[i] = power(f);
        factors[i] = (uint16_t)(d >= -14 ? (15 + d) << 10 : 1 << (24 + d));
    }
    if ((n & 63) && threadIdx.x < 32) factors[n + threadIdx.x] = 0;  // (n is a multiple of 32)
    if (threadIdx.x == 0) {
        split[n] = 1.0f;
        split[n + 1] = power(e);
    }
}

// ---- one row on the masters, without a copy of them -------------------------------------------------------------------------

struct GatedMastersParams {
    const void* W[2];         // masters gate, up [F, K]
    const void* b[2];
    const void* X;            // [K]
    void* H;                  // [F]
    int bias_dtype, x_dtype;
    float tf, clamp_min;
    int F, K;
};

template <int XT, bool RAG, int ITERS>
__device__ __forceinline__ void load_row(const void* X, int lane, int K, float (&x)[ITERS][8]) {
    Raw8<XT> in[ITERS];
#pragma unroll
    for (int i = 0; i < ITERS; i++) in[i] = load_raw8<XT>(X, piece_at((i * 64 + lane) * 8, K));
#pragma unroll
    for (int i = 0; i < ITERS; i++) widen_piece<XT, RAG>(in[i], (i * 64 + lane) * 8, K, x[i]);
}

// Forward alone: the masters are read once, ternarised in registers and multiplied there.  A wave takes one feature at a time, the gate's
// row and up's (as gated_quantize_kernel holds them), the next one's on their way; a lane's columns are the same for every feature, so
// the activations stay in its registers.  A product is the activation or its negative or nothing, a sum 8 ITERS terms in a lane and a tree
// over the lanes, in fp32.  Bound by the masters' bytes, and by whole features for the waves of the chip: 2 x 6912 x 2560 bf16 (71 MB), 3.4
// features a wave, 18.7 us, 34 through the copies and the tiled product; 2 x 11008 x 4096 bf16 43 and 63, fp32 masters of 2 x 6912 x 2560
// 31 and 45.  (More rows share the masters' pass there: 34 us up to 32 of them.)
template <int DT, int ITERS, bool RAG>
__global__ __launch_bounds__(512) void gated_masters_kernel(GatedMastersParams p) {
    constexpr int ST = master_storage(DT);
    constexpr bool AHEAD = ITERS * (ST == BT_F32 ? 2 : 1) <= 10;  // (registers for a second pair of rows)
    const int lane = threadIdx.x & 63, first = (int)blockIdx.x * 8 + (int)(threadIdx.x >> 6), step = (int)gridDim.x * 8;
    const int K = p.K, F = p.F;
    struct Rows {
        Raw8<ST> d[2][ITERS];
    };
    auto load = [&](int f, Rows& to) {
        const int64_t row = (int64_t)(f < F ? f : F - 1) * K;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < ITERS; i++) to.d[h][i] = load_raw8<ST>(p.W[h], row + piece_at((i * 64 + lane) * 8, K));
    };
    Rows in, next;
    load(first, AHEAD ? next : in);
    float x[ITERS][8];
    if (p.x_dtype == BT_F32) load_row<BT_F32, RAG>(p.X, lane, K, x);
    else if (p.x_dtype == BT_F16) load_row<BT_F16, RAG>(p.X, lane, K, x);
    else load_row<BT_BF16, RAG>(p.X, lane, K, x);
    for (int f = first; f < F; f += step) {
        if constexpr (AHEAD) {
            in = next;
            load(f + step, next);
        }
        auto values = [&](int h, int i, float (&v)[8]) {
            widen_piece<ST, RAG>(in.d[h][i], (i * 64 + lane) * 8, K, v);
            if constexpr (DT == BT_F32_AS_F16) {
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = round_to_dtype(v[e], BT_F16);
            }
        };
        float y[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float amax = 0.0f, sum = 0.0f;
#pragma unroll
            for (int i = 0; i < ITERS; i++) {
                float v[8];
                values(h, i, v);
#pragma unroll
                for (int e = 0; e < 8; e++) amax = fmaxf(amax, fabsf(v[e]));
            }
            const float s = fmaxf(wave_max(amax), p.clamp_min);
            const float thr = round_to_dtype(__fmul_rn(p.tf, s), DT == BT_F32_AS_F16 ? BT_F16 : DT);
            // (widened again, not kept in fp32 from above: half the registers)
#pragma unroll
            for (int i = 0; i < ITERS; i++)
#pragma unroll
                for (int q = 0; q < (ST == BT_F32 ? 2 : 1); q++) asm volatile("" : "+v"(in.d[h][i].d[q]));
#pragma unroll
            for (int i = 0; i < ITERS; i++) {
                float v[8];
                values(h, i, v);
#pragma unroll
                for (int e = 0; e < 8; e++) sum = __builtin_fmaf(x[i][e], fabsf(v[e]) > thr ? copysignf(1.0f, v[e]) : 0.0f, sum);
            }
            y[h] = epi_float(wave_sum_f32(sum), s, p.b[h] ? load_elem_rt(p.b[h], p.bias_dtype, f) : 0.0f);
        }
        if constexpr (!AHEAD) load(f + step, in);
        if (lane == 0) {
            if (p.x_dtype == BT_F32) store_elem<BT_F32>(p.H, f, __fdiv_rn(y[0], __fadd_rn(1.0f, exp_fixed(-y[0]))) * y[1]);
            else if (p.x_dtype == BT_F16) store_elem<BT_F16>(p.H, f, y[0] * sigmoid_fast(y[0]) * y[1]);
            else store_elem<BT_BF16>(p.H, f, y[0] * sigmoid_fast(y[0]) * y[1]);
        }
    }
}

template <int DT, int ITERS>
static void launch_gated_masters_cfg(const GatedMastersParams& p, hipStream_t st, dim3 grid) {
    if (p.K % 8 == 0) hipLaunchKernelGGL((gated_masters_kernel<DT, ITERS, false>), grid, dim3(512), 0, st, p);
    else hipLaunchKernelGGL((gated_masters_kernel<DT, ITERS, true>), grid, dim3(512), 0, st, p);
}
template <int DT>
static void launch_gated_masters(const GatedMastersParams& p, hipStream_t st) {
    const dim3 grid((unsigned)std::min<int64_t>(ceil_div(p.F, 8), gemm_compute_units()));
    if (p.K <= 1024) launch_gated_masters_cfg<DT, 2>(p, st, grid);
    else if (p.K <= 2560) launch_gated_masters_cfg<DT, 5>(p, st, grid);
    else if constexpr (master_storage(DT) != BT_F32) hipLaunchKernelGGL((gated_masters_kernel<DT, 8, false>), grid, dim3(512), 0, st, p);
}
// Rows of masters that a wave holds twice beside the activations, with a scale each
static bool masters_serve(int64_t B, int64_t K, int w_dtype, bool per_channel) {
    return per_channel && B == 1 && K >= 8 && (K <= 2560 || (K <= 4096 && K % 8 == 0 && (w_dtype == BT_F16 || w_dtype == BT_BF16)));
}

// ---- gradient of silu(g) u ------------------------------------------------------------------------------------------------

struct GatedGradParams {
    const void* dH;       // [B, F]
    const void* pre;      // 16-bit rows: [B, 3 Fp / 2] dwords, column pairs of gate and up in turn in 24 bits; fp32 rows: [B, 2 Fp], gate | up
    const float* scale;   // [2 Fp + 1]: what dg | du are multiplied by, over the last one
    void* G;              // [B, 2 Fp]
    float* parts;         // [gridDim.y, 2 F] sums of dg | du, or null
    int64_t B, rows;      // rows: of a workgroup
    int F, Fp;
};

// dh, g, u -> dg, du
template <int DT>
__device__ __forceinline__ void gated_grad_value(float dh, float g, float u, float& dg, float& du) {
    const float sig = DT == BT_F32 ? __fdiv_rn(1.0f, __fadd_rn(1.0f, exp_fixed(-g))) : sigmoid_fast(g);
    dg = dh * u * (sig * __builtin_fmaf(g, 1.0f - sig, 1.0f));
    du = dh * (g * sig);
}

// A thread takes eight features of a run of rows; the biases' sums stay in its registers.  Bound by memory: dh and both projections in, G
// out once.  RAG: F is not a multiple of 8.
template <int DT, bool RAG>
__global__ __launch_bounds__(256) void gated_grad_kernel(GatedGradParams p) {
    const int k = ((int)blockIdx.x * 256 + (int)threadIdx.x) * 8, F = p.F, Fp = p.Fp;
    if (k >= Fp) return;
    const int64_t first = (int64_t)blockIdx.y * p.rows, last = std::min(first + p.rows, p.B);
    float ag[8], au[8], bg[8], bu[8];
    const float unit = __fdiv_rn(1.0f, p.scale[2 * Fp]);
#pragma unroll
    for (int e = 0; e < 8; e++) {
        ag[e] = p.scale[k + e] * unit;
        au[e] = p.scale[Fp + k + e] * unit;
        bg[e] = bu[e] = 0.0f;
    }
#pragma unroll 2
    for (int64_t row = first; row < last; row++) {
        float dh[8], g[8], u[8];
        const Raw8<DT> dh_in = load_raw8<DT>(p.dH, row * F + piece_at(k, F));
        if constexpr (DT == BT_F32) {
            widen8<DT>(load_raw8<DT>(p.pre, row * 2 * Fp + k), g);
            widen8<DT>(load_raw8<DT>(p.pre, row * 2 * Fp + Fp + k), u);
        } else {
            const u32x4* at = (const u32x4*)((const uint32_t*)p.pre + (row * Fp + k) / 2 * 3);
            const u32x4 a = at[0], b = at[1], c = at[2];
            const uint32_t d[12] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3], c[0], c[1], c[2], c[3]};
#pragma unroll
            for (int q = 0; q < 4; q++) {
                float v[4];
                unpack24(d[3 * q], d[3 * q + 1], d[3 * q + 2], v);
                g[2 * q] = v[0]; g[2 * q + 1] = v[1];
                u[2 * q] = v[2]; u[2 * q + 1] = v[3];
            }
        }
        widen_piece<DT, RAG>(dh_in, k, F, dh);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            float dg, du;
            gated_grad_value<DT>(dh[e], g[e], u[e], dg, du);
            bg[e] += dg;
            bu[e] += du;
            g[e] = dg * ag[e];
            u[e] = du * au[e];
        }
        store8u<DT>(p.G, row * 2 * Fp + k, g);
        store8u<DT>(p.G, row * 2 * Fp + Fp + k, u);
    }
    if (!p.parts) return;
    float* out = p.parts + (int64_t)blockIdx.y * 2 * F;
    store_piece<BT_F32, RAG>(out, 0, k, F, bg);
    store_piece<BT_F32, RAG>(out, F, k, F, bu);
}

// F < 8: element by element
template <int DT>
__global__ __launch_bounds__(64) void gated_grad_narrow_kernel(GatedGradParams p) {
    const int k = threadIdx.x, F = p.F, Fp = p.Fp;
    if (k >= Fp) return;
    const int64_t first = (int64_t)blockIdx.y * p.rows, last = std::min(first + p.rows, p.B);
    float bg = 0.0f, bu = 0.0f;
    const float unit = __fdiv_rn(1.0f, p.scale[2 * Fp]);
    for (int64_t row = first; row < last; row++) {
        float dg = 0.0f, du = 0.0f;
        if (k < F) {
            float v[4];
            if constexpr (DT == BT_F32) {
                v[k & 1] = ((const float*)p.pre)[row * 2 * Fp + k];
                v[2 + (k & 1)] = ((const float*)p.pre)[row * 2 * Fp + Fp + k];
            } else {
                const uint32_t* at = (const uint32_t*)p.pre + row * (Fp / 2 * 3) + 3 * (k >> 1);
                unpack24(at[0], at[1], at[2], v);
            }
            gated_grad_value<DT>(load_elem<DT>(p.dH, row * F + k), v[k & 1], v[2 + (k & 1)], dg, du);
        }
        bg += dg;
        bu += du;
        store_elem<DT>(p.G, row * 2 * Fp + k, dg * (p.scale[k] * unit));
        store_elem<DT>(p.G, row * 2 * Fp + Fp + k, du * (p.scale[Fp + k] * unit));
    }
    if (!p.parts || k >= F) return;
    p.parts[(int64_t)blockIdx.y * 2 * F + k] = bg;
    p.parts[(int64_t)blockIdx.y * 2 * F + F + k] = bu;
}

// Runs of rows of the gradient kernel: eight workgroups a compute unit; two where each leaves sums behind
static int64_t grad_runs(int64_t B, int64_t F, bool sums) {
    return std::min<int64_t>(B, std::max<int64_t>(1, (sums ? 2 : 8) * gemm_compute_units() / ceil_div(F, 2048)));
}

template <int DT>
static void launch_gated_grad(const GatedGradParams& p, int64_t runs, hipStream_t st) {
    if (p.F < 8) {
        hipLaunchKernelGGL(gated_grad_narrow_kernel<DT>, dim3(1, (unsigned)runs), dim3(64), 0, st, p);
        return;
    }
    const dim3 grid((unsigned)ceil_div(p.Fp, 2048), (unsigned)runs);
    if (p.F % 8 == 0) hipLaunchKernelGGL((gated_grad_kernel<DT, false>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((gated_grad_kernel<DT, true>), grid, dim3(256), 0, st, p);
}

}  // namespace bt

using namespace bt;

extern "C" size_t bt_gated_quantize_workspace_bytes(int64_t F, int64_t K, int per_channel) {
    if (F <= 0 || K <= 0 || gated_quantizes(K, per_channel != 0)) return 0;
    return (size_t)(2 * ceil_div(ceil_div(K, 4) * F, 256) * 256 + 2 * (per_channel ? F : 1) * 4);  // [gate's bytes][up's][scales]
}

extern "C" int bt_gated_quantize(const void* gate, const void* up, int w_dtype, int64_t F, int64_t K, double threshold_factor, int per_channel,
                                 const void* gate_bias, const void* up_bias, int bias_dtype, uint8_t* W_pairs, uint8_t* W_back,
                                 float* scale, float* bias, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "bt_gated_quantize";
    if (!gate || !up || !scale || !W_pairs || F <= 0 || K <= 0) {
        set_error("%s: null pointer or empty shape", who);
        return BT_ERR_INVALID;
    }
    if (w_dtype != BT_F32 && w_dtype != BT_F16 && w_dtype != BT_BF16 && w_dtype != BT_F32_AS_F16) {
        set_error("%s: unsupported weight dtype %d", who, w_dtype);
        return BT_ERR_INVALID;
    }
    if ((gate_bias || up_bias) && (!bias || (bias_dtype != BT_F32 && bias_dtype != BT_F16 && bias_dtype != BT_BF16))) {
        set_error("%s: a bias without room for it or of an unsupported dtype", who);
        return BT_ERR_INVALID;
    }
    const int64_t Fp = padded(F);
    if (F >= (1ll << 23) || K >= (1ll << 23) || bt_tiled_weights_bytes(2 * Fp, K) >= (1ull << 32) || bt_tiled_weights_bytes(K, 2 * Fp) >= (1ull << 32) ||
        (((uintptr_t)W_pairs) | ((uintptr_t)W_back)) % 256 != 0) {
        set_error("%s: F and K below 2^23, copies 256-byte aligned and below 4 GiB (F=%lld, K=%lld)", who, (long long)F, (long long)K);
        return BT_ERR_INVALID;
    }
    const size_t need = bt_gated_quantize_workspace_bytes(F, K, per_channel);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace) % 256 != 0)) {
        set_error("%s: workspace of %zu bytes (256-byte aligned) needed, %zu given", who, need, workspace_bytes);
        return BT_ERR_WORKSPACE;
    }
    hipStream_t st = (hipStream_t)stream;
    const int64_t Kb = ceil_div(K, 4);
    const uint32_t steps = (uint32_t)ceil_div(Kb, 16), back_steps = (uint32_t)ceil_div(2 * Fp, 64);
    if (!need) {
        GatedQuantizeParams p = {};
        p.W[0] = gate; p.W[1] = up; p.b[0] = gate_bias; p.b[1] = up_bias; p.bias_dtype = bias_dtype;
        p.tf = (float)threshold_factor; p.clamp_min = quantize_clamp_min(w_dtype);
        p.F = (int)F; p.K = (int)K; p.Fp = (int)Fp; p.tiles = (int)(2 * ceil_div(F, 16)); p.per_xcd = (int)ceil_div(p.tiles, 8);
        p.pairs = W_pairs; p.back = W_back; p.scale = scale; p.bias = bias; p.steps = steps; p.back_steps = back_steps;
        if (w_dtype == BT_F32) launch_gated_quantize<BT_F32>(p, st);
        else if (w_dtype == BT_F16) launch_gated_quantize<BT_F16>(p, st);
        else if (w_dtype == BT_BF16) launch_gated_quantize<BT_BF16>(p, st);
        else launch_gated_quantize<BT_F32_AS_F16>(p, st);
        return check_launch(who);
    }
    uint8_t* codes[2] = {(uint8_t*)workspace, (uint8_t*)workspace + ceil_div(Kb * F, 256) * 256};
    float* absmax[2];
    absmax[0] = (float*)((uint8_t*)workspace + 2 * ceil_div(Kb * F, 256) * 256);
    absmax[1] = absmax[0] + (per_channel ? F : 1);
    for (int i = 0; i < 2; i++)
        if (int rc = bt_quantize_pack(i ? up : gate, w_dtype, F, K, threshold_factor, per_channel, codes[i], absmax[i], nullptr, stream)) return rc;
    GatedWeightsParams p = {};
    p.W[0] = codes[0]; p.W[1] = codes[1]; p.a[0] = absmax[0]; p.a[1] = absmax[1]; p.b[0] = gate_bias; p.b[1] = up_bias;
    p.bias_dtype = bias_dtype; p.one_scale = !per_channel;
    p.F = F; p.Fp = Fp; p.K = K; p.Kb = Kb;
    p.pairs = W_pairs; p.back = W_back; p.scale = scale; p.bias = bias;
    p.steps = steps; p.back_steps = back_steps;
    p.n_pairs = (uint32_t)(2 * steps * ceil_div(Fp, 256));
    p.n_back = W_back ? (uint32_t)(ceil_div(K, 16) * ceil_div(back_steps, 16)) : 0;
    hipLaunchKernelGGL(gated_weights_kernel, dim3(p.n_pairs + p.n_back + (unsigned)(2 * Fp / 256 + 1)), dim3(256), 0, st, p);
    return check_launch(who);
}

extern "C" int bt_gated_range(float* scale, int64_t F, void* stream) {
    const char* who = "bt_gated_range";
    if (!scale || F <= 0 || F >= (1ll << 23)) {
        set_error("%s: null pointer, or F not between 1 and 2^23", who);
        return BT_ERR_INVALID;
    }
    hipLaunchKernelGGL(gated_range_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, scale, (int)(2 * padded(F)), nullptr);
    return check_launch(who);
}

extern "C" size_t bt_gated_split_bytes(int64_t F) {
    return F > 0 && F < (1ll << 23) ? (size_t)(4 * (4 * padded(F) + 16) + 128 * ceil_div(2 * padded(F), 64)) : 0;
}

extern "C" int bt_gated_split(float* scale, int64_t F, float* split, void* stream) {
    const char* who = "bt_gated_split";
    if (!scale || !split || F <= 0 || F >= (1ll << 23) || ((uintptr_t)split) % 16 != 0) {
        set_error("%s: null pointer, split not 16-byte aligned, or F not between 1 and 2^23", who);
        return BT_ERR_INVALID;
    }
    hipLaunchKernelGGL(gated_range_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, scale, (int)(2 * padded(F)), split);
    return check_launch(who);
}

extern "C" size_t bt_gated_grad_input_workspace_bytes(int64_t B, int64_t F, int64_t K) {
    return B > 0 && F > 0 && K > 0 ? gemm_f16_factors_workspace_bytes(B, K, 2 * padded(F)) : 0;
}

extern "C" int bt_gated_grad_input(const void* G, const uint8_t* W_back, const float* split, void* dX, int64_t B, int64_t F, int64_t K, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    const char* who = "bt_gated_grad_input";
    if (!G || !W_back || !split || !dX || B <= 0 || F <= 0 || K <= 0) {
        set_error("%s: null pointer or empty shape", who);
        return BT_ERR_INVALID;
    }
    const int64_t n = 2 * padded(F);  // (below 2^24: 32-bit byte offsets span 128 rows of G)
    if (F >= (1ll << 23) || K >= (1ll << 23) || B >= (1ll << 31) || n >= (1ll << 24) || bt_tiled_weights_bytes(K, n) >= (1ull << 32) ||
        ((uintptr_t)W_back) % 256 != 0 || (((uintptr_t)G) | ((uintptr_t)split) | ((uintptr_t)dX)) % 16 != 0) {
        set_error("%s: F and K below 2^23, B below 2^31, buffers 16-byte and the copy 256-byte aligned and below 4 GiB (F=%lld, K=%lld)", who,
                  (long long)F, (long long)K);
        return BT_ERR_INVALID;
    }
    const size_t need = bt_gated_grad_input_workspace_bytes(B, F, K);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace) % 256 != 0)) {
        set_error("%s: workspace of %zu bytes (256-byte aligned) needed, %zu given", who, need, workspace_bytes);
        return BT_ERR_WORKSPACE;
    }
    return launch_gemm_f16_factors(G, W_back, (const uint16_t*)(split + 2 * n + 16), split + n + 1, dX, B, K, n, workspace, (hipStream_t)stream);
}

extern "C" int bt_ternary_gated_forward(const void* X, int x_dtype, void* X_padded, const uint8_t* W_pairs, const float* scale, const float* bias, void* H,
                                        void* pre, int64_t B, int64_t F, int64_t K, void* stream) {
    const char* who = "bt_ternary_gated_forward";
    if (!X || !W_pairs || !scale || !H || B <= 0 || F <= 0 || K <= 0 || (x_dtype != BT_F16 && x_dtype != BT_BF16)) {
        set_error("%s: null pointer, empty shape or bad dtype (fp16 and bf16 rows)", who);
        return BT_ERR_INVALID;
    }
    const int64_t Fp = padded(F);
    const void* rows = X_padded ? X_padded : X;
    const int64_t Kr = X_padded ? ceil_div(K, 8) * 8 : K;  // values of a row of them
    if (F >= (1ll << 23) || K >= (1ll << 23) || B >= (1ll << 31) || ((uintptr_t)W_pairs) % 256 != 0 || bt_tiled_weights_bytes(2 * Fp, K) >= (1ull << 32) ||
        ((uintptr_t)X) % 2 != 0 || ((uintptr_t)pre) % 16 != 0 || !gemm_f16_supported(2 * Fp, Kr, rows, W_pairs, H, true)) {
        set_error("%s: rows whose length is no multiple of 8 or that are not 16-byte aligned need X_padded; F and K below 2^23, buffers 16-byte "
                  "and the weights 256-byte aligned (F=%lld, K=%lld)", who, (long long)F, (long long)K);
        return BT_ERR_INVALID;
    }
    if (X_padded)
        if (int rc = launch_pad_rows(X, B, K, X_padded, (hipStream_t)stream)) return rc;
    Epilogue epi = {};
    epi.scale = scale; epi.scale_dtype = BT_F32;
    epi.bias = bias; epi.bias_dtype = BT_F32;
    return launch_gemm_f16_gated(x_dtype == BT_F16 ? MODE_F16 : MODE_BF16, rows, W_pairs, epi, H, (uint32_t*)pre, F, B, 2 * Fp, Kr, (hipStream_t)stream);
}

extern "C" int bt_gated_masters_serves(int64_t B, int64_t K, int w_dtype, int per_channel) { return masters_serve(B, K, w_dtype, per_channel != 0); }

extern "C" int bt_gated_masters_forward(const void* X, int x_dtype, const void* gate, const void* up, int w_dtype, double threshold_factor,
                                        const void* gate_bias, const void* up_bias, int bias_dtype, void* H, int64_t F, int64_t K, void* stream) {
    const char* who = "bt_gated_masters_forward";
    if (!X || !gate || !up || !H || F <= 0 || K <= 0 || (x_dtype != BT_F32 && x_dtype != BT_F16 && x_dtype != BT_BF16)) {
        set_error("%s: null pointer, empty shape or bad dtype", who);
        return BT_ERR_INVALID;
    }
    if ((w_dtype != BT_F32 && w_dtype != BT_F16 && w_dtype != BT_BF16 && w_dtype != BT_F32_AS_F16) ||
        ((gate_bias || up_bias) && bias_dtype != BT_F32 && bias_dtype != BT_F16 && bias_dtype != BT_BF16)) {
        set_error("%s: unsupported weight or bias dtype", who);
        return BT_ERR_INVALID;
    }
    if (!masters_serve(1, K, w_dtype, true) || F >= (1ll << 23)) {
        set_error("%s: a row that bt_gated_masters_serves takes, F below 2^23 (F=%lld, K=%lld)", who, (long long)F, (long long)K);
        return BT_ERR_INVALID;
    }
    GatedMastersParams p = {};
    p.W[0] = gate; p.W[1] = up; p.b[0] = gate_bias; p.b[1] = up_bias; p.bias_dtype = bias_dtype; p.X = X; p.x_dtype = x_dtype; p.H = H;
    p.tf = (float)threshold_factor; p.clamp_min = quantize_clamp_min(w_dtype);
    p.F = (int)F; p.K = (int)K;
    hipStream_t st = (hipStream_t)stream;
    if (w_dtype == BT_F32) launch_gated_masters<BT_F32>(p, st);
    else if (w_dtype == BT_F16) launch_gated_masters<BT_F16>(p, st);
    else if (w_dtype == BT_BF16) launch_gated_masters<BT_BF16>(p, st);
    else launch_gated_masters<BT_F32_AS_F16>(p, st);
    return check_launch(who);
}

extern "C" size_t bt_gated_grad_workspace_bytes(int64_t B, int64_t F) {
    return B > 0 && F > 0 ? (size_t)grad_runs(B, F, true) * 2 * (size_t)F * 4 : 0;
}

extern "C" int bt_gated_grad(const void* dH, int dtype, const void* pre, const float* scale, void* G, void* dBias, int bias_dtype, int64_t B,
                             int64_t F, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "bt_gated_grad";
    if (!dH || !pre || !G || B <= 0 || F <= 0 || (dtype != BT_F32 && dtype != BT_F16 && dtype != BT_BF16) || !scale) {
        set_error("%s: null pointer, empty shape or bad dtype", who);
        return BT_ERR_INVALID;
    }
    if (F >= (1ll << 23) || B >= (1ll << 31) || (((uintptr_t)pre) | ((uintptr_t)G)) % 16 != 0) {
        set_error("%s: F below 2^23, B below 2^31, the projections and G 16-byte aligned", who);
        return BT_ERR_INVALID;
    }
    if (dBias && (bias_dtype != BT_F32 && bias_dtype != BT_F16 && bias_dtype != BT_BF16)) {
        set_error("%s: unsupported bias dtype", who);
        return BT_ERR_INVALID;
    }
    if (dBias && (!workspace || workspace_bytes < bt_gated_grad_workspace_bytes(B, F) || ((uintptr_t)workspace) % 256 != 0)) {
        set_error("%s: workspace of %zu bytes (256-byte aligned) needed, %zu given", who, bt_gated_grad_workspace_bytes(B, F), workspace_bytes);
        return BT_ERR_WORKSPACE;
    }
    GatedGradParams p = {};
    int64_t runs = grad_runs(B, F, dBias != nullptr);
    p.rows = ceil_div(B, runs);
    runs = ceil_div(B, p.rows);  // (so that none is empty)
    p.dH = dH; p.pre = pre; p.scale = scale; p.G = G; p.parts = dBias ? (float*)workspace : nullptr;
    p.B = B; p.F = (int)F; p.Fp = (int)padded(F);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == BT_F32) launch_gated_grad<BT_F32>(p, runs, st);
    else if (dtype == BT_F16) launch_gated_grad<BT_F16>(p, runs, st);
    else launch_gated_grad<BT_BF16>(p, runs, st);
    const int rc = check_launch(who);
    return rc || !dBias ? rc : launch_column_sum(p.parts, runs, 2 * F, dBias, bias_dtype, st, who);
}
