// The residual connection and the norm behind it in one pass over the rows, and their gradient, for gfx950 (HBM-bound):
//
//   s = rd_r(x + residual)                                  the stream, in the residual's type
//   y = rd_x((s * r) * w),  r = 1 / sqrt(float(sum_k double(s)^2) / K + eps)
//   optionally q, s_x: y quantized per row to int8, as the row kernels of row_ops.hip do it
// (rd = round to that type; every fp32 operation of the forward rounded on its own).  The norm is that of the sum as it is stored:
// what the next block reads, what the backward pass reads, and bit for bit what an addition followed by bt_rmsnorm gives.
//
// Gradient, for incoming ds (of s) and dy (of y), with xhat = s * r and c = mean_k(dy w xhat):
//   dx = dresidual = ds + r (dy w - xhat c),      dw = sum_rows dy xhat
// in fp32 from the stored s and the stored r (four bytes a row instead of a pass over it); one rounding at the end.
//
// Both directions read every operand once: a row's values stay in registers between its reduction and what follows.
#include "row_vec.h"

namespace bt {

struct AddNormParams {
    const void* X;        // [B, K], row stride ldx
    const void* R;        // [B, K], row stride ldr; null: s = x, and S is not written
    const void* W;        // [K] or null (ones)
    int64_t ldx, ldr;
    void* S;              // [B, K]
    void* Y;              // [B, K] or null
    float* rstd;          // [B] or null
    int8_t* Q;            // [B, K] or null
    float* s_x;           // [B] with Q
    int32_t* rowsum;      // [B] or null
    float eps;
    int K;
    int w_f32;            // W is fp32 (otherwise of x's type)
    int q_layout;
};

// HIP takes fewer than 2^32 threads along x and wraps beyond: workgroups that there may be 2^22 and more of go over x and y.
static dim3 wide_grid(int64_t n) { return dim3((unsigned)std::min<int64_t>(n, 1 << 20), (unsigned)ceil_div(n, 1 << 20)); }
__device__ __forceinline__ int64_t wide_block() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

// WPR waves to a row (4: a workgroup per row; 1: four rows to a workgroup, without LDS or barriers), ITERS pieces of eight values a
// lane: K <= 512 ITERS WPR.  All loads go out before the first value is used.
template <int DT, int RT, int ITERS, int WPR, bool QUANT, bool RAG>
__global__ __launch_bounds__(256) void add_rmsnorm_kernel(AddNormParams p, int64_t B) {
    __shared__ double part_d[4];
    __shared__ float part_f[4];
    __shared__ int part_i[4];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, t = WPR == 1 ? lane : (int)threadIdx.x;
    const int K = p.K;
    const int64_t row = wide_block() * (4 / WPR) + (WPR == 1 ? wave : 0);
    if (row >= B) return;  // (WPR = 1: whole waves, and no barrier below; 4: whole workgroups)
    auto at = [&](int i) { return (i * 64 * WPR + t) * 8; };
    float v[ITERS][8];
    Raw8<DT> x[ITERS], w16[ITERS];
    Raw8<BT_F32> w32[ITERS];
#pragma unroll
    for (int i = 0; i < ITERS; i++) x[i] = load_raw8<DT>(p.X, row * p.ldx + piece_at(at(i), K));
    const bool has_r = p.R != nullptr, has_w = p.W != nullptr, wide_w = DT == BT_F32 || p.w_f32;  // (uniform)
    Raw8<RT> r_in[ITERS];
    if (has_r) {
#pragma unroll
        for (int i = 0; i < ITERS; i++) r_in[i] = load_raw8<RT>(p.R, row * p.ldr + piece_at(at(i), K));
    }
    if (has_w && wide_w) {
#pragma unroll
        for (int i = 0; i < ITERS; i++) w32[i] = load_raw8<BT_F32>(p.W, piece_at(at(i), K));
    } else if (has_w) {
#pragma unroll
        for (int i = 0; i < ITERS; i++) w16[i] = load_raw8<DT>(p.W, piece_at(at(i), K));
    }
#pragma unroll
    for (int i = 0; i < ITERS; i++) widen_piece<DT, RAG>(x[i], at(i), K, v[i]);
    if (has_r) {
#pragma unroll
        for (int i = 0; i < ITERS; i++) {
            float r[8];
            widen_piece<RT, RAG>(r_in[i], at(i), K, r);
#pragma unroll
            for (int e = 0; e < 8; e++) v[i][e] = round_to_dtype(__fadd_rn(v[i][e], r[e]), RT);
            store_piece<RT, RAG>(p.S, row * (int64_t)K, at(i), K, v[i]);
        }
    }
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < ITERS; i++)
#pragma unroll
        for (int e = 0; e < 8; e++) ss += (double)v[i][e] * (double)v[i][e];
    ss = wave_sum_f64(ss);
    if constexpr (WPR > 1) {
        if (lane == 0) part_d[wave] = ss;
        __syncthreads();
        ss = (part_d[0] + part_d[1]) + (part_d[2] + part_d[3]);
    }
    const float r = rms_rstd(ss, K, p.eps);
    if (p.rstd && t == 0) p.rstd[row] = r;
    if (has_w) {
#pragma unroll
        for (int i = 0; i < ITERS; i++) {
            float w[8];
            if (wide_w) widen_piece<BT_F32, RAG>(w32[i], at(i), K, w);
            else widen_piece<DT, RAG>(w16[i], at(i), K, w);
#pragma unroll
            for (int e = 0; e < 8; e++) v[i][e] = rmsnorm_value(v[i][e], r, w[e], DT);
        }
    } else {
#pragma unroll
        for (int i = 0; i < ITERS; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) v[i][e] = rmsnorm_value(v[i][e], r, 1.0f, DT);
    }
    if (p.Y) {
#pragma unroll
        for (int i = 0; i < ITERS; i++) store_piece<DT, RAG>(p.Y, row * (int64_t)K, at(i), K, v[i]);
    }
    if constexpr (!QUANT) return;
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < ITERS; i++)
#pragma unroll
        for (int e = 0; e < 8; e++) amax = fmaxf(amax, at(i) + e < K ? fabsf(v[i][e]) : 0.0f);
    amax = wave_max(amax);
    if constexpr (WPR > 1) {
        if (lane == 0) part_f[wave] = amax;
        __syncthreads();
        amax = fmaxf(fmaxf(part_f[0], part_f[1]), fmaxf(part_f[2], part_f[3]));
    }
    const float s = (amax > 1e-6f) ? __fdiv_rn(amax, 127.0f) : 1.0f;
    const float inv = __fdiv_rn(1.0f, s);
    if (t == 0) p.s_x[row] = s;
    int qsum = 0;
#pragma unroll
    for (int i = 0; i < ITERS; i++) {
        const int k = at(i);
        uint32_t d[2] = {0u, 0u};
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int8_t qv = quant_i8(v[i][e], inv);
            if (k + e < K) qsum += (int)qv;
            d[e >> 2] |= (uint32_t)(uint8_t)qv << (8 * (e & 3));
        }
        // (operand order: K % 16 == 0, so that both lanes of a group of sixteen are inside the row or outside)
        const uint2 o = p.q_layout == Q_OPERAND_ORDER ? q_to_operand_order(d[0], d[1], lane & 1) : make_uint2(d[0], d[1]);
        int8_t* dst = p.Q + row * (int64_t)K + k;
        if (k + 8 <= K) {
            typedef uint32_t u32x2_a1 __attribute__((ext_vector_type(2), aligned(1)));
            u32x2_a1 b;
            b[0] = o.x; b[1] = o.y;
            __builtin_nontemporal_store(b, (u32x2_a1*)dst);
        } else if (RAG && k < K) {
#pragma unroll
            for (int e = 0; e < 7; e++)
                if (k + e < K) dst[e] = (int8_t)((e < 4 ? o.x : o.y) >> (8 * (e & 3)));
        }
    }
    if (p.rowsum) {  // (uniform)
        qsum = wave_sum_i32(qsum);
        if constexpr (WPR > 1) {
            if (lane == 0) part_i[wave] = qsum;
            __syncthreads();
            qsum = (part_i[0] + part_i[1]) + (part_i[2] + part_i[3]);
        }
        if (t == 0) p.rowsum[row] = qsum;
    }
}

// Rows below 8 or above 16384 values: a workgroup per row, element by element; the passes behind the first read the stored sum again.
template <int DT, int RT>
__global__ __launch_bounds__(256) void add_rmsnorm_any_kernel(AddNormParams p, int64_t B) {
    __shared__ double part_d[4];
    __shared__ float part_f[4];
    __shared__ int part_i[4];
    const int tid = threadIdx.x, K = p.K;
    const int64_t row = wide_block();
    if (row >= B) return;  // (whole workgroups)
    auto sum = [&](int k) {
        const float x = load_elem<DT>(p.X, row * p.ldx + k);
        return p.R ? round_to_dtype(__fadd_rn(x, load_elem<RT>(p.R, row * p.ldr + k)), RT) : x;
    };
    double ss = 0.0;
    for (int k = tid; k < K; k += 256) {
        const float s = sum(k);
        if (p.R) store_elem<RT>(p.S, row * (int64_t)K + k, s);
        ss += (double)s * (double)s;
    }
    ss = wave_sum_f64(ss);
    if ((tid & 63) == 0) part_d[tid >> 6] = ss;
    __syncthreads();
    ss = (part_d[0] + part_d[1]) + (part_d[2] + part_d[3]);
    const float r = rms_rstd(ss, K, p.eps);
    if (p.rstd && tid == 0) p.rstd[row] = r;
    auto value = [&](int k) {  // (a thread's own elements, as it has stored them)
        const float s = p.R ? load_elem<RT>(p.S, row * (int64_t)K + k) : sum(k);
        return rmsnorm_value(s, r, p.W ? load_elem_rt(p.W, p.w_f32 ? BT_F32 : DT, k) : 1.0f, DT);
    };
    float amax = 0.0f;
    for (int k = tid; k < K; k += 256) {
        const float v = value(k);
        if (p.Y) store_elem<DT>(p.Y, row * (int64_t)K + k, v);
        amax = fmaxf(amax, fabsf(v));
    }
    if (!p.Q) return;  // (uniform)
    amax = wave_max(amax);
    if ((tid & 63) == 0) part_f[tid >> 6] = amax;
    __syncthreads();
    amax = fmaxf(fmaxf(part_f[0], part_f[1]), fmaxf(part_f[2], part_f[3]));
    const float s = (amax > 1e-6f) ? __fdiv_rn(amax, 127.0f) : 1.0f;
    const float inv = __fdiv_rn(1.0f, s);
    if (tid == 0) p.s_x[row] = s;
    int qsum = 0;
    for (int k = tid; k < K; k += 256) {
        const int8_t qv = quant_i8(value(k), inv);
        qsum += (int)qv;
        p.Q[row * (int64_t)K + (p.q_layout == Q_OPERAND_ORDER ? q_operand_order_pos(k) : k)] = qv;
    }
    if (!p.rowsum) return;  // (uniform)
    qsum = wave_sum_i32(qsum);
    if ((tid & 63) == 0) part_i[tid >> 6] = qsum;
    __syncthreads();
    if (tid == 0) p.rowsum[row] = (part_i[0] + part_i[1]) + (part_i[2] + part_i[3]);
}

template <int DT, int RT, int ITERS, int WPR>
static void launch_add_rmsnorm_cfg(const AddNormParams& p, int64_t B, hipStream_t st) {
    const dim3 grid = wide_grid(ceil_div(B, 4 / WPR)), block(256);
    if (p.K % 8 == 0) {
        if (p.Q) hipLaunchKernelGGL((add_rmsnorm_kernel<DT, RT, ITERS, WPR, true, false>), grid, block, 0, st, p, B);
        else hipLaunchKernelGGL((add_rmsnorm_kernel<DT, RT, ITERS, WPR, false, false>), grid, block, 0, st, p, B);
    } else {
        if (p.Q) hipLaunchKernelGGL((add_rmsnorm_kernel<DT, RT, ITERS, WPR, true, true>), grid, block, 0, st, p, B);
        else hipLaunchKernelGGL((add_rmsnorm_kernel<DT, RT, ITERS, WPR, false, true>), grid, block, 0, st, p, B);
    }
}
template <int DT, int RT>
static void launch_add_rmsnorm_dt(const AddNormParams& p, int64_t B, hipStream_t st) {
    if (p.K < 8 || p.K > 16384 || option(OPT_ROWOP_GENERIC)) {
        hipLaunchKernelGGL((add_rmsnorm_any_kernel<DT, RT>), wide_grid(B), dim3(256), 0, st, p, B);
        return;
    }
    // A wave to a row where there are rows for all of them and it holds the row in few registers; a workgroup's barriers and idle lanes
    // cost the short rows most.  us, a workgroup / a wave to a row, bf16: 65536 x 256 89.4 / 32.7, 16384 x 768 27.4 / 17.3 (with int8 36.5 /
    // 19.3), 8192 x 1024 15.5 / 12.0, 4096 x 2560 19.2 / 17.0 (20.7 / 17.7); an fp32 stream 8192 x 1536 29.1 / 30.4, 4096 x 2560 25.4 / 25.8.
    if (B >= 1024 && p.K <= (RT == BT_F32 ? 1024 : 2560)) {
        if (p.K <= 512) launch_add_rmsnorm_cfg<DT, RT, 1, 1>(p, B, st);
        else if (p.K <= 1024) launch_add_rmsnorm_cfg<DT, RT, 2, 1>(p, B, st);
        else if constexpr (RT != BT_F32) {
            if (p.K <= 1536) launch_add_rmsnorm_cfg<DT, RT, 3, 1>(p, B, st);
            else launch_add_rmsnorm_cfg<DT, RT, 5, 1>(p, B, st);
        }
        return;
    }
    if (p.K <= 2048) launch_add_rmsnorm_cfg<DT, RT, 1, 4>(p, B, st);
    else if (p.K <= 4096) launch_add_rmsnorm_cfg<DT, RT, 2, 4>(p, B, st);
    else if (p.K <= 8192) launch_add_rmsnorm_cfg<DT, RT, 4, 4>(p, B, st);
    else launch_add_rmsnorm_cfg<DT, RT, 8, 4>(p, B, st);
}

// ---- gradient -----------------------------------------------------------------------------------------------------------

struct AddNormGradParams {
    const void* S;        // [B, K] the stored sum, of the stream's type
    const float* rstd;    // [B]
    const void* W;        // [K] or null
    const void* dY;       // [B, K] of x's type
    const void* dS;       // [B, K] of the stream's type, or null
    void* dX;             // [B, K] of x's type, or null
    void* dR;             // [B, K] of the stream's type, or null
    float* parts;         // [gridDim.x, K] sums of dy xhat, or null
    int64_t B;
    int K;
    int w_f32;
};

// A workgroup of eight waves takes rows blockIdx.x, + gridDim.x, ... in groups of 8 / WPR, WPR waves to a row; a lane owns the same
// columns of every row, so that the weight's gradient gathers in its registers and leaves once, as a row of `parts`.  The rows stay as
// they were loaded until they are used, and the weight lies in LDS in fp32: registers are what bounds the rows in flight.
// Dynamic LDS: fp32 [max(K rounded up to pieces, 4096 for the last sums)].
template <int DT, int RT, int ITERS, int WPR, bool RAG>
__global__ __launch_bounds__(512) void add_rmsnorm_grad_kernel(AddNormGradParams p) {
    constexpr int GROUPS = 8 / WPR, C = 512 * WPR;  // columns of a piece of the whole group
    extern __shared__ __attribute__((aligned(16))) float lds_w[];
    __shared__ float part[2][8];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int group = wave / WPR, t = (wave % WPR) * 64 + lane;
    const int K = p.K;
    auto at = [&](int i) { return i * C + t * 8; };
    float dw[ITERS][8];
#pragma unroll
    for (int i = 0; i < ITERS; i++)
#pragma unroll
        for (int e = 0; e < 8; e++) dw[i][e] = 0.0f;
    for (int k = threadIdx.x; k < ITERS * C; k += 512)
        lds_w[k] = k >= K ? 0.0f : p.W ? load_elem_rt(p.W, p.w_f32 ? BT_F32 : DT, k) : 1.0f;
    __syncthreads();
    const float inv_k = 1.0f / (float)K;
    const bool has_g = p.dS != nullptr;
    const void* const dS = has_g ? p.dS : p.S;  // (without it the loads read the sum once more and their values are not used)
    struct Row {
        Raw8<RT> s[ITERS], g[ITERS];
        Raw8<DT> dy[ITERS];
        float r;
    };
    auto load = [&](int64_t row, Row& to) {
        row = row < p.B ? row : p.B - 1;
        to.r = p.rstd[row];
#pragma unroll
        for (int i = 0; i < ITERS; i++) to.s[i] = load_raw8<RT>(p.S, row * K + piece_at(at(i), K));
#pragma unroll
        for (int i = 0; i < ITERS; i++) to.dy[i] = load_raw8<DT>(p.dY, row * K + piece_at(at(i), K));
#pragma unroll
        for (int i = 0; i < ITERS; i++) to.g[i] = load_raw8<RT>(dS, row * K + piece_at(at(i), K));
    };
    constexpr bool AHEAD = ITERS + (RAG ? 1 : 0) < (RT == BT_F32 ? 4 : 5);  // (registers for a second row)
    int turn = 0;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    Row next;
    if constexpr (AHEAD) load((int64_t)blockIdx.x * GROUPS + group, next);
    for (int64_t row0 = (int64_t)blockIdx.x * GROUPS; row0 < p.B; row0 += step, turn ^= 1) {
        // (every group passes the barriers; one past the last row computes that row again and stores nothing)
        const bool ok = row0 + group < p.B;
        const int64_t row = ok ? row0 + group : p.B - 1;
        Row now;
        if constexpr (AHEAD) {
            now = next;
            load(row0 + step + group, next);  // in flight while this row is worked on (4096 x 2560 bf16: 21.9 -> 19.9 us)
        } else {
            load(row, now);
        }
        const Raw8<RT> (&s_in)[ITERS] = now.s, (&g_in)[ITERS] = now.g;
        const Raw8<DT> (&dy_in)[ITERS] = now.dy;
        const float r = now.r;
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < ITERS; i++) {
            float s[8], dy[8], piece = 0.0f;  // (a sum of its own for each piece: the chain of roundings is shorter)
            widen_piece<RT, RAG>(s_in[i], at(i), K, s);
            widen_piece<DT, RAG>(dy_in[i], at(i), K, dy);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float dy_xhat = dy[e] * (s[e] * r);
                if (ok) dw[i][e] += dy_xhat;
                piece = __builtin_fmaf(dy_xhat, lds_w[at(i) + e], piece);
            }
            dot += piece;
        }
        dot = wave_sum_f32(dot);
        if constexpr (WPR > 1) {
            if (lane == 0) part[turn][wave] = dot;
            __syncthreads();  // (one a row: the other half of `part` is written next, and this one behind the next barrier)
            dot = 0.0f;
#pragma unroll
            for (int i = 0; i < WPR; i++) dot += part[turn][group * WPR + i];
        }
        const float rc = r * (dot * inv_k);
        if (!ok) continue;  // (whole groups; the barrier of this turn is behind)
#pragma unroll
        for (int i = 0; i < ITERS; i++) {
            float s[8], dy[8], g[8];
            widen_piece<RT, RAG>(s_in[i], at(i), K, s);
            widen_piece<DT, RAG>(dy_in[i], at(i), K, dy);
            widen_piece<RT, RAG>(g_in[i], at(i), K, g);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float d = r * __builtin_fmaf(-s[e], rc, dy[e] * lds_w[at(i) + e]);
                g[e] = has_g ? g[e] + d : d;
            }
            if (p.dR) store_piece<RT, RAG>(p.dR, row * K, at(i), K, g);
            if (p.dX) store_piece<DT, RAG>(p.dX, row * K, at(i), K, g);
        }
    }
    if (!p.parts) return;  // (uniform)
    float* const out = p.parts + (int64_t)blockIdx.x * K;
#pragma unroll
    for (int i = 0; i < ITERS; i++) {
        if constexpr (GROUPS == 1) {
            store_piece<BT_F32, RAG>(out, 0, at(i), K, dw[i]);
        } else {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 8; e++) lds_w[group * C + t * 8 + e] = dw[i][e];
            __syncthreads();
            for (int c = threadIdx.x; c < C; c += 512) {
                float v = lds_w[c];
#pragma unroll
                for (int q = 1; q < GROUPS; q++) v += lds_w[q * C + c];
                if (i * C + c < K) out[i * C + c] = v;
            }
        }
    }
}

// Any K: the inputs' gradient, a workgroup per row, element by element
template <int DT, int RT>
__global__ __launch_bounds__(256) void add_rmsnorm_grad_any_kernel(AddNormGradParams p) {
    __shared__ float part[4];
    const int tid = threadIdx.x, K = p.K;
    const int64_t row = wide_block(), at = row * (int64_t)K;
    if (row >= p.B) return;  // (whole workgroups)
    const float r = p.rstd[row];
    auto weighted = [&](int k) { return load_elem<DT>(p.dY, at + k) * (p.W ? load_elem_rt(p.W, p.w_f32 ? BT_F32 : DT, k) : 1.0f); };
    float dot = 0.0f;
    for (int k = tid; k < K; k += 256) dot = __builtin_fmaf(weighted(k), load_elem<RT>(p.S, at + k) * r, dot);
    dot = wave_sum_f32(dot);
    if ((tid & 63) == 0) part[tid >> 6] = dot;
    __syncthreads();
    const float c = ((part[0] + part[1]) + (part[2] + part[3])) / (float)K;
    for (int k = tid; k < K; k += 256) {
        const float d = r * __builtin_fmaf(-(load_elem<RT>(p.S, at + k) * r), c, weighted(k));
        const float v = p.dS ? load_elem<RT>(p.dS, at + k) + d : d;
        if (p.dR) store_elem<RT>(p.dR, at + k, v);
        if (p.dX) store_elem<DT>(p.dX, at + k, v);
    }
}
// ... and the sums of the weight's gradient over a run of rows: a thread per column
template <int DT, int RT>
__global__ __launch_bounds__(256) void add_rmsnorm_gradw_any_kernel(AddNormGradParams p, int64_t rows) {
    const int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (k >= p.K) return;
    const int64_t first = (int64_t)blockIdx.y * rows, last = std::min(first + rows, p.B);
    float sum = 0.0f;
    for (int64_t row = first; row < last; row++)
        sum = __builtin_fmaf(load_elem<DT>(p.dY, row * p.K + k), load_elem<RT>(p.S, row * p.K + k) * p.rstd[row], sum);
    p.parts[(int64_t)blockIdx.y * p.K + k] = sum;
}

// Sums over the rows of `parts`: a workgroup takes 64 columns, its sixteen waves every sixteenth row each (a row of them at a time in
// flight: with four waves 256 rows of 2560 took 6.5 us, most of it waiting).
__global__ __launch_bounds__(1024) void column_sum_kernel(const float* __restrict__ parts, int64_t n, int64_t K, void* out, int dtype) {
    __shared__ float sums[16][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t k = wide_block() * 64 + lane;
    float a[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // (four loads in flight)
    if (k < K) {
        int64_t i = wave;
        for (; i + 48 < n; i += 64)
#pragma unroll
            for (int u = 0; u < 4; u++) a[u] += parts[(i + 16 * u) * K + k];
        for (; i < n; i += 16) a[0] += parts[i * K + k];
    }
    sums[wave][lane] = (a[0] + a[1]) + (a[2] + a[3]);
    __syncthreads();
    if (wave == 0 && k < K) {
        float v = 0.0f;
#pragma unroll
        for (int q = 0; q < 16; q += 4) v += (sums[q][lane] + sums[q + 1][lane]) + (sums[q + 2][lane] + sums[q + 3][lane]);
        if (dtype == BT_F32) store_elem<BT_F32>(out, k, v);
        else if (dtype == BT_F16) store_elem<BT_F16>(out, k, v);
        else store_elem<BT_BF16>(out, k, v);
    }
}
int launch_column_sum(const float* parts, int64_t n, int64_t K, void* out, int out_dtype, hipStream_t st, const char* who) {
    hipLaunchKernelGGL(column_sum_kernel, wide_grid(ceil_div(K, 64)), dim3(1024), 0, st, parts, n, K, out, out_dtype);
    return check_launch(who);
}

// Waves to a row: a lane holds at most three pieces (four of the longest rows), with more of them the registers of a row's operands
// and sums run over.
static bool grad_any(int64_t K) { return K < 8 || K > 16384 || option(OPT_ROWOP_GENERIC); }
static int grad_waves(int64_t K) { return K <= 3 * 512 ? 1 : K <= 6 * 512 ? 2 : K <= 12 * 512 ? 4 : 8; }
// Rows of `parts`: workgroups of the gradient kernel, one for each compute unit at most (their sums are K floats each)
static int64_t grad_parts(int64_t B, int64_t K) {
    if (grad_any(K)) return std::min<int64_t>(B, 64);
    return std::min<int64_t>(ceil_div(B, 8 / grad_waves(K)), gemm_compute_units());
}

template <int DT, int RT, int ITERS, int WPR>
static void launch_add_rmsnorm_grad_cfg(const AddNormGradParams& p, int64_t n, hipStream_t st) {
    const size_t lds = 4 * std::max(512 * ITERS * WPR, WPR < 8 ? 4096 : 0);
    if (p.K % 8 == 0) hipLaunchKernelGGL((add_rmsnorm_grad_kernel<DT, RT, ITERS, WPR, false>), dim3((unsigned)n), dim3(512), lds, st, p);
    else hipLaunchKernelGGL((add_rmsnorm_grad_kernel<DT, RT, ITERS, WPR, true>), dim3((unsigned)n), dim3(512), lds, st, p);
}
template <int DT, int RT>
static void launch_add_rmsnorm_grad(const AddNormGradParams& p, int64_t n, hipStream_t st) {
    const int K = p.K;
    if (grad_any(K)) {
        hipLaunchKernelGGL((add_rmsnorm_grad_any_kernel<DT, RT>), wide_grid(p.B), dim3(256), 0, st, p);
        if (p.parts) hipLaunchKernelGGL((add_rmsnorm_gradw_any_kernel<DT, RT>), dim3((unsigned)ceil_div(K, 256), (unsigned)n), dim3(256), 0, st, p, ceil_div(p.B, n));
        return;
    }
    const int waves = grad_waves(K), iters = (int)ceil_div(K, 512 * waves);
    if (waves == 1) {
        if (iters == 1) launch_add_rmsnorm_grad_cfg<DT, RT, 1, 1>(p, n, st);
        else if (iters == 2) launch_add_rmsnorm_grad_cfg<DT, RT, 2, 1>(p, n, st);
        else launch_add_rmsnorm_grad_cfg<DT, RT, 3, 1>(p, n, st);
    } else if (waves == 2) {
        if (iters == 2) launch_add_rmsnorm_grad_cfg<DT, RT, 2, 2>(p, n, st);
        else launch_add_rmsnorm_grad_cfg<DT, RT, 3, 2>(p, n, st);
    } else if (waves == 4) {
        if (iters == 2) launch_add_rmsnorm_grad_cfg<DT, RT, 2, 4>(p, n, st);
        else launch_add_rmsnorm_grad_cfg<DT, RT, 3, 4>(p, n, st);
    } else {
        if (iters == 2) launch_add_rmsnorm_grad_cfg<DT, RT, 2, 8>(p, n, st);
        else if (iters == 3) launch_add_rmsnorm_grad_cfg<DT, RT, 3, 8>(p, n, st);
        else launch_add_rmsnorm_grad_cfg<DT, RT, 4, 8>(p, n, st);
    }
}

static bool types_ok(int x_dtype, int r_dtype, int w_dtype, bool has_w) {
    auto known = [](int d) { return d == BT_F32 || d == BT_F16 || d == BT_BF16; };
    return known(x_dtype) && (r_dtype == x_dtype || r_dtype == BT_F32) && (!has_w || w_dtype == x_dtype || w_dtype == BT_F32);
}

}  // namespace bt

using namespace bt;

extern "C" int bt_add_rmsnorm(const void* X, int64_t ld_x, int x_dtype, const void* residual, int64_t ld_r, int r_dtype,
                              const void* weight, int w_dtype, float eps, int64_t B, int64_t K, void* sum, void* Y, float* rstd,
                              int8_t* Q, float* s_x, int32_t* q_rowsum, int q_layout, void* stream) {
    const char* who = "bt_add_rmsnorm";
    if (!X || B <= 0 || K <= 0 || (residual && !sum) || !types_ok(x_dtype, residual ? r_dtype : x_dtype, w_dtype, weight != nullptr)) {
        set_error("%s: null pointer, empty shape or bad dtype (the residual and the weight are of x's dtype or fp32)", who);
        return BT_ERR_INVALID;
    }
    if (ld_x < K || (residual && ld_r < K) || K > 0x7fffff00 || B > 0x7fffffff) {
        set_error("%s: row stride below K=%lld, or shape beyond 2^31", who, (long long)K);
        return BT_ERR_INVALID;
    }
    if (!Y && !Q) {
        set_error("%s: no output requested (Y and Q both null)", who);
        return BT_ERR_INVALID;
    }
    if ((Q && !s_x) || (q_rowsum && !Q)) {
        set_error("%s: Q given without s_x, or q_rowsum without Q", who);
        return BT_ERR_INVALID;
    }
    if (Q && q_layout != Q_ROW_MAJOR && (q_layout != Q_OPERAND_ORDER || K % 16 != 0 || ((uintptr_t)Q) % 16 != 0)) {
        set_error("%s: operand order needs K %% 16 == 0 and a 16-byte aligned Q (layout %d, K=%lld)", who, q_layout, (long long)K);
        return BT_ERR_INVALID;
    }
    AddNormParams p;
    p.X = X; p.R = residual; p.W = weight; p.ldx = ld_x; p.ldr = ld_r; p.S = sum; p.Y = Y; p.rstd = rstd; p.Q = Q; p.s_x = s_x;
    p.rowsum = q_rowsum; p.eps = eps; p.K = (int)K; p.w_f32 = w_dtype == BT_F32; p.q_layout = q_layout;
    hipStream_t st = (hipStream_t)stream;
    const bool wide = residual && r_dtype == BT_F32;
    if (x_dtype == BT_F32) launch_add_rmsnorm_dt<BT_F32, BT_F32>(p, B, st);
    else if (x_dtype == BT_F16) wide ? launch_add_rmsnorm_dt<BT_F16, BT_F32>(p, B, st) : launch_add_rmsnorm_dt<BT_F16, BT_F16>(p, B, st);
    else wide ? launch_add_rmsnorm_dt<BT_BF16, BT_F32>(p, B, st) : launch_add_rmsnorm_dt<BT_BF16, BT_BF16>(p, B, st);
    return check_launch(who);
}

extern "C" size_t bt_add_rmsnorm_backward_workspace_bytes(int64_t B, int64_t K) {
    return B > 0 && K > 0 ? (size_t)grad_parts(B, K) * (size_t)K * 4 : 0;
}

extern "C" int bt_add_rmsnorm_backward(const void* sum, int r_dtype, const float* rstd, const void* weight, int w_dtype, const void* dY,
                                       int x_dtype, const void* dSum, int64_t B, int64_t K, void* dX, void* dResidual, void* dWeight,
                                       void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "bt_add_rmsnorm_backward";
    if (!sum || !rstd || !dY || B <= 0 || K <= 0 || (!dX && !dResidual && !dWeight) ||
        !types_ok(x_dtype, r_dtype, w_dtype, weight != nullptr || dWeight != nullptr)) {
        set_error("%s: null pointer, empty shape or bad dtype (the sum and the weight are of x's dtype or fp32)", who);
        return BT_ERR_INVALID;
    }
    if (K > 0x7fffff00 || B > 0x7fffffff) {
        set_error("%s: shape beyond 2^31", who);
        return BT_ERR_INVALID;
    }
    const int64_t n = grad_parts(B, K);
    if (dWeight && (!workspace || workspace_bytes < bt_add_rmsnorm_backward_workspace_bytes(B, K) || ((uintptr_t)workspace) % 256 != 0)) {
        set_error("%s: workspace of %zu bytes (256-byte aligned) needed, %zu given", who, bt_add_rmsnorm_backward_workspace_bytes(B, K),
                  workspace_bytes);
        return BT_ERR_WORKSPACE;
    }
    AddNormGradParams p;
    p.S = sum; p.rstd = rstd; p.W = weight; p.dY = dY; p.dS = dSum; p.dX = dX; p.dR = dResidual; p.parts = dWeight ? (float*)workspace : nullptr;
    p.B = B; p.K = (int)K; p.w_f32 = w_dtype == BT_F32;
    hipStream_t st = (hipStream_t)stream;
    const bool wide = r_dtype == BT_F32;
    if (x_dtype == BT_F32) launch_add_rmsnorm_grad<BT_F32, BT_F32>(p, n, st);
    else if (x_dtype == BT_F16) wide ? launch_add_rmsnorm_grad<BT_F16, BT_F32>(p, n, st) : launch_add_rmsnorm_grad<BT_F16, BT_F16>(p, n, st);
    else wide ? launch_add_rmsnorm_grad<BT_BF16, BT_F32>(p, n, st) : launch_add_rmsnorm_grad<BT_BF16, BT_BF16>(p, n, st);
    int rc = check_launch(who);
    return rc || !dWeight ? rc : launch_column_sum(p.parts, n, K, dWeight, w_dtype, st, who);
}
