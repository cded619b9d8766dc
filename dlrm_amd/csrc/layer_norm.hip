// Layer norm over the rows of an activation, forward and backward.
//
//   forward    mean = sum x / N, rstd = 1 / sqrt(sum (x - mean)^2 / N + eps), xh = (x - mean) rstd, y = act(gamma xh + beta)
//   backward   d = dy where the ReLU let y through, else 0;  c1 = sum gamma d / N, c2 = sum gamma d xh / N
//              dx = rstd (gamma d - c1 - xh c2),  dgamma = sum over rows of d xh,  dbeta = sum over rows of d
//
// Both are bound by memory, so a row is read once: a team of lanes holds it in registers between the sums and the output
// (4 to 64 lanes of a wave for rows up to 1024 float32 or 512 bf16 elements, 128 to 1024 threads up to 16384).  Deviations
// are squared after the mean is known, not as sum x^2 - N mean^2, which loses everything when the mean is large.  Statistics and
// sums are float32 whatever the activation's type.  Longer rows are read again for every sum (the *_long kernels).
//
// The backward kernel's teams walk over many rows and keep their columns' share of dgamma and dbeta in registers; a
// workgroup leaves one partial row of each in the workspace and param_sums_kernel adds those in a fixed order: no
// atomics, the same bits every time.
//
// Measured (a 1 GiB copy reaches 5.1 to 5.4 TB/s here): forward 65536 x 1024 float32 97 us = 5.5 TB/s, with both checkpoints
// 138 us = 4.9; backward 202 us = 5.3 TB/s from x with a mask, 124 us = 5.4 from the checkpoints; bf16 56 us = 4.8 forward,
// 104 us = 5.2 backward from x.  Backward 4096 x 16384, a workgroup of 1024 threads per row: float32 216 us = 5.0 from x,
// 146 us = 4.6 from the checkpoints; bf16 137 us = 3.9 and 109 us = 3.7 (one row in flight per compute unit).  bf16 rows of
// 1030 to 16384 columns, 33.5 million elements: forward 2.9 (6714 columns) to 5.2 TB/s (2048), backward 3.2 (5029, from
// checkpoints) to 5.3 (2048, from x); a row takes 3 to 16 waves that meet at its sums, and what holds the slow widths was not traced.
#include "act8.h"

namespace dlrm {

constexpr int kLongRow = 16384;      // longest row that stays in registers

struct NormFwd {
    const void *x;
    int64_t x_ld;
    const float *gamma, *beta;
    void *y;
    int64_t y_ld;
    float *mean, *rstd;
    dlrm_act8 xhat8, y8;
    float *y_max;
    int64_t M;
    int N;
    float eps;
    int relu;
};

struct NormBwd {
    const void *x;              // or NULL: xhat8
    int64_t x_ld;
    dlrm_act8 xhat8;
    const float *mean, *rstd, *gamma;
    const void *dy;
    int64_t dy_ld;
    const void *mask;           // y of the forward pass, or NULL
    int64_t mask_ld;
    dlrm_act8 mask8;
    void *dx;
    int64_t dx_ld;
    float *part_g, *part_b;     // [workgroups][part_stride] partial sums, or NULL
    int64_t part_stride;
    float *dx_max;
    int64_t M;
    int N;
};

// Teams of 256 lanes and more are a workgroup of as many waves as the row needs, TEAM lanes at most; the sums of waves that
// it does not have are zeros from the start.  bf16, us with a power of two of waves and with those that the row needs: 6672 x
// 5029 forward 61.5, 47.1, 14827 x 2263 backward from x 93.7, 75.6, 32577 x 1030 91.6, 79.2.
template <int TEAM>
__device__ inline int team_lanes() { return TEAM >= 256 ? (int)blockDim.x : TEAM; }
template <int TEAM, int SLOTS>
__device__ inline void clear_slots(float (&slots)[2][SLOTS]) {
    if constexpr (TEAM >= 256) {
        if (threadIdx.x < 2 * SLOTS) slots[threadIdx.x / SLOTS][threadIdx.x % SLOTS] = 0.f;
        __syncthreads();
    }
}
// sum over the TEAM lanes that share a row, the same bits in all of them.  Teams of several waves meet in `slot` (a float
// for each wave of the workgroup): the caller alternates between slots, so that a slot is written again only behind a later barrier.
template <int TEAM>
__device__ inline float team_sum(float x, float *slot) {
    if constexpr (TEAM <= 64) return group_sum<TEAM>(x);
    else {
        constexpr int W = TEAM / 64;
        slot += threadIdx.x / TEAM * W;
        x = group_sum<64>(x);
        if ((threadIdx.x & 63) == 0) slot[(threadIdx.x >> 6) % W] = x;
        __syncthreads();
        float t = slot[0];
#pragma unroll
        for (int w = 1; w < W; w++) t += slot[w];
        return t;
    }
}
template <int TEAM>
__device__ inline void team_sum2(float &x, float &y, float *slot) {     // slot: two floats a wave
    if constexpr (TEAM <= 64) {
        x = group_sum<TEAM>(x);
        y = group_sum<TEAM>(y);
    } else {
        constexpr int W = TEAM / 64;
        slot += threadIdx.x / TEAM * 2 * W;
        x = group_sum<64>(x);
        y = group_sum<64>(y);
        if ((threadIdx.x & 63) == 0) {
            slot[(threadIdx.x >> 6) % W] = x;
            slot[W + (threadIdx.x >> 6) % W] = y;
        }
        __syncthreads();
        x = slot[0];
        y = slot[W];
#pragma unroll
        for (int w = 1; w < W; w++) {
            x += slot[w];
            y += slot[W + w];
        }
    }
}

// VEC elements of gamma or beta, `none` where there is none; VEC sums to their place
template <int VEC>
__device__ inline void param_elems(const float *param, int c, int N, float (&v)[VEC], float none) {
#pragma unroll
    for (int h = 0; h < VEC; h += 4) {
        float q[4] = {none, none, none, none};
        if (param) elems_of<float, 4>(request_elems<float, 4>(param, c + h, N), c + h, N, q, none);
#pragma unroll
        for (int j = 0; j < 4; j++) v[h + j] = q[j];
    }
}
template <int VEC>
__device__ inline void store_sums(float *row, int c, int N, const float (&v)[VEC]) {
#pragma unroll
    for (int h = 0; h < VEC; h += 4) {
        const float q[4] = {v[h], v[h + 1], v[h + 2], v[h + 3]};
        store_elems<float, 4>(row, c + h, N, q);
    }
}

// largest magnitude of VEC elements as they are stored
template <typename T, int VEC>
__device__ inline void fold_elems(const float (&v)[VEC], int c, int N, float &vmax) {
    float t[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) t[j] = v[j];
    round_elems<T, VEC>(t);
#pragma unroll
    for (int j = 0; j < VEC; j++) vmax = fmaxf(vmax, c + j < N ? fabsf(t[j]) : 0.f);
}

__device__ inline float relu_keeping_nan(float y) { return y <= 0.f ? 0.f : y; }

template <typename T, int VEC>
__device__ inline void norm_output(const NormFwd &p, int64_t row, int c, bool live, const float (&xh)[VEC], const float (&g)[VEC],
                                   const float (&b)[VEC], float &vmax) {
    if (p.xhat8.d_codes)
        act8_store<VEC>(xh, p.xhat8.d_codes + row * p.xhat8.ld, p.xhat8.d_exps + row * p.xhat8.exps_ld, c, act8_blocks(p.N), live);
    float y[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) {
        y[j] = __builtin_fmaf(xh[j], g[j], b[j]);
        if (p.relu) y[j] = relu_keeping_nan(y[j]);
    }
    round_elems<T, VEC>(y);
    if (c + VEC > p.N) {
#pragma unroll
        for (int j = 0; j < VEC; j++) y[j] = c + j < p.N ? y[j] : 0.f;
    }
    if (p.y_max) fold_elems<T, VEC>(y, c, p.N, vmax);
    // (the checkpoint of the stored value, so that it equals what dlrm_act8_pack makes of y)
    if (p.y8.d_codes)
        act8_store<VEC>(y, p.y8.d_codes + row * p.y8.ld, p.y8.d_exps + row * p.y8.exps_ld, c, act8_blocks(p.N), live);
    if (live) store_elems<T, VEC>(static_cast<T *>(p.y) + row * p.y_ld, c, p.N, y);
}

template <typename T, int V, int TEAM>
__global__ __launch_bounds__((TEAM > 256 ? TEAM : 256)) void norm_fwd_kernel(NormFwd p) {
    constexpr int VEC = kWide<T>, kThreads = TEAM > 256 ? TEAM : 256, kTeams = kThreads / TEAM;
    __shared__ float slots[2][TEAM > 64 ? kThreads / 64 : 1];
    const int lanes = team_lanes<TEAM>(), lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    clear_slots<TEAM>(slots);
    float g[V][VEC], b[V][VEC];
#pragma unroll
    for (int v = 0; v < V; v++) {
        const int c = (v * lanes + lane) * VEC;
        param_elems<VEC>(p.gamma, c, p.N, g[v], 1.f);
        param_elems<VEC>(p.beta, c, p.N, b[v], 0.f);
    }
    float vmax = 0.f;
    for (int64_t r0 = (int64_t)blockIdx.x * kTeams; r0 < p.M; r0 += (int64_t)gridDim.x * kTeams) {
        const bool live = r0 + team < p.M;            // (the other teams of the wave go along: exchanges need every lane)
        const int64_t row = live ? r0 + team : p.M - 1;
        const T *xr = static_cast<const T *>(p.x) + row * p.x_ld;
        u32x4 raw[V];
        float x[V][VEC], s = 0.f, q = 0.f;
#pragma unroll
        for (int v = 0; v < V; v++) raw[v] = request_elems<T, VEC>(xr, (v * lanes + lane) * VEC, p.N);
#pragma unroll
        for (int v = 0; v < V; v++) elems_of<T, VEC>(raw[v], (v * lanes + lane) * VEC, p.N, x[v]);
#pragma unroll
        for (int v = 0; v < V; v++)
#pragma unroll
            for (int j = 0; j < VEC; j++) s += x[v][j];
        const float mean = team_sum<TEAM>(s, slots[0]) / (float)p.N;
#pragma unroll
        for (int v = 0; v < V; v++)
#pragma unroll
            for (int j = 0; j < VEC; j++) x[v][j] -= mean;
        if (p.N < V * lanes * VEC) {        // (uniform: a row that fills its team has no columns to take out)
#pragma unroll
            for (int v = 0; v < V; v++)
#pragma unroll
                for (int j = 0; j < VEC; j++) x[v][j] = (v * lanes + lane) * VEC + j < p.N ? x[v][j] : 0.f;
        }
#pragma unroll
        for (int v = 0; v < V; v++)
#pragma unroll
            for (int j = 0; j < VEC; j++) q = __builtin_fmaf(x[v][j], x[v][j], q);
        const float rstd = 1.f / sqrtf(team_sum<TEAM>(q, slots[1]) / (float)p.N + p.eps);
        if (lane == 0 && live) {
            if (p.mean) p.mean[row] = mean;
            if (p.rstd) p.rstd[row] = rstd;
        }
#pragma unroll
        for (int v = 0; v < V; v++) {
#pragma unroll
            for (int j = 0; j < VEC; j++) x[v][j] *= rstd;
            float top = 0.f;
            norm_output<T, VEC>(p, row, (v * lanes + lane) * VEC, live, x[v], g[v], b[v], top);
            if (live) vmax = fmaxf(vmax, top);      // (y may be x: a team without a row may have read a finished one)
        }
    }
    if (p.y_max) fold_absmax(vmax, p.y_max);
}

// rows beyond kLongRow: a workgroup of 1024 threads per row, the row read once for each sum and once for the output
template <typename T>
__global__ __launch_bounds__(1024) void norm_fwd_long_kernel(NormFwd p) {
    constexpr int VEC = kWide<T>;
    __shared__ float slots[2][16];
    const int first = threadIdx.x * VEC, width = act8_blocks(p.N) * kAct8Block;
    float vmax = 0.f;
    for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x) {
        const T *xr = static_cast<const T *>(p.x) + row * p.x_ld;
        float s = 0.f, q = 0.f;
        for (int c = first; c < p.N; c += 1024 * VEC) {
            float x[VEC];
            elems_of<T, VEC>(request_elems<T, VEC>(xr, c, p.N), c, p.N, x);
#pragma unroll
            for (int j = 0; j < VEC; j++) s += x[j];
        }
        const float mean = team_sum<1024>(s, slots[0]) / (float)p.N;
        for (int c = first; c < p.N; c += 1024 * VEC) {
            float x[VEC];
            elems_of<T, VEC>(request_elems<T, VEC>(xr, c, p.N), c, p.N, x);
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                const float d = c + j < p.N ? x[j] - mean : 0.f;
                q = __builtin_fmaf(d, d, q);
            }
        }
        const float rstd = 1.f / sqrtf(team_sum<1024>(q, slots[1]) / (float)p.N + p.eps);
        if (threadIdx.x == 0) {
            if (p.mean) p.mean[row] = mean;
            if (p.rstd) p.rstd[row] = rstd;
        }
        // (whole waves take the last turn together: a block's lanes exchange its largest magnitude)
        for (int base = 0; base < width; base += 1024 * VEC) {
            const int c = base + first;
            float x[VEC], g[VEC], b[VEC];
            elems_of<T, VEC>(request_elems<T, VEC>(xr, c, p.N), c, p.N, x);
#pragma unroll
            for (int j = 0; j < VEC; j++) x[j] = c + j < p.N ? (x[j] - mean) * rstd : 0.f;
            param_elems<VEC>(p.gamma, c, p.N, g, 1.f);
            param_elems<VEC>(p.beta, c, p.N, b, 0.f);
            norm_output<T, VEC>(p, row, c, true, x, g, b, vmax);
        }
    }
    if (p.y_max) fold_absmax(vmax, p.y_max);
}

// What VEC elements of a row's backward pass read, requested at once, and their xh and d
template <typename T, int VEC, bool FROM8, int MASK>
struct NormGradPiece {
    u32x4 x, dy, y;
    unsigned codes[VEC / 4], marks[VEC / 4];
    int e;
    __device__ inline void request(const NormBwd &p, int64_t row, int c) {
        const int blocks = act8_blocks(p.N);
        if constexpr (FROM8) {
            act8_load<VEC>(p.xhat8.d_codes + row * p.xhat8.ld, c, blocks, codes);
            e = p.xhat8.d_exps[row * p.xhat8.exps_ld + min(c / kAct8Block, blocks - 1)];
        } else x = request_elems<T, VEC>(static_cast<const T *>(p.x) + row * p.x_ld, c, p.N);
        dy = request_elems<T, VEC>(static_cast<const T *>(p.dy) + row * p.dy_ld, c, p.N);
        if constexpr (MASK == 1) y = request_elems<T, VEC>(static_cast<const T *>(p.mask) + row * p.mask_ld, c, p.N);
        else if constexpr (MASK == 2) act8_load<VEC>(p.mask8.d_codes + row * p.mask8.ld, c, blocks, marks);
    }
    __device__ inline void values(const NormBwd &p, int c, float mean, float rstd, float (&xh)[VEC], float (&d)[VEC]) const {
        if constexpr (FROM8) act8_values<VEC>(codes, act8_step(c < p.N ? e : 0), xh);
        else {
            elems_of<T, VEC>(x, c, p.N, xh, mean);
#pragma unroll
            for (int j = 0; j < VEC; j++) xh[j] = (xh[j] - mean) * rstd;
        }
        elems_of<T, VEC>(dy, c, p.N, d);
        if constexpr (MASK == 1) {
            float v[VEC];
            elems_of<T, VEC>(y, c, p.N, v);
#pragma unroll
            for (int j = 0; j < VEC; j++) d[j] = v[j] > 0.f ? d[j] : 0.f;
        } else if constexpr (MASK == 2) {
#pragma unroll
            for (int j = 0; j < VEC; j++) d[j] = act8_positive((marks[j / 4] >> (8 * (j % 4))) & 0xff) ? d[j] : 0.f;
        }
    }
};

// MASK: 0 no ReLU behind the norm, 1 its output, 2 the checkpoint of its output
template <typename T, int V, int TEAM, bool FROM8, int MASK>
__global__ __launch_bounds__((TEAM > 256 ? TEAM : 256)) void norm_bwd_kernel(NormBwd p) {
    constexpr int VEC = kWide<T>, kThreads = TEAM > 256 ? TEAM : 256, kTeams = kThreads / TEAM;
    __shared__ float slots[2][TEAM > 64 ? kThreads / 32 : 1];
    const int lanes = team_lanes<TEAM>(), lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    clear_slots<TEAM>(slots);
    // (workgroups of 8 waves and more have no registers for more than one piece: read again per row.  Held, one piece takes bf16
    // 14827 x 2263 from x from 119 to 93 us)
    constexpr bool kHoldGamma = TEAM < 512 || V == 1;
    float g[V][VEC], acc_g[V][VEC], acc_b[V][VEC];
#pragma unroll
    for (int v = 0; v < V; v++) {
        const int c = (v * lanes + lane) * VEC;
        if (kHoldGamma) param_elems<VEC>(p.gamma, c, p.N, g[v], 1.f);
#pragma unroll
        for (int j = 0; j < VEC; j++) acc_g[v][j] = acc_b[v][j] = 0.f;
    }
    float vmax = 0.f;
    int turn = 0;
    for (int64_t r0 = (int64_t)blockIdx.x * kTeams; r0 < p.M; r0 += (int64_t)gridDim.x * kTeams, turn ^= 1) {
        const bool live = r0 + team < p.M;
        // (a lane number that the compiler has to take as new per row: what it makes from it, addresses and conditions of every
        // piece, would otherwise be held from row to row and spill where the row takes 80 of 128 registers: 4096 x 16384 from
        // checkpoints 211 us instead of 146).  No float32 instance spills so; the four bf16 ones with a mask keep 1 to 5
        // registers a lane in scratch.
        int at = lane;
        if constexpr (TEAM == 1024 && V * VEC == 16) asm volatile("" : "+v"(at));
        const int64_t row = live ? r0 + team : p.M - 1;
        const float rstd = p.rstd[row], mean = FROM8 ? 0.f : p.mean[row];
        float xh[V][VEC], d[V][VEC], s1 = 0.f, s2 = 0.f;
        NormGradPiece<T, VEC, FROM8, MASK> piece[V];
#pragma unroll
        for (int v = 0; v < V; v++) piece[v].request(p, row, (v * lanes + at) * VEC);
#pragma unroll
        for (int v = 0; v < V; v++) piece[v].values(p, (v * lanes + at) * VEC, mean, rstd, xh[v], d[v]);
#pragma unroll
        for (int v = 0; v < V; v++) {
            if (!kHoldGamma) param_elems<VEC>(p.gamma, (v * lanes + at) * VEC, p.N, g[v], 1.f);
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                if (live) {
                    acc_b[v][j] += d[v][j];
                    acc_g[v][j] = __builtin_fmaf(d[v][j], xh[v][j], acc_g[v][j]);
                }
                d[v][j] *= g[v][j];
                s1 += d[v][j];
                s2 = __builtin_fmaf(d[v][j], xh[v][j], s2);
            }
        }
        team_sum2<TEAM>(s1, s2, slots[turn]);
        const float c1 = s1 / (float)p.N, c2 = s2 / (float)p.N;
#pragma unroll
        for (int v = 0; v < V; v++) {
            const int c = (v * lanes + at) * VEC;
#pragma unroll
            for (int j = 0; j < VEC; j++) d[v][j] = rstd * (d[v][j] - c1 - xh[v][j] * c2);
            if (p.dx_max && live) fold_elems<T, VEC>(d[v], c, p.N, vmax);
            if (live) store_elems<T, VEC>(static_cast<T *>(p.dx) + row * p.dx_ld, c, p.N, d[v]);
        }
    }
    if (p.dx_max) fold_absmax(vmax, p.dx_max);
    if (p.part_g == nullptr && p.part_b == nullptr) return;
    // the teams' columns, added in team order
    if constexpr (kTeams > 1) {
        constexpr int W = V * TEAM * VEC;
        __shared__ float meet[kTeams * W];
#pragma unroll
        for (int which = 0; which < 2; which++) {
            float *part = which == 0 ? p.part_g : p.part_b;
            __syncthreads();
#pragma unroll
            for (int v = 0; v < V; v++)
#pragma unroll
                for (int j = 0; j < VEC; j++)
                    meet[team * W + (v * TEAM + lane) * VEC + j] = which == 0 ? acc_g[v][j] : acc_b[v][j];
            __syncthreads();
            if (part)
                for (int c = threadIdx.x; c < p.N; c += kThreads) {
                    float t = meet[c];
                    for (int k = 1; k < kTeams; k++) t += meet[k * W + c];
                    part[(int64_t)blockIdx.x * p.part_stride + c] = t;
                }
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; v++) {
            const int c = (v * lanes + lane) * VEC;
            if (p.part_g) store_sums<VEC>(p.part_g + (int64_t)blockIdx.x * p.part_stride, c, p.N, acc_g[v]);
            if (p.part_b) store_sums<VEC>(p.part_b + (int64_t)blockIdx.x * p.part_stride, c, p.N, acc_b[v]);
        }
    }
}

// rows beyond kLongRow.  Parameter gradients: a thread per 16 bytes of columns walks over a share of the rows (before dx is written:
// dx may be dy's own memory) ...
template <typename T, bool FROM8, int MASK>
__global__ __launch_bounds__(256) void norm_bwd_long_params_kernel(NormBwd p, int64_t rows_per_part) {
    constexpr int VEC = kWide<T>;
    const int c = (blockIdx.x * 256 + threadIdx.x) * VEC;
    if (c >= p.N) return;
    const int64_t begin = blockIdx.y * rows_per_part;
    const int64_t end = begin + rows_per_part < p.M ? begin + rows_per_part : p.M;
    float ag[VEC], ab[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) ag[j] = ab[j] = 0.f;
    for (int64_t row = begin; row < end; row++) {
        float xh[VEC], d[VEC];
        NormGradPiece<T, VEC, FROM8, MASK> piece;
        piece.request(p, row, c);
        piece.values(p, c, FROM8 ? 0.f : p.mean[row], p.rstd[row], xh, d);
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            ab[j] += d[j];
            ag[j] = __builtin_fmaf(d[j], xh[j], ag[j]);
        }
    }
    if (p.part_g) store_sums<VEC>(p.part_g + blockIdx.y * p.part_stride, c, p.N, ag);
    if (p.part_b) store_sums<VEC>(p.part_b + blockIdx.y * p.part_stride, c, p.N, ab);
}
// ... and dx with a workgroup per row, which is read once for the sums and once for the output
template <typename T, bool FROM8, int MASK>
__global__ __launch_bounds__(1024) void norm_bwd_long_kernel(NormBwd p) {
    constexpr int VEC = kWide<T>;
    __shared__ float slots[2][32];
    float vmax = 0.f;
    int turn = 0;
    for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x, turn ^= 1) {
        const float rstd = p.rstd[row], mean = FROM8 ? 0.f : p.mean[row];
        float xh[VEC], d[VEC], g[VEC], s1 = 0.f, s2 = 0.f;
        for (int c = threadIdx.x * VEC; c < p.N; c += 1024 * VEC) {
            NormGradPiece<T, VEC, FROM8, MASK> piece;
            piece.request(p, row, c);
            piece.values(p, c, mean, rstd, xh, d);
            param_elems<VEC>(p.gamma, c, p.N, g, 1.f);
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                const float gd = d[j] * g[j];
                s1 += gd;
                s2 = __builtin_fmaf(gd, xh[j], s2);
            }
        }
        team_sum2<1024>(s1, s2, slots[turn]);
        const float c1 = s1 / (float)p.N, c2 = s2 / (float)p.N;
        for (int c = threadIdx.x * VEC; c < p.N; c += 1024 * VEC) {
            NormGradPiece<T, VEC, FROM8, MASK> piece;
            piece.request(p, row, c);
            piece.values(p, c, mean, rstd, xh, d);
            param_elems<VEC>(p.gamma, c, p.N, g, 1.f);
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                const float gd = d[j] * g[j];
                d[j] = rstd * (gd - c1 - xh[j] * c2);
            }
            if (p.dx_max) fold_elems<T, VEC>(d, c, p.N, vmax);
            store_elems<T, VEC>(static_cast<T *>(p.dx) + row * p.dx_ld, c, p.N, d);
        }
    }
    if (p.dx_max) fold_absmax(vmax, p.dx_max);
}

// out[c] = sum over the partial rows of a column, for both gradients: a workgroup takes 32 columns, its 32 groups of 32
// lanes every 32nd partial row, and the groups meet in LDS in a fixed order
struct ParamSums {
    const float *part[2];
    float *out[2];
    int64_t stride;
    int parts, N;
};
__global__ __launch_bounds__(1024) void param_sums_kernel(ParamSums p) {
    __shared__ float meet[32][33];
    const int e = threadIdx.x & 31, q = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + e;
    const float *part = p.part[blockIdx.y];
    float *out = p.out[blockIdx.y];
    if (out == nullptr) return;
    float a = 0.f;
    if (c < p.N) {
        int k = q;
        for (; k + 224 < p.parts; k += 256) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; u++) v[u] = part[(k + 32 * u) * p.stride + c];
#pragma unroll
            for (int u = 0; u < 8; u++) a += v[u];
        }
        for (; k < p.parts; k += 32) a += part[k * p.stride + c];
    }
    meet[q][e] = a;
    __syncthreads();
    if (q == 0 && c < p.N) {
        for (int k = 1; k < 32; k++) a += meet[k][e];
        out[c] = a;
    }
}

// ---- launches.
static int row_threads(int N, int elems) { return (int)ceil_div(N, 64 * elems) * 64; }

// Most partial rows that a backward launch leaves, which are its workgroups: as many whole ones as give a compute unit 1024
// threads, or 512 where a lane has more than one piece of float32 (us for 256 / 512 / 1024 workgroups): of 256 threads, float32
// 131072 x 256 165 / 102 / 106 from x, 146 / 86 / 67 from checkpoints, 8192 x 1024 from x 24.3 / 21.7 / 23.7, bf16 65536 x
// 1024 from x 142 with 512, 104 with 1024; of 512, bf16 8192 x 4096 79 / 61 / 66, float32 4096 x 8192 112 / 119 / 129; of 1024,
// bf16 61 / 66 / 81.  Requesting the next row ahead of a row's sums gained nothing to 7 % from x and cost as much from
// checkpoints: other waves cover the wait.
static int64_t norm_bwd_cap(int N, bool bf16) {
    if (N > kLongRow) return 64;
    const int threads = N <= (bf16 ? 1024 : 2048) ? 256 : row_threads(N, bf16 && N <= 8192 ? 8 : 16);
    return 256 * ((!bf16 && N > 256 && N <= 8192 ? 512 : 1024) / threads);
}
static int64_t norm_bwd_parts(int64_t M, int N, bool bf16) {
    const int64_t cap = norm_bwd_cap(N, bf16);
    return M < cap ? (M < 1 ? 1 : M) : cap;
}
// ... of either type, which a workspace holds
static int64_t norm_bwd_parts(int64_t M, int N) {
    const int64_t a = norm_bwd_parts(M, N, false), b = norm_bwd_parts(M, N, true);
    return a > b ? a : b;
}

// Forward workgroups at most, each with several rows: as many as give a compute unit 4096 threads, 2048 where a lane has four
// pieces of float32 (us, 2048 / 4096 / 8192 workgroups of 256 threads: bf16 65536 x 1024 66.6 / 56.2 / 56.7, 32768 x 512 16.6 /
// 16.2 / 18.2, float32 262144 x 256 120 / 105 / 99; 16384 x 1024 24.2 / 25.9 / 25.7, 65536 x 1024 97.7 / 96.0 / 92.6).  Lanes
// with 16 elements have the registers for 1024 threads at a time, and a second round that is not full costs more than second
// rows do: 8160 x 514 float32 16.1 us with 2040 workgroups, 13.6 with 1024, 349 x 12000 14.7 and 12.4.
template <typename T, int V, int TEAM>
static void launch_fwd(const NormFwd &p, hipStream_t s) {
    // (lanes with 16 elements: 5 or 6 waves leave places free beside one another that 2 x 8 fill, 6672 x 5029 float32 73 or 78
    // against 65 us)
    const int threads = TEAM == 512 && V * kWide<T> == 16 ? 512 : TEAM >= 256 ? row_threads(p.N, V * kWide<T>) : 256;
    const int64_t want = TEAM >= 256 ? p.M : ceil_div(p.M, 256 / TEAM), at_once = 256 * (1024 / threads);
    const int64_t cap = V * kWide<T> == 16 && want <= 2 * at_once ? at_once : (V <= 2 ? 4 : 2) * at_once;
    hipLaunchKernelGGL((norm_fwd_kernel<T, V, TEAM>), dim3((unsigned)(want < cap ? want : cap)), dim3(threads), 0, s, p);
}

template <typename T, int V, int TEAM, bool FROM8, int MASK>
static void launch_bwd_as(const NormBwd &p, unsigned grid, hipStream_t s) {
    const int threads = TEAM >= 256 ? row_threads(p.N, V * kWide<T>) : 256;
    hipLaunchKernelGGL((norm_bwd_kernel<T, V, TEAM, FROM8, MASK>), dim3(grid), dim3(threads), 0, s, p);
}
template <typename T, int V, int TEAM>
static void launch_bwd(NormBwd p, float *dgamma, float *dbeta, int64_t *parts, hipStream_t s) {
    constexpr int kTeams = TEAM > 256 ? 1 : 256 / TEAM;
    const int64_t want = ceil_div(p.M, kTeams), cap = norm_bwd_parts(p.M, p.N, sizeof(T) == 2);
    const unsigned grid = (unsigned)(want < cap ? want : cap);
    *parts = grid;
    if (grid == 1) {            // a single workgroup's sums are the gradients
        p.part_g = dgamma;
        p.part_b = dbeta;
    }
    const int mask = p.mask8.d_codes ? 2 : (p.mask ? 1 : 0);
    if (p.x == nullptr) {
        if (mask == 0) launch_bwd_as<T, V, TEAM, true, 0>(p, grid, s);
        else if (mask == 1) launch_bwd_as<T, V, TEAM, true, 1>(p, grid, s);
        else launch_bwd_as<T, V, TEAM, true, 2>(p, grid, s);
    } else {
        if (mask == 0) launch_bwd_as<T, V, TEAM, false, 0>(p, grid, s);
        else if (mask == 1) launch_bwd_as<T, V, TEAM, false, 1>(p, grid, s);
        else launch_bwd_as<T, V, TEAM, false, 2>(p, grid, s);
    }
}

template <typename T, bool FROM8, int MASK>
static void launch_bwd_long_as(const NormBwd &p, int64_t parts, hipStream_t s) {
    if (p.part_g || p.part_b)
        hipLaunchKernelGGL((norm_bwd_long_params_kernel<T, FROM8, MASK>), dim3((unsigned)ceil_div(p.N, 256 * kWide<T>), (unsigned)parts),
                           dim3(256), 0, s, p, ceil_div(p.M, parts));
    hipLaunchKernelGGL((norm_bwd_long_kernel<T, FROM8, MASK>), dim3((unsigned)(p.M < 512 ? p.M : 512)), dim3(1024), 0, s, p);
}
template <typename T>
static void launch_bwd_long(NormBwd p, float *dgamma, float *dbeta, int64_t *parts, hipStream_t s) {
    const int64_t n = ceil_div(p.M, ceil_div(p.M, norm_bwd_parts(p.M, p.N)));      // (every part has a row)
    *parts = n;
    if (n == 1) {
        p.part_g = dgamma;
        p.part_b = dbeta;
    }
    const int mask = p.mask8.d_codes ? 2 : (p.mask ? 1 : 0);
    if (p.x == nullptr) {
        if (mask == 0) launch_bwd_long_as<T, true, 0>(p, n, s);
        else if (mask == 1) launch_bwd_long_as<T, true, 1>(p, n, s);
        else launch_bwd_long_as<T, true, 2>(p, n, s);
    } else {
        if (mask == 0) launch_bwd_long_as<T, false, 0>(p, n, s);
        else if (mask == 1) launch_bwd_long_as<T, false, 1>(p, n, s);
        else launch_bwd_long_as<T, false, 2>(p, n, s);
    }
}

// One team shape per width: the smallest that holds the row with up to 16 float32 or 8 bf16 elements a lane.  More elements
// cost registers and with them waves in flight: bf16 backward 65536 x 1024 from x 168 us with 16 a lane, 104 us with 8.
// Four lanes where nothing needs the 8 lanes of a float32 checkpoint's block together (HALF): 4194304 x 16 forward
// float32 109 us with 4, 154 with 8, bf16 94 and 164, its backward from x 142 and 249.
#define DLRM_NORM_SHAPES(T, N, HALF, CALL, LONG, ...)                          \
    do {                                                                       \
        constexpr int W = kWide<T>, F = W / 4;                                 \
        if ((N) <= 4 * W && (HALF)) CALL<T, 1, 4>(__VA_ARGS__);                \
        else if ((N) <= 8 * W) CALL<T, 1, 8>(__VA_ARGS__);                          \
        else if ((N) <= 16 * W) CALL<T, 1, 16>(__VA_ARGS__);                   \
        else if ((N) <= 32 * W) CALL<T, 1, 32>(__VA_ARGS__);                   \
        else if ((N) <= 64 * W) CALL<T, 1, 64>(__VA_ARGS__);                   \
        else if ((N) <= 512) CALL<T, 2 / F, 64>(__VA_ARGS__);                  \
        else if ((N) <= 1024) CALL<T, 4 / (F * F), 64 * F>(__VA_ARGS__);       \
        else if ((N) <= 2048) CALL<T, 4 / (F * F), 128 * F>(__VA_ARGS__);      \
        else if ((N) <= 4096) CALL<T, 4 / (F * F), 256 * F>(__VA_ARGS__);      \
        else if ((N) <= 8192) CALL<T, 4 / (F * F), 512 * F>(__VA_ARGS__);      \
        else if ((N) <= kLongRow) CALL<T, 4 / F, 1024>(__VA_ARGS__);           \
        else LONG<T>(__VA_ARGS__);                                             \
    } while (0)

template <typename T>
static void launch_fwd_long(const NormFwd &p, hipStream_t s) {
    hipLaunchKernelGGL((norm_fwd_long_kernel<T>), dim3((unsigned)(p.M < 512 ? p.M : 512)), dim3(1024), 0, s, p);
}

template <typename T>
static void norm_fwd(const NormFwd &p, hipStream_t s) {
    const bool half = sizeof(T) == 2 || (p.xhat8.d_codes == nullptr && p.y8.d_codes == nullptr);
    DLRM_NORM_SHAPES(T, p.N, half, launch_fwd, launch_fwd_long, p, s);
}
template <typename T>
static void norm_bwd(const NormBwd &p, float *dgamma, float *dbeta, int64_t *parts, hipStream_t s) {
    DLRM_NORM_SHAPES(T, p.N, true, launch_bwd, launch_bwd_long, p, dgamma, dbeta, parts, s);
}

static bool rows_aligned(const void *p, int size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }

static int norm_shape(int64_t M, int32_t N, int32_t dtype) {
    DLRM_REQUIRE(M >= 0 && N >= 1 && N <= (1 << 30), "bad shape: %lld rows of %d columns", (long long)M, N);
    DLRM_REQUIRE(dtype == DLRM_F32 || dtype == DLRM_BF16, "dtype %d is neither DLRM_F32 nor DLRM_BF16", dtype);
    return DLRM_OK;
}

}  // namespace dlrm

using namespace dlrm;

extern "C" int dlrm_layer_norm_forward(const dlrm_layer_norm *l, dlrm_stream_t stream) {
    DLRM_REQUIRE(l != nullptr, "layer_norm descriptor is NULL");
    if (int rc = norm_shape(l->M, l->N, l->dtype)) return rc;
    DLRM_REQUIRE(l->act == DLRM_ACT_NONE || l->act == DLRM_ACT_RELU, "act must be DLRM_ACT_NONE or DLRM_ACT_RELU, got %d", l->act);
    DLRM_REQUIRE(l->eps >= 0.f, "eps must not be negative");
    if (l->M == 0) return DLRM_OK;
    const int size = l->dtype == DLRM_F32 ? 4 : 2;
    DLRM_REQUIRE(l->d_x && l->d_y, "NULL operand");
    DLRM_REQUIRE(l->x_ld >= l->N && l->y_ld >= l->N, "leading dimension too small");
    DLRM_REQUIRE(rows_aligned(l->d_x, size) && rows_aligned(l->d_y, size), "operand is not aligned to its elements");
    if (l->xhat8.d_codes)
        if (int rc = act8_check(&l->xhat8, l->N, "checkpoint of the normalised rows")) return rc;
    if (l->y8.d_codes)
        if (int rc = act8_check(&l->y8, l->N, "checkpoint of the output")) return rc;
    NormFwd p{};
    p.x = l->d_x; p.x_ld = l->x_ld; p.gamma = l->d_gamma; p.beta = l->d_beta; p.y = l->d_y; p.y_ld = l->y_ld;
    p.mean = l->d_mean; p.rstd = l->d_rstd; p.xhat8 = l->xhat8; p.y8 = l->y8; p.y_max = l->d_y_absmax;
    p.M = l->M; p.N = l->N; p.eps = l->eps; p.relu = l->act == DLRM_ACT_RELU;
    if (l->dtype == DLRM_F32) norm_fwd<float>(p, as_stream(stream));
    else norm_fwd<uint16_t>(p, as_stream(stream));
    DLRM_LAUNCH_CHECK();
    return DLRM_OK;
}

extern "C" int dlrm_layer_norm_backward_workspace_bytes(int64_t M, int32_t N, size_t *bytes) {
    DLRM_REQUIRE(bytes != nullptr, "bytes is NULL");
    if (int rc = norm_shape(M, N, DLRM_F32)) return rc;
    *bytes = sizeof(float) * 2 * (size_t)norm_bwd_parts(M, N) * (size_t)N;
    return DLRM_OK;
}

extern "C" int dlrm_layer_norm_backward(const dlrm_layer_norm_bwd *l, void *d_workspace, size_t workspace_bytes,
                                        dlrm_stream_t stream) {
    DLRM_REQUIRE(l != nullptr, "layer_norm_bwd descriptor is NULL");
    if (int rc = norm_shape(l->M, l->N, l->dtype)) return rc;
    const int size = l->dtype == DLRM_F32 ? 4 : 2;
    const bool params = l->d_dgamma != nullptr || l->d_dbeta != nullptr;
    NormBwd p{};
    int64_t parts = 0;
    hipStream_t s = as_stream(stream);
    if (l->M > 0) {
        DLRM_REQUIRE(l->d_dy && l->d_dx && l->d_rstd, "NULL operand");
        DLRM_REQUIRE((l->d_x != nullptr) != (l->xhat8.d_codes != nullptr),
                     "exactly one of the input and the checkpoint of the normalised rows must be given");
        DLRM_REQUIRE(l->d_x == nullptr || l->d_mean != nullptr, "the input needs the rows' means");
        DLRM_REQUIRE(l->d_relu_mask == nullptr || l->relu_mask8.d_codes == nullptr, "two ReLU masks given");
        DLRM_REQUIRE(l->dy_ld >= l->N && l->dx_ld >= l->N && (l->d_x == nullptr || l->x_ld >= l->N) &&
                         (l->d_relu_mask == nullptr || l->relu_mask_ld >= l->N),
                     "leading dimension too small");
        DLRM_REQUIRE(rows_aligned(l->d_x, size) && rows_aligned(l->d_dy, size) && rows_aligned(l->d_dx, size) &&
                         rows_aligned(l->d_relu_mask, size),
                     "operand is not aligned to its elements");
        if (l->xhat8.d_codes)
            if (int rc = act8_check(&l->xhat8, l->N, "checkpoint of the normalised rows")) return rc;
        if (l->relu_mask8.d_codes)
            if (int rc = act8_check(&l->relu_mask8, l->N, "checkpoint of the output")) return rc;
        if (params) {
            size_t need = 0;
            if (int rc = dlrm_layer_norm_backward_workspace_bytes(l->M, l->N, &need)) return rc;
            DLRM_REQUIRE(d_workspace != nullptr && workspace_bytes >= need, "workspace too small: %zu < %zu", workspace_bytes, need);
            DLRM_REQUIRE(reinterpret_cast<uintptr_t>(d_workspace) % 16 == 0, "workspace must be 16-byte aligned");
        }
        p.x = l->d_x; p.x_ld = l->x_ld; p.xhat8 = l->xhat8; p.mean = l->d_mean; p.rstd = l->d_rstd; p.gamma = l->d_gamma;
        p.dy = l->d_dy; p.dy_ld = l->dy_ld; p.mask = l->d_relu_mask; p.mask_ld = l->relu_mask_ld; p.mask8 = l->relu_mask8;
        p.dx = l->d_dx; p.dx_ld = l->dx_ld; p.dx_max = l->d_dx_absmax; p.M = l->M; p.N = l->N;
        float *ws = static_cast<float *>(d_workspace);
        p.part_stride = l->N;
        p.part_g = l->d_dgamma ? ws : nullptr;
        p.part_b = l->d_dbeta ? ws + norm_bwd_parts(l->M, l->N) * l->N : nullptr;
        if (l->dtype == DLRM_F32) norm_bwd<float>(p, l->d_dgamma, l->d_dbeta, &parts, s);
        else norm_bwd<uint16_t>(p, l->d_dgamma, l->d_dbeta, &parts, s);
        DLRM_LAUNCH_CHECK();
        if (parts == 1) return DLRM_OK;
    }
    if (!params) return DLRM_OK;
    ParamSums q{};                      // (no rows: the sums over none of them are zero)
    q.part[0] = p.part_g; q.part[1] = p.part_b; q.out[0] = l->d_dgamma; q.out[1] = l->d_dbeta;
    q.stride = l->N; q.parts = (int)parts; q.N = l->N;
    hipLaunchKernelGGL(param_sums_kernel, dim3((unsigned)ceil_div(l->N, 32), 2), dim3(1024), 0, s, q);
    DLRM_LAUNCH_CHECK();
    return DLRM_OK;
}
