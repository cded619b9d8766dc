// Activations into 8-bit checkpoints and back (format and rounding: act8.h).
//
// Both directions are one pass bound by memory: float32 in or out 4 bytes an element, the checkpoint 1 1/32.  A row is
// shared by the smallest power of two of lanes that covers it (at most a wave) and every lane moves 16 bytes of the
// activation per step, so the 32 columns of a block sit in 8 (float32) or 4 (bf16) neighbouring lanes and its largest
// magnitude is three (two) exchanges on the vector unit's own lane paths.
#include "act8.h"

namespace dlrm {

int act8_check(const dlrm_act8 *a, int cols, const char *what) {
    DLRM_REQUIRE(a->d_codes != nullptr && a->d_exps != nullptr, "%s: NULL codes or exponents", what);
    DLRM_REQUIRE(cols <= (1 << 30), "%s: %d columns are more than 2^30", what, cols);
    const int64_t blocks = act8_blocks(cols);
    DLRM_REQUIRE(reinterpret_cast<uintptr_t>(a->d_codes) % 16 == 0 && a->ld % 16 == 0,
                 "%s: code rows must start on 16-byte boundaries (leading dimension %lld)", what, (long long)a->ld);
    DLRM_REQUIRE(a->ld >= blocks * kAct8Block && a->exps_ld >= blocks,
                 "%s: leading dimensions %lld (codes) and %lld (exponents) are too small for %d columns", what, (long long)a->ld,
                 (long long)a->exps_ld, cols);
    return DLRM_OK;
}

struct Act8Pass {
    const void *src;
    void *dst;
    int64_t ld;            // of the activation
    int8_t *codes;
    int64_t codes_ld;
    uint8_t *exps;
    int64_t exps_ld;
    int64_t rows;
    int cols, blocks;
    int lanes_log2;        // lanes that share a row: 2^lanes_log2, a wave at most
    int chunks;            // of four steps in a row that is longer than one
};

// S: steps that a lane takes per row, 4 meaning "four at a time": longer rows are cut into chunks of four steps
// (blocks do not depend on one another), which spread over the grid's second axis where there are few rows: 42 x 14764
// float32 there and back 31.6 us with a wave for a whole row, 13.3 this way (two launches from the host).  With S = 1 or 2 a
// lane takes four or two rows at a time, so that four loads are in flight per lane whatever the row's width.
template <typename T, int S>
__global__ __launch_bounds__(256) void act8_pack_kernel(Act8Pass p) {
    constexpr int VEC = kWide<T>, R = 4 / S;
    const int lane = threadIdx.x & 63, lanes = 1 << p.lanes_log2;
    const int first = (lane & (lanes - 1)) * VEC, step = lanes * VEC;
    const int rows_per_wave = 64 >> p.lanes_log2;
    const int64_t n_waves = (int64_t)gridDim.x * 4;
    for (int64_t r0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * rows_per_wave * R; r0 < p.rows; r0 += n_waves * rows_per_wave * R)
    for (int chunk = blockIdx.y; chunk < p.chunks; chunk += gridDim.y) {
        // (every lane of the wave takes every step: the exchanges inside act8_store need the neighbours)
        const int base = chunk * (S * step) + first;
        u32x4 x[4];
        int64_t row[R];
        bool live[R];
#pragma unroll
        for (int k = 0; k < R; k++) {
            row[k] = r0 + k * rows_per_wave + (lane >> p.lanes_log2);
            live[k] = row[k] < p.rows;
            if (!live[k]) row[k] = p.rows - 1;
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
            x[u] = request_elems<T, VEC>(static_cast<const T *>(p.src) + row[u / S] * p.ld, base + (u % S) * step, p.cols);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int c = base + (u % S) * step;
            float v[VEC];
            elems_of<T, VEC>(x[u], c, p.cols, v);
            act8_store<VEC>(v, p.codes + row[u / S] * p.codes_ld, p.exps + row[u / S] * p.exps_ld, c, p.blocks, live[u / S]);
        }
    }
}

template <typename T, int S>
__global__ __launch_bounds__(256) void act8_unpack_kernel(Act8Pass p) {
    constexpr int VEC = kWide<T>, R = 4 / S;
    const int lane = threadIdx.x & 63, lanes = 1 << p.lanes_log2;
    const int first = (lane & (lanes - 1)) * VEC, step = lanes * VEC;
    const int rows_per_wave = 64 >> p.lanes_log2;
    const int64_t n_waves = (int64_t)gridDim.x * 4;
    for (int64_t r0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * rows_per_wave * R; r0 < p.rows; r0 += n_waves * rows_per_wave * R)
    for (int chunk = blockIdx.y; chunk < p.chunks; chunk += gridDim.y) {
        const int base = chunk * (S * step) + first;
        unsigned w[4][VEC / 4];
        int e[4];
        int64_t row[R];
#pragma unroll
        for (int k = 0; k < R; k++) row[k] = r0 + k * rows_per_wave + (lane >> p.lanes_log2);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int64_t r = row[u / S] < p.rows ? row[u / S] : p.rows - 1;
            const int c = base + (u % S) * step;
            act8_load<VEC>(p.codes + r * p.codes_ld, c, p.blocks, w[u]);
            e[u] = p.exps[r * p.exps_ld + min(c / kAct8Block, p.blocks - 1)];
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int c = base + (u % S) * step;
            float v[VEC];
            act8_values<VEC>(w[u], act8_step(e[u]), v);
            if (c < p.cols && row[u / S] < p.rows) store_elems<T, VEC>(static_cast<T *>(p.dst) + row[u / S] * p.ld, c, p.cols, v);
        }
    }
}

// lanes per row (a block's stay together), steps of a lane per row, chunks of a row and workgroups
static dim3 act8_grid(Act8Pass &p, int vec, int *steps) {
    const int per_row = p.blocks * (kAct8Block / vec);
    p.lanes_log2 = vec == 8 ? 2 : 3;
    while (p.lanes_log2 < 6 && (1 << p.lanes_log2) < per_row) p.lanes_log2++;
    const int s = (per_row + (1 << p.lanes_log2) - 1) >> p.lanes_log2;
    *steps = s <= 2 ? s : 4;
    p.chunks = (int)ceil_div(s, *steps);
    const int64_t want = ceil_div(p.rows, (int64_t)4 * (64 >> p.lanes_log2) * (4 / *steps));
    const unsigned gx = (unsigned)(want < 4096 ? want : 4096), gy = 4096 / gx;
    return dim3(gx, gy < (unsigned)p.chunks ? gy : (unsigned)p.chunks);
}

static int act8_args(const void *d_x, int32_t dtype, int64_t rows, int32_t cols, int64_t x_ld, const dlrm_act8 *a) {
    DLRM_REQUIRE(a != nullptr, "checkpoint descriptor is NULL");
    DLRM_REQUIRE(dtype == DLRM_F32 || dtype == DLRM_BF16, "dtype %d is neither DLRM_F32 nor DLRM_BF16", dtype);
    DLRM_REQUIRE(rows >= 0 && cols >= 1 && cols <= (1 << 30) && x_ld >= cols, "bad shape: %lld rows of %d columns, leading dimension %lld",
                 (long long)rows, cols, (long long)x_ld);
    DLRM_REQUIRE(rows == 0 || d_x != nullptr, "NULL activation");
    DLRM_REQUIRE(reinterpret_cast<uintptr_t>(d_x) % (dtype == DLRM_F32 ? 4 : 2) == 0, "activation is not aligned to its elements");
    return rows == 0 ? DLRM_OK : act8_check(a, cols, "checkpoint");
}

static Act8Pass act8_pass(const dlrm_act8 *a, int64_t rows, int cols, int64_t x_ld) {
    Act8Pass p{};
    p.ld = x_ld; p.codes = a->d_codes; p.codes_ld = a->ld; p.exps = a->d_exps; p.exps_ld = a->exps_ld;
    p.rows = rows; p.cols = cols; p.blocks = act8_blocks(cols);
    return p;
}

}  // namespace dlrm

using namespace dlrm;

#define DLRM_ACT8_LAUNCH(KERNEL, T)                                                                       \
    do {                                                                                                  \
        int steps = 1;                                                                                    \
        const dim3 grid = act8_grid(p, kWide<T>, &steps);                                             \
        if (steps == 1) hipLaunchKernelGGL((KERNEL<T, 1>), grid, dim3(256), 0, as_stream(stream), p);      \
        else if (steps == 2) hipLaunchKernelGGL((KERNEL<T, 2>), grid, dim3(256), 0, as_stream(stream), p); \
        else hipLaunchKernelGGL((KERNEL<T, 4>), grid, dim3(256), 0, as_stream(stream), p);          \
        DLRM_LAUNCH_CHECK();                                                                              \
    } while (0)

extern "C" int dlrm_act8_pack(const void *d_x, int32_t dtype, int64_t rows, int32_t cols, int64_t x_ld, const dlrm_act8 *out,
                              dlrm_stream_t stream) {
    if (int rc = act8_args(d_x, dtype, rows, cols, x_ld, out)) return rc;
    if (rows == 0) return DLRM_OK;
    Act8Pass p = act8_pass(out, rows, cols, x_ld);
    p.src = d_x;
    if (dtype == DLRM_F32) DLRM_ACT8_LAUNCH(act8_pack_kernel, float);
    else DLRM_ACT8_LAUNCH(act8_pack_kernel, uint16_t);
    return DLRM_OK;
}

extern "C" int dlrm_act8_unpack(const dlrm_act8 *a, int64_t rows, int32_t cols, void *d_x, int32_t dtype, int64_t x_ld,
                                dlrm_stream_t stream) {
    if (int rc = act8_args(d_x, dtype, rows, cols, x_ld, a)) return rc;
    if (rows == 0) return DLRM_OK;
    Act8Pass p = act8_pass(a, rows, cols, x_ld);
    p.dst = d_x;
    if (dtype == DLRM_F32) DLRM_ACT8_LAUNCH(act8_unpack_kernel, float);
    else DLRM_ACT8_LAUNCH(act8_unpack_kernel, uint16_t);
    return DLRM_OK;
}
