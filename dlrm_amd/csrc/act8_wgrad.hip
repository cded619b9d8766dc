// Weight gradient from an 8-bit checkpoint of the layer's input: dW = dz^T x [N,K], reduction over the batch.
//
// A code times its block's power-of-two step is an exact bf16 number, so x enters v_mfma_f32_32x32x16_bf16 as it is and
// only dz is cut into three bf16 pieces (common.h: split3_pair): three terms instead of the six that two float32 operands
// take, every product exact in float32, float32 accumulation -- the accuracy of the bf16x3 evaluation at half its matrix
// work and with a quarter of x's bytes.
//
// A 256-thread workgroup owns TM columns of dz x TN columns of x (TM, TN in {128, 64}; 2 x 2 waves, each with
// (TM/64) x (TN/64) MFMA tiles) for a range of rows and walks it in steps of 32 rows: the next step's operands are
// requested into registers, the present step's MFMAs run out of one LDS stage, then the requested operands are split /
// widened to bf16 and written to the other stage.  Both operands have the reduction index as their row, so LDS holds
// [32 rows][TM or TN] bf16 planes and the fragments come out of the transposing read ds_read_b64_tr_b16.  Row ranges
// leave partial sums that the caller adds in a fixed order.
#include "act8.h"

namespace dlrm {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr int kStepRows = 32;

// byte offset of 16-byte chunk ch of row `row` in a [32][R] bf16 plane.  The transposing read takes four rows x 64 bytes
// per 32 lanes; the exchange of chunks puts those on different banks.
template <int R>
__device__ inline int plane_off(int row, int ch) {
    if constexpr (R == 64) return 128 * row + 16 * (ch ^ ((((row >> 1) & 1) << 2) | ((row >> 2) & 3)));
    else return 2 * R * row + 16 * (ch ^ (((row & 3) << 2) | ((row >> 2) & 3)));
}

// reduction rows 16 slice + 8 (lane / 32) .. +7 of column base + lane % 32
template <int R>
__device__ inline bf16x8 plane_frag(const unsigned char *plane, int base, int slice) {
    const int lane = threadIdx.x & 63;
    const int li = lane & 15, g = lane >> 4;
    const int ch = (base >> 3) + 2 * (g & 1) + ((li & 3) >> 1);
    const int row = 16 * slice + 8 * (g >> 1) + (li >> 2);
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(plane + plane_off<R>(row, ch) + 8 * (li & 1)));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(plane + plane_off<R>(row + 4, ch) + 8 * (li & 1)));
    const s16x8 t = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(bf16x8, t);
}

// two values that bf16 holds exactly, packed
__device__ inline unsigned exact_bf16_pair(float a, float b) {
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

template <int TM, int TN>
__global__ __launch_bounds__(256, 2) void wgrad8_kernel(Wgrad8 p) {
    constexpr int MI = TM / 64, NI = TN / 64;
    constexpr int PA = TM / 32, LA = TM / 4;              // dz: 16-byte pieces per thread and step, lanes per row
    constexpr int CP = TN == 64 ? 8 : 16, LB = TN / CP;   // x: codes per piece (one per thread), lanes per row
    constexpr int kPlaneA = kStepRows * TM * 2, kPlaneB = kStepRows * TN * 2, kStage = 3 * kPlaneA + kPlaneB;
    static_assert(kStepRows * TN == 256 * CP, "one piece of x per thread and step");
    __shared__ __attribute__((aligned(16))) unsigned char smem[2 * kStage];

    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int wr = wave >> 1, wc = wave & 1;
    // consecutive tiles of one row range on one XCD (workgroups are dealt to the eight in turn): they share its operands
    const int nwg = p.gx * p.gy * p.gz;
    const int lin = blockIdx.x, xcd = lin & 7, q8 = nwg >> 3, r8 = nwg & 7;
    const int tile = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (lin >> 3);
    const int bx = tile % p.gx, by = (tile / p.gx) % p.gy, bz = tile / (p.gx * p.gy);
    const int n0 = by * TM, k0 = bx * TN;
    const int begin = bz * p.rows_per_split, end = min(p.M, begin + p.rows_per_split);
    const int steps = (end - begin + kStepRows - 1) / kStepRows;

    // columns past the operands only feed outputs that are never stored: their loads are moved inside the row
    int ca = n0 + 4 * (tid % LA);
    if (p.dz_vec && ca + 4 > p.dz_ld) ca = (int)p.dz_ld - 4;
    const int ra = tid / LA;
    int cb = k0 + CP * (tid % LB);
    if (cb + CP > p.blocks * kAct8Block) cb = p.blocks * kAct8Block - CP;
    const int rb = tid / LB;

    f32x16 acc[MI][NI];
#pragma unroll
    for (int mi = 0; mi < MI; mi++)
#pragma unroll
        for (int ni = 0; ni < NI; ni++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[mi][ni][r] = 0.f;
    const bool sums = p.colsum != nullptr && bx == 0;
    f32x4 colsum = {0.f, 0.f, 0.f, 0.f};

    f32x4 xa[PA];
    unsigned xb[CP / 4];
    int eb;
    auto load = [&](int t) {
        const int r0 = begin + t * kStepRows;
#pragma unroll
        for (int v = 0; v < PA; v++) {
            const int r = r0 + ra + (1024 / TM) * v;
            const float *row = p.dz + (int64_t)min(r, end - 1) * p.dz_ld;
            f32x4 x;
            if (p.dz_vec) x = *reinterpret_cast<const f32x4 *>(row + ca);
            else
#pragma unroll
                for (int q = 0; q < 4; q++) x[q] = row[min(ca + q, p.N - 1)];
#pragma unroll
            for (int q = 0; q < 4; q++) xa[v][q] = r < end ? x[q] : 0.f;
        }
        const int r = r0 + rb;
        const int64_t rc = min(r, end - 1);
        if constexpr (CP == 16) {
            const u32x4 w = *reinterpret_cast<const u32x4 *>(p.codes + rc * p.codes_ld + cb);
#pragma unroll
            for (int q = 0; q < 4; q++) xb[q] = w[q];
        } else {
            const u32x2 w = *reinterpret_cast<const u32x2 *>(p.codes + rc * p.codes_ld + cb);
            xb[0] = w[0];
            xb[1] = w[1];
        }
        eb = p.exps[rc * p.exps_ld + cb / kAct8Block];
        if (r >= end) eb = 0;                  // (a row that is none of this range's counts as zeros)
    };
    auto stage = [&](unsigned char *s) {
#pragma unroll
        for (int v = 0; v < PA; v++) {
            unsigned h0, m0, l0, h1, m1, l1;
            split3_pair(f32x2{xa[v][0], xa[v][1]}, h0, m0, l0);
            split3_pair(f32x2{xa[v][2], xa[v][3]}, h1, m1, l1);
            const int off = plane_off<TM>(ra + (1024 / TM) * v, (tid % LA) >> 1) + 8 * (tid & 1);
            *reinterpret_cast<u32x2 *>(s + off) = u32x2{h0, h1};
            *reinterpret_cast<u32x2 *>(s + kPlaneA + off) = u32x2{m0, m1};
            *reinterpret_cast<u32x2 *>(s + 2 * kPlaneA + off) = u32x2{l0, l1};
            if (sums) colsum += xa[v];
        }
        const float step = act8_step(eb);
        unsigned char *b = s + 3 * kPlaneA;
#pragma unroll
        for (int c = 0; c < CP / 8; c++) {
            unsigned o[4];
#pragma unroll
            for (int q = 0; q < 2; q++) {
                const unsigned w = act8_clear_marks(xb[2 * c + q]);
                o[2 * q] = exact_bf16_pair(act8_value(w, 0, step), act8_value(w, 1, step));
                o[2 * q + 1] = exact_bf16_pair(act8_value(w, 2, step), act8_value(w, 3, step));
            }
            *reinterpret_cast<u32x4 *>(b + plane_off<TN>(rb, (tid % LB) * (CP / 8) + c)) = u32x4{o[0], o[1], o[2], o[3]};
        }
    };
    auto multiply = [&](const unsigned char *s) {
#pragma unroll
        for (int sl = 0; sl < 2; sl++) {
            bf16x8 a[MI][3], b[NI];
#pragma unroll
            for (int ni = 0; ni < NI; ni++) b[ni] = plane_frag<TN>(s + 3 * kPlaneA, wc * (TN / 2) + 32 * ni, sl);
#pragma unroll
            for (int mi = 0; mi < MI; mi++)
#pragma unroll
                for (int k = 2; k >= 0; k--) a[mi][k] = plane_frag<TM>(s + k * kPlaneA, wr * (TM / 2) + 32 * mi, sl);
#pragma unroll
            for (int k = 2; k >= 0; k--)                // smallest terms first
#pragma unroll
                for (int mi = 0; mi < MI; mi++)
#pragma unroll
                    for (int ni = 0; ni < NI; ni++)
                        acc[mi][ni] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[mi][k], b[ni], acc[mi][ni], 0, 0, 0);
        }
    };

    load(0);
    stage(smem);
    __syncthreads();
    for (int t = 0; t < steps; t++) {
        unsigned char *now = smem + (t & 1) * kStage, *next = smem + ((t + 1) & 1) * kStage;
        if (t + 1 < steps) load(t + 1);
        multiply(now);
        if (t + 1 < steps) stage(next);
        __syncthreads();
    }

    if (sums) {         // this thread's four columns over its rows -> the tile's, in a fixed order
        float *meet = reinterpret_cast<float *>(smem);
        *reinterpret_cast<f32x4 *>(meet + ra * TM + 4 * (tid % LA)) = colsum;
        __syncthreads();
        if (tid < TM && n0 + tid < p.N) {
            float a = 0.f;
#pragma unroll
            for (int w = 0; w < 1024 / TM; w++) a += meet[w * TM + tid];
            p.colsum[(int64_t)bz * p.N + n0 + tid] = a;
        }
    }
    // register r of a lane: row (r & 3) + 8 (r >> 2) + 4 (lane / 32), column lane % 32 of its tile: 128 bytes of a row at once
    float *C = p.C + (int64_t)bz * p.slab_stride;
#pragma unroll
    for (int mi = 0; mi < MI; mi++)
#pragma unroll
        for (int ni = 0; ni < NI; ni++) {
            const int k = k0 + wc * (TN / 2) + 32 * ni + (lane & 31);
            const int n = n0 + wr * (TM / 2) + 32 * mi + 4 * (lane >> 5);
            if (k >= p.K) continue;
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int row = n + (r & 3) + 8 * (r >> 2);
                if (row < p.N) C[(int64_t)row * p.ldc + k] = acc[mi][ni][r];
            }
        }
}

int launch_wgrad8(Wgrad8 p, int tm, int tn, hipStream_t s) {
    p.gx = (int)ceil_div(p.K, tn);
    p.gy = (int)ceil_div(p.N, tm);
    const int64_t nwg = (int64_t)p.gx * p.gy * p.gz;
    DLRM_REQUIRE(nwg < (1ll << 31), "GEMM grid too large");
    const dim3 grid((unsigned)nwg), block(256);
    if (tm == 128 && tn == 128) hipLaunchKernelGGL((wgrad8_kernel<128, 128>), grid, block, 0, s, p);
    else if (tm == 128) hipLaunchKernelGGL((wgrad8_kernel<128, 64>), grid, block, 0, s, p);
    else if (tn == 128) hipLaunchKernelGGL((wgrad8_kernel<64, 128>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((wgrad8_kernel<64, 64>), grid, block, 0, s, p);
    DLRM_LAUNCH_CHECK();
    return DLRM_OK;
}

}  // namespace dlrm
