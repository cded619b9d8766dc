// Weight gradient from an 8-bit checkpoint of the layer's input: dW = dz^T x [N,K], reduction over the batch.
//
// A code times its block's power-of-two step is an exact bf16 number, so x enters v_mfma_f32_32x32x16_bf16 as it is and
// only dz is cut into three bf16 pieces (common.h: split3_pair): three terms instead of the six that two float32 operands
// take, every product exact in float32, float32 accumulation -- the accuracy of the bf16x3 evaluation at half its matrix
// work and with a quarter of x's bytes.
//
// A 256-thread workgroup owns TM columns of dz x TN columns of x (2 x 2 waves, each with (TM/64) x (TN/64) MFMA tiles) for a
// range of rows and walks it in steps of 16: the operands of the step after next are requested into registers, those of the
// next step are cut into pieces / widened to bf16 and written to one LDS stage, the present step's MFMAs run out of the
// other.  Both operands have the reduction index as their row, so LDS holds [16 rows][TM or TN] bf16 planes and the
// fragments come out of the transposing read ds_read_b64_tr_b16.  Row ranges leave partial sums that the caller adds in a
// fixed order.  x costs a third of dz's LDS traffic and half its conversions per column, so the tile is wider in x.
//
// What bounds it: 65536 x 1024 x 1024, 412 GF of bf16 MFMA: 339 us with the addition of the ranges (65536-row N(0,1) data),
// 1.22 PF/s, where a large bf16 product of the library sustains 1.17 to 1.34 on the same card.  Counters at 380 us: the MFMA
// pipe busy 55 % of the cycles at 1.87 GHz, 4.7 vector instructions per MFMA (the conversions), LDS 28 %.
#include "act8.h"

namespace dlrm {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4u __attribute__((aligned(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr int kStepRows = 16;

// byte offset of 16-byte chunk ch of row `row` in a [16][R] bf16 plane.  The transposing read takes four rows x 64 bytes
// per 32 lanes; the exchange of chunks puts those on different banks.
template <int R>
__device__ inline int plane_off(int row, int ch) {
    if constexpr (R == 64) return 128 * row + 16 * (ch ^ ((((row >> 1) & 1) << 2) | ((row >> 2) & 3)));
    else return 2 * R * row + 16 * (ch ^ (((row & 3) << 2) | ((row >> 2) & 3)));
}

// reduction rows 8 (lane / 32) .. +7 of column base + lane % 32
template <int R>
__device__ inline bf16x8 plane_frag(const unsigned char *plane, int base) {
    const int lane = threadIdx.x & 63;
    const int li = lane & 15, g = lane >> 4;
    const int ch = (base >> 3) + 2 * (g & 1) + ((li & 3) >> 1);
    const int row = 8 * (g >> 1) + (li >> 2);
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(plane + plane_off<R>(row, ch) + 8 * (li & 1)));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(plane + plane_off<R>(row + 4, ch) + 8 * (li & 1)));
    const s16x8 t = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(bf16x8, t);
}

// Scheduling recipe of a step: the fragment reads, then the next step's conversions spread evenly behind the MFMAs, its LDS
// writes behind the last ones
template <int I, int MFMAS, int VALU, int WRITES>
__device__ inline void interleave() {
    if constexpr (I < MFMAS) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, (VALU * (I + 1)) / MFMAS - (VALU * I) / MFMAS, 0);
        if constexpr (I == MFMAS / 2 - 1 || I == MFMAS - 1) __builtin_amdgcn_sched_group_barrier(0x200, (WRITES + 1) / 2, 0);
        interleave<I + 1, MFMAS, VALU, WRITES>();
    }
}

// a compiler fence for register values: their uses stay in the step they are written in
__device__ inline void pin(f32x4 &a) { asm volatile("" : "+v"(a)); }
__device__ inline void pin(unsigned &a) { asm volatile("" : "+v"(a)); }

// two values that bf16 holds exactly, packed
__device__ inline unsigned exact_bf16_pair(float a, float b) {
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

// CUT: N is no multiple of four, so the last tile along it has pieces that N cuts through
template <int TM, int TN, bool CUT>
__global__ __launch_bounds__(256, 2) void wgrad8_kernel(Wgrad8 p) {
    constexpr int MI = TM / 64, NI = TN / 64;
    constexpr int PA = TM / 64, LA = TM / 4, RA = 256 / LA;     // dz: 16-byte pieces per thread and step, lanes per row, rows per piece
    constexpr int CP = TN / 16, LB = 16;                        // x: codes per thread and step, lanes per row
    constexpr int kPlaneA = kStepRows * TM * 2, kPlaneB = kStepRows * TN * 2, kStage = 3 * kPlaneA + kPlaneB;
    __shared__ __attribute__((aligned(16))) unsigned char smem[2 * kStage];

    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int wr = wave >> 1, wc = wave & 1;
    // consecutive tiles of one row range on one XCD (workgroups are dealt to the eight in turn): they share its operands
    const int nwg = p.gx * p.gy * p.gz;
    const int lin = blockIdx.x, xcd = lin & 7, q8 = nwg >> 3, r8 = nwg & 7;
    const int tile = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (lin >> 3);
    const int bx = tile % p.gx, by = (tile / p.gx) % p.gy, bz = tile / (p.gx * p.gy);
    const int n0 = by * TM, k0 = bx * TN;
    const int begin = bz * p.rows_per_split, end = begin + min(p.M - begin, p.rows_per_split);    // (no sum passes M < 2^31)
    const int full = (end - begin) / kStepRows, steps = full + ((end - begin) % kStepRows != 0);

    // Columns past the operands only feed outputs that are never stored: their loads are moved inside the row.  A piece of dz
    // that N cuts through is moved back too and put in its place in registers.
    const int ca = n0 + 4 * (tid % LA), ca_in = max(min(ca, p.N - 4), 0), shift = ca < p.N ? ca - ca_in : 0;
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

    struct Raw {                              // one step's operands on their way
        f32x4 a[PA];
        unsigned b[CP / 4], e;
    };
    // a wave-uniform origin and 32-bit offsets that no step changes (the launch bounds the row lengths)
    const unsigned oa = ((unsigned)ra * (unsigned)p.dz_ld + (unsigned)ca_in) * 4u, ob = (unsigned)rb * (unsigned)p.codes_ld + (unsigned)cb;
    const unsigned oe = (unsigned)rb * (unsigned)p.exps_ld + (unsigned)(cb / kAct8Block);
    auto request = [&](int t, Raw &x) {       // a whole step of rows of at least four (16-byte loads at any alignment)
        const int64_t r0 = begin + t * kStepRows;
        const char *a = reinterpret_cast<const char *>(p.dz + r0 * p.dz_ld);
        const int8_t *b = p.codes + r0 * p.codes_ld;
#pragma unroll
        for (int v = 0; v < PA; v++) x.a[v] = *reinterpret_cast<const f32x4u *>(a + (oa + (unsigned)(RA * v) * (unsigned)p.dz_ld * 4u));
        if constexpr (CP == 16) {
            const u32x4 w = *reinterpret_cast<const u32x4 *>(b + ob);
#pragma unroll
            for (int q = 0; q < 4; q++) x.b[q] = w[q];
        } else if constexpr (CP == 8) {
            const u32x2 w = *reinterpret_cast<const u32x2 *>(b + ob);
            x.b[0] = w[0];
            x.b[1] = w[1];
        } else x.b[0] = *reinterpret_cast<const unsigned *>(b + ob);
        x.e = (p.exps + r0 * p.exps_ld)[oe];
    };
    auto request_any = [&](int t, Raw &x) {   // any step: rows past the range count as zeros
        const int r0 = begin + t * kStepRows;
#pragma unroll
        for (int v = 0; v < PA; v++) {
            const int r = r0 + ra + RA * v;
            const float *row = p.dz + (int64_t)min(r, end - 1) * p.dz_ld;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const float f = row[min(ca + q, p.N - 1)];
                x.a[v][q] = r < end ? f : 0.f;
            }
        }
        const int r = r0 + rb;
        const int64_t rc = min(r, end - 1);
#pragma unroll
        for (int q = 0; q < CP / 4; q++) x.b[q] = reinterpret_cast<const unsigned *>(p.codes + rc * p.codes_ld + cb)[q];
        const unsigned e = p.exps[rc * p.exps_ld + cb / kAct8Block];
        x.e = r < end ? e : 0u;
    };
    auto stage = [&](unsigned char *s, Raw &x, auto with_sums) {
#pragma unroll
        for (int v = 0; v < PA; v++) {
            unsigned h0, m0, l0, h1, m1, l1;
            split3_pair(f32x2{x.a[v][0], x.a[v][1]}, h0, m0, l0);
            split3_pair(f32x2{x.a[v][2], x.a[v][3]}, h1, m1, l1);
            const int off = plane_off<TM>(ra + RA * v, (tid % LA) >> 1) + 8 * (tid & 1);
            *reinterpret_cast<u32x2 *>(s + off) = u32x2{h0, h1};
            *reinterpret_cast<u32x2 *>(s + kPlaneA + off) = u32x2{m0, m1};
            *reinterpret_cast<u32x2 *>(s + 2 * kPlaneA + off) = u32x2{l0, l1};
            if constexpr (decltype(with_sums)::value) colsum += x.a[v];
        }
        unsigned char *b = s + 3 * kPlaneA;
        const float step = act8_step((int)x.e);
        unsigned o[CP / 2];
#pragma unroll
        for (int q = 0; q < CP / 4; q++) {
            const unsigned w = act8_clear_marks(x.b[q]);
            o[2 * q] = exact_bf16_pair(act8_value(w, 0, step), act8_value(w, 1, step));
            o[2 * q + 1] = exact_bf16_pair(act8_value(w, 2, step), act8_value(w, 3, step));
        }
        if constexpr (CP == 4) *reinterpret_cast<u32x2 *>(b + plane_off<TN>(rb, (tid % LB) >> 1) + 8 * (tid & 1)) = u32x2{o[0], o[1]};
        else
#pragma unroll
            for (int c = 0; c < CP / 8; c++)
                *reinterpret_cast<u32x4 *>(b + plane_off<TN>(rb, (tid % LB) * (CP / 8) + c)) = u32x4{o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]};
    };
    bf16x8 fa[MI][3], fb[NI];
    auto fragments = [&](const unsigned char *s) {
#pragma unroll
        for (int ni = 0; ni < NI; ni++) fb[ni] = plane_frag<TN>(s + 3 * kPlaneA, wc * (TN / 2) + 32 * ni);
#pragma unroll
        for (int k = 2; k >= 0; k--)
#pragma unroll
            for (int mi = 0; mi < MI; mi++) fa[mi][k] = plane_frag<TM>(s + k * kPlaneA, wr * (TM / 2) + 32 * mi);
    };
    auto multiply = [&]() {
#pragma unroll
        for (int k = 2; k >= 0; k--)                // smallest terms first
#pragma unroll
            for (int mi = 0; mi < MI; mi++)
#pragma unroll
                for (int ni = 0; ni < NI; ni++)
                    acc[mi][ni] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[mi][k], fb[ni], acc[mi][ni], 0, 0, 0);
    };

    // Steps [t0, t1) by one way of requesting them.  During step t the operands of t + 2 are requested, those of t + 1 (which
    // arrived meanwhile) converted and written to the other stage, and the MFMAs of t run.  Requests past the last step repeat it.
    auto run = [&](auto whole, auto with_sums, int t0, int t1) {
        constexpr bool kWhole = decltype(whole)::value;
        auto get = [&](int t, Raw &x) {
            if constexpr (kWhole) request(min(t, t1 - 1), x);
            else request_any(min(t, t1 - 1), x);
        };
        auto place = [&](Raw &x) {
            if constexpr (kWhole && CUT)
#pragma unroll
                for (int v = 0; v < PA; v++) {
                    f32x4 a = x.a[v];
                    if (shift & 1) a = f32x4{a[1], a[2], a[3], a[3]};
                    if (shift & 2) a = f32x4{a[2], a[3], a[3], a[3]};
                    x.a[v] = a;
                }
        };
        Raw u, w;
        auto step = [&](int t, unsigned char *now, unsigned char *next, Raw &gone, Raw &come) {
            get(t + 2, gone);
            __builtin_amdgcn_sched_barrier(0);
            fragments(now);
#pragma unroll
            for (int v = 0; v < PA; v++) pin(come.a[v]);
#pragma unroll
            for (int q = 0; q < CP / 4; q++) pin(come.b[q]);
            pin(come.e);
            place(come);
            stage(next, come, with_sums);
            multiply();
            __builtin_amdgcn_sched_group_barrier(0x100, 2 * (3 * MI + NI), 0);
            interleave<0, 3 * MI * NI, 24 * PA + 4 * CP, 3 * PA + (CP + 7) / 8>();
            __builtin_amdgcn_sched_barrier(0);
            __syncthreads();
        };
        get(t0, u);
        get(t0 + 1, w);
        place(u);
        stage(smem, u, with_sums);
        __syncthreads();
        int t = t0;
        for (; t + 2 < t1; t += 2) {
            step(t, smem, smem + kStage, u, w);
            step(t + 1, smem + kStage, smem, w, u);
        }
        if (t + 1 < t1) {
            step(t, smem, smem + kStage, u, w);
            fragments(smem + kStage);
        } else fragments(smem);
        multiply();
        __syncthreads();
    };
    auto run_all = [&](auto with_sums) {
        const int fast = p.N >= 4 ? full : 0;
        if (fast > 0) run(std::true_type{}, with_sums, 0, fast);
        if (fast < steps) run(std::false_type{}, with_sums, fast, steps);
    };
    if (sums) run_all(std::true_type{});
    else run_all(std::false_type{});

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

// Tile and ranges: the least of a model of the time over the four tiles, each with the ranges that give about 256, 512, 768 or
// 1024 workgroups.  A step of 16 rows takes a workgroup `alone` us; at_once of them share a compute unit and then take
// `each` us of it apiece, their tiles are stored at 5 outputs a ns, and the addition of the ranges is a launch and 4 bytes an
// output and range at 4.2 TB/s.  The constants are a fit to 1100 measured pairs of tile and ranges (60 shapes, 512 to 65536
// rows, 1 to 1024 columns; 5 % root mean square near a shape's best), and what the model takes is 2 % slower on average than
// the fastest of a shape's pairs, 14 % at most.  Taking the widest tile that fills 512 workgroups was 17 % slower on average:
// 53205 x 720 x 34 61 us with 128 x 256 tiles, 34 with 64 x 64; 25089 x 679 x 143 56 us with 294 workgroups of 128 x 256, 45
// with 759 of 64 x 64; 11515 x 643 x 255 39 and 30.
Wgrad8Shape wgrad8_shape(int64_t M, int N, int K, size_t max_bytes) {
    static const struct { int tm, tn; float alone, each; int at_once; } tiles[4] = {
        {128, 256, .74f, .58f, 2}, {128, 128, .48f, .375f, 2}, {64, 128, .28f, .225f, 3}, {64, 64, .21f, .145f, 4}};
    const int64_t rows_in = M < 1 ? 1 : M, unit = (int64_t)N * K + N;
    const size_t slab = sizeof(float) * (size_t)unit;
    int64_t most = rows_in / 64 < 1 ? 1 : (rows_in / 64 > 256 ? 256 : rows_in / 64);
    if (max_bytes != 0 && (size_t)most * slab > max_bytes) most = max_bytes < 2 * slab ? 1 : (int64_t)(max_bytes / slab);
    Wgrad8Shape w{};
    float least = 0.f;
    for (const auto &t : tiles) {
        const int64_t n = ceil_div(N, t.tm) * ceil_div(K, t.tn);
        for (int want = 256; want <= 1024; want += 256) {
            int64_t s = (want + n / 2) / n;
            s = s < 1 ? 1 : (s > most ? most : s);
            const int64_t up = ceil_div(ceil_div(rows_in, s), 32) * 32, rows = up < rows_in ? up : rows_in;
            s = ceil_div(rows_in, rows);
            const int64_t wave = 256 * t.at_once, left = n * s % wave;
            float step = (float)(n * s / wave) * t.each * t.at_once;        // us that one step of all workgroups takes
            if (left > 0) step += fmaxf(t.alone, t.each * (float)ceil_div(left, 256));
            const float us = step * (float)(up / kStepRows) + 2e-7f * (float)((n * s < wave ? n * s : wave) * t.tm * t.tn) +
                             (s > 1 ? 4.f + (float)(s * unit) * 0.95e-6f : 0.f);
            if (w.splits == 0 || us < least) {
                least = us;
                w.tm = t.tm;
                w.tn = t.tn;
                w.splits = (int)s;
                w.rows_per_split = (int)rows;
            }
        }
    }
    w.bytes = w.splits * slab + 256;
    return w;
}

int launch_wgrad8(Wgrad8 p, int tm, int tn, hipStream_t s) {
    p.gx = (int)ceil_div(p.K, tn);
    p.gy = (int)ceil_div(p.N, tm);
    const int64_t nwg = (int64_t)p.gx * p.gy * p.gz;
    DLRM_REQUIRE(nwg < (1ll << 31), "GEMM grid too large");
    DLRM_REQUIRE(p.dz_ld <= (1 << 24) && p.codes_ld <= (1 << 24) && p.exps_ld <= (1 << 24), "leading dimension above 2^24");
    const dim3 grid((unsigned)nwg), block(256);
#define DLRM_WGRAD8(TM, TN)                                                                                   \
    do {                                                                                                      \
        if (p.N % 4 == 0) hipLaunchKernelGGL((wgrad8_kernel<TM, TN, false>), grid, block, 0, s, p);           \
        else hipLaunchKernelGGL((wgrad8_kernel<TM, TN, true>), grid, block, 0, s, p);                         \
    } while (0)
    if (tn == 256) DLRM_WGRAD8(128, 256);
    else if (tm == 128) DLRM_WGRAD8(128, 128);
    else if (tn == 128) DLRM_WGRAD8(64, 128);
    else DLRM_WGRAD8(64, 64);
#undef DLRM_WGRAD8
    DLRM_LAUNCH_CHECK();
    return DLRM_OK;
}

}  // namespace dlrm
