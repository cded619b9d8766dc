// The 8-bit activation checkpoint (dlrm_act8): per 32 consecutive columns of a row one power-of-two step 2^(E-127) and
// one signed byte per element, the element's value divided by the step and rounded to the nearest integer (ties to even).
//
// The step is the smallest power of two with max |x| < 127.5 steps, so no code leaves [-127, 127] and every element is
// within half a step of its value: at most max |x| / 127.5 (the largest magnitude lies in [63.75, 127.5) steps; at the two
// ends of float32's range see act8_exponent).  A power
// of two, not max |x| / 127: dividing by it and multiplying with it are exact, so packing is a function of the input
// alone (no rounding of a scale in between), and a code times its step is an exact bf16 number (7 significant bits),
// which the weight gradient multiplies on the matrix cores without splitting it.
// Code -128 marks a positive element that rounds to zero: its value is 0, and a ReLU mask still sees it as positive.
#pragma once
#include <type_traits>

#include "common.h"

namespace dlrm {

constexpr int kAct8Block = 32;

__host__ __device__ inline int act8_blocks(int cols) { return (cols + kAct8Block - 1) / kAct8Block; }

// what a launch that reads or writes a checkpoint of `cols` columns asks of its descriptor
int act8_check(const dlrm_act8 *a, int cols, const char *what);

// dW = dz^T x and the column sums of dz over ranges of rows_per_split rows (act8_wgrad.hip), x from its checkpoint: range z
// writes [N,K] at C + z slab_stride and [N] at colsum + z N.  The caller has checked the shapes and adds the ranges up.
struct Wgrad8 {
    const float *dz;
    int64_t dz_ld;
    const int8_t *codes;
    int64_t codes_ld;
    const uint8_t *exps;
    int64_t exps_ld;
    int blocks;              // of 32 columns in a row of the checkpoint
    float *C;
    int64_t ldc, slab_stride;
    float *colsum;           // or NULL
    int M, N, K;
    int rows_per_split;      // a multiple of 32, or all rows
    int gx, gy, gz;          // gz: ranges; gx, gy are filled in by the launch
};
int launch_wgrad8(Wgrad8 p, int tm, int tn, hipStream_t s);
// output tile, ranges of the batch and the bytes of their partial sums; max_bytes != 0: at most so many
struct Wgrad8Shape {
    int tm, tn, splits, rows_per_split;
    size_t bytes;
};
Wgrad8Shape wgrad8_shape(int64_t M, int N, int K, size_t max_bytes);

// exponent byte of a block whose largest magnitude has the bits `amax` (sign cleared): the mantissa carries into the
// exponent from 127.5/128 of the next power of two on.  At most 248: 64 steps of 2^122 would be an infinity, so blocks that
// close to the end of float32 keep the step 2^121 and their codes stop at 127.  255: the block holds an infinity or a NaN.
__device__ inline int act8_exponent(unsigned amax) {
    if (amax >= 0x7f800000u) return 255;
    const int e = (int)((amax + 0x10000u) >> 23) - 6;
    return e < 1 ? 1 : (e > 248 ? 248 : e);
}
// 1 / step and step as floats
__device__ inline float act8_inverse(int e) { return e == 255 ? 0.f : __uint_as_float((unsigned)(254 - e) << 23); }
__device__ inline float act8_step(int e) { return __uint_as_float(e == 255 ? 0x7fc00000u : (unsigned)e << 23); }

// Codes of four elements of a block of exponent e, packed.  Adding 1.5 * 2^23 rounds x / step (exact: a power of two) to an
// integer, ties to even, and leaves its two's complement in the low bits: one fma per element.  0 < x <= step / 2 is the
// mark; on the bits, as unsigned numbers less one, it is one comparison.
__device__ inline unsigned act8_codes(const float *x, int e) {
    const float inverse = act8_inverse(e);
    const unsigned half = e == 255 ? 0x7f800000u : (e == 1 ? 0x00400000u : (unsigned)(e - 1) << 23);
    unsigned b[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        float v = x[j];
        if (e >= 248) {        // the top of the range; a block with an infinity or a NaN: zeros and marks
            const float top = 127.f * __uint_as_float(248u << 23);
            v = e == 255 ? (v > 0.f ? 1.f : 0.f) : fminf(fmaxf(v, -top), top);
        }
        b[j] = __float_as_uint(v) - 1u < half ? 0x80u : __float_as_uint(__builtin_fmaf(v, inverse, 12582912.f));
    }
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u), __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u),
                                 0x05040100u);
}
// x > 0 of the element behind a code: 1 .. 127 and -128
__device__ inline bool act8_positive(int code) { return (unsigned)(code - 1) % 256u < 128u; }

// four codes in a dword with every -128 replaced by 0
__device__ inline unsigned act8_clear_marks(unsigned w) {
    return w & (((w & 0x7f7f7f7fu) + 0x7f7f7f7fu) | 0x7f7f7f7fu);
}
// value of code j of a dword of codes with the marks cleared
__device__ inline float act8_value(unsigned cleared, int j, float step) {
    return (float)(signed char)(cleared >> (8 * j)) * step;
}

// ---- exchanges between lanes.  The first four steps of a butterfly run on the data-parallel-primitive path of the vector
// unit (no LDS traffic): exchange with lane ^ 1, ^ 2 (quad permutes), then mirrored halves of 8 and of 16 lanes, which are
// lane ^ 4 and ^ 8 once the smaller groups agree.
template <int CTRL>
__device__ inline float dpp_move(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
// sum / maximum over the aligned group of G lanes a lane belongs to, in every lane, the same bits in all of them
template <int G>
__device__ inline float group_sum(float x) {
    if constexpr (G >= 2) x += dpp_move<0xB1>(x);
    if constexpr (G >= 4) x += dpp_move<0x4E>(x);
    if constexpr (G >= 8) x += dpp_move<0x141>(x);
    if constexpr (G >= 16) x += dpp_move<0x140>(x);
    if constexpr (G >= 32) x += __shfl_xor(x, 16, 64);
    if constexpr (G >= 64) x += __shfl_xor(x, 32, 64);
    return x;
}
template <int G>
__device__ inline unsigned group_umax(unsigned x) {
    auto fold = [](unsigned a, unsigned b) { return a > b ? a : b; };
    auto mv = [](unsigned a, auto ctrl) {
        return (unsigned)__builtin_amdgcn_update_dpp(0, (int)a, decltype(ctrl)::value, 0xf, 0xf, true);
    };
    if constexpr (G >= 2) x = fold(x, mv(x, std::integral_constant<int, 0xB1>{}));
    if constexpr (G >= 4) x = fold(x, mv(x, std::integral_constant<int, 0x4E>{}));
    if constexpr (G >= 8) x = fold(x, mv(x, std::integral_constant<int, 0x141>{}));
    if constexpr (G >= 16) x = fold(x, mv(x, std::integral_constant<int, 0x140>{}));
    static_assert(G <= 16, "a block's lanes");
    return x;
}

// ---- rows of float32 or bf16 elements, 16 bytes' worth of consecutive ones per lane
template <typename T> constexpr int kWide = 16 / (int)sizeof(T);      // float: 4, bf16 (uint16_t): 8

__device__ inline float to_f32(float x) { return x; }
__device__ inline float to_f32(uint16_t x) { return bf16_bits_to_f32(x); }
// two values as bf16, packed (rounded to nearest even)
__device__ inline unsigned bf16_pair(float a, float b) { return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{a, b}, bf16x2)); }
// values as they are once they are stored as T
template <typename T, int VEC>
__device__ inline void round_elems(float (&v)[VEC]) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
            const unsigned w = bf16_pair(v[j], v[j + 1]);
            v[j] = __uint_as_float(w << 16);
            v[j + 1] = __uint_as_float(w & 0xffff0000u);
        }
    }
}

// Aligned to its elements only: global memory takes 16-byte accesses at any address here, and one that straddles two cache
// lines costs far less than the four (eight) accesses of single elements: rows of 479 bf16 elements, packed, 8191 of them
// through the layer norm: 12.6 us element by element, 8.8 us this way.
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 piece4 __attribute__((aligned(4)));      // (in memory: 16 bytes of float32 or bf16 elements)
typedef u32x4 piece2 __attribute__((aligned(2)));
template <typename T> struct PieceIn { typedef piece4 type; };
template <> struct PieceIn<uint16_t> { typedef piece2 type; };

// Elements c .. c+VEC-1 of a row of N (VEC: 16 bytes' worth) in two steps, so that a kernel can have all of its requests
// under way before it looks at the first: the request has no branch that depends on the lane (a piece that would pass the
// end of the row is moved back inside it), and elems_of puts such a piece in its place and `fill` where there is no element.
template <typename T, int VEC>
__device__ inline u32x4 request_elems(const T *row, int c, int N) {
    static_assert(VEC == kWide<T>, "a piece is 16 bytes");
    if (N >= VEC) return *reinterpret_cast<const typename PieceIn<T>::type *>(row + (c + VEC <= N ? c : N - VEC));
    u32x4 w = {0, 0, 0, 0};
    for (int j = 0; j < N; j++) {
        const unsigned e = sizeof(T) == 2 ? (unsigned)reinterpret_cast<const uint16_t *>(row)[j] << (16 * (j & 1))
                                          : reinterpret_cast<const unsigned *>(row)[j];
        const int at = sizeof(T) == 2 ? j >> 1 : j;
        if (at == 0) w[0] |= e;
        else if (at == 1) w[1] |= e;
        else if (at == 2) w[2] |= e;
        else w[3] |= e;
    }
    return w;
}
template <typename T, int VEC>
__device__ inline void elems_of(u32x4 w, int c, int N, float (&v)[VEC], float fill = 0.f) {
    if (c + VEC > N && N % VEC != 0) {         // (waves without the end of the row skip it)
        const int back = N >= VEC ? c - (N - VEC) : c;
        if constexpr (sizeof(T) == 2)
            if (back & 1) {
#pragma unroll
                for (int j = 0; j < 4; j++) w[j] = __builtin_amdgcn_alignbit(j < 3 ? w[j + 1] : 0u, w[j], 16);
            }
        const int words = sizeof(T) == 2 ? back >> 1 : back;
        if (words & 1) w = u32x4{w[1], w[2], w[3], w[3]};
        if (words & 2) w = u32x4{w[2], w[3], w[3], w[3]};
    }
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            v[2 * j] = __uint_as_float(w[j] << 16);
            v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = __uint_as_float(w[j]);
    }
    if (c + VEC > N) {
#pragma unroll
        for (int j = 0; j < VEC; j++) v[j] = c + j < N ? v[j] : fill;
    }
}
template <typename T, int VEC>
__device__ inline void store_elems(T *row, int c, int N, const float (&v)[VEC]) {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if constexpr (sizeof(T) == 2) w[j] = bf16_pair(v[2 * j], v[2 * j + 1]);
        else w[j] = __float_as_uint(v[j]);
    }
    if (c + VEC <= N) *reinterpret_cast<typename PieceIn<T>::type *>(row + c) = w;
    else {
#pragma unroll
        for (int j = 0; j < VEC; j++)
            if (c + j < N) {
                if constexpr (sizeof(T) == 2) row[c + j] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
                else row[c + j] = v[j];
            }
    }
}

// VEC elements of one lane (zero at N and beyond) to their place in a checkpoint row: 32 / VEC neighbouring lanes hold a
// block and all of them call this.  Blocks past the last one are not written.
template <int VEC>
__device__ inline void act8_store(const float (&v)[VEC], int8_t *codes, uint8_t *exps, int c, int blocks, bool live) {
    float top = fabsf(v[0]);
#pragma unroll
    for (int j = 1; j < VEC; j++) top = __builtin_elementwise_maximum(top, fabsf(v[j]));        // (a NaN stays one)
    const int e = act8_exponent(group_umax<kAct8Block / VEC>(__float_as_uint(top)));
    const int block = c / kAct8Block;
    if (!live || block >= blocks) return;
    unsigned w[VEC / 4];
#pragma unroll
    for (int j = 0; j < VEC / 4; j++) w[j] = act8_codes(v + 4 * j, e);
    if constexpr (VEC == 4) *reinterpret_cast<unsigned *>(codes + c) = w[0];
    else *reinterpret_cast<uint2 *>(codes + c) = make_uint2(w[0], w[1]);
    if (c % kAct8Block == 0) exps[block] = (uint8_t)e;
}
// the raw codes of VEC elements from column c of a checkpoint row, in dwords of four (past the last block: some of its last)
template <int VEC>
__device__ inline void act8_load(const int8_t *codes, int c, int blocks, unsigned (&w)[VEC / 4]) {
    const int8_t *at = codes + min(c, blocks * kAct8Block - VEC);
    if constexpr (VEC == 4) w[0] = *reinterpret_cast<const unsigned *>(at);
    else {
        const uint2 t = *reinterpret_cast<const uint2 *>(at);
        w[0] = t.x;
        w[1] = t.y;
    }
}
template <int VEC>
__device__ inline void act8_values(const unsigned (&w)[VEC / 4], float step, float (&v)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; j++) v[j] = act8_value(act8_clear_marks(w[j / 4]), j % 4, step);
}

}  // namespace dlrm
