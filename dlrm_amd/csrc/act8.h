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
    int dz_vec;              // rows of dz start on 16-byte boundaries
    const int8_t *codes;
    int64_t codes_ld;
    const uint8_t *exps;
    int64_t exps_ld;
    int blocks;              // of 32 columns in a row of the checkpoint
    float *C;
    int64_t ldc, slab_stride;
    float *colsum;           // or NULL
    int M, N, K;
    int rows_per_split;      // a multiple of 32
    int gx, gy, gz;          // gz: ranges; gx, gy are filled in by the launch
};
int launch_wgrad8(Wgrad8 p, int tm, int tn, hipStream_t s);      // output tile tm x tn, each 128 or 64

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

// code of one element, in the low byte (in a block of exponent 255: 0, or -128 where x > 0)
__device__ inline unsigned act8_code(float x, float inverse) {
    const float t = x * inverse;
    const int q = (t == t) ? (int)fminf(fmaxf(rintf(t), -127.f), 127.f) : 0;
    return (unsigned)((q == 0 && x > 0.f) ? -128 : q) & 0xffu;
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
    if constexpr (G >= 32) x = fold(x, (unsigned)__shfl_xor((int)x, 16, 64));
    return x;
}

// ---- rows of float32 or bf16 elements, VEC consecutive ones per lane (VEC: 16 bytes' worth, or 1)
template <typename T> constexpr int kWide = 16 / (int)sizeof(T);      // float: 4, bf16 (uint16_t): 8

__device__ inline float to_f32(float x) { return x; }
__device__ inline float to_f32(uint16_t x) { return bf16_bits_to_f32(x); }
__device__ inline void from_f32(float v, float &x) { x = v; }
__device__ inline void from_f32(float v, uint16_t &x) { x = (uint16_t)f32_to_bf16_bits(v); }
// the value an element has once it is stored as T
template <typename T>
__device__ inline float rounded_to(float v) {
    T t;
    from_f32(v, t);
    return to_f32(t);
}

template <typename T, int VEC> struct alignas(VEC * sizeof(T)) Pack { T e[VEC]; };

// elements c .. c+VEC-1 of a row of N; what lies at N or beyond is `fill` and is not touched in memory
template <typename T, int VEC>
__device__ inline void load_elems(const T *row, int c, int N, float (&v)[VEC], float fill = 0.f) {
    if (VEC == 1 || c + VEC <= N) {
        if (VEC > 1 || c < N) {
            const Pack<T, VEC> p = *reinterpret_cast<const Pack<T, VEC> *>(row + c);
#pragma unroll
            for (int j = 0; j < VEC; j++) v[j] = to_f32(p.e[j]);
        } else v[0] = fill;
    } else {
#pragma unroll
        for (int j = 0; j < VEC; j++) v[j] = c + j < N ? to_f32(row[c + j]) : fill;
    }
}
template <typename T, int VEC>
__device__ inline void store_elems(T *row, int c, int N, const float (&v)[VEC]) {
    if (VEC == 1 || c + VEC <= N) {
        if (VEC > 1 || c < N) {
            Pack<T, VEC> p;
#pragma unroll
            for (int j = 0; j < VEC; j++) from_f32(v[j], p.e[j]);
            *reinterpret_cast<Pack<T, VEC> *>(row + c) = p;
        }
    } else {
#pragma unroll
        for (int j = 0; j < VEC; j++)
            if (c + j < N) from_f32(v[j], row[c + j]);
    }
}

// VEC elements of one lane (zero at N and beyond) to their place in a checkpoint row: 32 / VEC neighbouring lanes hold a
// block and all of them call this.  Blocks past the last one are not written.
template <int VEC>
__device__ inline void act8_store(const float (&v)[VEC], int8_t *codes, uint8_t *exps, int c, int blocks, bool live) {
    unsigned amax = 0;
#pragma unroll
    for (int j = 0; j < VEC; j++) {
        const unsigned b = __float_as_uint(v[j]) & 0x7fffffffu;
        amax = b > amax ? b : amax;
    }
    const int e = act8_exponent(group_umax<kAct8Block / VEC>(amax));
    const float inverse = act8_inverse(e);
    const int block = c / kAct8Block;
    if (!live || block >= blocks) return;
    if constexpr (VEC == 1) codes[c] = (int8_t)act8_code(v[0], inverse);
    else {
        unsigned w[VEC / 4];
#pragma unroll
        for (int j = 0; j < VEC / 4; j++)
            w[j] = act8_code(v[4 * j], inverse) | act8_code(v[4 * j + 1], inverse) << 8 | act8_code(v[4 * j + 2], inverse) << 16 |
                   act8_code(v[4 * j + 3], inverse) << 24;
        if constexpr (VEC == 4) *reinterpret_cast<unsigned *>(codes + c) = w[0];
        else *reinterpret_cast<uint2 *>(codes + c) = make_uint2(w[0], w[1]);
    }
    if (c % kAct8Block == 0) exps[block] = (uint8_t)e;
}
// the raw codes of VEC elements from column c of a checkpoint row (0 past the last block), in dwords of four (VEC = 1: one)
template <int VEC>
__device__ inline void act8_load(const int8_t *codes, int c, int blocks, unsigned (&w)[VEC == 8 ? 2 : 1]) {
#pragma unroll
    for (int j = 0; j < (VEC == 8 ? 2 : 1); j++) w[j] = 0;
    if (c >= blocks * kAct8Block) return;
    if constexpr (VEC == 1) w[0] = (uint8_t)codes[c];
    else if constexpr (VEC == 4) w[0] = *reinterpret_cast<const unsigned *>(codes + c);
    else {
        const uint2 t = *reinterpret_cast<const uint2 *>(codes + c);
        w[0] = t.x;
        w[1] = t.y;
    }
}
template <int VEC>
__device__ inline void act8_values(const unsigned (&w)[VEC == 8 ? 2 : 1], float step, float (&v)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; j++) v[j] = act8_value(act8_clear_marks(w[j / 4]), j % 4, step);
}

}  // namespace dlrm
