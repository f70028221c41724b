// rac_mma.hpp — 32 x 32 matrix-core tiles of fp32, bf16 and fp16 operands for
// the attention kernels, one interface for the three types.
//
// A fragment is 16 bytes a lane: row (or column) l % 32 of an operand, and of
// every KF consecutive k the KF / 2 that lane half h = l / 32 holds.  For the
// 16-bit types it is one 32x32x16 instruction (8 values); for fp32 four
// 32x32x2 (4 values, value j of the two halves being the two k of instruction
// j).  The accumulator of a product has column l % 32 and, in register 4 b + j,
// row 8 b + 4 h + j: KF k of a following product are KF / 2 neighbouring
// registers, so an accumulator turns into that product's right operand (pack)
// without leaving its lane, as long as the left operand's fragments hold their k
// in the same order: of every KF the half h the rows 4 h + j, and for the 16-bit
// types 8 + 4 h + j, j = 0 .. 3 (Tile::cols).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace rac {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Mma;

template <>
struct Mma<float> {
    using Frag = f32x4;
    static constexpr int KF = 8;              // k of a fragment
    static constexpr int VEC = 4;             // values of a 16-byte vector
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
#pragma unroll
        for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ Frag pack(const f32x16& c, int f) {
        return Frag{c[4 * f], c[4 * f + 1], c[4 * f + 2], c[4 * f + 3]};
    }
    static __device__ __forceinline__ float to_f32(float v) { return v; }
    static __device__ __forceinline__ float from_f32(float v) { return v; }
};

// a transposing read of LDS: 16 lanes bring 4 rows of 16 columns (lane i the
// four columns from 4 (i % 4) of row i / 4), lane i keeps column i
__device__ __forceinline__ s16x4 lds_read_tr(const void* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
}

// 16-bit operands: T's bits travel as shorts, the instruction knows the type
template <typename T, typename V8>
struct MmaHalf {
    using Frag = V8;
    static constexpr int KF = 16;
    static constexpr int VEC = 8;
    static __device__ __forceinline__ Frag pack(const f32x16& c, int f) {
        Frag r;
#pragma unroll
        for (int j = 0; j < 8; j++) r[j] = (T)c[8 * f + j];      // to nearest even
        return r;
    }
    static __device__ __forceinline__ float to_f32(T v) { return (float)v; }
    static __device__ __forceinline__ T from_f32(float v) { return (T)v; }
};

template <>
struct Mma<__bf16> : MmaHalf<__bf16, bf16x8> {
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Mma<_Float16> : MmaHalf<_Float16, f16x8> {
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; i++) z[i] = 0.0f;
    return z;
}

// the lower half's value and the upper half's, in every lane
__device__ __forceinline__ void both_halves(float v, float& lo, float& hi) {
    const uint32_t a = __builtin_bit_cast(uint32_t, v);
    const u32x2 r = __builtin_amdgcn_permlane32_swap(a, a, false, false);
    const uint32_t r0 = r[0], r1 = r[1];     // scalars: a bit_cast of r[1] itself reads r[0]
    lo = __builtin_bit_cast(float, r0);
    hi = __builtin_bit_cast(float, r1);
}
__device__ __forceinline__ float half_sum(float v) {
    float lo, hi;
    both_halves(v, lo, hi);
    return lo + hi;
}
__device__ __forceinline__ float half_max(float v) {
    float lo, hi;
    both_halves(v, lo, hi);
    return fmaxf(lo, hi);
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// 2^x, x <= 0 or NaN: the hardware's exponential (1 ulp; results below the
// least normal become 0, which no sum here can tell)
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// 16 bytes of a row in global memory from element c on, elements past d as
// zeros; vec: the row is 16-byte aligned and d a multiple of the vector
template <typename T>
__device__ __forceinline__ u32x4 load_chunk(const T* row, int c, int d, bool vec) {
    constexpr int VEC = Mma<T>::VEC;
    u32x4 r = {0, 0, 0, 0};
    if (vec) {
        if (c < d) r = *reinterpret_cast<const u32x4*>(row + c);
        return r;
    }
    union { T e[VEC]; u32x4 v; } u;
    u.v = r;
#pragma unroll
    for (int j = 0; j < VEC; j++)
        if (c + j < d) u.e[j] = row[c + j];
    return u.v;
}

}  // namespace rac
