// rac_attn.hpp — what the attention kernels on the matrix cores share: tiles
// of rows through registers into LDS, rows as fragments, accumulators into
// rows, and the rows done again on the VALU where the matrix cores' products
// met a value that is not finite.
#pragma once
#include "rac_mma.hpp"

namespace rac {

constexpr int kAttnThreads = 256, kAttnWaves = 4;

// BN rows of a [total, heads, d] array's head (rows first .. of a sequence of
// len rows; past it zeros) through registers into LDS rows of LD values
template <typename T, int DP, int BN>
struct TileStage {
    static constexpr int VEC = Mma<T>::VEC, CPR = DP / VEC, N = BN * CPR / kAttnThreads;
    static_assert(N >= 1 && BN * CPR % kAttnThreads == 0, "a tile is a whole number of vectors a thread");
    u32x4 r[N];
    __device__ __forceinline__ void load(const T* base, long stride, int first, int len, int d, bool vec) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int v = threadIdx.x + i * kAttnThreads, row = first + v / CPR, c = v % CPR * VEC;
            r[i] = row < len ? load_chunk(base + (long)row * stride, c, d, vec) : u32x4{0, 0, 0, 0};
        }
    }
    template <int LD>
    __device__ __forceinline__ void store(T* lds) const {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int v = threadIdx.x + i * kAttnThreads;
            *reinterpret_cast<u32x4*>(lds + v / CPR * LD + v % CPR * VEC) = r[i];
        }
    }
};

// a row's fragments: value KF f + KF / 2 half of row `row` (global memory)
template <typename T, int DP>
__device__ __forceinline__ void load_frags(typename Mma<T>::Frag (&fr)[DP / Mma<T>::KF], const T* row, bool there,
                                           int d, int half, bool vec) {
    constexpr int KF = Mma<T>::KF;
#pragma unroll
    for (int f = 0; f < DP / KF; f++)
        fr[f] = __builtin_bit_cast(typename Mma<T>::Frag,
                                   there ? load_chunk(row, f * KF + half * (KF / 2), d, vec) : u32x4{0, 0, 0, 0});
}

// a 32-column accumulator set (DP rows of d) times f into one contiguous row
template <typename T, int ND>
__device__ __forceinline__ void attn_store(T* row, const f32x16 (&acc)[ND], float f, int d, int half, bool vec) {
#pragma unroll
    for (int n = 0; n < ND; n++)
#pragma unroll
        for (int b = 0; b < 4; b++) {
            const int c = 32 * n + 8 * b + 4 * half;
            union { T e[4]; u32x2 v2; u32x4 v4; } u;
#pragma unroll
            for (int j = 0; j < 4; j++) u.e[j] = Mma<T>::from_f32(acc[n][4 * b + j] * f);
            if (vec) {
                if (c < d) {
                    if constexpr (sizeof(T) == 2) *reinterpret_cast<u32x2*>(row + c) = u.v2;
                    else *reinterpret_cast<u32x4*>(row + c) = u.v4;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (c + j < d) row[c + j] = u.e[j];
            }
        }
}

// whether a column of the accumulators holds a value that is not finite
template <int N>
__device__ __forceinline__ bool not_finite(const f32x16 (&acc)[N]) {
    float t = 0.0f;
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
        for (int i = 0; i < 16; i++) t = __builtin_fmaf(acc[n][i], 0.0f, t);
    return t != 0.0f;                   // NaN
}

// dot product of two rows of d values, and its partner's values times f added
// to lane e's columns e, e + 64, ...: the parts of a row done again on the VALU
template <typename T>
__device__ float row_dot(const T* x, const T* y, int d) {
    float s = 0.0f;
    for (int c = 0; c < d; c++) s = __builtin_fmaf(Mma<T>::to_f32(x[c]), Mma<T>::to_f32(y[c]), s);
    return s;
}
template <typename T, int DP>
__device__ void row_axpy(float (&acc)[(DP + 63) / 64], float f, const T* y, int d) {
#pragma unroll
    for (int n = 0; n < (DP + 63) / 64; n++) {
        const int c = (threadIdx.x & 63) + 64 * n;
        if (c < d) acc[n] = __builtin_fmaf(f, Mma<T>::to_f32(y[c]), acc[n]);
    }
}
// out = f sum of w(j) rows(j) over j in [j0, j1): the weights of 64 j at a time,
// one to a lane, then their rows one by one; nothing of a j outside is read
// (with SKIP, nor of a j whose weight is below 0)
template <typename T, int DP, bool SKIP = false, typename O, typename W, typename R>
__device__ void attn_again(O* out, float f, int d, int j0, int j1, W w, R rows) {
    float acc[(DP + 63) / 64] = {};
    for (int j = j0; j < j1; j += 64) {
        const int mine = j + (threadIdx.x & 63);
        const float wt = mine < j1 ? w(mine) : 0.0f;
        for (int i = 0; i < min(64, j1 - j); i++) {
            const float wi = __shfl(wt, i);
            if (!SKIP || !(wi < 0.0f)) row_axpy<T, DP>(acc, wi, rows(j + i), d);
        }
    }
#pragma unroll
    for (int n = 0; n < (DP + 63) / 64; n++) {
        const int c = (threadIdx.x & 63) + 64 * n;
        if (c < d) out[c] = Mma<O>::from_f32(acc[n] * f);
    }
}

}  // namespace rac
