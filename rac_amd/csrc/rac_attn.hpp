// rac_attn.hpp — what the attention kernels on the matrix cores share: tiles
// of rows through registers into LDS, rows as fragments, accumulators into
// rows, and the rows done again on the VALU where the matrix cores' products
// met a value that is not finite.
#pragma once
#include "rac_mma.hpp"

namespace rac {

// for the lambdas of the kernels: a call of one would lose what is uniform
#define ATTN_INLINE __attribute__((always_inline))

constexpr int kAttnThreads = 256, kAttnWaves = 4;

// v, as a value of its own: addresses made of it are made where they are used
// and hold no registers between
__device__ __forceinline__ int attn_fresh(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// A tile of rows in LDS: row r's 16-byte vectors lie in it without padding,
// vector c at place c ^ tile_swz(r), so that both ways of reading a tile, 32
// rows at the same vector (rows as a left operand) and 4 rows by 32 values
// (transposed), touch every bank equally often.
template <int CPR>
__device__ __forceinline__ int tile_swz(int r) {
    if constexpr (CPR % 16 == 0) return ((r & 3) << 2) | ((r >> 2) & 3);
    else if constexpr (CPR % 8 == 0) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    else return (r >> 2) & 3;
}

template <typename T, int DP>
struct Tile {
    using M = Mma<T>;
    using Frag = typename M::Frag;
    static constexpr int RB = DP * (int)sizeof(T), CPR = RB / 16;     // bytes and vectors of a row

    // fragment f of row r of the tile's rows from `row` on (row % 16 == 0), r = lane % 32
    static __device__ __forceinline__ Frag rows(const char* lds, int row, int f, int lane) {
        const int r = lane & 31;
        return *reinterpret_cast<const Frag*>(lds + (row + r) * RB + ((2 * f + (lane >> 5)) ^ tile_swz<CPR>(r)) * 16);
    }
    // Mma's transposed fragment f of the 32 rows from `row` on, columns 32 n + lane % 32
    static __device__ __forceinline__ Frag cols(const char* lds, int row, int f, int n, int lane) {
        const int h = lane >> 5;
        if constexpr (sizeof(T) == 4) {
            Frag v;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int r = 8 * f + 4 * h + j;
                v[j] = *reinterpret_cast<const float*>(lds + (row + r) * RB +
                                                       ((8 * n + ((lane & 31) >> 2)) ^ tile_swz<CPR>(r)) * 16 + 4 * (lane & 3));
            }
            return v;
        } else {
            const int i = lane & 15, c = 4 * n + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1), r = 16 * f + 4 * h + (i >> 2);
            const char* p = lds + (row + r) * RB + 8 * (i & 1);
            union { s16x4 s[2]; Frag f; } u;
            u.s[0] = lds_read_tr(p + (c ^ tile_swz<CPR>(r)) * 16);
            u.s[1] = lds_read_tr(p + 8 * RB + (c ^ tile_swz<CPR>(r + 8)) * 16);
            return u.f;
        }
    }
};

// ROWS rows of an array (element stride between rows) into LDS, 16 bytes a
// thread and load, rows past the last and columns past d as zeros: issue()
// before the work on the tile before, commit() behind it.
// DIRECT: straight into LDS, which spares registers and instructions, else
// through registers.  Before a transposing read (16-bit types) the compiler
// waits for every load into LDS, whatever its place, so that a direct load has
// only the time up to the first of them: enough where the rows come from L2 and
// the scores stand between, too little where they come from HBM.
template <typename T, int DP, int ROWS, bool DIRECT = sizeof(T) == 4>
struct TileLoad {
    static constexpr int VEC = Mma<T>::VEC, RB = DP * (int)sizeof(T), CPR = RB / 16, N = ROWS * CPR / kAttnThreads;
    static_assert(N >= 1 && ROWS * CPR % kAttnThreads == 0, "a tile is a whole number of vectors a thread");
    // Loads i and i + P of a thread read the same vector of rows whose distance
    // is uniform: one offset serves them, on bases apart.
    static constexpr int STEP = kAttnThreads / CPR;        // rows a load of the workgroup covers
    static constexpr int P = kAttnThreads % CPR ? N : STEP % 16 == 0 ? 1 : STEP % 8 == 0 && N > 1 ? 2 : N;
    uint32_t off[P];
    u32x4 r[DIRECT ? 1 : N];
    __device__ __forceinline__ void init(long stride, int d) {
#pragma unroll
        for (int i = 0; i < P; i++) {
            const int v = threadIdx.x + i * kAttnThreads, r = v / CPR, c = v % CPR ^ tile_swz<CPR>(r);
            // an offset past any buffer's end reads as 0
            off[i] = c * VEC < d ? (uint32_t)(r * (int)stride * (int)sizeof(T)) + c * 16 : 0x80000000u;
        }
    }
    __device__ __forceinline__ void load(char* lds, int i, __amdgpu_buffer_rsrc_t rs, int base, int wave) {
        if constexpr (DIRECT)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                rs, (__attribute__((address_space(3))) void*)(lds + (wave * 64 + i * kAttnThreads) * 16), 16, (int)off[i % P],
                base, 0, 0);
        else
            r[i] = __builtin_amdgcn_raw_buffer_load_b128(rs, (int)off[i % P], base, 0);
    }
    // the tile's first row at `row`, `left` rows from there on (uniform)
    __device__ __forceinline__ void issue(char* lds, const T* row, int left, long stride, int d, bool vec, int wave) {
        if (vec && left >= ROWS) {
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)row, 0, 0x7fffffff, 0x00027000);
#pragma unroll
            for (int i = 0; i < N; i++) load(lds, i, rs, i / P * P * STEP * (int)stride * (int)sizeof(T), wave);
        } else if (vec) {
            // the buffer ends with the last row
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int skip = i / P * P * STEP, n = left - skip;
                const int bytes = n <= 0 ? 0 : ((n - 1) * (int)stride + d) * (int)sizeof(T);
                load(lds, i, __builtin_amdgcn_make_buffer_rsrc((void*)(row + skip * stride), 0, bytes, 0x00027000), 0, wave);
            }
        }
    }
    // the same tile's arguments
    __device__ __forceinline__ void commit(char* lds, const T* row, int left, long stride, int d, bool vec) {
        if (!vec) {
            const int tid = attn_fresh(threadIdx.x);
#pragma unroll 1
            for (int i = 0; i < N; i++) {
                const int v = tid + i * kAttnThreads, r = v / CPR, c = v % CPR ^ tile_swz<CPR>(r);
                *reinterpret_cast<u32x4*>(lds + v * 16) =
                    r < left ? load_chunk(row + (long)r * stride, c * VEC, d, false) : u32x4{0, 0, 0, 0};
            }
        } else if constexpr (!DIRECT) {
#pragma unroll
            for (int i = 0; i < N; i++) *reinterpret_cast<u32x4*>(lds + (threadIdx.x + i * kAttnThreads) * 16) = r[i];
        }
    }
};

// keeps a rare, uniform branch one: its body would else be done every time,
// and its results selected
__device__ __forceinline__ void attn_branch() { asm volatile(""); }

// every load into LDS so far has landed, for all the workgroup's waves
__device__ __forceinline__ void tiles_landed() {
    __builtin_amdgcn_s_waitcnt(0x0f70);            // vmcnt(0)
    __syncthreads();
}

// The key groups' (or row groups') accumulators of the same columns added
// into group 0's, 32 rows at a time through `lds` (16 KB a group past the
// first and column set); all the workgroup's waves call it.
template <int KG, int WR, int ND>
__device__ __forceinline__ void join_groups(f32x16 (&o)[ND], float f, char* lds, int wr, int kg, int lane) {
    float* jo = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int i = 0; i < ND; i++) {
        __syncthreads();
        if (kg) {
#pragma unroll
            for (int e = 0; e < 16; e++) jo[(((kg - 1) * WR + wr) * 16 + e) * 64 + lane] = o[i][e] * f;
        }
        __syncthreads();
        if (!kg) {
#pragma unroll
            for (int e = 0; e < 16; e++) {
                float t = o[i][e] * f;
#pragma unroll
                for (int k = 1; k < KG; k++) t += jo[(((k - 1) * WR + wr) * 16 + e) * 64 + lane];
                o[i][e] = t;
            }
        }
    }
}

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

// 4 values at columns c .. of a row
template <typename T>
__device__ __forceinline__ void store4(T* row, int c, const float (&v)[4], int d, bool vec) {
    union { T e[4]; u32x2 v2; u32x4 v4; } u;
#pragma unroll
    for (int j = 0; j < 4; j++) u.e[j] = Mma<T>::from_f32(v[j]);
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

// a 32-column accumulator set (DP rows of d) times f into one contiguous row
template <typename T, int ND>
__device__ __forceinline__ void attn_store(T* row, const f32x16 (&acc)[ND], float f, int d, int half, bool vec) {
#pragma unroll
    for (int n = 0; n < ND; n++)
#pragma unroll
        for (int b = 0; b < 4; b++) {
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = acc[n][4 * b + j] * f;
            store4(row, 32 * n + 8 * b + 4 * half, v, d, vec);
        }
}
// what the rounding to T took from that
template <typename T, int ND>
__device__ __forceinline__ void attn_store_rest(T* row, const f32x16 (&acc)[ND], float f, int d, int half, bool vec) {
#pragma unroll
    for (int n = 0; n < ND; n++)
#pragma unroll
        for (int b = 0; b < 4; b++) {
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                v[j] = acc[n][4 * b + j] * f;
                v[j] -= Mma<T>::to_f32(Mma<T>::from_f32(v[j]));
            }
            store4(row, 32 * n + 8 * b + 4 * half, v, d, vec);
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

// The wave's columns (bit r: column r) of which a lane says so.
__device__ __forceinline__ uint32_t columns_of(bool lane_says) {
    const uint64_t b = __ballot(lane_says);
    return (uint32_t)b | (uint32_t)(b >> 32);
}

// dot product of two rows of d values, and its partner's values times f added
// to lane e's columns e, e + 64, ...: the parts of a row done again on the VALU
template <typename T>
__device__ __forceinline__ float row_dot(const T* x, const T* y, int d) {
    float s = 0.0f;
    for (int c = 0; c < d; c++) s = __builtin_fmaf(Mma<T>::to_f32(x[c]), Mma<T>::to_f32(y[c]), s);
    return s;
}
template <typename T, int DP>
__device__ __forceinline__ void row_axpy(float (&acc)[(DP + 63) / 64], float f, const T* y, int d) {
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
__device__ __forceinline__ void attn_again(O* out, float f, int d, int j0, int j1, W w, R rows, O* lo = nullptr) {
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
        if (c < d) {
            const float v = acc[n] * f;
            out[c] = Mma<O>::from_f32(v);
            if (lo) lo[c] = Mma<O>::from_f32(v - Mma<O>::to_f32(out[c]));
        }
    }
}

}  // namespace rac
