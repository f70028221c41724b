// rac_logprob.hip — log probabilities of given tokens, the entropy and the
// likeliest tokens of rows of logits, and the gradient.
//
// Of a row x of V logits with m = max x, z_j = x_j - m, l = sum_j exp(z_j):
//   logp_j = z_j - log l,  lse = m + log l,
//   entropy = -sum_j p_j logp_j = log l - sum_j exp(z_j) z_j / l
// and, with g and h the gradients of logp_token and of the entropy,
//   dx_j = g ([j = token] - p_j) - h p_j (logp_j + entropy).
// One pass over the logits keeps a running maximum, both sums and a wave's
// list of its largest values; the sums of a row are fp32 sums of at most 32
// values a lane at a time.  In powers of two: e = 2^(x log2 e - r) with r =
// m log2 e rounded once, whose rounding is a factor of every e and so of l.  Logits of -inf have probability 0 and no part in
// the entropy; a row of nothing else has log probabilities of -inf, entropy 0
// and gradients 0.
//
// The list lives one entry to a lane, best first: keys are the logits' bits
// mapped to integers in their order (NaN as -inf, -0 as 0), equal keys go to
// the lower token.  Lanes offer their values in token order, so that a later
// value enters only if it is larger than the last entry.
#include <hip/hip_runtime.h>
#include "rac_internal.hpp"
#include "rac_mma.hpp"

namespace rac {

constexpr int kLpThreads = 256, kLpWaves = 4;

__device__ __forceinline__ uint32_t lp_key(float x) {
    if (!(x == x)) x = -__builtin_inff();
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
    return (int32_t)u < 0 ? ~u : u | 0x80000000u;
}
// the same of bits that are uniform, on the scalar side
__device__ __forceinline__ uint32_t lp_key_bits(uint32_t u) {
    if ((u & 0x7fffffffu) > 0x7f800000u) u = 0xff800000u;
    if (u == 0x80000000u) u = 0;
    return (int32_t)u < 0 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float lp_value(uint32_t k) {
    return __builtin_bit_cast(float, (int32_t)k < 0 ? k & 0x7fffffffu : ~k);
}

// a row's running statistics
struct LpStat {
    float m, l, s;                            // maximum times log2 e (r), sum e, sum e (x log2 e - r)
};
constexpr float kLpLn2 = 0.69314718f;
__device__ __forceinline__ void lp_join(LpStat& a, float m, float l, float s) {
    const float mt = fmaxf(a.m, m);
    const float da = a.m - mt, db = m - mt;   // NaN where both are -inf: l is 0 there
    const float fa = a.l == 0.0f ? 0.0f : exp2_hw(da), fb = l == 0.0f ? 0.0f : exp2_hw(db);
    // sum e (z + d), for a part with nothing in it d may be -inf
    const float sa = fa == 0.0f ? 0.0f : fa * __builtin_fmaf(a.l, da, a.s);
    const float sb = fb == 0.0f ? 0.0f : fb * __builtin_fmaf(l, db, s);
    a.l = a.l * fa + l * fb;
    a.s = sa + sb;
    a.m = mt;
}

// the wave's lanes joined, the same bits in all
__device__ __forceinline__ void lp_wave_join(LpStat& r) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const float m = __shfl_xor(r.m, o), l = __shfl_xor(r.l, o), s = __shfl_xor(r.s, o);
        // the same order of the two in both lanes
        LpStat p = {lane & o ? m : r.m, lane & o ? l : r.l, lane & o ? s : r.s};
        lp_join(p, lane & o ? r.m : m, lane & o ? r.l : l, lane & o ? r.s : s);
        r = p;
    }
}

// the value of the lane below (lane 0 keeps its own)
__device__ __forceinline__ int lane_below(int v) {
    return __builtin_amdgcn_update_dpp(v, v, 0x138, 0xf, 0xf, false);        // wave_shr:1
}

// entry (key, tok) into the wave's list
__device__ __forceinline__ void lp_insert(uint32_t& lk, int& lt, uint32_t key, int tok, int lane) {
    const int at = __popcll(__ballot(lk > key || (lk == key && lt < tok)));
    const uint32_t pk = (uint32_t)lane_below((int)lk);
    const int pt = lane_below(lt);
    lk = lane == at ? key : lane > at ? pk : lk;
    lt = lane == at ? tok : lane > at ? pt : lt;
}

// A threshold that at least `top` of the wave's values exceed (0: none such):
// just below the top-th largest of the lanes' own maxima.
__device__ __forceinline__ uint32_t lp_start(uint32_t mine, int top) {
    int above = 0;
    for (int i = 0; i < 64; i++) {
        const uint32_t k = (uint32_t)__builtin_amdgcn_readlane((int)mine, i);
        above += k > mine || (k == mine && i < (int)(threadIdx.x & 63));
    }
    const uint64_t at = __ballot(above == top - 1);
    const uint32_t k = (uint32_t)__builtin_amdgcn_readlane((int)mine, __ffsll((unsigned long long)at) - 1);
    return k ? k - 1 : 0;
}

// the lists of the workgroup's waves into the `top` best, rank by rank
__device__ __forceinline__ void lp_rank(uint32_t lk, int lt, int top, uint32_t (*sk)[kLogprobMaxTop],
                                        int (*st)[kLogprobMaxTop], uint32_t* ok, int* ot) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    sk[wave][lane] = lk;
    st[wave][lane] = lt;
    __syncthreads();
    if (lane < top) {
        int rank = 0;
#pragma unroll
        for (int w = 0; w < kLpWaves; w++)
            for (int i = 0; i < top; i += 4) {
                const u32x4 k4 = *reinterpret_cast<const u32x4*>(&sk[w][i]);
                const u32x4 t4 = *reinterpret_cast<const u32x4*>(&st[w][i]);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    // empty entries alike but for their place
                    const uint32_t k = k4[j];
                    const int t = (int)t4[j];
                    rank += i + j < top &&
                            (k > lk || (k == lk && (t < lt || (t == lt && 64 * w + i + j < 64 * wave + lane))));
                }
            }
        if (rank < top) {
            ok[rank] = lk;
            ot[rank] = lt;
        }
    }
    __syncthreads();
}

// row results from the whole row's statistics
template <typename T>
__device__ __forceinline__ void lp_finish(const LogprobArgs& a, long row, const LpStat& r, const uint32_t* ok,
                                          const int* ot) {
    const bool empty = r.m == -__builtin_inff() && r.l == 0.0f;
    const float ll = __builtin_logf(r.l), lse = empty ? -__builtin_inff() : __builtin_fmaf(r.m, kLpLn2, ll);
    auto logp = [&](float x) {
        return x == -__builtin_inff() && r.l == r.l ? x : __builtin_fmaf(x, kLog2e, -r.m) * kLpLn2 - ll;
    };
    if (threadIdx.x == 0) {
        const long t = a.tok[row];
        float lp = 0.0f;                      // a negative token: none
        if (t >= a.vocab) lp = __builtin_nanf("");
        else if (t >= 0) lp = logp(Mma<T>::to_f32(((const T*)a.x)[row * a.stride + t]));
        a.lp[row] = lp;
        a.ent[row] = empty ? 0.0f : ll - r.s / r.l * kLpLn2;
        if (a.lse) a.lse[row] = lse;
    }
    if ((int)threadIdx.x < a.top) {
        a.top_lp[row * a.top + threadIdx.x] = logp(lp_value(ok[threadIdx.x]));
        a.top_tok[row * a.top + threadIdx.x] = ot[threadIdx.x];
    }
}

// One workgroup per row and split: columns [c0, c1) of the row.
template <typename T, bool TOP>
__global__ __launch_bounds__(kLpThreads) void logprob_kernel(const LogprobArgs a) {
    constexpr int VEC = Mma<T>::VEC, U = 4;                // U vectors of a thread in flight
    __shared__ __attribute__((aligned(16))) uint32_t sk[TOP ? kLpWaves : 1][kLogprobMaxTop], ok[kLogprobMaxTop];
    __shared__ __attribute__((aligned(16))) int st[TOP ? kLpWaves : 1][kLogprobMaxTop], ot[kLogprobMaxTop];
    __shared__ float red[kLpWaves][3];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long row = blockIdx.x;
    const int split = blockIdx.y;
    const T* x = (const T*)a.x + row * a.stride;
    // vectors on 16-byte boundaries: vector v is the values VEC v - off ..
    const int off = (int)(((uintptr_t)x / sizeof(T)) % VEC);
    const long nv = (a.vocab + off + VEC - 1) / VEC, per = (nv + a.splits - 1) / a.splits;
    const long v0 = split * per, v1 = v0 + per < nv ? v0 + per : nv;
    LpStat r = {-__builtin_inff(), 0.0f, 0.0f};
    uint32_t lk = 0;                                       // 0: nothing yet
    int lt = 0x7fffffff;
    uint32_t thr = 0;
    for (long b = v0; b < v1; b += U * kLpThreads) {
        float f[U][VEC];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long v = b + u * kLpThreads + tid, c = v * VEC - off;
            union { u32x4 w; T e[VEC]; } in;
            if (v < v1 && c >= 0 && c + VEC <= a.vocab) {
                in.w = *reinterpret_cast<const u32x4*>(x + c);
#pragma unroll
                for (int e = 0; e < VEC; e++) f[u][e] = Mma<T>::to_f32(in.e[e]);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; e++)
                    f[u][e] = v < v1 && c + e >= 0 && c + e < a.vocab ? Mma<T>::to_f32(x[c + e]) : -__builtin_inff();
            }
        }
        float mx = f[0][0];
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                mx = fmaxf(mx, f[u][e]);
            }
        if constexpr (TOP) {
            if (__any(lp_key(mx) > thr)) {
                // keys of places past the row are never offered, but count as
                // -inf here, which at worst is too low a threshold
                if (b == v0) thr = lp_start(lp_key(mx), a.top);
#pragma unroll
                for (int u = 0; u < U; u++) {
                    float um = f[u][0];
#pragma unroll
                    for (int e = 1; e < VEC; e++) um = fmaxf(um, f[u][e]);
                    const long v = b + u * kLpThreads + tid, c = v * VEC - off;
                    const uint32_t uk = v < v1 ? lp_key(um) : 0;
                    for (uint64_t cand = __ballot(uk > thr); cand;) {
                        const int src = __ffsll((unsigned long long)cand) - 1;
#pragma unroll
                        for (int e = 0; e < VEC; e++) {
                            const float fe = f[u][e];
                            const uint32_t key = lp_key_bits(__builtin_amdgcn_readlane(__builtin_bit_cast(int, fe), src));
                            if (key > thr) {
                                const int tok = __builtin_amdgcn_readlane((int)(c + e), src);
                                if (tok >= 0 && tok < a.vocab) {
                                    lp_insert(lk, lt, key, tok, lane);
                                    const uint32_t last = __builtin_amdgcn_readlane(lk, a.top - 1);
                                    if (last > thr) thr = last;
                                }
                            }
                        }
                        // the lanes behind that still have one
                        cand = src == 63 ? 0 : __ballot(uk > thr) & (~0ull << (src + 1));
                    }
                }
            }
        }
        mx *= kLog2e;
        if (mx > r.m) {
            const float d = r.m - mx;
            const float g = exp2_hw(d);
            r.s = g == 0.0f ? 0.0f : g * __builtin_fmaf(r.l, d, r.s);
            r.l *= g;
            r.m = mx;
        }
        const float mu = r.m == -__builtin_inff() ? 0.0f : r.m;
        float bl = 0.0f, bs = 0.0f;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const float z = __builtin_fmaf(f[u][e], kLog2e, -mu), p = exp2_hw(z);
                bl += p;
                bs = __builtin_fmaf(p, fmaxf(z, -1e4f), bs);       // p is 0 there, z may be -inf
            }
        r.l += bl;
        r.s += bs;
    }
    // NaN came through l; infinity less itself did too
    lp_wave_join(r);
    if (lane == 0) {
        red[wave][0] = r.m;
        red[wave][1] = r.l;
        red[wave][2] = r.s;
    }
    if constexpr (TOP) lp_rank(lk, lt, a.top, sk, st, ok, ot);
    else __syncthreads();
    r = {red[0][0], red[0][1], red[0][2]};
#pragma unroll
    for (int w = 1; w < kLpWaves; w++) lp_join(r, red[w][0], red[w][1], red[w][2]);
    if (a.splits == 1) {
        lp_finish<T>(a, row, r, ok, ot);
        return;
    }
    float* p = a.part + (row * a.splits + split) * (3 + 2 * a.top);
    if (tid == 0) {
        p[0] = r.m;
        p[1] = r.l;
        p[2] = r.s;
    }
    if (TOP && tid < a.top) {
        reinterpret_cast<uint32_t*>(p)[3 + tid] = ok[tid];
        reinterpret_cast<int*>(p)[3 + a.top + tid] = ot[tid];
    }
}

// The splits of a row joined.
template <typename T, bool TOP>
__global__ __launch_bounds__(kLpThreads) void logprob_join_kernel(const LogprobArgs a) {
    __shared__ __attribute__((aligned(16))) uint32_t sk[TOP ? kLpWaves : 1][kLogprobMaxTop], ok[kLogprobMaxTop];
    __shared__ __attribute__((aligned(16))) int st[TOP ? kLpWaves : 1][kLogprobMaxTop], ot[kLogprobMaxTop];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long row = blockIdx.x;
    const int width = 3 + 2 * a.top;
    const float* p = a.part + row * a.splits * width;
    LpStat r = {-__builtin_inff(), 0.0f, 0.0f};
    for (int s = lane; s < a.splits; s += 64) lp_join(r, p[s * width], p[s * width + 1], p[s * width + 2]);
    lp_wave_join(r);
    if constexpr (TOP) {
        // the wave's first list as it stands; the next one's loads ahead of its turn
        const uint32_t* list = reinterpret_cast<const uint32_t*>(p) + 3;
        auto load = [&](int s, uint32_t& k, int& t) {
            const bool there = s < a.splits && lane < a.top;
            k = there ? list[s * width + lane] : 0;
            t = there ? (int)list[s * width + a.top + lane] : 0x7fffffff;
        };
        uint32_t lk, mk;
        int lt, mt;
        load(wave, lk, lt);
        load(wave + kLpWaves, mk, mt);
        for (int s = wave + kLpWaves; s < a.splits; s += kLpWaves) {
            uint32_t nk;
            int nt;
            load(s + kLpWaves, nk, nt);
            for (int i = 0; i < a.top; i++) {
                const uint32_t key = __builtin_amdgcn_readlane(mk, i);
                // splits come in token order: an equal key's token is higher
                if (key <= __builtin_amdgcn_readlane(lk, a.top - 1)) break;
                lp_insert(lk, lt, key, __builtin_amdgcn_readlane(mt, i), lane);
            }
            mk = nk;
            mt = nt;
        }
        lp_rank(lk, lt, a.top, sk, st, ok, ot);
    }
    lp_finish<T>(a, row, r, ok, ot);
}

// dx of a piece of a row: VEC values a thread and step.
template <typename T>
__global__ __launch_bounds__(kLpThreads) void logprob_backward_kernel(const void* __restrict__ xv, long stride,
                                                                     const long* __restrict__ tok,
                                                                     const float* __restrict__ lse_in,
                                                                     const float* __restrict__ ent_in,
                                                                     const float* __restrict__ g_lp,
                                                                     const float* __restrict__ g_ent, void* dxv,
                                                                     long vocab, long per) {
    constexpr int VEC = Mma<T>::VEC;
    const long row = blockIdx.x;
    const T* x = (const T*)xv + row * stride;
    T* dx = (T*)dxv + row * vocab;
    const float lse = lse_in[row], ent = ent_in[row];
    const long t = tok[row];
    float g = g_lp && t >= 0 ? g_lp[row] : 0.0f;
    if (t >= vocab) g = __builtin_nanf("");
    const float h = g_ent ? g_ent[row] : 0.0f;
    const float a0 = -(g + h * ent);                       // dx = p (a0 - h logp) (+ g at the token)
    const bool empty = lse == -__builtin_inff();
    auto grad = [&](float v, long c) {
        const float lp = v - lse, p = exp2_hw(lp * kLog2e);
        float d = p == 0.0f || empty ? 0.0f : p * __builtin_fmaf(-h, lp, a0);
        if (c == t && !empty) d += g;
        return Mma<T>::from_f32(d);
    };
    // vectors on the output's 16-byte boundaries; the input's where it shares them
    const int off = (int)(((uintptr_t)dx / sizeof(T)) % VEC);
    const bool same = (uintptr_t)x % 16 == (uintptr_t)dx % 16;
    const long nv = (vocab + off + VEC - 1) / VEC;
    const long v0 = blockIdx.y * per, v1 = v0 + per < nv ? v0 + per : nv;
    for (long v = v0 + threadIdx.x; v < v1; v += kLpThreads) {
        const long c = v * VEC - off;
        if (c >= 0 && c + VEC <= vocab) {
            union { u32x4 w; T e[VEC]; } in, out;
            if (same) {
                in.w = *reinterpret_cast<const u32x4*>(x + c);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; e++) in.e[e] = x[c + e];
            }
#pragma unroll
            for (int e = 0; e < VEC; e++) out.e[e] = grad(Mma<T>::to_f32(in.e[e]), c + e);
            *reinterpret_cast<u32x4*>(dx + c) = out.w;
        } else {
            for (int e = 0; e < VEC; e++)
                if (c + e >= 0 && c + e < vocab) dx[c + e] = grad(Mma<T>::to_f32(x[c + e]), c + e);
        }
    }
}

// Workgroups of few rows: about four to a CU, each of at least 2048 values.
static int logprob_splits(long rows, long vocab) {
    long s = (4 * device_cus() + rows - 1) / rows;
    const long most = (vocab + 2047) / 2048;
    if (s > most) s = most;
    return s < 1 ? 1 : (int)s;
}

long token_logprobs_workspace(long rows, long vocab, int top, int dtype) {
    const int s = logprob_splits(rows, vocab);
    return s > 1 ? 4L * rows * s * (3 + 2 * top) : 0;
}

template <typename T>
static void logprob_launch_t(const LogprobArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)a.rows, a.splits), t(kLpThreads);
    if (a.top) hipLaunchKernelGGL((logprob_kernel<T, true>), grid, t, 0, s, a);
    else hipLaunchKernelGGL((logprob_kernel<T, false>), grid, t, 0, s, a);
    if (a.splits > 1) {
        if (a.top) hipLaunchKernelGGL((logprob_join_kernel<T, true>), dim3((unsigned)a.rows), t, 0, s, a);
        else hipLaunchKernelGGL((logprob_join_kernel<T, false>), dim3((unsigned)a.rows), t, 0, s, a);
    }
}

hipError_t token_logprobs_launch(LogprobArgs a, int dtype, hipStream_t s) {
    a.splits = logprob_splits(a.rows, a.vocab);
    if (dtype == 0) logprob_launch_t<float>(a, s);
    else if (dtype == 1) logprob_launch_t<__bf16>(a, s);
    else logprob_launch_t<_Float16>(a, s);
    return hipGetLastError();
}

hipError_t token_logprobs_backward_launch(const void* x, long stride, const long* tok, const float* lse,
                                          const float* ent, const float* g_lp, const float* g_ent, void* dx, long rows,
                                          long vocab, int dtype, hipStream_t s) {
    const int vec = dtype == 0 ? 4 : 8;
    const long nv = (vocab + 2 * vec - 2) / vec;           // of the worst offset
    long pieces = (nv + 4 * kLpThreads - 1) / (4 * kLpThreads);
    if (pieces > 65535) pieces = 65535;
    const long per = (nv + pieces - 1) / pieces;
    const dim3 grid((unsigned)rows, (unsigned)pieces), t(kLpThreads);
#define RAC_LP_BACKWARD(T)                                                                                           \
    hipLaunchKernelGGL((logprob_backward_kernel<T>), grid, t, 0, s, x, stride, tok, lse, ent, g_lp, g_ent, dx, vocab, per)
    if (dtype == 0) RAC_LP_BACKWARD(float);
    else if (dtype == 1) RAC_LP_BACKWARD(__bf16);
    else RAC_LP_BACKWARD(_Float16);
#undef RAC_LP_BACKWARD
    return hipGetLastError();
}

}  // namespace rac
