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
// the lower token.
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
constexpr uint32_t kLpLowest = 0x007fffffu;              // -inf's key
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

// the wave's own LDS writes are there for its other lanes' reads
__device__ __forceinline__ void wave_lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
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

// An entry of a list: the key above, and the token so that of equal keys the
// lower one is the larger entry; 0 is none.
typedef unsigned long long lp_t;
__device__ __forceinline__ lp_t lp_entry(uint32_t key, int tok) {
    return (lp_t)key << 32 | (uint32_t)(0x7fffffff - tok);
}
__device__ __forceinline__ float lp_entry_value(lp_t e) { return lp_value((uint32_t)(e >> 32)); }
__device__ __forceinline__ int lp_entry_token(lp_t e) { return 0x7fffffff - (int)(uint32_t)e; }
__device__ __forceinline__ lp_t lp_lane(lp_t v, int lane) {                      // lane uniform
    return (lp_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}

// entry e (uniform) into the wave's list, best first, one to a lane
__device__ __forceinline__ void lp_insert(lp_t& list, lp_t e, int lane) {
    const int at = __popcll(__ballot(list > e));
    // the entry of the lane below (wave_shr:1)
    const int hi = (int)(list >> 32), lo = (int)list;
    const lp_t below = (lp_t)(uint32_t)__builtin_amdgcn_update_dpp(hi, hi, 0x138, 0xf, 0xf, false) << 32 |
                       (uint32_t)__builtin_amdgcn_update_dpp(lo, lo, 0x138, 0xf, 0xf, false);
    list = lane == at ? e : lane > at ? below : list;
}

// how many of the n entries at p (LDS, best first) beat e
__device__ __forceinline__ int lp_above(const lp_t* p, int n, lp_t e) {
    int lo = 0;
    for (int step = 32; step; step >>= 1)
        if (lo + step <= n && p[lo + step - 1] > e) lo += step;
    return lo == 63 && n == 64 && p[63] > e ? 64 : lo;
}

// The wave's c entries of no order, one to each of its first lanes, best first:
// each counts those that beat it, with no step waiting for the one before.
// buf: 64 entries of LDS of the wave's own.
__device__ __forceinline__ lp_t lp_sort(lp_t e, int c, lp_t* buf, int lane) {
    int rank = 0;
#pragma unroll 4
    for (int i = 0; i < c; i++) rank += lp_lane(e, i) > e;
    wave_lds_sync();
    if (lane < c) buf[rank] = e;
    wave_lds_sync();
    return lane < c ? buf[lane] : 0;
}

// the best `top` of two lists (c entries in `more`), each best first
__device__ __forceinline__ void lp_merge(lp_t& list, lp_t more, int top, int c, lp_t* buf, lp_t* buf2, int lane) {
    wave_lds_sync();
    buf[lane] = list;
    buf2[lane] = more;
    wave_lds_sync();
    const int a = lane + lp_above(buf2, c, list), b = lane + lp_above(buf, top, more);
    wave_lds_sync();
    if (lane < top && a < top) buf[a] = list;
    if (lane < c && b < top) buf[b] = more;
    wave_lds_sync();
    list = lane < top ? buf[lane] : 0;
}

// A key that at least `top` of the wave's values reach: the top-th largest of
// the lanes' own maxima, in its upper 16 bits.
__device__ __forceinline__ uint32_t lp_start(uint32_t mine, int top) {
    uint32_t t = 0;
#pragma unroll
    for (int bit = 31; bit >= 16; bit--) {
        const uint32_t more = t | 1u << bit;
        if (__popcll(__ballot(mine >= more)) >= top) t = more;
    }
    return t;
}

// the lists of the workgroup's waves into the `top` best, out[rank]
__device__ __forceinline__ void lp_rank(lp_t list, int top, lp_t (*all)[kLogprobMaxTop], lp_t* out) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    all[wave][lane] = list;
    __syncthreads();
    int rank = lane;
#pragma unroll
    for (int w = 1; w < kLpWaves; w++) {
        const int o = (wave + w) % kLpWaves;
        // empty entries behind those of the waves before
        int n = lp_above(all[o], top, list);
        if (list == 0 && o < wave) n = top;
        rank += n;
    }
    if (lane < top && rank < top) out[rank] = list;
    __syncthreads();
}

// row results from the whole row's statistics
template <typename T>
__device__ __forceinline__ void lp_finish(const LogprobArgs& a, long row, const LpStat& r, const lp_t* best) {
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
        a.top_lp[row * a.top + threadIdx.x] = logp(lp_entry_value(best[threadIdx.x]));
        a.top_tok[row * a.top + threadIdx.x] = lp_entry_token(best[threadIdx.x]);
    }
}

// floats of a split's part: three statistics, a gap, `top` entries
__host__ __device__ constexpr int lp_width(int top) { return 4 + 2 * top; }

// One workgroup per row and split: vectors [v0, v1) of the row.  Bound by reading
// the logits: 2048 bf16 rows of 128000 with 5 alternatives 121 us (4.3 TB/s;
// without 109, 4.8), 1001 fp32 rows of 50001 36 us (5.5 TB/s, part
// of it from cache).  One batch of loads is under way while the one before is
// summed (130 us in graph replay; loaded where used 153).
template <typename T, bool TOP>
__global__ __launch_bounds__(kLpThreads) void logprob_kernel(const LogprobArgs a) {
    constexpr int VEC = Mma<T>::VEC, U = 4;                // U vectors of a thread in flight
    __shared__ lp_t all[TOP ? kLpWaves : 1][kLogprobMaxTop], two[TOP ? kLpWaves : 1][64], best[kLogprobMaxTop];
    __shared__ float red[kLpWaves][3];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const long row = blockIdx.x;
    const int split = blockIdx.y;
    const T* x = (const T*)a.x + row * a.stride;
    // vectors on 16-byte boundaries: vector v is the values VEC v - off ..
    const int off = (int)(((uintptr_t)x / sizeof(T)) % VEC);
    const long nv = (a.vocab + off + VEC - 1) / VEC, per = (nv + a.splits - 1) / a.splits;
    const long v0 = split * per, v1 = v0 + per < nv ? v0 + per : nv;
    LpStat r = {-__builtin_inff(), 0.0f, 0.0f};
    lp_t list = 0, last = 0;                               // its last entry: what a value has to beat
    uint32_t thr = 0;                                      // the key that it has to reach
    // batches that lie within the row are loaded one ahead, 16 bytes a load
    u32x4 next[U];
    auto whole = [&](long b) { return b * VEC >= off && b + U * kLpThreads <= v1 && (b + U * kLpThreads) * VEC - off <= a.vocab; };
    auto fetch = [&](long b) {
#pragma unroll
        for (int u = 0; u < U; u++)
            next[u] = *reinterpret_cast<const u32x4*>(x + ((b + u * kLpThreads + tid) * VEC - off));
    };
    bool ahead = whole(v0);
    if (ahead) fetch(v0);
    for (long b = v0; b < v1; b += U * kLpThreads) {
        float f[U][VEC];
        if (ahead) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                union { u32x4 w; T e[VEC]; } in;
                in.w = next[u];
#pragma unroll
                for (int e = 0; e < VEC; e++) f[u][e] = Mma<T>::to_f32(in.e[e]);
            }
        } else {
#pragma unroll
            for (int u = 0; u < U; u++) {
                const long v = b + u * kLpThreads + tid, c = v * VEC - off;
                if (v < v1 && c >= 0 && c + VEC <= a.vocab) {
                    union { u32x4 w; T e[VEC]; } in;
                    in.w = *reinterpret_cast<const u32x4*>(x + c);
#pragma unroll
                    for (int e = 0; e < VEC; e++) f[u][e] = Mma<T>::to_f32(in.e[e]);
                } else {
#pragma unroll
                    for (int e = 0; e < VEC; e++)
                        f[u][e] = v < v1 && c + e >= 0 && c + e < a.vocab ? Mma<T>::to_f32(x[c + e]) : -__builtin_inff();
                }
            }
        }
        ahead = whole(b + U * kLpThreads);
        if (ahead) fetch(b + U * kLpThreads);
        float mx = f[0][0];
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                mx = fmaxf(mx, f[u][e]);
            }
        if constexpr (TOP) {
            const uint32_t mk = lp_key(mx);
            if (b == v0) thr = lp_start(mk, a.top);
            // NaN beside a number counts as -inf, which a maximum hides
            if (__any(mk >= thr) || thr <= kLpLowest) {
                lp_t* const cand = all[wave];
                int c = 0;
#pragma unroll
                for (int u = 0; u < U; u++) {
                    float um = f[u][0];
#pragma unroll
                    for (int e = 1; e < VEC; e++) um = fmaxf(um, f[u][e]);
                    const long v = b + u * kLpThreads + tid;
                    const int t0 = (int)(v * VEC - off);
                    if (!__any(v < v1 && lp_key(um) >= thr) && thr > kLpLowest) continue;
#pragma unroll
                    for (int e = 0; e < VEC; e++) {
                        const uint32_t key = lp_key(f[u][e]);
                        const int tok = t0 + e;
                        const lp_t entry = lp_entry(key, tok);
                        const bool in = v < v1 && tok >= 0 && tok < a.vocab && key >= thr && entry > last;
                        const uint64_t at = __ballot(in);
                        if (!at) continue;
                        const int place = c + __popcll(at & ((1ull << lane) - 1));
                        if (in && place < 64) cand[place] = entry;
                        c += __popcll(at);
                        if (c > 64) {
                            // what has no place goes into the list by itself
                            for (uint64_t rest = __ballot(in && place >= 64); rest; rest &= rest - 1)
                                lp_insert(list, lp_lane(entry, __ffsll((unsigned long long)rest) - 1), lane);
                            c = 64;
                        }
                    }
                }
                wave_lds_sync();
                lp_t more = lane < c ? cand[lane] : 0;
                if (c > 2) {
                    more = lp_sort(more, c, cand, lane);
                    lp_merge(list, more, a.top, c, cand, two[wave], lane);
                } else {
                    for (int i = 0; i < c; i++) lp_insert(list, lp_lane(more, i), lane);
                }
                last = lp_lane(list, a.top - 1);
                // a later batch's equal key has a higher token
                if ((uint32_t)(last >> 32) >= thr) thr = (uint32_t)(last >> 32) + 1;
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
    if constexpr (TOP) lp_rank(lane < a.top ? list : 0, a.top, all, best);
    else __syncthreads();
    r = {red[0][0], red[0][1], red[0][2]};
#pragma unroll
    for (int w = 1; w < kLpWaves; w++) lp_join(r, red[w][0], red[w][1], red[w][2]);
    if (a.splits == 1) {
        lp_finish<T>(a, row, r, best);
        return;
    }
    float* p = a.part + (row * a.splits + split) * lp_width(a.top);
    if (tid == 0) {
        p[0] = r.m;
        p[1] = r.l;
        p[2] = r.s;
    }
    if (TOP && tid < a.top) reinterpret_cast<lp_t*>(p + 4)[tid] = best[tid];
}

// The splits of a row joined.
template <typename T, bool TOP>
__global__ __launch_bounds__(kLpThreads) void logprob_join_kernel(const LogprobArgs a) {
    __shared__ lp_t all[TOP ? kLpWaves : 1][kLogprobMaxTop], two[TOP ? kLpWaves : 1][64], best[kLogprobMaxTop];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long row = blockIdx.x;
    const int width = lp_width(a.top);
    const float* p = a.part + row * a.splits * width;
    lp_t list = 0, more = 0;
    // the wave's first list as it stands; the next one's load ahead of its turn
    auto load = [&](int s) {
        return s < a.splits && lane < a.top ? reinterpret_cast<const lp_t*>(p + (long)s * width + 4)[lane] : 0;
    };
    if constexpr (TOP) {
        list = load(wave);
        more = load(wave + kLpWaves);
    }
    LpStat r = {-__builtin_inff(), 0.0f, 0.0f};
    for (int s = lane; s < a.splits; s += 64) {
        const float* q = p + (long)s * width;
        lp_join(r, q[0], q[1], q[2]);
    }
    lp_wave_join(r);
    if constexpr (TOP) {
        for (int s = wave + kLpWaves; s < a.splits; s += kLpWaves) {
            const lp_t next = load(s + kLpWaves);
            const int c = __popcll(__ballot(more > lp_lane(list, a.top - 1)));
            if (c > 2) {
                lp_merge(list, more, a.top, c, all[wave], two[wave], lane);
            } else {
                for (int i = 0; i < c; i++) lp_insert(list, lp_lane(more, i), lane);
            }
            more = next;
        }
        lp_rank(lane < a.top ? list : 0, a.top, all, best);
    }
    lp_finish<T>(a, row, r, best);
}

// dx of a piece of a row: VEC values a thread and step, four steps.  Reads the
// logits and writes as much: 1001 fp32 rows of 50001 84 us, 4096 bf16 rows of
// 32000 110 (4.7 TB/s both, a large copy's rate).  One step to a thread 85 and
// 113, sixteen 87 and 109, and 64 bf16 rows of 32000 4.1 and 10.2 against 4.9.
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

// Workgroups of few rows: about two to a CU, each of at least 4096 values.  us
// without alternatives, with 20 in the first two (MI355X), in two to a CU, four
// and one: 16 bf16 rows of 128000 21.4, 25, 18.9; 4 fp32 rows of 32000 14.5 in
// each; 64 fp32 rows of 128000 10.9, 11.2, 12.5; 1001 fp32 rows of 50001 36, 38,
// 36.  In pieces of 2048 at least the 4 rows take 15.7, in 8192 18.2.
static int logprob_splits(long rows, long vocab) {
    long s = (2 * device_cus() + rows - 1) / rows;
    const long most = (vocab + 4095) / 4096;
    if (s > most) s = most;
    return s < 1 ? 1 : (int)s;
}

long token_logprobs_workspace(long rows, long vocab, int top, int dtype) {
    const int s = logprob_splits(rows, vocab);
    return s > 1 ? 4L * rows * s * lp_width(top) : 0;
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
