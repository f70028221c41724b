// rac_tree.hip — attention of a tree of drafted tokens over a key/value cache.
//
// Of sequence b the cache holds len tokens, positions 0 .. len - 1, and the
// keys and values of its T drafted tokens at positions len .. len + T - 1.
// Drafted token t continues token parents[t] < t, or the cache itself (-1); it
// sees the cache, its ancestors and itself:
//   o_t = sum_j p_j v_j,  p = softmax_j(scale q_t . k_j),
//   j < len or j = len + u with u on t's path to the root.
// A decode step is T = 1, a chain of tokens parents[t] = t - 1.
//
// The queries of all heads that share a key / value head are rows over the
// same keys: row t rep + r of group g is token t of head g rep + r, so the
// cache is read once for up to 32 rows a wave.  Few rows: the workgroup's
// waves take different keys; many: different rows of the same keys.  The keys
// are split over workgroups, which leave their rows' running maximum, sum and
// unnormalised output; a second launch joins them.
#include <hip/hip_runtime.h>
#include "rac_attn.hpp"
#include "rac_internal.hpp"

namespace rac {

constexpr int kTreeThreads = kAttnThreads;
constexpr int kTreeWords = kTreeMaxTokens / 32 + 1;       // one more, always 0, for reads of 32 bits at any place

// keys a wave takes at a time, and those of a tile: one such set for each of
// the workgroup's key groups
constexpr int tree_bn(int es, int wr) { return es == 2 && wr == kAttnWaves ? 64 : 32; }
constexpr int tree_tile(int es, int wr) { return tree_bn(es, wr) * (kAttnWaves / wr); }

// the tiles that split s of `splits` takes out of `tiles`: `per` from s per on
__device__ __forceinline__ int tree_per(int tiles, int splits) { return (tiles + splits - 1) / splits; }

template <typename T, int DP, int WR>
__global__ __launch_bounds__(kTreeThreads, DP * sizeof(T) <= 256 ? 2 : 1) void tree_kernel(const TreeArgs a) {
    using M = Mma<T>;
    using Frag = typename M::Frag;
    constexpr int KF = M::KF, NF = DP / KF, ND = DP / 32, LD = DP + M::VEC;
    constexpr int BN = tree_bn(sizeof(T), WR), NS = BN / 32;
    constexpr int KG = kAttnWaves / WR, TILE = BN * KG;
    // the waves' outputs are joined where the tiles were
    constexpr int TILES = 2 * TILE * LD * (int)sizeof(T), JOIN = KG > 1 ? (KG - 1) * WR * 64 * 16 * 4 : 0;
    __shared__ __attribute__((aligned(16))) char lds[TILES > JOIN ? TILES : JOIN];
    __shared__ uint32_t anc[kTreeMaxTokens][kTreeWords];
    __shared__ int up[2][kTreeMaxTokens];
    __shared__ float sm[kAttnWaves][32], sl[kAttnWaves][32];
    T* const sk = (T*)lds;
    T* const sv = sk + TILE * LD;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;
    const int wr = wave % WR, kg = wave / WR;
    const int rep = a.heads / a.kv_heads, rows = rep * a.tokens;
    const int split = blockIdx.x, rb = blockIdx.y, b = blockIdx.z / a.kv_heads, g = blockIdx.z % a.kv_heads;
    const int r = (rb * WR + wr) * 32 + (lane & 31);                    // the lane's row
    const bool there = r < rows;
    const int tok = there ? r / rep : 0, head = g * rep + (there ? r % rep : 0);
    const int len = a.len[b];
    T* out = (T*)a.out + (((long)b * a.tokens + tok) * a.heads + head) * a.d;
    const bool ok = len >= 0 && (long)len + a.tokens <= a.cap;
    const int n = ok ? len + a.tokens : 0;
    const int tiles = (n + TILE - 1) / TILE, per = tree_per(tiles, a.splits);
    const int j0 = split * per, j1 = min(tiles, j0 + per);
    if (!ok) {
        // a length outside the cache: NaN, nothing read
        if (split == 0 && there && kg == 0)
            for (int c = half; c < a.d; c += 2) out[c] = M::from_f32(__builtin_nanf(""));
        return;
    }
    if (j0 >= j1) return;
    const T* K = (const T*)a.k + (long)b * a.sk_b + (long)g * a.sk_g;
    const T* V = (const T*)a.v + (long)b * a.sv_b + (long)g * a.sv_g;
    const T* qrow = (const T*)a.q + (long)b * a.sq_b + (long)tok * a.sq_t + (long)head * a.sq_h;
    TileStage<T, DP, TILE> rk, rv;
    rk.load(K, a.sk_t, j0 * TILE, n, a.d, a.vec);
    rv.load(V, a.sv_t, j0 * TILE, n, a.d, a.vec);
    Frag qf[NF];
    load_frags<T, DP>(qf, qrow, there, a.d, half, a.vec);
    const bool tail = j1 * TILE > len;                   // the split holds drafted tokens
    if (tail) {
        // paths to the root, a step that doubles what is known at a time
        int p = -1;
        if (tid < a.tokens) {
            p = a.parents[(long)b * a.parents_b + tid];
            if (p >= tid) p = -1;
            up[0][tid] = p;
#pragma unroll
            for (int w = 0; w < kTreeWords; w++) anc[tid][w] = w == tid / 32 ? 1u << (tid & 31) : 0u;
        }
        for (int hop = 1, cur = 0; hop < a.tokens; hop *= 2, cur ^= 1) {
            __syncthreads();
            uint32_t m[kTreeWords];
            if (tid < a.tokens && p >= 0) {
#pragma unroll
                for (int w = 0; w < kTreeWords; w++) m[w] = anc[tid][w] | anc[p][w];
                p = up[cur][p];
            }
            __syncthreads();
            if (tid < a.tokens) {
                if (up[cur][tid] >= 0) {
#pragma unroll
                    for (int w = 0; w < kTreeWords; w++) anc[tid][w] = m[w];
                }
                up[cur ^ 1][tid] = p;
            }
        }
    }
    const float c = a.scale * kLog2e;
    f32x16 o[ND];
#pragma unroll
    for (int i = 0; i < ND; i++) o[i] = zero16();
    float m = -__builtin_inff(), l = 0.0f;
    // bits of positions len + u .. + 31 that the row sees, ones before the drafts
    auto seen = [&](int u) -> uint32_t {
        if (u >= a.tokens) return 0u;
        if (u <= -32) return ~0u;
        const uint32_t* w = anc[tok];
        if (u < 0) return (1u << -u) - 1u | w[0] << -u;
        const uint64_t two = w[u >> 5] | (uint64_t)w[(u >> 5) + 1] << 32;
        return (uint32_t)(two >> (u & 31));
    };
    for (int j = j0; j < j1; j++) {
        __syncthreads();
        rk.template store<LD>(sk);
        rv.template store<LD>(sv);
        __syncthreads();
        if (j + 1 < j1) {
            rk.load(K, a.sk_t, (j + 1) * TILE, n, a.d, a.vec);
            rv.load(V, a.sv_t, (j + 1) * TILE, n, a.d, a.vec);
        }
        const int first = j * TILE + kg * BN;             // the wave's keys
        if (first >= n) continue;
        const T* ks = sk + kg * BN * LD;
        const T* vs = sv + kg * BN * LD;
        f32x16 s[NS];
#pragma unroll
        for (int u = 0; u < NS; u++) {
            s[u] = zero16();
#pragma unroll
            for (int f = 0; f < NF; f++)
                s[u] = M::mma(*reinterpret_cast<const Frag*>(ks + (32 * u + (lane & 31)) * LD + f * KF +
                                                             half * (KF / 2)), qf[f], s[u]);
        }
        if (first + BN > len) {
#pragma unroll
            for (int u = 0; u < NS; u++) {
                const uint32_t bits = seen(first + 32 * u - len);
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (!(bits >> (8 * (i / 4) + 4 * half + i % 4) & 1)) s[u][i] = -__builtin_inff();
            }
        }
        float mx = s[0][0];
#pragma unroll
        for (int u = 0; u < NS; u++)
#pragma unroll
            for (int i = 0; i < 16; i++) mx = fmaxf(mx, s[u][i]);
        mx = fmaxf(m, half_max(mx) * c);
        const float mu = mx == -__builtin_inff() ? 0.0f : mx;
        const float al = exp2_hw(m - mu);
        m = mx;
        float ls = 0.0f;
#pragma unroll
        for (int u = 0; u < NS; u++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                s[u][i] = exp2_hw(__builtin_fmaf(s[u][i], c, -mu));
                ls += s[u][i];
            }
        l = __builtin_fmaf(l, al, ls);
#pragma unroll
        for (int i = 0; i < ND; i++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[i][e] *= al;
#pragma unroll
        for (int u = 0; u < NS; u++)
#pragma unroll
            for (int f = 0; f < 32 / KF; f++) {
                const Frag pf = M::pack(s[u], f);
#pragma unroll
                for (int i = 0; i < ND; i++)
                    o[i] = M::mma(M::load_tr(vs + 32 * u * LD + 32 * i, LD, f, lane), pf, o[i]);
            }
    }
    l = half_sum(l);
    if constexpr (KG > 1) {
        // the key groups' rows into group 0's, 32 columns of d at a time
        float* jo = (float*)lds;
        if (half == 0) {
            sm[wave][lane] = m;
            sl[wave][lane] = l;
        }
        __syncthreads();
        float mt = -__builtin_inff();
#pragma unroll
        for (int k = 0; k < KG; k++) mt = fmaxf(mt, sm[k * WR + wr][lane & 31]);
        const float mu = mt == -__builtin_inff() ? 0.0f : mt;
        l = 0.0f;
#pragma unroll
        for (int k = 0; k < KG; k++) l = __builtin_fmaf(sl[k * WR + wr][lane & 31], exp2_hw(sm[k * WR + wr][lane & 31] - mu), l);
        const float f = exp2_hw(m - mu);
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
        m = mt;
        if (kg) return;
    }
    // rows that met a value that is not finite: again, over what they see
    uint64_t again = __ballot(not_finite(o) && there);
    again = (again | again >> 32) & 0xffffffffull;
    const bool store = there && !(again >> (lane & 31) & 1);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const bool whole = per >= tiles;                      // no other split has keys
    float* po = a.part + (((long)b * a.kv_heads + g) * a.splits + split) * rows * (a.d + 2);
    if (whole) {
        if (store) attn_store<T, ND>(out, o, inv, a.d, half, a.vec_out);
    } else {
        if (there && half == 0) {
            po[(long)r * (a.d + 2) + a.d] = m;
            po[(long)r * (a.d + 2) + a.d + 1] = l;
        }
        if (store) attn_store<float, ND>(po + (long)r * (a.d + 2), o, 1.0f, a.d, half, false);
    }
    for (; again; again &= again - 1) {
        const int rl = __ffsll((unsigned long long)again) - 1, rr = (rb * WR + wr) * 32 + rl;
        const int t = rr / rep, hh = g * rep + rr % rep;
        const float mr = __shfl(m, rl), ir = __shfl(inv, rl);
        const T* q = (const T*)a.q + (long)b * a.sq_b + (long)t * a.sq_t + (long)hh * a.sq_h;
        auto w = [&](int j) {
            if (j >= len && !(anc[t][(j - len) >> 5] >> ((j - len) & 31) & 1)) return -1.0f;
            return exp2_hw(__builtin_fmaf(row_dot(q, K + (long)j * a.sk_t, a.d), c, -mr));
        };
        auto vrow = [&](int j) { return V + (long)j * a.sv_t; };
        const int ja = j0 * TILE, jb = min(n, j1 * TILE);
        if (whole)
            attn_again<T, DP, true>((T*)a.out + (((long)b * a.tokens + t) * a.heads + hh) * a.d, ir, a.d, ja, jb, w, vrow);
        else
            attn_again<T, DP, true>(po + (long)rr * (a.d + 2), 1.0f, a.d, ja, jb, w, vrow);
    }
}

// Splits joined: a wave per row.
template <typename T>
__global__ __launch_bounds__(kTreeThreads) void tree_join_kernel(const TreeArgs a, int tile) {
    const int lane = threadIdx.x & 63, rep = a.heads / a.kv_heads, rows = rep * a.tokens;
    const int r = blockIdx.x * kAttnWaves + (threadIdx.x >> 6), b = blockIdx.y / a.kv_heads, g = blockIdx.y % a.kv_heads;
    if (r >= rows) return;
    const int len = a.len[b];
    if (len < 0 || (long)len + a.tokens > a.cap) return;
    const int tiles = (len + a.tokens + tile - 1) / tile, per = tree_per(tiles, a.splits);
    if (per >= tiles) return;                              // one split: it stored the rows itself
    const int live = (tiles + per - 1) / per;
    const float* p = a.part + ((long)b * a.kv_heads + g) * a.splits * rows * (a.d + 2) + (long)r * (a.d + 2);
    const long step = (long)rows * (a.d + 2);
    float m = -__builtin_inff();
    for (int s = lane; s < live; s += 64) m = fmaxf(m, p[s * step + a.d]);
#pragma unroll
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if (m == -__builtin_inff()) m = 0.0f;
    float l = 0.0f, acc[4] = {};
    for (int s = 0; s < live; s++) {
        const float f = exp2_hw(p[s * step + a.d] - m);
        l = __builtin_fmaf(f, p[s * step + a.d + 1], l);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (lane + 64 * i < a.d) acc[i] = __builtin_fmaf(f, p[s * step + lane + 64 * i], acc[i]);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* out = (T*)a.out + (((long)b * a.tokens + r / rep) * a.heads + g * rep + r % rep) * a.d;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (lane + 64 * i < a.d) out[lane + 64 * i] = Mma<T>::from_f32(acc[i] * inv);
}

// Rows of a wave set: one wave's 32 while all fit there, else four waves' 128;
// d past 128 in fp32 leaves LDS for one key group only.
struct TreePlan {
    int wr, tile, splits;
};
static TreePlan tree_plan(const TreeArgs& a, int dtype) {
    const int rows = a.heads / a.kv_heads * a.tokens, es = dtype == 0 ? 4 : 2;
    const int dp = a.d <= 32 ? 32 : a.d <= 64 ? 64 : a.d <= 128 ? 128 : 256;
    TreePlan p;
    p.wr = rows <= 32 && dp * es <= 512 ? 1 : 4;
    p.tile = tree_tile(es, p.wr);
    const long groups = (long)a.batch * a.kv_heads * ((rows + 32 * p.wr - 1) / (32 * p.wr));
    const long most = (a.cap + p.tile - 1) / p.tile;
    long s = (2 * device_cus() + groups - 1) / groups;
    if (s > most) s = most;
    if (s > 64) s = 64;
    p.splits = s < 1 ? 1 : (int)s;
    return p;
}

template <typename T, int DP>
static void tree_launch_dp(const TreeArgs& a, const TreePlan& p, hipStream_t s) {
    const int rows = a.heads / a.kv_heads * a.tokens;
    const dim3 grid(p.splits, (rows + 32 * p.wr - 1) / (32 * p.wr), a.batch * a.kv_heads);
    if constexpr (DP * sizeof(T) <= 512) {
        if (p.wr == 1) {
            hipLaunchKernelGGL((tree_kernel<T, DP, 1>), grid, dim3(kTreeThreads), 0, s, a);
            return;
        }
    }
    hipLaunchKernelGGL((tree_kernel<T, DP, 4>), grid, dim3(kTreeThreads), 0, s, a);
}

template <typename T>
static void tree_launch_t(const TreeArgs& a, const TreePlan& p, hipStream_t s) {
    if (a.d <= 32) tree_launch_dp<T, 32>(a, p, s);
    else if (a.d <= 64) tree_launch_dp<T, 64>(a, p, s);
    else if (a.d <= 128) tree_launch_dp<T, 128>(a, p, s);
    else tree_launch_dp<T, 256>(a, p, s);
    if (p.splits > 1) {
        const int rows = a.heads / a.kv_heads * a.tokens;
        hipLaunchKernelGGL((tree_join_kernel<T>), dim3((rows + kAttnWaves - 1) / kAttnWaves, a.batch * a.kv_heads),
                           dim3(kTreeThreads), 0, s, a, p.tile);
    }
}

long tree_attention_workspace(const TreeArgs& a, int dtype) {
    const TreePlan p = tree_plan(a, dtype);
    return p.splits > 1 ? 4L * p.splits * a.batch * a.tokens * a.heads * (a.d + 2) : 0;
}

hipError_t tree_attention_launch(TreeArgs a, int dtype, hipStream_t s) {
    const TreePlan p = tree_plan(a, dtype);
    a.splits = p.splits;
    if (dtype == 0) tree_launch_t<float>(a, p, s);
    else if (dtype == 1) tree_launch_t<__bf16>(a, p, s);
    else tree_launch_t<_Float16>(a, p, s);
    return hipGetLastError();
}

}  // namespace rac
