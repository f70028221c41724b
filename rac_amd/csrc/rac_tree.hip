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

// A workgroup's four waves are WR sets of 32 rows times KG = 4 / WR groups that
// take different keys of a tile: BN a wave.
constexpr int tree_bn(int es, int dp, int wr) { return es == 2 && wr == kAttnWaves && dp <= 128 ? 64 : 32; }
constexpr int tree_tile(int es, int dp, int wr) { return tree_bn(es, dp, wr) * (kAttnWaves / wr); }

// the tiles that split s of `splits` takes out of `tiles`: `per` from s per on
__device__ __forceinline__ int tree_per(int tiles, int splits) { return (tiles + splits - 1) / splits; }

// part: unnormalised outputs [batch, kv_heads, splits, rows, d], then their
// maxima and sums [.., rows, 2] from here on
__host__ __device__ inline long tree_stats(const TreeArgs& a) {
    return (long)a.batch * a.splits * a.heads * a.tokens * a.d;
}

// Bound by the two products where rows are many (16 bf16 caches of up to 8001
// positions, 64 drafts each, 32/8 heads of 128: 152 us, the sum of the caches'
// lengths at 0.68 PFLOP/s), by latency where they are few (a token over 515
// positions, 8 heads of 64 in fp32: 9.4 us and 3.2 of the join).
template <typename T, int DP, int WR>
__global__ __launch_bounds__(kTreeThreads, DP * sizeof(T) <= 256 ? 2 : 1) void tree_kernel(const TreeArgs a) {
    using M = Mma<T>;
    using Frag = typename M::Frag;
    using TL = Tile<T, DP>;
    constexpr int NF = DP / M::KF, ND = DP / 32, FS = 32 / M::KF;
    constexpr int KG = kAttnWaves / WR, BN = tree_bn(sizeof(T), DP, WR), NS = BN / 32, TILE = BN * KG;
    constexpr int BYTES = TILE * DP * (int)sizeof(T);
    __shared__ __attribute__((aligned(16))) char ka[BYTES], va[BYTES], kb[BYTES], vb[BYTES];
    __shared__ uint32_t anc[kTreeMaxTokens][kTreeWords];
    __shared__ int up[2][kTreeMaxTokens];
    __shared__ float sm[kAttnWaves][32], sl[kAttnWaves][32];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    const int wr = wave % WR, kg = wave / WR;
    const int rep = a.heads / a.kv_heads, rows = rep * a.tokens;
    // workgroup L runs on XCD L % 8: the row blocks over the same keys follow
    // each other on one XCD and share its L2
    const int nb = (rows + 32 * WR - 1) / (32 * WR), i8 = blockIdx.x / 8, rb = i8 % nb, unit = i8 / nb * 8 + blockIdx.x % 8;
    const int split = unit % a.splits, bg = unit / a.splits, b = bg / a.kv_heads, g = bg % a.kv_heads;
    if (b >= a.batch) return;
    const int rw = (rb * WR + wr) * 32, r = rw + (lane & 31);           // the wave's first row, the lane's
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
    // 16 bits through registers: 16 bf16 caches of up to 8001 positions, 64 drafts
    // each (32/8 heads of 128), 167 us, direct 236
    TileLoad<T, DP, TILE> lk, lv;
    lk.init(a.sk_t, a.d);
    lv.init(a.sv_t, a.d);
    auto issue = [&](int j, char* kd, char* vd) ATTN_INLINE {
        lk.issue(kd, K + (long)j * TILE * a.sk_t, n - j * TILE, a.sk_t, a.d, a.vec, wave);
        lv.issue(vd, V + (long)j * TILE * a.sv_t, n - j * TILE, a.sv_t, a.d, a.vec, wave);
    };
    auto commit = [&](int j, char* kd, char* vd) ATTN_INLINE {
        lk.commit(kd, K + (long)j * TILE * a.sk_t, n - j * TILE, a.sk_t, a.d, a.vec);
        lv.commit(vd, V + (long)j * TILE * a.sv_t, n - j * TILE, a.sv_t, a.d, a.vec);
    };
    // a workgroup begins within its tiles at a place of its own and goes round:
    // caches whose sequences lie a power of two apart would else be walked in
    // step, all on the same memory channels at a time (16 bf16 caches of up to
    // 8001 positions, 8192 apart: 173 us from the first tile on, 167 so)
    const int cnt = j1 - j0, turn = (7 * bg + 3 * split) % cnt;
    auto tile_of = [&](int i) ATTN_INLINE { return j0 + (i + turn < cnt ? i + turn : i + turn - cnt); };
    issue(tile_of(0), ka, va);
    Frag qf[NF];
    load_frags<T, DP>(qf, qrow, there, a.d, half, a.vec);
    if (j1 * TILE > len) {
        // the split holds drafted tokens: their paths to the root, in steps
        // that double what is known
        int p = -1;
        if (tid < a.tokens) {
            p = a.parents[(long)b * a.parents_b + tid];
            if (p >= tid) p = -1;
            up[0][tid] = p;
#pragma unroll
            for (int w = 0; w < kTreeWords; w++) anc[tid][w] = w == tid / 32 ? 1u << (tid & 31) : 0u;
        }
        for (int hop = 1, cur = 0; hop < a.tokens; hop *= 2, cur ^= 1) {
            if (!__syncthreads_or(p >= 0)) break;          // every path known
            uint32_t m[kTreeWords];
            const bool had = p >= 0;
            if (had) {
#pragma unroll
                for (int w = 0; w < kTreeWords; w++) m[w] = anc[tid][w] | anc[p][w];
                p = up[cur][p];
            }
            __syncthreads();
            if (tid < a.tokens) {
                if (had) {
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
    auto seen = [&](int u) ATTN_INLINE -> uint32_t {
        if (u >= a.tokens) return 0u;
        if (u <= -32) return ~0u;
        const uint32_t* w = anc[tok];
        if (u < 0) return (1u << -u) - 1u | w[0] << -u;
        const uint64_t two = w[u >> 5] | (uint64_t)w[(u >> 5) + 1] << 32;
        return (uint32_t)(two >> (u & 31));
    };
    auto work = [&](int i, const char* ks, const char* vs) ATTN_INLINE {
        const int first = tile_of(i) * TILE + kg * BN;    // the wave's keys
        if (first >= n || rw >= rows) return;
        f32x16 s[NS];
#pragma unroll
        for (int u = 0; u < NS; u++) s[u] = zero16();
#pragma unroll
        for (int f = 0; f < NF; f++)
#pragma unroll
            for (int u = 0; u < NS; u++) s[u] = M::mma(TL::rows(ks, kg * BN + 32 * u, f, lane), qf[f], s[u]);
        if (first + BN > len) {
            attn_branch();
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
        mx = half_max(mx) * c;
        // the maximum that exponents refer to may lag behind by a factor of 2^8
        if (__any(mx > m + 8.0f)) {
            const float mt = fmaxf(m, mx);
            // nothing but -inf so far: exponents of -inf, not NaN
            const float al = exp2_hw(m - (mt == -__builtin_inff() ? 0.0f : mt));
            m = mt;
            l *= al;
#pragma unroll
            for (int i = 0; i < ND; i++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[i][e] *= al;
        }
        const float mu = m == -__builtin_inff() ? 0.0f : m;
        float ls = 0.0f;
#pragma unroll
        for (int u = 0; u < NS; u++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                s[u][i] = exp2_hw(__builtin_fmaf(s[u][i], c, -mu));
                ls += s[u][i];
            }
        l += ls;
#pragma unroll
        for (int u = 0; u < NS; u++)
#pragma unroll
            for (int f = 0; f < FS; f++) {
                const Frag pf = M::pack(s[u], f);
#pragma unroll
                for (int i = 0; i < ND; i++) o[i] = M::mma(TL::cols(vs, kg * BN + 32 * u, f, i, lane), pf, o[i]);
            }
    };
    auto step = [&](int i, const char* ks, const char* vs, char* kn, char* vn) ATTN_INLINE {
        tiles_landed();
        if (i + 1 < cnt) issue(tile_of(i + 1), kn, vn);
        work(i, ks, vs);
        if (i + 1 < cnt) commit(tile_of(i + 1), kn, vn);
    };
    commit(tile_of(0), ka, va);
    for (int i = 0; i < cnt; i += 2) {
        step(i, ka, va, kb, vb);
        if (i + 1 < cnt) step(i + 1, kb, vb, ka, va);
    }
    l = half_sum(l);
    if constexpr (KG > 1) {
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
        for (int k = 0; k < KG; k++)
            l = __builtin_fmaf(sl[k * WR + wr][lane & 31], exp2_hw(sm[k * WR + wr][lane & 31] - mu), l);
        join_groups<KG, WR, ND>(o, exp2_hw(m - mu), ka, wr, kg, lane);
        m = mt;
        if (kg) return;
    }
    // rows that met a value that is not finite in a split with drafts, which may
    // be one they do not see: again, over what they do
    uint32_t again = j1 * TILE > len ? columns_of(not_finite(o) && there && l == l) : 0;
    const bool store = there && !(again >> (lane & 31) & 1);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const bool whole = per >= tiles;                      // no other split has keys
    const long part = ((long)bg * a.splits + split) * rows;
    float* po = a.part + part * a.d;
    if (whole) {
        if (store) attn_store<T, ND>(out, o, inv, a.d, half, a.vec_out);
    } else {
        if (there && half == 0) {
            float* ps = a.part + tree_stats(a) + 2 * (part + r);
            ps[0] = m;
            ps[1] = l;
        }
        if (store) attn_store<float, ND>(po + (long)r * a.d, o, 1.0f, a.d, half, a.d % 4 == 0);
    }
    for (; again; again &= again - 1) {
        const int rl = __ffs((int)again) - 1, rr = rw + rl;
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
            attn_again<T, DP, true>(po + (long)rr * a.d, 1.0f, a.d, ja, jb, w, vrow);
    }
}

// Splits joined: a thread per 4 values of a row.
template <typename T>
__global__ __launch_bounds__(kTreeThreads) void tree_join_kernel(const TreeArgs a, int tile) {
    const int rep = a.heads / a.kv_heads, rows = rep * a.tokens, d4 = (a.d + 3) / 4;
    const long i = (long)blockIdx.x * kTreeThreads + threadIdx.x;
    const int bg = blockIdx.y, b = bg / a.kv_heads, g = bg % a.kv_heads;
    const int len = a.len[b];
    if (i >= (long)rows * d4 || len < 0 || (long)len + a.tokens > a.cap) return;
    const int tiles = (len + a.tokens + tile - 1) / tile, per = tree_per(tiles, a.splits);
    if (per >= tiles) return;                              // one split: it stored the rows itself
    const int live = (tiles + per - 1) / per, r = (int)(i / d4), c = (int)(i % d4) * 4;
    const float* po = a.part + ((long)bg * a.splits * rows + r) * a.d + c;
    const float* ps = a.part + tree_stats(a) + ((long)bg * a.splits * rows + r) * 2;
    const long so = (long)rows * a.d, ss = 2L * rows;
    float m = -__builtin_inff();
#pragma unroll 4
    for (int s = 0; s < live; s++) m = fmaxf(m, ps[s * ss]);
    if (m == -__builtin_inff()) m = 0.0f;
    float l = 0.0f, acc[4] = {};
    const bool vec = a.d % 4 == 0;
#pragma unroll 4
    for (int s = 0; s < live; s++) {
        const float f = exp2_hw(ps[s * ss] - m);
        l = __builtin_fmaf(f, ps[s * ss + 1], l);
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
        if (vec) {
            v = *reinterpret_cast<const f32x4*>(po + s * so);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (c + e < a.d) v[e] = po[s * so + e];
        }
#pragma unroll
        for (int e = 0; e < 4; e++) acc[e] = __builtin_fmaf(f, v[e], acc[e]);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* out = (T*)a.out + (((long)b * a.tokens + r / rep) * a.heads + g * rep + r % rep) * a.d + c;
    union { T e[4]; u32x2 v2; u32x4 v4; } u;
#pragma unroll
    for (int e = 0; e < 4; e++) u.e[e] = Mma<T>::from_f32(acc[e] * inv);
    if (a.vec_out) {
        if constexpr (sizeof(T) == 2) *reinterpret_cast<u32x2*>(out) = u.v2;
        else *reinterpret_cast<u32x4*>(out) = u.v4;
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (c + e < a.d) out[e] = u.e[e];
    }
}

// Row sets: one while all rows fit there (two where four groups' tiles do not
// fit LDS), else four.
struct TreePlan {
    int wr, tile, splits;
};
constexpr int tree_few_sets(int es, int dp) { return dp * es <= 256 ? 1 : dp * es <= 512 ? 2 : 4; }
static TreePlan tree_plan(const TreeArgs& a, int dtype) {
    const int rows = a.heads / a.kv_heads * a.tokens, es = dtype == 0 ? 4 : 2;
    const int dp = a.d <= 32 ? 32 : a.d <= 64 ? 64 : a.d <= 96 ? 96 : a.d <= 128 ? 128 : 256;
    TreePlan p;
    p.wr = tree_few_sets(es, dp);
    if (rows > 32 * p.wr) p.wr = 4;
    p.tile = tree_tile(es, dp, p.wr);
    const long groups = (long)a.batch * a.kv_heads * ((rows + 32 * p.wr - 1) / (32 * p.wr));
    // two workgroups to a CU, but two tiles to each at least: 24 drafts over 2019
    // positions in fp32 (32/4 heads of 64) 22.4 us in 32 splits, 32.5 in 64 and
    // 23.4 in 16; 16 bf16 caches of up to 8001 (32/8 heads of 128) 168 us in 2,
    // 196 in one
    // (one row set's tile is four groups' already: a token over 515 positions in
    // fp32, 8 heads of 64, 13.1 us in splits of one tile, 15.2 of two)
    const long least = p.wr == kAttnWaves ? 2L * p.tile : p.tile, most = (a.cap + least - 1) / least;
    long s = (2 * device_cus() + groups - 1) / groups;
    if (s > most) s = most;
    if (s > 64) s = 64;
    p.splits = s < 1 ? 1 : (int)s;
    return p;
}

template <typename T, int DP>
static void tree_launch_dp(const TreeArgs& a, const TreePlan& p, hipStream_t s) {
    const int rows = a.heads / a.kv_heads * a.tokens;
    const long units = ((long)p.splits * a.batch * a.kv_heads + 7) / 8 * 8;
    const dim3 grid((unsigned)(units * ((rows + 32 * p.wr - 1) / (32 * p.wr))));
    constexpr int FEW = tree_few_sets(sizeof(T), DP);
    if (p.wr == FEW) hipLaunchKernelGGL((tree_kernel<T, DP, FEW>), grid, dim3(kTreeThreads), 0, s, a);
    else hipLaunchKernelGGL((tree_kernel<T, DP, 4>), grid, dim3(kTreeThreads), 0, s, a);
}

template <typename T>
static void tree_launch_t(const TreeArgs& a, const TreePlan& p, hipStream_t s) {
    if (a.d <= 32) tree_launch_dp<T, 32>(a, p, s);
    else if (a.d <= 64) tree_launch_dp<T, 64>(a, p, s);
    else if (a.d <= 96) tree_launch_dp<T, 96>(a, p, s);
    else if (a.d <= 128) tree_launch_dp<T, 128>(a, p, s);
    else tree_launch_dp<T, 256>(a, p, s);
    if (p.splits > 1) {
        const long threads = (long)(a.heads / a.kv_heads) * a.tokens * ((a.d + 3) / 4);
        hipLaunchKernelGGL((tree_join_kernel<T>), dim3((unsigned)((threads + kTreeThreads - 1) / kTreeThreads),
                           a.batch * a.kv_heads), dim3(kTreeThreads), 0, s, a, p.tile);
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
