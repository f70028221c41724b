// rac_packed.hip — causal attention over packed sequences with grouped heads,
// forward and backward, on the matrix cores.
//
// Rows of all sequences lie one after the other: sequence i is the rows
// cu[i] .. cu[i + 1] - 1.  For its row t, query head h and key / value head
// g = h / (H / G):
//   s_j = scale q_t . k_j  (j <= t),  lse = log sum_j exp(s_j),
//   p_j = exp(s_j - lse),  o_t = sum_j p_j v_j
// and with do_t given:  D = do_t . o_t,  dp_j = do_t . v_j,
//   ds_j = p_j (dp_j - D),  dq_t = scale sum_j ds_j k_j,
//   dk_j = scale sum_{h in g, t >= j} ds_j q_t,  dv_j = sum p_j do_t.
//
// One pass over the keys with a running maximum and sum; no score leaves the
// registers.  A wave holds 32 query rows (forward, dq) or 32 keys (dk, dv) as
// the columns of its products, so a softmax row is a lane pair, a probability
// tile is the next product's right operand as it stands (rac_mma.hpp), and the
// left operands come from tiles of the other side in LDS that the workgroup's
// four waves share.  Backward recomputes the probabilities from lse, once for
// dq and once for dk and dv: seven products where five would do with atomic
// sums of dq, whose order, and so whose result, would change from call to call.
//
// Values in places the mask takes away do not reach a result, NaN and
// infinities among them: masked scores are replaced before the exponential;
// where a tile's product would still multiply such a value by a probability of
// 0, the row's accumulators show it (they are not finite), and its wave does
// that row again over the keys it sees and no others (attn_again).
#include <hip/hip_runtime.h>
#include "rac_internal.hpp"
#include "rac_attn.hpp"

namespace rac {

constexpr int kPkThreads = kAttnThreads;

struct PackedSeg {
    int start, len, row0;      // first row of the sequence, its length, the tile's first row in it
    int kind;                  // 0 none, 1 a sequence, 2 rows outside every sequence
};

__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
    return __builtin_amdgcn_readfirstlane(v);
}

__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v = max(v, __shfl_xor(v, o));
    return __builtin_amdgcn_readfirstlane(v);
}

// Tile `idx` of all sequences' tiles, `rows` rows to a tile and each sequence
// started anew; behind them the tiles of the rows before the first sequence
// and behind the last.  Tile t of a sequence costs the forward pass (and dq) t
// + 1 tiles of keys and, counted from the end, the keys' kernel (`back`) as
// many of queries: the costly ones come first, of all sequences up to 64 (a
// list one to a lane), else sequence by sequence.  Boundaries are held within
// [0, total], so that no row out of range is touched whatever cu holds.
__device__ __forceinline__ PackedSeg packed_tile(const int* __restrict__ cu, int n, int total, int idx, int rows,
                                                 bool back) {
    const int lane = threadIdx.x & 63;
    auto bound = [&](int i) { return min(max(cu[i], 0), total); };
    int before = 0;
    for (int base = 0; base < n; base += 64) {
        int b = 0, e = 0;
        if (base + lane < n) {
            b = bound(base + lane);
            e = max(bound(base + lane + 1), b);
        }
        const int tiles = (e - b + rows - 1) / rows, sum = wave_sum(tiles);
        if (idx < before + sum) {
            int l, t, k = idx - before;              // sequence, its tile's number in the order of cost
            if (n <= 64) {
                // the least level lo with at most k tiles above it
                int lo = 0, hi = wave_max(tiles) - 1;
                while (lo < hi) {
                    const int mid = (lo + hi) / 2;
                    if (wave_sum(max(0, tiles - 1 - mid)) <= k) hi = mid;
                    else lo = mid + 1;
                }
                t = lo;
                k -= wave_sum(max(0, tiles - 1 - lo));
                uint64_t at = __ballot(tiles > lo);
                for (; k; k--) at &= at - 1;
                l = __ffsll((unsigned long long)at) - 1;
            } else {
                int inc = tiles;
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const int up = __shfl_up(inc, o);
                    if (lane >= o) inc += up;
                }
                l = __ffsll((unsigned long long)__ballot(inc > k)) - 1;
                t = __builtin_amdgcn_readlane(inc, l) - 1 - k;
            }
            PackedSeg r;
            r.start = __builtin_amdgcn_readlane(b, l);
            r.len = __builtin_amdgcn_readlane(e, l) - r.start;
            r.row0 = (back ? __builtin_amdgcn_readlane(tiles, l) - 1 - t : t) * rows;
            r.kind = 1;
            return r;
        }
        before += sum;
    }
    const int b0 = bound(0), e1 = max(bound(n), b0), t0 = (b0 + rows - 1) / rows, t1 = (total - e1 + rows - 1) / rows;
    idx -= before;
    if (idx < t0) return PackedSeg{0, b0, idx * rows, 2};
    if (idx < t0 + t1) return PackedSeg{e1, total - e1, (idx - t0) * rows, 2};
    return PackedSeg{0, 0, 0, 0};
}

// Workgroup b of heads x tiles -> (head, tile).  Workgroup b runs on XCD b % 8:
// where the heads divide by 8, each XCD takes whole neighbouring heads, so that
// the heads that share keys and values share an L2.
__device__ __forceinline__ void packed_block(int heads, int& head, int& tile) {
    const int b = blockIdx.x;
    if (heads % 8 == 0) {
        const int per = heads / 8, i = b / 8;
        head = (b % 8) * per + i % per;
        tile = i / per;
    } else {
        head = b % heads;
        tile = b / heads;
    }
}

// zeros in rows r0 .. of a [total, heads, d] array's head (d contiguous)
template <typename T>
__device__ __forceinline__ void packed_zero(T* p, int row0, int rows, int heads, int head, int d) {
    for (long i = threadIdx.x; i < (long)rows * d; i += kPkThreads)
        p[((long)(row0 + i / d) * heads + head) * d + i % d] = (T)0.0f;
}

// The workgroup's four waves are WR sets of 32 rows (keys, in the keys'
// kernel) times KG = 4 / WR groups that take turns at the other side's tiles.
// WR = 4 reads a tile once for 128 rows; WR = 1 and 2 make four and two times
// the workgroups, with a critical path as much shorter, and pay with LDS and a
// sum over the groups at the end.
// Rows of the other side a wave takes from a tile, and a tile's.
template <typename T, int DP, int WR>
struct PackedShape {
    static constexpr int KG = kAttnWaves / WR;
    static constexpr int BN = sizeof(T) == 2 && WR == 4 && DP <= 128 ? 64 : 32;
    static constexpr int TILE = BN * KG, BYTES = TILE * DP * (int)sizeof(T), ROWS = 32 * WR;
    static constexpr int ND = DP / 32, NF = DP / Mma<T>::KF, NS = BN / 32, FS = 32 / Mma<T>::KF;
};

// ── forward ──────────────────────────────────────────────────────────────

template <typename T, int DP, int WR>
__global__ __launch_bounds__(kPkThreads, DP * sizeof(T) <= 256 ? 2 : 1) void packed_fwd_kernel(const PackedArgs a) {
    using M = Mma<T>;
    using Frag = typename M::Frag;
    using S = PackedShape<T, DP, WR>;
    using TL = Tile<T, DP>;
    constexpr int KG = S::KG, BN = S::BN, TILE = S::TILE, ND = S::ND, NF = S::NF, NS = S::NS, FS = S::FS;
    __shared__ __attribute__((aligned(16))) char ka[S::BYTES], va[S::BYTES], kb[S::BYTES], vb[S::BYTES];
    __shared__ float sm[KG > 1 ? kAttnWaves : 1][32], sl[KG > 1 ? kAttnWaves : 1][32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int wr = wave % WR, kg = wave / WR;
    int h, tile;
    packed_block(a.heads, h, tile);
    const PackedSeg seg = packed_tile(a.cu, a.n_seqs, a.total, tile, S::ROWS, false);
    if (seg.kind == 0) return;
    T* out = (T*)a.out;
    if (seg.kind == 2) {
        if (a.zero_rest) packed_zero(out, seg.start + seg.row0, min(S::ROWS, seg.len - seg.row0), a.heads, h, a.d);
        return;
    }
    const int q0 = seg.row0, qw = q0 + 32 * wr, qrow = qw + (lane & 31);
    const int g = h / (a.heads / a.kv_heads);
    const T* K = (const T*)a.k + (long)seg.start * a.sk_t + (long)g * a.sk_h;
    const T* V = (const T*)a.v + (long)seg.start * a.sv_t + (long)g * a.sv_h;
    const int nt = (min(seg.len, q0 + S::ROWS) + TILE - 1) / TILE;
    TileLoad<T, DP, TILE> lk, lv;
    lk.init(a.sk_t, a.d);
    lv.init(a.sv_t, a.d);
    auto issue = [&](int j, char* kd, char* vd) {
        lk.issue(kd, K + (long)j * TILE * a.sk_t, seg.len - j * TILE, a.sk_t, a.d, a.vec, wave);
        lv.issue(vd, V + (long)j * TILE * a.sv_t, seg.len - j * TILE, a.sv_t, a.d, a.vec, wave);
    };
    issue(0, ka, va);
    Frag qf[NF];
    load_frags<T, DP>(qf, (const T*)a.q + (long)(seg.start + qrow) * a.sq_t + (long)h * a.sq_h, qrow < seg.len, a.d,
                      half, a.vec);
    const float c = a.scale * kLog2e;
    f32x16 o[ND];
#pragma unroll
    for (int n = 0; n < ND; n++) o[n] = zero16();
    float m = -__builtin_inff(), l = 0.0f;

    auto step = [&](int j, const char* ks, const char* vs, char* kn, char* vn) {
        tiles_landed();
        if (j + 1 < nt) issue(j + 1, kn, vn);
        const int first = j * TILE + kg * BN;             // the wave's keys
        if (first > qw + 31) return;
        f32x16 s[NS];
#pragma unroll
        for (int u = 0; u < NS; u++) s[u] = zero16();
#pragma unroll
        for (int f = 0; f < NF; f++)
#pragma unroll
            for (int u = 0; u < NS; u++) s[u] = M::mma(TL::rows(ks, kg * BN + 32 * u, f, lane), qf[f], s[u]);
        if (first + BN - 1 > qw) {
#pragma unroll
            for (int u = 0; u < NS; u++)
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (first + 32 * u + 8 * (i / 4) + 4 * half + i % 4 > qrow) s[u][i] = -__builtin_inff();
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
            for (int n = 0; n < ND; n++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[n][i] *= al;
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
                for (int n = 0; n < ND; n++) o[n] = M::mma(TL::cols(vs, kg * BN + 32 * u, f, n, lane), pf, o[n]);
            }
    };
    for (int j = 0; j < nt; j += 2) {
        step(j, ka, va, kb, vb);
        if (j + 1 < nt) step(j + 1, kb, vb, ka, va);
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
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const bool bad = not_finite(o) && qrow < seg.len;
    uint64_t again = __ballot(bad);
    again = (again | again >> 32) & 0xffffffffull;
    if (qrow < seg.len) {
        const long row = seg.start + qrow;
        if (!(again >> (lane & 31) & 1)) attn_store<T, ND>(out + (row * a.heads + h) * a.d, o, inv, a.d, half, a.vec_out);
        if (a.lse && half == 0) a.lse[(long)h * a.total + row] = (m + __builtin_amdgcn_logf(l)) * kLn2;
    }
    for (; again; again &= again - 1) {
        const int r = __ffsll((unsigned long long)again) - 1, t = qw + r;
        const float mr = __shfl(m, r), ir = __shfl(inv, r);
        const T* q = (const T*)a.q + (long)(seg.start + t) * a.sq_t + (long)h * a.sq_h;
        attn_again<T, DP>(out + ((long)(seg.start + t) * a.heads + h) * a.d, ir, a.d, 0, t + 1,
                          [&](int j) { return exp2_hw(__builtin_fmaf(row_dot(q, K + (long)j * a.sk_t, a.d), c, -mr)); },
                          [&](int j) { return V + (long)j * a.sv_t; });
    }
}

// ── backward: dq (and D) ─────────────────────────────────────────────────

template <typename T, int DP, int WR>
__global__ __launch_bounds__(kPkThreads, DP * sizeof(T) <= 256 ? 2 : 1) void packed_dq_kernel(const PackedArgs a) {
    using M = Mma<T>;
    using Frag = typename M::Frag;
    using S = PackedShape<T, DP, WR>;
    using TL = Tile<T, DP>;
    constexpr int KG = S::KG, BN = S::BN, TILE = S::TILE, ND = S::ND, NF = S::NF, NS = S::NS, FS = S::FS;
    __shared__ __attribute__((aligned(16))) char ka[S::BYTES], va[S::BYTES], kb[S::BYTES], vb[S::BYTES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int wr = wave % WR, kg = wave / WR;
    int h, tile;
    packed_block(a.heads, h, tile);
    const PackedSeg seg = packed_tile(a.cu, a.n_seqs, a.total, tile, S::ROWS, false);
    if (seg.kind == 0) return;
    T* dq = (T*)a.dq;
    if (seg.kind == 2) {
        if (a.zero_rest) packed_zero(dq, seg.start + seg.row0, min(S::ROWS, seg.len - seg.row0), a.heads, h, a.d);
        return;
    }
    const int q0 = seg.row0, qw = q0 + 32 * wr, qrow = qw + (lane & 31);
    const bool there = qrow < seg.len;
    const long row = seg.start + qrow;
    const int g = h / (a.heads / a.kv_heads);
    const T* K = (const T*)a.k + (long)seg.start * a.sk_t + (long)g * a.sk_h;
    const T* V = (const T*)a.v + (long)seg.start * a.sv_t + (long)g * a.sv_h;
    const int nt = (min(seg.len, q0 + S::ROWS) + TILE - 1) / TILE;
    TileLoad<T, DP, TILE> lk, lv;
    lk.init(a.sk_t, a.d);
    lv.init(a.sv_t, a.d);
    auto issue = [&](int j, char* kd, char* vd) {
        lk.issue(kd, K + (long)j * TILE * a.sk_t, seg.len - j * TILE, a.sk_t, a.d, a.vec, wave);
        lv.issue(vd, V + (long)j * TILE * a.sv_t, seg.len - j * TILE, a.sv_t, a.d, a.vec, wave);
    };
    issue(0, ka, va);
    Frag qf[NF], gf[NF];
    load_frags<T, DP>(qf, (const T*)a.q + row * a.sq_t + (long)h * a.sq_h, there, a.d, half, a.vec);
    load_frags<T, DP>(gf, (const T*)a.grad + (row * a.heads + h) * a.d, there, a.d, half, a.vec);
    // D = do . o, kept for the keys' kernel
    float dl = 0.0f;
    {
        Frag of[NF];
        load_frags<T, DP>(of, (const T*)a.out + (row * a.heads + h) * a.d, there, a.d, half, a.vec);
#pragma unroll
        for (int f = 0; f < NF; f++)
#pragma unroll
            for (int e = 0; e < M::VEC; e++) dl = __builtin_fmaf(M::to_f32(gf[f][e]), M::to_f32(of[f][e]), dl);
    }
    dl = half_sum(dl);
    if (there && half == 0 && kg == 0) a.delta[(long)h * a.total + row] = dl;
    // rows without a key that counts (lse -inf) and rows past the sequence: p = 0
    float lse = there ? a.lse[(long)h * a.total + row] * kLog2e : __builtin_inff();
    if (lse == -__builtin_inff()) lse = __builtin_inff();
    const float c = a.scale * kLog2e;
    f32x16 acc[ND];
#pragma unroll
    for (int n = 0; n < ND; n++) acc[n] = zero16();

    auto step = [&](int j, const char* ks, const char* vs, char* kn, char* vn) {
        tiles_landed();
        if (j + 1 < nt) issue(j + 1, kn, vn);
        const int first = j * TILE + kg * BN;
        if (first > qw + 31) return;
        const bool diag = first + BN - 1 > qw;
#pragma unroll
        for (int u = 0; u < NS; u++) {
            f32x16 s = zero16(), dp = zero16();
#pragma unroll
            for (int f = 0; f < NF; f++) {
                s = M::mma(TL::rows(ks, kg * BN + 32 * u, f, lane), qf[f], s);
                dp = M::mma(TL::rows(vs, kg * BN + 32 * u, f, lane), gf[f], dp);
            }
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float p = exp2_hw(__builtin_fmaf(s[i], c, -lse));
                s[i] = p * (dp[i] - dl);
            }
            if (diag) {
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (first + 32 * u + 8 * (i / 4) + 4 * half + i % 4 > qrow) s[i] = 0.0f;
            }
#pragma unroll
            for (int f = 0; f < FS; f++) {
                const Frag df = M::pack(s, f);
#pragma unroll
                for (int n = 0; n < ND; n++) acc[n] = M::mma(TL::cols(ks, kg * BN + 32 * u, f, n, lane), df, acc[n]);
            }
        }
    };
    for (int j = 0; j < nt; j += 2) {
        step(j, ka, va, kb, vb);
        if (j + 1 < nt) step(j + 1, kb, vb, ka, va);
    }
    if constexpr (KG > 1) {
        join_groups<KG, WR, ND>(acc, 1.0f, ka, wr, kg, lane);
        if (kg) return;
    }
    const bool bad = not_finite(acc) && there;
    uint64_t again = __ballot(bad);
    again = (again | again >> 32) & 0xffffffffull;
    if (there && !(again >> (lane & 31) & 1))
        attn_store<T, ND>(dq + (row * a.heads + h) * a.d, acc, a.scale, a.d, half, a.vec_out);
    for (; again; again &= again - 1) {
        const int r = __ffsll((unsigned long long)again) - 1;
        const long t = qw + r, at = ((seg.start + t) * a.heads + h) * a.d;
        const float lr = __shfl(lse, r), dr = __shfl(dl, r);
        const T* q = (const T*)a.q + (seg.start + t) * a.sq_t + (long)h * a.sq_h;
        const T* go = (const T*)a.grad + at;
        attn_again<T, DP>(dq + at, a.scale, a.d, 0, (int)t + 1,
                          [&](int j) {
                              const float p = exp2_hw(__builtin_fmaf(row_dot(q, K + (long)j * a.sk_t, a.d), c, -lr));
                              return p * (row_dot(go, V + (long)j * a.sv_t, a.d) - dr);
                          },
                          [&](int j) { return K + (long)j * a.sk_t; });
    }
}

// ── backward: dk, dv ─────────────────────────────────────────────────────

// WHICH: 1 dv, 2 dk, 3 both (d past 128 in fp32 has no registers for both)
template <typename T, int DP, int WR, int WHICH>
__global__ __launch_bounds__(kPkThreads, DP * sizeof(T) <= 128 ? 2 : 1) void packed_dkv_kernel(const PackedArgs a) {
    using M = Mma<T>;
    using Frag = typename M::Frag;
    using S = PackedShape<T, DP, WR>;
    using TL = Tile<T, DP>;
    constexpr int KG = S::KG, BQ = S::BN, TILE = S::TILE, ND = S::ND, NF = S::NF, NS = S::NS, FS = S::FS;
    constexpr bool WV = WHICH & 1, WK = WHICH & 2;
    __shared__ __attribute__((aligned(16))) char qa[S::BYTES], ga[S::BYTES], qb[S::BYTES], gb[S::BYTES];
    __shared__ __attribute__((aligned(16))) float sa[2][TILE], sb[2][TILE];      // lse and D
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int wr = wave % WR, kg = wave / WR;
    int g, tile;
    packed_block(a.kv_heads, g, tile);
    const PackedSeg seg = packed_tile(a.cu, a.n_seqs, a.total, tile, S::ROWS, true);
    if (seg.kind == 0) return;
    T* dk = (T*)a.dk;
    T* dv = (T*)a.dv;
    if (seg.kind == 2) {
        const int rows = min(S::ROWS, seg.len - seg.row0);
        if (a.zero_rest) {
            if (WK) packed_zero(dk, seg.start + seg.row0, rows, a.kv_heads, g, a.d);
            if (WV) packed_zero(dv, seg.start + seg.row0, rows, a.kv_heads, g, a.d);
        }
        return;
    }
    const int k0 = seg.row0, kw = k0 + 32 * wr, key = kw + (lane & 31);
    const int rep = a.heads / a.kv_heads;
    const bool there = key < seg.len;
    const long row = seg.start + key;
    // steps: the tiles of queries from the diagonal on, for one head of the group after the other
    const int t0 = k0 / TILE, per = (seg.len + TILE - 1) / TILE - t0, steps = per * rep;
    const T* const Q = (const T*)a.q + (long)seg.start * a.sq_t + (long)g * rep * a.sq_h;
    const T* const G = (const T*)a.grad + ((long)seg.start * a.heads + (long)g * rep) * a.d;
    TileLoad<T, DP, TILE> lq, lg;
    lq.init(a.sq_t, a.d);
    lg.init((long)a.heads * a.d, a.d);
    int ih = 0, it = t0;                                  // head and tile of the next issue
    auto issue = [&](char* qd, char* gd, float (*st)[TILE]) {
        const int first = it * TILE;
        lq.issue(qd, Q + (long)ih * a.sq_h + (long)first * a.sq_t, seg.len - first, a.sq_t, a.d, a.vec, wave);
        lg.issue(gd, G + (long)ih * a.d + (long)first * a.heads * a.d, seg.len - first, (long)a.heads * a.d, a.d, a.vec,
                 wave);
        if (threadIdx.x < TILE) {
            const int t = first + threadIdx.x;
            float rl = __builtin_inff(), rd = 0.0f;
            if (t < seg.len) {
                const long at = (long)(g * rep + ih) * a.total + seg.start + t;
                rl = a.lse[at] * kLog2e;
                if (rl == -__builtin_inff()) rl = __builtin_inff();
                rd = a.delta[at];
            }
            st[0][threadIdx.x] = rl;
            st[1][threadIdx.x] = rd;
        }
        if (++it == t0 + per) {
            it = t0;
            ih++;
        }
    };
    issue(qa, ga, sa);
    Frag kf[NF], vf[WK ? NF : 1];
    load_frags<T, DP>(kf, (const T*)a.k + row * a.sk_t + (long)g * a.sk_h, there, a.d, half, a.vec);
    if constexpr (WK) load_frags<T, DP>(vf, (const T*)a.v + row * a.sv_t + (long)g * a.sv_h, there, a.d, half, a.vec);
    const float c = a.scale * kLog2e;
    f32x16 ak[WK ? ND : 1], av[WV ? ND : 1];
#pragma unroll
    for (int n = 0; n < ND; n++) {
        if constexpr (WK) ak[n] = zero16();
        if constexpr (WV) av[n] = zero16();
    }
    int ct = t0;                                          // tile of this step
    auto step = [&](int st, const char* qs, const char* gs, const float (*ss)[TILE], char* qn, char* gn,
                    float (*sn)[TILE]) {
        tiles_landed();
        if (st + 1 < steps) issue(qn, gn, sn);
        const int first = ct * TILE + kg * BQ;
        if (++ct == t0 + per) ct = t0;
#pragma unroll
        for (int u = 0; u < NS; u++) {
            const int q0 = first + 32 * u, at = kg * BQ + 32 * u;
            if (q0 + 31 < kw || q0 >= seg.len) continue;     // before the wave's keys, or past the sequence
            f32x16 s = zero16(), dp = zero16();
#pragma unroll
            for (int f = 0; f < NF; f++) {
                s = M::mma(TL::rows(qs, at, f, lane), kf[f], s);
                if constexpr (WK) dp = M::mma(TL::rows(gs, at, f, lane), vf[f], dp);
            }
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const f32x4 le = *reinterpret_cast<const f32x4*>(&ss[0][at + 8 * b + 4 * half]);
                const f32x4 de = *reinterpret_cast<const f32x4*>(&ss[1][at + 8 * b + 4 * half]);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int i = 4 * b + j;
                    s[i] = exp2_hw(__builtin_fmaf(s[i], c, -le[j]));
                    if constexpr (WK) dp[i] = s[i] * (dp[i] - de[j]);
                }
            }
            if (q0 < kw + 31) {
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (q0 + 8 * (i / 4) + 4 * half + i % 4 < key) {
                        s[i] = 0.0f;
                        if constexpr (WK) dp[i] = 0.0f;
                    }
            }
#pragma unroll
            for (int f = 0; f < FS; f++) {
                Frag pf, df;
                if constexpr (WV) pf = M::pack(s, f);
                if constexpr (WK) df = M::pack(dp, f);
#pragma unroll
                for (int n = 0; n < ND; n++) {
                    if constexpr (WV) av[n] = M::mma(TL::cols(gs, at, f, n, lane), pf, av[n]);
                    if constexpr (WK) ak[n] = M::mma(TL::cols(qs, at, f, n, lane), df, ak[n]);
                }
            }
        }
    };
    for (int st = 0; st < steps; st += 2) {
        step(st, qa, ga, sa, qb, gb, sb);
        if (st + 1 < steps) step(st + 1, qb, gb, sb, qa, ga, sa);
    }
    if constexpr (KG > 1) {
        if constexpr (WK) join_groups<KG, WR, ND>(ak, 1.0f, qa, wr, kg, lane);
        if constexpr (WV) join_groups<KG, WR, ND>(av, 1.0f, qa, wr, kg, lane);
        if (kg) return;
    }
    bool bad = false;
    if constexpr (WK) bad |= not_finite(ak);
    if constexpr (WV) bad |= not_finite(av);
    uint64_t again = __ballot(bad && there);
    again = (again | again >> 32) & 0xffffffffull;
    if (there && !(again >> (lane & 31) & 1)) {
        const long at = (row * a.kv_heads + g) * a.d;
        if constexpr (WK) attn_store<T, ND>(dk + at, ak, a.scale, a.d, half, a.vec_out);
        if constexpr (WV) attn_store<T, ND>(dv + at, av, 1.0f, a.d, half, a.vec_out);
    }
    for (; again; again &= again - 1) {
        const int kr = kw + __ffsll((unsigned long long)again) - 1, from = kr, n = seg.len - from;
        const long at = ((long)(seg.start + kr) * a.kv_heads + g) * a.d;
        const T* kk = (const T*)a.k + (long)(seg.start + kr) * a.sk_t + (long)g * a.sk_h;
        const T* vv = (const T*)a.v + (long)(seg.start + kr) * a.sv_t + (long)g * a.sv_h;
        // queries from .. of head 0 of the group, then of head 1, ...
        auto qrow = [&](int i) { return Q + (long)(i / n) * a.sq_h + (long)(from + i % n) * a.sq_t; };
        auto grow = [&](int i) { return G + ((long)(from + i % n) * a.heads + i / n) * a.d; };
        auto stat = [&](int i) { return (long)(g * rep + i / n) * a.total + seg.start + from + i % n; };
        auto prob = [&](int i) {
            const float lr = a.lse[stat(i)] * kLog2e;
            return lr == -__builtin_inff() ? 0.0f : exp2_hw(__builtin_fmaf(row_dot(qrow(i), kk, a.d), c, -lr));
        };
        if constexpr (WV) attn_again<T, DP>(dv + at, 1.0f, a.d, 0, n * rep, prob, grow);
        if constexpr (WK)
            attn_again<T, DP>(dk + at, a.scale, a.d, 0, n * rep,
                                [&](int i) { return prob(i) * (row_dot(grow(i), vv, a.d) - a.delta[stat(i)]); }, qrow);
    }
}

// ── launches ─────────────────────────────────────────────────────────────

// tiles of `rows` rows: at most this many, whatever the sequences' lengths
static long packed_tiles(const PackedArgs& a, int rows) { return (long)a.total / rows + a.n_seqs + 2; }

// Row sets of a workgroup: 4 while that makes a workgroup for every CU, else as
// few as LDS allows (128 KB of it hold the two tiles twice).
template <typename T, int DP, int WR>
constexpr bool packed_fits() {
    return 4 * PackedShape<T, DP, WR>::BYTES <= (128 << 10);
}
static bool packed_few(const PackedArgs& a, int heads) {
    return ((long)a.total / 128 + (a.n_seqs + 1) / 2) * heads < device_cus();
}

template <typename T, int DP, int WR>
static void packed_launch_fwd(const PackedArgs& a, hipStream_t s) {
    hipLaunchKernelGGL((packed_fwd_kernel<T, DP, WR>), dim3((unsigned)(packed_tiles(a, 32 * WR) * a.heads)),
                       dim3(kPkThreads), 0, s, a);
}
template <typename T, int DP, int WR>
static void packed_launch_dq(const PackedArgs& a, hipStream_t s) {
    hipLaunchKernelGGL((packed_dq_kernel<T, DP, WR>), dim3((unsigned)(packed_tiles(a, 32 * WR) * a.heads)),
                       dim3(kPkThreads), 0, s, a);
}
template <typename T, int DP, int WR>
static void packed_launch_dkv(const PackedArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)(packed_tiles(a, 32 * WR) * a.kv_heads)), t(kPkThreads);
    if constexpr (DP * sizeof(T) > 512) {
        hipLaunchKernelGGL((packed_dkv_kernel<T, DP, WR, 1>), grid, t, 0, s, a);
        hipLaunchKernelGGL((packed_dkv_kernel<T, DP, WR, 2>), grid, t, 0, s, a);
    } else {
        hipLaunchKernelGGL((packed_dkv_kernel<T, DP, WR, 3>), grid, t, 0, s, a);
    }
}

template <typename T, int DP>
static void packed_launch_dp(const PackedArgs& a, bool backward, hipStream_t s) {
    constexpr int FEW = packed_fits<T, DP, 1>() ? 1 : packed_fits<T, DP, 2>() ? 2 : 4;
    const bool rows = packed_few(a, a.heads), keys = packed_few(a, a.kv_heads);
    if (!backward) {
        if (rows) packed_launch_fwd<T, DP, FEW>(a, s);
        else packed_launch_fwd<T, DP, 4>(a, s);
        return;
    }
    if (rows) packed_launch_dq<T, DP, FEW>(a, s);
    else packed_launch_dq<T, DP, 4>(a, s);
    if (keys) packed_launch_dkv<T, DP, FEW>(a, s);
    else packed_launch_dkv<T, DP, 4>(a, s);
}

template <typename T>
static void packed_launch_t(const PackedArgs& a, bool backward, hipStream_t s) {
    if (a.d <= 32) packed_launch_dp<T, 32>(a, backward, s);
    else if (a.d <= 64) packed_launch_dp<T, 64>(a, backward, s);
    else if (a.d <= 96) packed_launch_dp<T, 96>(a, backward, s);
    else if (a.d <= 128) packed_launch_dp<T, 128>(a, backward, s);
    else packed_launch_dp<T, 256>(a, backward, s);
}

hipError_t packed_attention_launch(const PackedArgs& a, int dtype, bool backward, hipStream_t s) {
    if (dtype == 0) packed_launch_t<float>(a, backward, s);
    else if (dtype == 1) packed_launch_t<__bf16>(a, backward, s);
    else packed_launch_t<_Float16>(a, backward, s);
    return hipGetLastError();
}

}  // namespace rac
