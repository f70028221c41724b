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
constexpr int kPkRows = 32 * kAttnWaves;        // rows (or keys) of a workgroup

struct PackedSeg {
    int start, len, row0;      // first row of the sequence, its length, the tile's first row in it
    int kind;                  // 0 none, 1 a sequence, 2 rows outside every sequence
};

// Tile `idx` of the list that the rows before the first sequence, every
// sequence and the rows behind the last make, `rows` rows to a tile and each
// started anew.  Boundaries are held within [0, total], so that no row out of
// range is touched whatever cu holds.
__device__ __forceinline__ PackedSeg packed_tile(const int* __restrict__ cu, int n, int total, int idx, int rows) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < n + 2; base += 64) {
        const int s = base + lane;
        int b = 0, e = 0;
        if (s < n + 2) {
            b = s == 0 ? 0 : cu[s - 1];
            e = s == n + 1 ? total : cu[s];
            b = min(max(b, 0), total);
            e = min(max(e, b), total);
        }
        const int tiles = (e - b + rows - 1) / rows;
        int inc = tiles;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int up = __shfl_up(inc, o);
            if (lane >= o) inc += up;
        }
        const uint64_t hit = __ballot(before + inc > idx);
        if (hit) {
            const int l = __ffsll((unsigned long long)hit) - 1;
            const int first = before + __shfl(inc - tiles, l);
            PackedSeg r;
            r.start = __shfl(b, l);
            r.len = __shfl(e, l) - r.start;
            r.row0 = (idx - first) * rows;
            const int seg = base + l;
            r.kind = seg == 0 || seg == n + 1 ? 2 : 1;
            return r;
        }
        before += __shfl(inc, 63);
    }
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

// ── forward ──────────────────────────────────────────────────────────────

template <typename T, int DP, int BN>
__global__ __launch_bounds__(kPkThreads, DP * sizeof(T) <= 256 ? 2 : 1) void packed_fwd_kernel(const PackedArgs a) {
    using M = Mma<T>;
    using Frag = typename M::Frag;
    constexpr int KF = M::KF, NF = DP / KF, ND = DP / 32, NS = BN / 32, LD = DP + M::VEC;
    __shared__ __attribute__((aligned(16))) T sk[2][BN * LD];
    __shared__ __attribute__((aligned(16))) T sv[2][BN * LD];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    int h, tile;
    packed_block(a.heads, h, tile);
    PackedSeg seg = packed_tile(a.cu, a.n_seqs, a.total, tile, kPkRows);
    if (seg.kind == 0) return;
    T* out = (T*)a.out;
    if (seg.kind == 2) {
        if (a.zero_rest) packed_zero(out, seg.start + seg.row0, min(kPkRows, seg.len - seg.row0), a.heads, h, a.d);
        return;
    }
    // the tiles of most keys first
    const int q0 = ((seg.len - 1) / kPkRows) * kPkRows - seg.row0;
    const int qw = q0 + 32 * wave, qrow = qw + (lane & 31);
    const int g = h / (a.heads / a.kv_heads);
    const T* K = (const T*)a.k + (long)seg.start * a.sk_t + (long)g * a.sk_h;
    const T* V = (const T*)a.v + (long)seg.start * a.sv_t + (long)g * a.sv_h;
    Frag qf[NF];
    load_frags<T, DP>(qf, (const T*)a.q + (long)(seg.start + qrow) * a.sq_t + (long)h * a.sq_h, qrow < seg.len, a.d,
                      half, a.vec);
    const float c = a.scale * kLog2e;
    const int nt = (min(seg.len, q0 + kPkRows) + BN - 1) / BN;

    f32x16 o[ND];
    float m, l;
    TileStage<T, DP, BN> rk, rv;
    {
#pragma unroll
        for (int n = 0; n < ND; n++) o[n] = zero16();
        m = -__builtin_inff();
        l = 0.0f;
        rk.load(K, a.sk_t, 0, seg.len, a.d, a.vec);
        rv.load(V, a.sv_t, 0, seg.len, a.d, a.vec);
        rk.template store<LD>(sk[0]);
        rv.template store<LD>(sv[0]);
        __syncthreads();
        for (int j = 0; j < nt; j++) {
            if (j + 1 < nt) {
                rk.load(K, a.sk_t, (j + 1) * BN, seg.len, a.d, a.vec);
                rv.load(V, a.sv_t, (j + 1) * BN, seg.len, a.d, a.vec);
            }
            if (j * BN <= qw + 31) {
                const T* ks = sk[j & 1];
                const T* vs = sv[j & 1];
                f32x16 s[NS];
#pragma unroll
                for (int u = 0; u < NS; u++) {
                    s[u] = zero16();
#pragma unroll
                    for (int f = 0; f < NF; f++) {
                        const Frag kf = *reinterpret_cast<const Frag*>(ks + (32 * u + (lane & 31)) * LD + f * KF +
                                                                       half * (KF / 2));
                        s[u] = M::mma(kf, qf[f], s[u]);
                    }
                }
                const bool diag = j * BN + BN - 1 > qw;
                if (diag) {
#pragma unroll
                    for (int u = 0; u < NS; u++)
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            if (j * BN + 32 * u + 8 * (i / 4) + 4 * half + i % 4 > qrow) s[u][i] = -__builtin_inff();
                }
                float mx = s[0][0];
#pragma unroll
                for (int u = 0; u < NS; u++)
#pragma unroll
                    for (int i = 0; i < 16; i++) mx = fmaxf(mx, s[u][i]);
                mx = fmaxf(m, half_max(mx) * c);
                // nothing but -inf so far: exponents of -inf, not NaN
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
                for (int n = 0; n < ND; n++)
#pragma unroll
                    for (int i = 0; i < 16; i++) o[n][i] *= al;
#pragma unroll
                for (int u = 0; u < NS; u++)
#pragma unroll
                    for (int f = 0; f < 32 / KF; f++) {
                        const Frag pf = M::pack(s[u], f);
#pragma unroll
                        for (int n = 0; n < ND; n++) {
                            const Frag vf = M::load_tr(vs + 32 * u * LD + 32 * n, LD, f, lane);
                            o[n] = M::mma(vf, pf, o[n]);
                        }
                    }
            }
            if (j + 1 < nt) {
                rk.template store<LD>(sk[(j + 1) & 1]);
                rv.template store<LD>(sv[(j + 1) & 1]);
            }
            __syncthreads();
        }
    }
    l = half_sum(l);
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

template <typename T, int DP, int BN>
__global__ __launch_bounds__(kPkThreads, DP * sizeof(T) <= 256 ? 2 : 1) void packed_dq_kernel(const PackedArgs a) {
    using M = Mma<T>;
    using Frag = typename M::Frag;
    constexpr int KF = M::KF, NF = DP / KF, ND = DP / 32, NS = BN / 32, LD = DP + M::VEC;
    __shared__ __attribute__((aligned(16))) T sk[BN * LD];
    __shared__ __attribute__((aligned(16))) T sv[BN * LD];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    int h, tile;
    packed_block(a.heads, h, tile);
    PackedSeg seg = packed_tile(a.cu, a.n_seqs, a.total, tile, kPkRows);
    if (seg.kind == 0) return;
    T* dq = (T*)a.dq;
    if (seg.kind == 2) {
        if (a.zero_rest) packed_zero(dq, seg.start + seg.row0, min(kPkRows, seg.len - seg.row0), a.heads, h, a.d);
        return;
    }
    const int q0 = ((seg.len - 1) / kPkRows) * kPkRows - seg.row0;
    const int qw = q0 + 32 * wave, qrow = qw + (lane & 31);
    const bool there = qrow < seg.len;
    const long row = seg.start + qrow;
    const int g = h / (a.heads / a.kv_heads);
    const T* K = (const T*)a.k + (long)seg.start * a.sk_t + (long)g * a.sk_h;
    const T* V = (const T*)a.v + (long)seg.start * a.sv_t + (long)g * a.sv_h;
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
    if (there && half == 0) a.delta[(long)h * a.total + row] = dl;
    // rows without a key that counts (lse -inf) and rows past the sequence: p = 0
    float lse = there ? a.lse[(long)h * a.total + row] * kLog2e : __builtin_inff();
    if (lse == -__builtin_inff()) lse = __builtin_inff();
    const float c = a.scale * kLog2e;
    const int nt = (min(seg.len, q0 + kPkRows) + BN - 1) / BN;

    f32x16 acc[ND];
    TileStage<T, DP, BN> rk, rv;
    {
#pragma unroll
        for (int n = 0; n < ND; n++) acc[n] = zero16();
        rk.load(K, a.sk_t, 0, seg.len, a.d, a.vec);
        rv.load(V, a.sv_t, 0, seg.len, a.d, a.vec);
        for (int j = 0; j < nt; j++) {
            __syncthreads();
            rk.template store<LD>(sk);
            rv.template store<LD>(sv);
            __syncthreads();
            if (j + 1 < nt) {
                rk.load(K, a.sk_t, (j + 1) * BN, seg.len, a.d, a.vec);
                rv.load(V, a.sv_t, (j + 1) * BN, seg.len, a.d, a.vec);
            }
            if (j * BN > qw + 31) continue;
            const bool diag = j * BN + BN - 1 > qw;
#pragma unroll
            for (int u = 0; u < NS; u++) {
                f32x16 s = zero16(), dp = zero16();
#pragma unroll
                for (int f = 0; f < NF; f++) {
                    const int at = (32 * u + (lane & 31)) * LD + f * KF + half * (KF / 2);
                    s = M::mma(*reinterpret_cast<const Frag*>(sk + at), qf[f], s);
                    dp = M::mma(*reinterpret_cast<const Frag*>(sv + at), gf[f], dp);
                }
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const float p = exp2_hw(__builtin_fmaf(s[i], c, -lse));
                    s[i] = p * (dp[i] - dl);
                }
                if (diag) {
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        if (j * BN + 32 * u + 8 * (i / 4) + 4 * half + i % 4 > qrow) s[i] = 0.0f;
                }
#pragma unroll
                for (int f = 0; f < 32 / KF; f++) {
                    const Frag df = M::pack(s, f);
#pragma unroll
                    for (int n = 0; n < ND; n++) {
                        const Frag kf = M::load_tr(sk + 32 * u * LD + 32 * n, LD, f, lane);
                        acc[n] = M::mma(kf, df, acc[n]);
                    }
                }
            }
        }
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
template <typename T, int DP, int BQ, int WHICH>
__global__ __launch_bounds__(kPkThreads, DP * sizeof(T) <= 128 ? 2 : 1) void packed_dkv_kernel(const PackedArgs a) {
    using M = Mma<T>;
    using Frag = typename M::Frag;
    constexpr int KF = M::KF, NF = DP / KF, ND = DP / 32, NS = BQ / 32, LD = DP + M::VEC;
    constexpr bool WV = WHICH & 1, WK = WHICH & 2;
    __shared__ __attribute__((aligned(16))) T sq[BQ * LD];
    __shared__ __attribute__((aligned(16))) T sg[BQ * LD];
    __shared__ __attribute__((aligned(16))) float sl[BQ];
    __shared__ __attribute__((aligned(16))) float sd[BQ];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    int g, tile;
    packed_block(a.kv_heads, g, tile);
    const PackedSeg seg = packed_tile(a.cu, a.n_seqs, a.total, tile, kPkRows);
    if (seg.kind == 0) return;
    T* dk = (T*)a.dk;
    T* dv = (T*)a.dv;
    if (seg.kind == 2) {
        const int rows = min(kPkRows, seg.len - seg.row0);
        if (a.zero_rest) {
            if (WK) packed_zero(dk, seg.start + seg.row0, rows, a.kv_heads, g, a.d);
            if (WV) packed_zero(dv, seg.start + seg.row0, rows, a.kv_heads, g, a.d);
        }
        return;
    }
    const int k0 = seg.row0, kw = k0 + 32 * wave, key = kw + (lane & 31);
    const int rep = a.heads / a.kv_heads;
    const bool there = key < seg.len;
    const long row = seg.start + key;
    Frag kf[NF], vf[WK ? NF : 1];
    load_frags<T, DP>(kf, (const T*)a.k + row * a.sk_t + (long)g * a.sk_h, there, a.d, half, a.vec);
    if constexpr (WK) load_frags<T, DP>(vf, (const T*)a.v + row * a.sv_t + (long)g * a.sv_h, there, a.d, half, a.vec);
    const float c = a.scale * kLog2e;
    const int t0 = k0 / BQ, nt = (seg.len + BQ - 1) / BQ, steps = (nt - t0) * rep;

    f32x16 ak[WK ? ND : 1], av[WV ? ND : 1];
    TileStage<T, DP, BQ> rq, rg;
    float rl = 0.0f, rd = 0.0f;
    const T* const Q = (const T*)a.q + (long)seg.start * a.sq_t + (long)g * rep * a.sq_h;
    const T* const G = (const T*)a.grad + ((long)seg.start * a.heads + (long)g * rep) * a.d;
    auto fetch = [&](int st) {
        const int r = st / (nt - t0), first = (t0 + st % (nt - t0)) * BQ;
        rq.load(Q + (long)r * a.sq_h, a.sq_t, first, seg.len, a.d, a.vec);
        rg.load(G + (long)r * a.d, (long)a.heads * a.d, first, seg.len, a.d, a.vec);
        if (threadIdx.x < BQ) {
            const int t = first + threadIdx.x;
            rl = __builtin_inff();
            rd = 0.0f;
            if (t < seg.len) {
                const long at = (long)(g * rep + r) * a.total + seg.start + t;
                rl = a.lse[at] * kLog2e;
                if (rl == -__builtin_inff()) rl = __builtin_inff();
                rd = a.delta[at];
            }
        }
    };
    {
#pragma unroll
        for (int n = 0; n < ND; n++) {
            if constexpr (WK) ak[n] = zero16();
            if constexpr (WV) av[n] = zero16();
        }
        fetch(0);
        for (int st = 0; st < steps; st++) {
            __syncthreads();
            rq.template store<LD>(sq);
            rg.template store<LD>(sg);
            if (threadIdx.x < BQ) {
                sl[threadIdx.x] = rl;
                sd[threadIdx.x] = rd;
            }
            __syncthreads();
            if (st + 1 < steps) fetch(st + 1);
            const int first = (t0 + st % (nt - t0)) * BQ;
#pragma unroll
            for (int u = 0; u < NS; u++) {
                const int qb = first + 32 * u;
                if (qb + 31 < kw) continue;              // every query of these is before the wave's keys
                f32x16 s = zero16(), dp = zero16();
#pragma unroll
                for (int f = 0; f < NF; f++) {
                    const int at = (32 * u + (lane & 31)) * LD + f * KF + half * (KF / 2);
                    s = M::mma(*reinterpret_cast<const Frag*>(sq + at), kf[f], s);
                    if constexpr (WK) dp = M::mma(*reinterpret_cast<const Frag*>(sg + at), vf[f], dp);
                }
                const bool diag = qb < kw + 31;
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    const f32x4 le = *reinterpret_cast<const f32x4*>(sl + 32 * u + 8 * b + 4 * half);
                    const f32x4 de = *reinterpret_cast<const f32x4*>(sd + 32 * u + 8 * b + 4 * half);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int i = 4 * b + j;
                        s[i] = exp2_hw(__builtin_fmaf(s[i], c, -le[j]));
                        if constexpr (WK) dp[i] = s[i] * (dp[i] - de[j]);
                        if (diag && qb + 8 * b + 4 * half + j < key) {
                            s[i] = 0.0f;
                            if constexpr (WK) dp[i] = 0.0f;
                        }
                    }
                }
#pragma unroll
                for (int f = 0; f < 32 / KF; f++) {
                    Frag pf, df;
                    if constexpr (WV) pf = M::pack(s, f);
                    if constexpr (WK) df = M::pack(dp, f);
#pragma unroll
                    for (int n = 0; n < ND; n++) {
                        if constexpr (WV) {
                            const Frag ga = M::load_tr(sg + 32 * u * LD + 32 * n, LD, f, lane);
                            av[n] = M::mma(ga, pf, av[n]);
                        }
                        if constexpr (WK) {
                            const Frag qa = M::load_tr(sq + 32 * u * LD + 32 * n, LD, f, lane);
                            ak[n] = M::mma(qa, df, ak[n]);
                        }
                    }
                }
            }
        }
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

static long packed_tiles(const PackedArgs& a) { return (long)a.total / kPkRows + a.n_seqs + 2; }

template <typename T, int DP>
static void packed_launch_dp(const PackedArgs& a, bool backward, hipStream_t s) {
    constexpr int BN = sizeof(T) == 2 ? 64 : 32;
    const dim3 gh((unsigned)(packed_tiles(a) * a.heads)), gk((unsigned)(packed_tiles(a) * a.kv_heads)), t(kPkThreads);
    if (!backward) {
        hipLaunchKernelGGL((packed_fwd_kernel<T, DP, BN>), gh, t, 0, s, a);
        return;
    }
    hipLaunchKernelGGL((packed_dq_kernel<T, DP, BN>), gh, t, 0, s, a);
    if constexpr (DP * sizeof(T) > 512) {
        hipLaunchKernelGGL((packed_dkv_kernel<T, DP, 32, 1>), gk, t, 0, s, a);
        hipLaunchKernelGGL((packed_dkv_kernel<T, DP, 32, 2>), gk, t, 0, s, a);
    } else {
        hipLaunchKernelGGL((packed_dkv_kernel<T, DP, BN, 3>), gk, t, 0, s, a);
    }
}

template <typename T>
static void packed_launch_t(const PackedArgs& a, bool backward, hipStream_t s) {
    if (a.d <= 32) packed_launch_dp<T, 32>(a, backward, s);
    else if (a.d <= 64) packed_launch_dp<T, 64>(a, backward, s);
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
