// rac_packed_dkv.hip — packed causal attention, the gradients of k and v.
#include "rac_packed.hpp"
#include <type_traits>

namespace rac {

// p and ds of 32 keys as columns, then dv += p do and dk += ds q: four products
// of a tile of q and do, each read both ways, over the group's query heads.  Both
// sums' accumulators and the keys' fragments leave a SIMD one wave in rows of 256
// bytes, whose matrix instructions wait for its own LDS reads (busy 0.28): six
// bf16 documents of 8192 rows (32/8 heads of 128) 568 - 627 us, fp32 rows of
// 777, 1, 1250 and 63 (12/4 heads of 80, by query head) 141 and the join 7.
// WHICH: 1 dv, 2 dk, 3 both (d past 128 in fp32 has no registers for both)
// BY_HEAD: a workgroup sums one query head's part, in fp32, for the join below
template <typename T, int DP, int WR, int WHICH, bool BY_HEAD>
__global__ __launch_bounds__(kPkThreads, DP * sizeof(T) <= 128 ? 2 : 1) void packed_dkv_kernel(const PackedArgs a) {
    using M = Mma<T>;
    using Frag = typename M::Frag;
    using S = PackedShape<T, DP, WR>;
    using TL = Tile<T, DP>;
    constexpr int KG = S::KG, BQ = S::BN, TILE = S::TILE, ND = S::ND, NF = S::NF, NS = S::NS, FS = S::FS;
    constexpr bool WV = WHICH & 1, WK = WHICH & 2;
    __shared__ __attribute__((aligned(16))) char qa[S::BYTES], ga[S::BYTES], qb[S::BYTES], gb[S::BYTES];
    __shared__ __attribute__((aligned(16))) float sa[2 * TILE], sb[2 * TILE];       // log2 sums and D
    const int lane0 = threadIdx.x & 63, lane = lane0, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int wr = wave % WR, kg = wave / WR;
    using O = typename std::conditional<BY_HEAD, float, T>::type;
    int h, tile;
    packed_block(BY_HEAD ? a.heads : a.kv_heads, h, tile);
    const int group = a.heads / a.kv_heads, g = BY_HEAD ? h / group : h;
    const PackedSeg seg = packed_tile(a.cu, a.n_seqs, a.total, tile, S::ROWS, true);
    if (seg.kind == 0) return;
    O* dk = BY_HEAD ? (O*)a.part : (O*)a.dk;
    O* dv = BY_HEAD ? (O*)(a.part + (long)a.total * a.heads * a.d) : (O*)a.dv;
    if (seg.kind == 2) {
        const int rows = min(S::ROWS, seg.len - seg.row0);
        if (!BY_HEAD && a.zero_rest) {
            if (WK) packed_zero(dk, seg.start + seg.row0, rows, a.kv_heads, g, a.d);
            if (WV) packed_zero(dv, seg.start + seg.row0, rows, a.kv_heads, g, a.d);
        }
        return;
    }
    const int k0 = seg.row0, kw = k0 + 32 * wr, key = kw + (lane & 31);
    const int rep = BY_HEAD ? 1 : group, h0 = BY_HEAD ? h : g * group;      // query heads of the sum
    const int oheads = BY_HEAD ? a.heads : a.kv_heads;
    const bool there = key < seg.len;
    const long row = seg.start + key;
    // steps: the tiles of queries from the diagonal on, for one head of the group after the other
    const int t0 = k0 / TILE, per = (seg.len + TILE - 1) / TILE - t0, steps = per * rep;
    const T* const Q = (const T*)a.q + (long)seg.start * a.sq_t + (long)h0 * a.sq_h;
    const T* const G = (const T*)a.grad + ((long)seg.start * a.heads + h0) * a.d;
    // direct also in 16 bits: 6 bf16 documents of 8192 rows (32/8 heads of 128)
    // 795 us, through registers 870
    TileLoad<T, DP, TILE, true> lq, lg;
    lq.init(a.sq_t, a.d);
    lg.init((long)a.heads * a.d, a.d);
    int ih = 0, it = t0;                                  // head and tile of the next issue
    const int slot = threadIdx.x;                         // a thread's value of a tile's log sums and D
    float stat_next = 0.0f;
    auto issue = [&](char* qd, char* gd) ATTN_INLINE {
        const int first = it * TILE, left = seg.len - first;
        lq.issue(qd, Q + (long)ih * a.sq_h + (long)first * a.sq_t, left, a.sq_t, a.d, a.vec, wave);
        lg.issue(gd, G + (long)ih * a.d + (long)first * a.heads * a.d, left, (long)a.heads * a.d, a.d, a.vec, wave);
        if (slot < 2 * TILE) {
            const float* base = a.stats + 2 * ((long)(h0 + ih) * a.total + seg.start + first);
            // rows past the sequence: 0, next to zeros of do no matter
            stat_next = slot < 2 * left ? base[slot] : 0.0f;
        }
    };
    // behind the work on the tile before
    auto commit = [&](char* qd, char* gd, float* st) ATTN_INLINE {
        if (slot < 2 * TILE) st[slot] = stat_next;
        const int first = it * TILE, left = seg.len - first;
        lq.commit(qd, Q + (long)ih * a.sq_h + (long)first * a.sq_t, left, a.sq_t, a.d, a.vec);
        lg.commit(gd, G + (long)ih * a.d + (long)first * a.heads * a.d, left, (long)a.heads * a.d, a.d, a.vec);
        if (++it == t0 + per) {
            it = t0;
            ih++;
        }
    };
    issue(qa, ga);
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
    auto work = [&](const char* qs, const char* gs, const float* ss) ATTN_INLINE {
        // rows this long fill the registers: no tile's address stays in one
        const int lane = DP * sizeof(T) >= 512 ? attn_fresh(lane0) : lane0, half = lane >> 5;
        const int first = ct * TILE + kg * BQ, row0 = kg * BQ;
        if (++ct == t0 + per) ct = t0;
        auto scores = [&](int u, f32x16& s, f32x16& dp) ATTN_INLINE {
            s = zero16();
            dp = zero16();
#pragma unroll
            for (int f = 0; f < NF; f++) {
                s = M::mma(TL::rows(qs, row0 + 32 * u, f, lane), kf[f], s);
                if constexpr (WK) dp = M::mma(TL::rows(gs, row0 + 32 * u, f, lane), vf[f], dp);
            }
        };
        auto weights = [&](int u, f32x16& s, f32x16& dp) ATTN_INLINE {
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const f32x4* st = reinterpret_cast<const f32x4*>(ss + 2 * (row0 + 32 * u + 8 * b + 4 * half));
                const f32x4 st0 = st[0], st1 = st[1];
                const float le[4] = {st0[0], st0[2], st1[0], st1[2]}, de[4] = {st0[1], st0[3], st1[1], st1[3]};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int i = 4 * b + j;
                    s[i] = exp2_hw(__builtin_fmaf(s[i], c, -le[j]));
                    if constexpr (WK) dp[i] = s[i] * (dp[i] - de[j]);
                }
            }
        };
        auto sums = [&](int u, const f32x16& s, const f32x16& dp) ATTN_INLINE {
#pragma unroll
            for (int f = 0; f < FS; f++) {
                Frag pf, df;
                if constexpr (WV) pf = M::pack(s, f);
                if constexpr (WK) df = M::pack(dp, f);
#pragma unroll
                for (int n = 0; n < ND; n++) {
                    if constexpr (WV) av[n] = M::mma(TL::cols(gs, row0 + 32 * u, f, n, lane), pf, av[n]);
                    if constexpr (WK) ak[n] = M::mma(TL::cols(qs, row0 + 32 * u, f, n, lane), df, ak[n]);
                }
            }
        };
        auto mask = [&](int q0, f32x16& s, f32x16& dp) ATTN_INLINE {
            attn_branch();
#pragma unroll
            for (int i = 0; i < 16; i++)
                if (q0 + 8 * (i / 4) + 4 * half + i % 4 < kw + (lane & 31)) {
                    s[i] = 0.0f;
                    if constexpr (WK) dp[i] = 0.0f;
                }
        };
        if (first + BQ - 1 < kw || first >= seg.len) return;      // before the wave's keys, or past the sequence
        f32x16 s[NS], dp[NS];
#pragma unroll
        for (int u = 0; u < NS; u++) scores(u, s[u], dp[u]);
#pragma unroll
        for (int u = 0; u < NS; u++) {
            weights(u, s[u], dp[u]);
            if (first + 32 * u < kw + 31) mask(first + 32 * u, s[u], dp[u]);
            sums(u, s[u], dp[u]);
        }
    };
    auto step = [&](int st, const char* qs, const char* gs, const float* ss, char* qn, char* gn, float* sn) ATTN_INLINE {
        tiles_landed();
        if (st + 1 < steps) issue(qn, gn);
        work(qs, gs, ss);
        if (st + 1 < steps) commit(qn, gn, sn);
    };
    commit(qa, ga, sa);
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
    uint32_t again = columns_of(bad && there);
    if (there && !(again >> (lane & 31) & 1)) {
        const long at = (row * oheads + h) * a.d;
        if constexpr (WK) attn_store<O, ND>(dk + at, ak, a.scale, a.d, half, BY_HEAD ? a.d % 4 == 0 : a.vec_out);
        if constexpr (WV) attn_store<O, ND>(dv + at, av, 1.0f, a.d, half, BY_HEAD ? a.d % 4 == 0 : a.vec_out);
    }
    for (; again; again &= again - 1) {
        const int kr = kw + __ffs((int)again) - 1, from = kr, n = seg.len - from;
        const long at = ((long)(seg.start + kr) * oheads + h) * a.d;
        const T* kk = (const T*)a.k + (long)(seg.start + kr) * a.sk_t + (long)g * a.sk_h;
        const T* vv = (const T*)a.v + (long)(seg.start + kr) * a.sv_t + (long)g * a.sv_h;
        // queries from .. of head 0 of the group, then of head 1, ...
        auto qrow = [&](int i) { return Q + (long)(i / n) * a.sq_h + (long)(from + i % n) * a.sq_t; };
        auto grow = [&](int i) { return G + ((long)(from + i % n) * a.heads + i / n) * a.d; };
        auto stats_of = [&](int i) { return a.stats + 2 * ((long)(h0 + i / n) * a.total + seg.start + from + i % n); };
        auto prob = [&](int i) { return exp2_hw(__builtin_fmaf(row_dot(qrow(i), kk, a.d), c, -*stats_of(i))); };
        auto score = [&](int i) { return prob(i) * (row_dot(grow(i), vv, a.d) - stats_of(i)[1]); };
        // a NaN weight of the key's own query: no head to sum over
        if constexpr (WV) {
            const float w = prob(0);
            attn_again<T, DP>(dv + at, w == w ? 1.0f : w, a.d, 0, w == w ? n * rep : 0, prob, grow);
        }
        if constexpr (WK) {
            const float w = score(0);
            attn_again<T, DP>(dk + at, w == w ? a.scale : w, a.d, 0, w == w ? n * rep : 0, score, qrow);
        }
    }
}

// dk and dv from their query heads' parts, in the order of the heads: a thread
// per value.
template <typename T>
__global__ __launch_bounds__(kPkThreads) void packed_join_kernel(const PackedArgs a) {
    const int rep = a.heads / a.kv_heads;
    const long i = (long)blockIdx.x * kPkThreads + threadIdx.x;
    if (i >= (long)a.total * a.kv_heads * a.d) return;
    const int row = (int)(i / ((long)a.kv_heads * a.d)), c = (int)(i % a.d), g = (int)(i / a.d % a.kv_heads);
    const int first = min(max(a.cu[0], 0), a.total), end = min(max(a.cu[a.n_seqs], first), a.total);
    const bool in = row >= first && row < end;
    if (!in && !a.zero_rest) return;
    float k = 0.0f, v = 0.0f;
    if (in) {
        const float* pk = a.part + ((long)row * a.heads + (long)g * rep) * a.d + c;
        const float* pv = pk + (long)a.total * a.heads * a.d;
        for (int r = 0; r < rep; r++) {
            k += pk[(long)r * a.d];
            v += pv[(long)r * a.d];
        }
    }
    ((T*)a.dk)[i] = Mma<T>::from_f32(k);
    ((T*)a.dv)[i] = Mma<T>::from_f32(v);
}

// ── launch ──────────────────────────────────────────────────────────────

namespace {
struct Launch {
    const PackedArgs& a;
    hipStream_t s;
    template <typename T, int DP, int WR, bool BY_HEAD>
    void sets() const {
        const dim3 grid((unsigned)(packed_tiles(a, 32 * WR) * (BY_HEAD ? a.heads : a.kv_heads))), t(kPkThreads);
        if constexpr (DP == 256) {
            hipLaunchKernelGGL((packed_dkv_kernel<T, DP, WR, 1, BY_HEAD>), grid, t, 0, s, a);
            hipLaunchKernelGGL((packed_dkv_kernel<T, DP, WR, 2, BY_HEAD>), grid, t, 0, s, a);
        } else {
            hipLaunchKernelGGL((packed_dkv_kernel<T, DP, WR, 3, BY_HEAD>), grid, t, 0, s, a);
        }
    }
    // The most row sets that still make a workgroup for every CU, in 16 bits two
    // at most and in rows of 64 bytes one: shorter tiles even out the triangle.
    // us of the backward pass in 4, 2 and 1 sets (MI355X): 6 bf16 documents of
    // 8192 rows, 32/8 heads of 128, 949, 819, 1420; 64 532, 430, 444; 32 372, 293,
    // 255; one of 8192, 32/4 heads of 128, 3497, 2327, 3949.
    template <typename T, int DP, bool BY_HEAD>
    void run_heads() const {
        constexpr int FEW = packed_few_sets<T, DP>();
        const int heads = BY_HEAD ? a.heads : a.kv_heads;
        if constexpr (sizeof(T) == 4 || DP == 256) {
            if (packed_enough(a, 128, heads, 1)) return sets<T, DP, 4, BY_HEAD>();
        }
        if constexpr (FEW < 2 && DP > 32) {
            if (packed_enough(a, 64, heads, 1)) return sets<T, DP, 2, BY_HEAD>();
        }
        sets<T, DP, FEW, BY_HEAD>();
    }
    template <typename T, int DP>
    void run() const {
        if (!packed_by_head_parts(a)) return run_heads<T, DP, false>();
        run_heads<T, DP, true>();
        const long n = (long)a.total * a.kv_heads * a.d;
        hipLaunchKernelGGL((packed_join_kernel<T>), dim3((unsigned)((n + kPkThreads - 1) / kPkThreads)), dim3(kPkThreads), 0,
                           s, a);
    }
};
}  // namespace

long packed_dkv_parts(const PackedArgs& a) { return packed_by_head_parts(a) ? 2L * a.total * a.heads * a.d : 0; }

hipError_t packed_dkv_launch(const PackedArgs& a, int dtype, hipStream_t s) {
    packed_by_type(dtype, a.d, Launch{a, s});
    return hipGetLastError();
}

}  // namespace rac
