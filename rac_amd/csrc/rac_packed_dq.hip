// rac_packed_dq.hip — packed causal attention, the gradient of q, and D = do . o.
#include "rac_packed.hpp"

namespace rac {

// ds = p (dp - D) of 32 rows as columns, then dq += ds k: three products of a
// tile of keys and values, of which k is read both ways.  Bound by matrix
// instructions (busy 0.41): six bf16 documents of 8192 rows (32/8 heads of 128)
// 342 - 360 us, fp32 rows of 777, 1, 1250 and 63 (12/4 heads of 80) 118.
template <typename T, int DP, int WR>
__global__ __launch_bounds__(kPkThreads, DP * sizeof(T) <= 256 ? 2 : 1) void packed_dq_kernel(const PackedArgs a) {
    using M = Mma<T>;
    using Frag = typename M::Frag;
    using S = PackedShape<T, DP, WR>;
    using TL = Tile<T, DP>;
    constexpr int KG = S::KG, BN = S::BN, TILE = S::TILE, ND = S::ND, NF = S::NF, NS = S::NS, FS = S::FS;
    __shared__ __attribute__((aligned(16))) char ka[S::BYTES], va[S::BYTES], kb[S::BYTES], vb[S::BYTES];
    const int lane0 = threadIdx.x & 63, lane = lane0, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
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
    // 16 bits through registers: 6 bf16 documents of 8192 rows (32/8 heads of
    // 128) 305 us, direct 386
    TileLoad<T, DP, TILE> lk, lv;
    lk.init(a.sk_t, a.d);
    lv.init(a.sv_t, a.d);
    auto issue = [&](int j, char* kd, char* vd) ATTN_INLINE {
        lk.issue(kd, K + (long)j * TILE * a.sk_t, seg.len - j * TILE, a.sk_t, a.d, a.vec, wave);
        lv.issue(vd, V + (long)j * TILE * a.sv_t, seg.len - j * TILE, a.sv_t, a.d, a.vec, wave);
    };
    auto commit = [&](int j, char* kd, char* vd) ATTN_INLINE {
        lk.commit(kd, K + (long)j * TILE * a.sk_t, seg.len - j * TILE, a.sk_t, a.d, a.vec);
        lv.commit(vd, V + (long)j * TILE * a.sv_t, seg.len - j * TILE, a.sv_t, a.d, a.vec);
    };
    // D = do . o, kept for the keys' kernel beside the log sums.  A rounded o
    // alone would leave D, and through it every ds of the row, off by as much as
    // all their own roundings together: what its rounding took is added.
    float dl = 0.0f;
    if (there) {
        const long at = (row * a.heads + h) * a.d;
#pragma unroll 4
        for (int f = 0; f < NF; f++) {
            const int at_f = f * M::KF + half * (M::KF / 2);
            auto chunk = [&](const void* p) ATTN_INLINE {
                return __builtin_bit_cast(Frag, load_chunk((const T*)p + at, at_f, a.d, a.vec));
            };
            const Frag go = chunk(a.grad), of = chunk(a.out), lo = sizeof(T) == 2 && a.out_lo ? chunk(a.out_lo) : Frag{};
#pragma unroll
            for (int e = 0; e < M::VEC; e++) {
                dl = __builtin_fmaf(M::to_f32(go[e]), M::to_f32(of[e]), dl);
                if (sizeof(T) == 2) dl = __builtin_fmaf(M::to_f32(go[e]), M::to_f32(lo[e]), dl);
            }
        }
    }
    issue(0, ka, va);
    Frag qf[NF], gf[NF];
    load_frags<T, DP>(qf, (const T*)a.q + row * a.sq_t + (long)h * a.sq_h, there, a.d, half, a.vec);
    load_frags<T, DP>(gf, (const T*)a.grad + (row * a.heads + h) * a.d, there, a.d, half, a.vec);
    dl = half_sum(dl);
    // rows without a key that counts (lse -inf) and rows past the sequence: p = 0
    float lse = there ? a.lse[(long)h * a.total + row] * kLog2e : __builtin_inff();
    if (lse == -__builtin_inff()) lse = __builtin_inff();
    if (there && half == 0 && kg == 0) {
        a.stats[2 * ((long)h * a.total + row)] = lse;
        a.stats[2 * ((long)h * a.total + row) + 1] = dl;
    }
    const float c = a.scale * kLog2e;
    f32x16 acc[ND];
#pragma unroll
    for (int n = 0; n < ND; n++) acc[n] = zero16();

    auto work = [&](int j, const char* ks, const char* vs) ATTN_INLINE {
        // rows this long fill the registers: no tile's address stays in one
        const int lane = DP * sizeof(T) >= 1024 ? attn_fresh(lane0) : lane0, half = lane >> 5;
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
                attn_branch();
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
    auto step = [&](int j, const char* ks, const char* vs, char* kn, char* vn) ATTN_INLINE {
        tiles_landed();
        if (j + 1 < nt) issue(j + 1, kn, vn);
        work(j, ks, vs);
        if (j + 1 < nt) commit(j + 1, kn, vn);
    };
    commit(0, ka, va);
    for (int j = 0; j < nt; j += 2) {
        step(j, ka, va, kb, vb);
        if (j + 1 < nt) step(j + 1, kb, vb, ka, va);
    }
    if constexpr (KG > 1) {
        join_groups<KG, WR, ND>(acc, 1.0f, ka, wr, kg, lane);
        if (kg) return;
    }
    uint32_t again = columns_of(not_finite(acc) && there && lse == lse && dl == dl);
    if (there && !(again >> (lane & 31) & 1))
        attn_store<T, ND>(dq + (row * a.heads + h) * a.d, acc, a.scale, a.d, half, a.vec_out);
    for (; again; again &= again - 1) {
        const int r = __ffs((int)again) - 1;
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

// ── launch ──────────────────────────────────────────────────────────────

namespace {
struct Launch {
    const PackedArgs& a;
    hipStream_t s;
    template <typename T, int DP, int WR>
    void sets() const {
        hipLaunchKernelGGL((packed_dq_kernel<T, DP, WR>), dim3((unsigned)(packed_tiles(a, 32 * WR) * a.heads)), dim3(kPkThreads), 0,
                           s, a);
    }
    template <typename T, int DP>
    void run() const {
        packed_by_sets<T, DP>(a, *this);
    }
};
}  // namespace

hipError_t packed_dq_launch(const PackedArgs& a, int dtype, hipStream_t s) {
    packed_by_type(dtype, a.d, Launch{a, s});
    return hipGetLastError();
}

}  // namespace rac
