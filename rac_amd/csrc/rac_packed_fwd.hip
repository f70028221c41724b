// rac_packed_fwd.hip — packed causal attention, forward.
#include "rac_packed.hpp"

namespace rac {

// Bound by matrix instructions and, in 16 bits, the exponentials beside them,
// which one wave's products and another's softmax overlap: two workgroups to a
// CU.  One bf16 prompt of 8192 (32/8 heads of 128) 521 - 558 us, 1.0 PFLOP/s of
// the triangle, matrix cores busy 0.57 of the time and the VALU 0.51; six fp32
// prompts of 4096 rows in all (32/4 heads of 64) 225 us, matrix cores 0.77.
template <typename T, int DP, int WR>
__global__ __launch_bounds__(kPkThreads, DP * sizeof(T) <= 256 ? 2 : 1) void packed_fwd_kernel(const PackedArgs a) {
    using M = Mma<T>;
    using Frag = typename M::Frag;
    using S = PackedShape<T, DP, WR>;
    using TL = Tile<T, DP>;
    constexpr int KG = S::KG, BN = S::BN, TILE = S::TILE, ND = S::ND, NF = S::NF, NS = S::NS, FS = S::FS;
    __shared__ __attribute__((aligned(16))) char ka[S::BYTES], va[S::BYTES], kb[S::BYTES], vb[S::BYTES];
    __shared__ float sm[KG > 1 ? kAttnWaves : 1][32], sl[KG > 1 ? kAttnWaves : 1][32];
    const int lane0 = threadIdx.x & 63, lane = lane0, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int wr = wave % WR, kg = wave / WR;
    int h, tile;
    packed_block(a.heads, h, tile);
    const PackedSeg seg = packed_tile(a.cu, a.n_seqs, a.total, tile, S::ROWS, false);
    if (seg.kind == 0) return;
    T* out = (T*)a.out;
    T* lo = (T*)a.out_lo;
    if (seg.kind == 2) {
        if (a.zero_rest) packed_zero(out, seg.start + seg.row0, min(S::ROWS, seg.len - seg.row0), a.heads, h, a.d);
        return;
    }
    const int q0 = seg.row0, qw = q0 + 32 * wr, qrow = qw + (lane & 31);
    const int g = h / (a.heads / a.kv_heads);
    const T* K = (const T*)a.k + (long)seg.start * a.sk_t + (long)g * a.sk_h;
    const T* V = (const T*)a.v + (long)seg.start * a.sv_t + (long)g * a.sv_h;
    const int nt = (min(seg.len, q0 + S::ROWS) + TILE - 1) / TILE;
    // direct also in 16 bits: one bf16 prompt of 8192 (32/8 heads of 128) 608 us,
    // through registers 634
    TileLoad<T, DP, TILE, true> lk, lv;
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
    issue(0, ka, va);
    Frag qf[NF];
    load_frags<T, DP>(qf, (const T*)a.q + (long)(seg.start + qrow) * a.sq_t + (long)h * a.sq_h, qrow < seg.len, a.d,
                      half, a.vec);
    const float c = a.scale * kLog2e;
    f32x16 o[ND];
#pragma unroll
    for (int n = 0; n < ND; n++) o[n] = zero16();
    float m = -__builtin_inff(), l = 0.0f;

    auto work = [&](int j, const char* ks, const char* vs) ATTN_INLINE {
        // rows this long fill the registers: no tile's address stays in one
        const int lane = DP * sizeof(T) >= 1024 ? attn_fresh(lane0) : lane0, half = lane >> 5;
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
            attn_branch();
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
    uint32_t again = columns_of(not_finite(o) && qrow < seg.len && l == l);
    if (qrow < seg.len) {
        const long row = seg.start + qrow;
        const long at = (row * a.heads + h) * a.d;
        if (!(again >> (lane & 31) & 1)) {
            attn_store<T, ND>(out + at, o, inv, a.d, half, a.vec_out);
            if (sizeof(T) == 2 && lo) attn_store_rest<T, ND>(lo + at, o, inv, a.d, half, a.vec_out);
        }
        if (a.lse && half == 0) a.lse[(long)h * a.total + row] = (m + __builtin_amdgcn_logf(l)) * kLn2;
    }
    for (; again; again &= again - 1) {
        const int r = __ffs((int)again) - 1, t = qw + r;
        const float mr = __shfl(m, r), ir = __shfl(inv, r);
        const T* q = (const T*)a.q + (long)(seg.start + t) * a.sq_t + (long)h * a.sq_h;
        const long at = ((long)(seg.start + t) * a.heads + h) * a.d;
        attn_again<T, DP>(out + at, ir, a.d, 0, t + 1,
                          [&](int j) { return exp2_hw(__builtin_fmaf(row_dot(q, K + (long)j * a.sk_t, a.d), c, -mr)); },
                          [&](int j) { return V + (long)j * a.sv_t; }, lo && sizeof(T) == 2 ? lo + at : nullptr);
    }
}

// ── launch ──────────────────────────────────────────────────────────────

namespace {
struct Launch {
    const PackedArgs& a;
    hipStream_t s;
    template <typename T, int DP, int WR>
    void sets() const {
        hipLaunchKernelGGL((packed_fwd_kernel<T, DP, WR>), dim3((unsigned)(packed_tiles(a, 32 * WR) * a.heads)), dim3(kPkThreads), 0,
                           s, a);
    }
    template <typename T, int DP>
    void run() const {
        packed_by_sets<T, DP>(a, *this);
    }
};
}  // namespace

hipError_t packed_fwd_launch(const PackedArgs& a, int dtype, hipStream_t s) {
    packed_by_type(dtype, a.d, Launch{a, s});
    return hipGetLastError();
}

}  // namespace rac
