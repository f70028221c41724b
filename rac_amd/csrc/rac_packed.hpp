// rac_packed.hpp — causal attention over packed sequences with grouped heads,
// forward and backward, on the matrix cores: what its three kernels
// (rac_packed_fwd.hip, rac_packed_dq.hip, rac_packed_dkv.hip) share.
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
// Scores, statistics and every sum are fp32.  The 16-bit types round p (in [0,
// 2^8] against the running maximum) and ds to themselves for the next product,
// each by half a step of its own value and independently of the others, because
// the matrix cores take 16-bit operands at seven times the fp32 rate: relative
// to their size, bf16 outputs are off by 0.0021 and dq by 0.0027 in all, of which
// the rounding of the results themselves is 0.0017.
//
// Values in places the mask takes away do not reach a result, NaN and
// infinities among them: masked scores are replaced before the exponential;
// where a tile's product would still multiply such a value by a probability of
// 0, the row's accumulators show it (they are not finite), and its wave does
// that row again over the keys it sees and no others (attn_again).  A row whose
// own weights are NaN is NaN throughout and stays so.
#pragma once
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

// tiles of `rows` rows: at most this many, whatever the sequences' lengths
inline long packed_tiles(const PackedArgs& a, int rows) { return (long)a.total / rows + a.n_seqs + 2; }

// LDS for the two tiles twice: 128 KB of it
template <typename T, int DP, int WR>
constexpr bool packed_fits() {
    return 4 * PackedShape<T, DP, WR>::BYTES <= (128 << 10);
}
// the fewest row sets (16-bit rows of 192 bytes and more: 128 KB to a workgroup
// cost more than its shorter path gains, 3 prompts of 2500 rows, 8 heads of
// 128, 39 us in one set, 22 in two)
template <typename T, int DP>
constexpr int packed_few_sets() {
    if (sizeof(T) == 2 && DP >= 96) return 2;
    return packed_fits<T, DP, 1>() ? 1 : packed_fits<T, DP, 2>() ? 2 : 4;
}
// about `each` workgroups for every CU, with `rows` rows to one
inline bool packed_enough(const PackedArgs& a, int rows, int heads, int each) {
    return ((long)a.total / rows + (a.n_seqs + 1) / 2) * heads >= each * device_cus();
}
// Whether the keys' kernel takes a workgroup for every query head, and a join:
// where heads share keys and the keys' tiles alone leave CUs idle.
inline bool packed_by_head_parts(const PackedArgs& a) {
    return a.heads > a.kv_heads && !packed_enough(a, 64, a.kv_heads, 1);
}

// Forward and dq: the most row sets that still make two workgroups for every
// CU.  us of the forward pass in 4, 2 and 1 sets (MI355X): bf16, heads x rows of
// 32 x 4096 x 128 156, 180, 454; 32 x 1400 x 64 28, 22, 33; 8 x 1000 x 64 21, 16,
// 12; fp32, 32 x 1500 x 64 137, 100, 137; 8 x 1000 x 64 77, 43, 28.
template <typename T, int DP, typename F>
void packed_by_sets(const PackedArgs& a, F f) {
    constexpr int FEW = packed_few_sets<T, DP>();
    if (packed_enough(a, 128, a.heads, 2)) return f.template sets<T, DP, 4>();
    if constexpr (FEW < 2) {
        if (packed_enough(a, 64, a.heads, 2)) return f.template sets<T, DP, 2>();
    }
    f.template sets<T, DP, FEW>();
}

// f.run<T, DP>() for a type and a head size
template <typename T, typename F>
void packed_by_head(int d, F f) {
    if (d <= 32) f.template run<T, 32>();
    else if (d <= 64) f.template run<T, 64>();
    else if (d <= 96) f.template run<T, 96>();
    else if (d <= 128) f.template run<T, 128>();
    else f.template run<T, 256>();
}
template <typename F>
void packed_by_type(int dtype, int d, F f) {
    if (dtype == 0) packed_by_head<float>(d, f);
    else if (dtype == 1) packed_by_head<__bf16>(d, f);
    else packed_by_head<_Float16>(d, f);
}

}  // namespace rac
