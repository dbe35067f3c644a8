// Backward of fmha_fwd on tcgen05 (formulas and the ownership of the sums: fmha_bwd_generic.cu).  hdim 128 / 64, every mask, batch
// and group mode, GQA, ALiBi, soft cap.  Two kernels; a work item is one 128-row tile whose gradient stays in tensor memory:
//
//   dQ    (bwd_dq_sm100_kernel):   128 queries of one head walk the key tiles:    S = Q K^T, dP = dO V^T, dQ += dS K
//   dK/dV (bwd_dkdv_sm100_kernel): 128 keys of one kv head walk the query tiles of the group's heads, transposed:
//                                  S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q
//
// Seven products where one pass with a shared sum for dQ has five; but that pass pays 64 KB of fp32 reductions per tile pair and
// order-dependent results.  Counted in the 128 bytes a clock of shared memory, which feeds both operands of an SS product and
// one of a TS product (128 x 128 x 128: 512 clocks of the tensor pipe, 512 or 256 of shared memory): dQ 3 x 256 + K/V copies 512
// = 1280 clocks beside 1536 of products (Q and dO live in tensor memory, so all three products are TS); dK/dV 2 x 512 + 2 x 256 +
// 512 = 2048 beside 2048.  P and dS go from registers to tensor memory as A operands and never through shared memory.
//
// The kernels are persistent (one CTA per SM).  Roles: warps 0-15 the elementwise work (thread = tensor memory lane = row; four
// warpgroups, 32 columns of a 128-column tile each: four warps per scheduler, in code of 32 elements, hide each other's round trips
// to tensor memory; with two warps of 64 elements 2 x 5000 tokens behind a window with a soft cap took 1100 us instead of 902, 16 x 1025
// of hdim 64 568 instead of 503), warp 16 issues S, warp 17 the other products (a single issuer spends as long on its waits and
// commits as the products take, and the tensor pipe takes instructions only about one ahead: 2 x 4096 causal tokens of 32 / 8
// heads 927 us instead of 789; dP follows the product that has read dS from its columns in one warp's order, without a
// barrier between them), warp 18 finds the work items, hands them to the others through a ring and
// issues the TMA copies, warp 19 requests the next item's O from memory (dQ) or
// fetches LSE and D of the query columns (dK/dV).  D is computed by the elementwise warps of dQ, eight rows each.
//   dQ works by halves h of 64 keys, each with its own barriers: one half's products run under the other's elementwise work.
//   dK/dV: two 128-column regions change roles from step to step: P(i) and dS(i) lie in the region that S(i) came in, so that S(i+1)
//   can take the other one as soon as dP(i) has been read from it.
// Every mbarrier wait is bounded; on expiry the CTA records a code in the device status word and drains.
#pragma once
#include "fmha_fwd_sm100.cuh"

namespace fck {

namespace sm100 {

struct BwdSm100Dev {
    const void* dout;
    const void* q;
    const void* o;
    const float* lse;
    const float* dlse;
    float* delta;
    void* dq;
    void* dk;
    void* dv;
    const int64_t* seqstart_q;
    const int64_t* seqstart_k;
    int* status;
    int batch, seqlen_q, seqlen_k, hq, hkv;
    int mask_type, wl, wr;
    float scale, scale_log2;
    const float* alibi;
    int alibi_rank;
    float soft_cap, inv_cap_log2;  // the soft cap c (0: off), 1 / (c log2(e))
    SoftCap cap;                   // constants of soft_cap_scores
    const void* bias;              // VAR 2: an elementwise bias, planes of bias_sq x bias_sk (group mode: the packed totals)
    void* dbias;
    int bias_rank;                 // 0 one plane, 1 one per head, 2 one per (batch, head)
    int64_t bias_sq, bias_sk;
    int listed;                    // a persistent grid finds the items, 1: in order of cost, 2: sequence after sequence; 0: one per CTA, by its index
    int max_tiles;                 // tiles of the longest sequence
};

struct BwdSeq {
    int q0, k0, sq, sk, shift;
};
__device__ __forceinline__ BwdSeq bwd_sequence(const BwdSm100Dev& p, int b) {
    BwdSeq s;
    const int64_t q0 = p.seqstart_q ? p.seqstart_q[b] : (int64_t)b * p.seqlen_q, k0 = p.seqstart_k ? p.seqstart_k[b] : (int64_t)b * p.seqlen_k;
    s.q0 = (int)q0;  // (rows fit 31 bits: checked on the host)
    s.k0 = (int)k0;
    s.sq = p.seqstart_q ? (int)max((int64_t)0, p.seqstart_q[b + 1] - q0) : p.seqlen_q;
    s.sk = p.seqstart_k ? (int)max((int64_t)0, p.seqstart_k[b + 1] - k0) : p.seqlen_k;
    s.shift = p.mask_type == 2 ? s.sk - s.sq : 0;
    return s;
}
// A row without keys (LSE -inf) gets +inf here: P = exp2(S - inf) = 0.
__device__ __forceinline__ float bwd_lse_base2(float lse) { return lse == -INFINITY ? INFINITY : lse * kLog2e; }

// D (+)= A B^T over `HDIM` columns, both operands K-major tiles of 128 rows in shared memory.
template <int HDIM>
__device__ __forceinline__ void bwd_issue_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
#pragma unroll
    for (int ks = 0; ks < HDIM / 16; ++ks) {
        const uint64_t off = (uint64_t)(((ks / 4) * HALF_BYTES + (ks % 4) * 32) >> 4);
        umma_ss(d, a + off, b + off, idesc, ks > 0 ? 1u : 0u);
    }
}
// The same with A in tensor memory (two elements a column).
template <int HDIM>
__device__ __forceinline__ void bwd_issue_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
#pragma unroll
    for (int ks = 0; ks < HDIM / 16; ++ks)
        umma_ts(d, a + ks * 8, b + (uint64_t)(((ks / 4) * HALF_BYTES + (ks % 4) * 32) >> 4), idesc, ks > 0 ? 1u : 0u);
}
// D += X B over 64 of 128 rows (half 0 / 1): X in tensor memory, every 32 rows 16 columns in steps of 32; B MN-major.
__device__ __forceinline__ void bwd_issue_xb(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, int half, bool accumulate) {
#pragma unroll
    for (int ks = half * 4; ks < half * 4 + 4; ++ks)
        umma_ts(d, a + (ks / 2) * 32 + (ks % 2) * 8, b + (uint64_t)((ks * 2048) >> 4), idesc, (accumulate || ks > half * 4) ? 1u : 0u);
}

// 2^x on the FMA pipe for two values: x = n + f, f in [-0.5, 0.5], 2^f by the polynomial of degree 4 of least relative error
// (2.7e-6 with its fp32 rounding), times 2^n put together from its bits.  x above -126 (2^-126 stands for everything below).  A NaN
// stays one: the maximum hands it on, and a product with it is NaN whatever the bits of n have become (added to the exponent,
// n would turn it into the largest finite number).
__device__ __forceinline__ float bwd_max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 bwd_exp2_poly(float2 x) {
    x.x = bwd_max_nan(x.x, -126.f);
    x.y = bwd_max_nan(x.y, -126.f);
    const float2 t = __fadd2_rn(x, make_float2(12582912.f, 12582912.f));  // 1.5 * 2^23: n lands in the low mantissa bits
    const float2 f = __fadd2_rn(x, __fadd2_rn(make_float2(12582912.f, 12582912.f), make_float2(-t.x, -t.y)));
    float2 q = __ffma2_rn(make_float2(0.009570076f, 0.009570076f), f, make_float2(0.05591789f, 0.05591789f));
    q = __ffma2_rn(q, f, make_float2(0.24024746f, 0.24024746f));
    q = __ffma2_rn(q, f, make_float2(0.6931218f, 0.6931218f));
    q = __ffma2_rn(q, f, make_float2(0.9999993f, 0.9999993f));
    return __fmul2_rn(q, make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3f800000), __int_as_float((__float_as_int(t.y) << 23) + 0x3f800000)));
}
// The exponentials of a pair: pairs `i` of every 8 below POLY go to the FMA pipe, the others to the exp2 unit, which alone would
// take 1024 clocks per 128 x 128 tile.  Shares of 8 measured (dQ, dK/dV; us of 2 x 4096 causal tokens of 32 / 8 heads, and of 37k ragged
// ones): (0, 3) 780, 2512; (1, 3) 773, 2489; (1, 4) 774, 2502; (2, 2) 780, 2525 (before the product that keeps a
// NaN, with which the packed ones take 1 % more).  None with a bias tensor: its -inf must give a P of 0.
constexpr int kPolyDq = 1, kPolyDkdv = 3;
template <int POLY>
__device__ __forceinline__ float2 bwd_exp2(float2 y, int i) {
    return (i & 7) < POLY ? bwd_exp2_poly(y) : make_float2(ex2_fast(y.x), ex2_fast(y.y));
}

// Score additions (template parameter VAR of the kernels): 0 none, 1 ALiBi and / or a soft cap, 2 a bias tensor and / or a soft cap.
// Base-2 exponent of a pair of scores (raw, or behind a soft cap what soft_cap_scores left of them), LSE subtracted; with a soft
// cap f is what dS gets from it, 1 - tanh^2.  `add`: distances from the diagonal, or bias values.
template <int VAR>
__device__ __forceinline__ float2 bwd_exponent(const BwdSm100Dev& p, float2 x, float slope_log2, float2 add, float2 neg_lse2, float2& f) {
    if constexpr (VAR == 0) return __ffma2_rn(x, make_float2(p.scale_log2, p.scale_log2), neg_lse2);
    float2 y = x;
    if (p.soft_cap > 0.f) {
        const float2 t = __fmul2_rn(x, make_float2(p.inv_cap_log2, p.inv_cap_log2));
        f = __ffma2_rn(make_float2(-t.x, -t.y), t, make_float2(1.f, 1.f));
    } else {
        y = __fmul2_rn(x, make_float2(p.scale_log2, p.scale_log2));
    }
    if constexpr (VAR == 2) y = __ffma2_rn(make_float2(kLog2e, kLog2e), add, y);
    else y = __ffma2_rn(make_float2(-slope_log2, -slope_log2), make_float2(fabsf(add.x), fabsf(add.y)), y);
    return __fadd2_rn(y, neg_lse2);
}
// Element (0, 0) of the bias block of a (sequence, head).
__device__ __forceinline__ int64_t bwd_bias_block(const BwdSm100Dev& p, int b, int h, int64_t q0, int64_t k0) {
    const int64_t plane = p.bias_sq * p.bias_sk;
    return (p.bias_rank >= 1 ? (int64_t)h * plane : 0) + (p.bias_rank == 2 ? (int64_t)b * p.hq * plane : 0) +
           (p.seqstart_q ? q0 * p.bias_sk + k0 : 0);
}

// A row of P 16-byte pieces per lane, P = 2, 4 or 8, to P lanes per row: lane l of a group of P lanes gets piece l of the rows of all
// its group's lanes.  A row's pieces straight from its lane touch 32 lines per store instruction, and the elementwise warps
// stood in the queue for them (4000 clocks per 128 x 128 tile); after the exchange an instruction writes whole lines.
template <int P>
__device__ __forceinline__ void bwd_exchange(uint4 (&x)[P], int lane) {
#pragma unroll
    for (int s = 1; s < P; s *= 2) {
        const bool up = lane & s;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            if (i & s) continue;
            uint4 a = up ? x[i] : x[i | s];
            a.x = __shfl_xor_sync(0xffffffffu, a.x, s);
            a.y = __shfl_xor_sync(0xffffffffu, a.y, s);
            a.z = __shfl_xor_sync(0xffffffffu, a.z, s);
            a.w = __shfl_xor_sync(0xffffffffu, a.w, s);
            if (up) x[i] = a;
            else x[i | s] = a;
        }
    }
}
// COLS fp32 accumulator columns from tensor memory, times f, packed to the element type, as the lane's row.
template <typename T, int COLS>
__device__ __forceinline__ void bwd_load_rows(uint32_t src, float f, uint4 (&x)[COLS / 8]) {
    constexpr int STEP = COLS < 32 ? COLS : 32;
#pragma unroll
    for (int c = 0; c < COLS; c += STEP) {
        uint32_t t[STEP];
        if constexpr (STEP == 32) tmem_ld32(src + c, t);
        else tmem_ld16(src + c, t);
        tmem_wait_ld();
#pragma unroll
        for (int v = 0; v < STEP / 8; ++v) {
            uint4& w = x[c / 8 + v];
            w.x = Elem<T>::pack2(__uint_as_float(t[8 * v]) * f, __uint_as_float(t[8 * v + 1]) * f);
            w.y = Elem<T>::pack2(__uint_as_float(t[8 * v + 2]) * f, __uint_as_float(t[8 * v + 3]) * f);
            w.z = Elem<T>::pack2(__uint_as_float(t[8 * v + 4]) * f, __uint_as_float(t[8 * v + 5]) * f);
            w.w = Elem<T>::pack2(__uint_as_float(t[8 * v + 6]) * f, __uint_as_float(t[8 * v + 7]) * f);
        }
    }
}
// The lanes' rows to a gradient tensor: dst is where the first of the 32 rows starts, `rows` of them exist.  Warp-collective.
template <typename T, int P>
__device__ __forceinline__ void bwd_store_rows(T* dst, int64_t row_stride, int rows, uint4 (&x)[P], int lane) {
    bwd_exchange<P>(x, lane);
    const int row0 = lane & ~(P - 1), piece = lane & (P - 1);
#pragma unroll
    for (int j = 0; j < P; ++j)
        if (row0 + j < rows) *reinterpret_cast<uint4*>(dst + (row0 + j) * row_stride + piece * 8) = x[j];
}
// Columns lo .. hi of 32 (either may lie outside) as bits.
__device__ __forceinline__ uint32_t bwd_column_bits(int lo, int hi) {
    const uint32_t upto = hi < 0 ? 0u : hi >= 31 ? 0xffffffffu : 0xffffffffu >> (31 - hi);
    return lo <= 0 ? upto : lo > 31 ? 0u : upto & (0xffffffffu << lo);
}
// Zeros to the hidden ones of 32 packed elements (whatever they hold: it may be a NaN).
__device__ __forceinline__ void bwd_hide(uint32_t (&w)[16], uint32_t bits) {
#pragma unroll
    for (int e = 0; e < 16; ++e) w[e] &= (bits >> (2 * e) & 1u ? 0xffffu : 0u) | (bits >> (2 * e + 1) & 1u ? 0xffff0000u : 0u);
}
// 128 rows of a K-major tile in shared memory to tensor memory as an A operand: 8 columns (16 elements a row) per instruction.
template <int HDIM>
__device__ __forceinline__ void bwd_copy_to_tmem(uint32_t d, uint64_t src) {
#pragma unroll
    for (int ks = 0; ks < HDIM / 16; ++ks)
        asm volatile("tcgen05.cp.cta_group::1.128x256b [%0], %1;\n" ::"r"(d + ks * 8), "l"(src + (uint64_t)(((ks / 4) * HALF_BYTES + (ks % 4) * 32) >> 4))
                     : "memory");
}

// One tile by TMA (64-column boxes of 128 rows).  Where the sequence ends inside it, the rows behind the end are set to zero before
// the tile is handed over: they belong to another sequence, and 0 times a NaN of it would not be 0.  Warp-collective.
template <int HDIM>
__device__ __forceinline__ bool bwd_load_tile(uint8_t* dst, const CUtensorMap* map, uint64_t* full, uint64_t* tail, uint32_t& tails, int head,
                                              int row, int valid, int lane, volatile int* abort_flag, int* status) {
    uint64_t* bar = valid < 128 ? tail : full;
    if (lane == 0) {
        mbar_expect_tx(bar, 128 * HDIM * 2);
#pragma unroll
        for (int hb = 0; hb < HDIM / 64; ++hb) tma_load_3d(dst + hb * HALF_BYTES, map, bar, hb * 64, head, row);
    }
    if (valid >= 128) return true;
    __syncwarp();
    const bool ok = __all_sync(0xffffffffu, mbar_wait_bounded(tail, tails++ & 1u, abort_flag, status, 0x10000));
    if (!ok) return false;
    for (int e = valid * 8 + lane; e < 128 * 8; e += 32)
#pragma unroll
        for (int hb = 0; hb < HDIM / 64; ++hb) reinterpret_cast<uint4*>(dst + hb * HALF_BYTES)[e] = make_uint4(0u, 0u, 0u, 0u);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(full);
    return true;
}

// A work item as the scheduling warp hands it out; row0: first row of the tile inside the sequence.
struct alignas(16) BwdItem {
    int valid, b, h, row0, q0, k0, sq, sk;
};
constexpr int kBwdItemRing = 4, kBwdMaxBatch = 256;

struct BwdCtrl {
    BwdItem items[kBwdItemRing];
    uint64_t item_full[kBwdItemRing], item_empty[kBwdItemRing];
    uint64_t a_full[3], a_empty[3], b_full[2], b_empty[2];  // rings: dQ K / V; dK/dV Q / dO
    uint64_t own_full[2], own_free[2];  // what an item owns: dK/dV the K / V tile; dQ: Q / dO on their way to tensor memory
    uint64_t s_full[2], s_free[2], dp_full[2], ds_full[2];  // dQ: by half; dK/dV: [0] (s_free[0]: dP has been read)
    uint64_t p_full[2];         // dK/dV, by step: the elementwise warps can be one step ahead of the products that read P
    uint64_t acc_full, acc_free, tail;
    uint64_t row_full[2], row_empty[2];
    uint32_t tmem_base;
    int abort_flag;
};

// The schedule, kept by the warp that issues the copies.  Items of a level cost the same under a causal mask: level l is the row tile
// l of dQ (the last tiles see the most keys), the tile l places in front of the last one of dK/dV (the first tiles are seen by
// the most queries).  Levels come in decreasing order, a level's sequences in order, their heads side by side (they share tiles
// through L2); rounds of the grid take the items in alternate directions.  Tile counts are held eight sequences a lane.  More sequences
// than that come in their own order, 32 at a time, the tiles of a sequence one after the other: the tiles that exist, not those that
// the longest sequence would have.
template <bool DQ>
struct BwdSchedule {
    int cnt[kBwdMaxBatch / 32], level, round;  // (listed 2: cnt[0] is sequence level + lane's)
    int64_t base;  // first item of the level (listed 2: of the 32 sequences)
    uint32_t k;    // items handed out

    __device__ __forceinline__ int tiles_of(const BwdSm100Dev& p, int b) {
        if (b >= p.batch) return 0;
        const BwdSeq s = bwd_sequence(p, b);
        return min(((DQ ? s.sq : s.sk) + 127) / 128, p.max_tiles);
    }

    __device__ __forceinline__ void init(const BwdSm100Dev& p, int lane) {
        k = 0;
        round = 0;
        base = 0;
        level = -1;
        if (!p.listed) return;
        if (p.listed == 2) {
            level = 0;
            cnt[0] = tiles_of(p, lane);
            return;
        }
        int most = 0;
#pragma unroll
        for (int u = 0; u < kBwdMaxBatch / 32; ++u) {
            cnt[u] = tiles_of(p, u * 32 + lane);
            most = max(most, cnt[u]);
        }
        level = (int)__reduce_max_sync(0xffffffffu, (unsigned)most) - 1;
    }
    // The next item, handed to the other warps as well; false: there is none (said to the others), or a wait ran out.
    __device__ __forceinline__ bool next(BwdCtrl* ctrl, const BwdSm100Dev& p, int lane, BwdItem& it) {
        const int heads = DQ ? p.hq : p.hkv;
        it = BwdItem{};
        if (!p.listed) {  // one item per CTA, by its index
            if (round++ == 0) {
                const int per_tile = heads * p.batch, t = (int)blockIdx.x / per_tile, rest = (int)blockIdx.x - t * per_tile;
                it.b = rest / heads;
                it.h = rest - it.b * heads;
                it.row0 = (DQ ? (int)gridDim.x / per_tile - 1 - t : t) * 128;
                it.valid = 1;
            }
        } else if (p.listed == 2) {
            const int64_t w = (int64_t)round * gridDim.x + blockIdx.x;
            ++round;
            int total;
            while (true) {
                total = __reduce_add_sync(0xffffffffu, cnt[0]);
                if (w < base + (int64_t)total * heads || level + 32 >= p.batch) break;
                base += (int64_t)total * heads;
                level += 32;
                cnt[0] = tiles_of(p, level + lane);
            }
            if (w < base + (int64_t)total * heads) {
                const int at = (int)((w - base) / heads);  // tile of the 32 sequences
                int end = cnt[0];                          // tiles up to and with the lane's
#pragma unroll
                for (int off = 1; off < 32; off *= 2) {
                    const int before = __shfl_up_sync(0xffffffffu, end, off);
                    if (lane >= off) end += before;
                }
                const int l = __ffs(__ballot_sync(0xffffffffu, end > at)) - 1;
                it.b = level + l;
                it.h = (int)(w - base) - at * heads;
                it.row0 = (at - __shfl_sync(0xffffffffu, end - cnt[0], l)) * 128;
                it.valid = 1;
            }
        } else {
            const int64_t w = (int64_t)round * gridDim.x + ((round & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
            ++round;
            for (; level >= 0; --level) {
                int n = 0;
#pragma unroll
                for (int u = 0; u < kBwdMaxBatch / 32; ++u) n += __popc(__ballot_sync(0xffffffffu, cnt[u] > level));
                if (w < base + (int64_t)n * heads) break;
                base += (int64_t)n * heads;
            }
            if (level >= 0) {
                int rank = (int)((w - base) / heads), tiles = 0;
                it.h = (int)(w - base) - rank * heads;
#pragma unroll
                for (int u = 0; u < kBwdMaxBatch / 32; ++u) {
                    const uint32_t m = __ballot_sync(0xffffffffu, cnt[u] > level);
                    const int c = __popc(m);
                    if (!it.valid && rank < c) {
                        const int l = __fns(m, 0, rank + 1);
                        it.b = u * 32 + l;
                        tiles = __shfl_sync(0xffffffffu, cnt[u], l);
                        it.valid = 1;
                    }
                    rank -= c;
                }
                it.row0 = (DQ ? level : tiles - 1 - level) * 128;
            }
        }
        if (it.valid) {
            const BwdSeq s = bwd_sequence(p, it.b);
            it.q0 = s.q0; it.k0 = s.k0; it.sq = s.sq; it.sk = s.sk;
            it.valid = it.row0 < (DQ ? s.sq : s.sk);
        }
        const int slot = k % kBwdItemRing;
        if (!__all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->item_empty[slot], ((k / kBwdItemRing) & 1u) ^ 1u, &ctrl->abort_flag, p.status, 0x10001))) return false;
        ++k;
        if (lane == 0) {
            ctrl->items[slot] = it;
            mbar_arrive(&ctrl->item_full[slot]);
        }
        __syncwarp();
        return it.valid != 0;
    }
};
// The next item of a consumer warp (false: no more, or a wait ran out).
__device__ __forceinline__ bool bwd_next_item(BwdCtrl* ctrl, const BwdSm100Dev& p, uint32_t& k, int lane, BwdItem& it) {
    const int slot = k % kBwdItemRing;
    if (!__all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->item_full[slot], (k / kBwdItemRing) & 1u, &ctrl->abort_flag, p.status, 0x10002))) return false;
    ++k;
    it = ctrl->items[slot];
    __syncwarp();
    if (lane == 0) mbar_arrive(&ctrl->item_empty[slot]);
    return it.valid != 0;
}
// Tiles of the other side that an item visits: [begin, begin + count)
struct BwdRange {
    int begin, count;
};
__device__ __forceinline__ BwdRange bwd_key_tiles(const BwdSm100Dev& p, const BwdItem& it) {
    int lo = 0, hi = it.sk - 1;
    const int shift = p.mask_type == 2 ? it.sk - it.sq : 0;
    if (p.mask_type != 0) {
        if (p.wl >= 0) lo = max(lo, it.row0 + shift - p.wl);
        if (p.wr >= 0) hi = min(hi, min(it.sq, it.row0 + 128) - 1 + shift + p.wr);
    }
    return hi >= lo ? BwdRange{lo / 128, hi / 128 + 1 - lo / 128} : BwdRange{0, 0};
}
__device__ __forceinline__ BwdRange bwd_query_tiles(const BwdSm100Dev& p, const BwdItem& it) {  // i + shift - wl <= j <= i + shift + wr
    int lo = 0, hi = it.sq - 1;
    const int shift = p.mask_type == 2 ? it.sk - it.sq : 0;
    if (p.mask_type != 0) {
        if (p.wr >= 0) lo = max(lo, it.row0 - shift - p.wr);
        if (p.wl >= 0) hi = min(hi, min(it.sk, it.row0 + 128) - 1 - shift + p.wl);
    }
    return hi >= lo ? BwdRange{lo / 128, hi / 128 + 1 - lo / 128} : BwdRange{0, 0};
}

// Rows that belong to no sequence (in front of the first, behind the last one) get zero gradients, a share per CTA.
template <int HDIM>
__device__ __forceinline__ void bwd_zero_outside(const BwdSm100Dev& p) {
    if (!p.seqstart_q) return;
    const int64_t tid = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, threads = (int64_t)gridDim.x * blockDim.x;
    auto zero = [&](void* t, int64_t from, int64_t to, int heads) {
        const int64_t per_row = (int64_t)heads * HDIM / 8;
        for (int64_t e = from * per_row + tid; e < to * per_row; e += threads) reinterpret_cast<uint4*>(t)[e] = make_uint4(0u, 0u, 0u, 0u);
    };
    auto clip = [](int64_t x, int64_t n) { return x < 0 ? (int64_t)0 : x > n ? n : x; };
    const int64_t q0 = clip(p.seqstart_q[0], p.seqlen_q), q1 = clip(p.seqstart_q[p.batch], p.seqlen_q);
    const int64_t k0 = clip(p.seqstart_k[0], p.seqlen_k), k1 = clip(p.seqstart_k[p.batch], p.seqlen_k);
    zero(p.dq, 0, q0, p.hq);
    zero(p.dq, q1, p.seqlen_q, p.hq);
    zero(p.dk, 0, k0, p.hkv);
    zero(p.dk, k1, p.seqlen_k, p.hkv);
    zero(p.dv, 0, k0, p.hkv);
    zero(p.dv, k1, p.seqlen_k, p.hkv);
}


constexpr int kBwdThreads = 640, kBwdConsumers = 19;  // (consumers of the item ring: every warp but the one that fills it)

// 2 x 4096 causal tokens of 32 / 8 heads of 128: 322 us, 1280 TFLOP/s of its three products, the tensor pipe busy 66 % of the time, at 1700
// clocks a step beside the 1536 of the products and 8-9k clocks between two items (code that runs once an item comes from memory
// again each time).
// ---- dQ -----------------------------------------------------------------------------------------------------------------
template <typename T, int HDIM, int VAR>
__global__ void __launch_bounds__(kBwdThreads, 1)
bwd_dq_sm100_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                    const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do, const BwdSm100Dev p) {
    constexpr int TILE = 128 * HDIM * 2, KS = 3, VS = 2;
    constexpr uint32_t cS = 0, cDP = 128, cDQ = 256, cQ = 384, cDO = 448;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* sK = smem_raw;  // (no room for slack: that it starts on a 1024-byte boundary is checked below)
    uint8_t* sV = sK + KS * TILE;
    uint8_t* sQ = sV + VS * TILE;                            // Q and dO of the next item on their way to tensor memory
    uint8_t* sDO = sQ + TILE;
    float* sDelta = reinterpret_cast<float*>(sDO + TILE);    // [2 items][128 rows]
    BwdCtrl* ctrl = reinterpret_cast<BwdCtrl*>(sDelta + 256);
    volatile int* abort_flag = &ctrl->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if ((smem_u32(smem_raw) & 1023u) != 0) {
        if (threadIdx.x == 0) atomicOr(p.status, 0x10100);
        pdl_wait();
        return;
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < kBwdItemRing; ++i) {
            mbar_init(&ctrl->item_full[i], 1);
            mbar_init(&ctrl->item_empty[i], kBwdConsumers);
        }
        for (int i = 0; i < KS; ++i) { mbar_init(&ctrl->a_full[i], 1); mbar_init(&ctrl->a_empty[i], 1); }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&ctrl->b_full[i], 1);
            mbar_init(&ctrl->b_empty[i], 1);
            mbar_init(&ctrl->s_full[i], 1);
            mbar_init(&ctrl->s_free[i], 8);
            mbar_init(&ctrl->dp_full[i], 1);
            mbar_init(&ctrl->ds_full[i], 8);
            mbar_init(&ctrl->row_full[i], 16);
        }
        mbar_init(&ctrl->own_full[0], 1);
        mbar_init(&ctrl->own_full[1], 1);
        mbar_init(&ctrl->own_free[0], 1);
        mbar_init(&ctrl->own_free[1], 17);  // copied to tensor memory, and read for D by the elementwise warps
        mbar_init(&ctrl->acc_full, 1);
        mbar_init(&ctrl->acc_free, 16);
        mbar_init(&ctrl->tail, 1);
        ctrl->abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_u32(&ctrl->tmem_base)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    }
    pdl_wait();
    pdl_launch_dependents();
    bwd_zero_outside<HDIM>(p);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctrl->tmem_base;
    uint32_t k_item = 0;
    BwdItem it{};

    // Registers: launched with 640 x 96 = 512 x 104 + 128 x 64.
    if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;\n" ::);
        if (warp == 18) {
            // ================================ items and TMA copies ================================
            BwdSchedule<true> schedule;
            schedule.init(p, lane);
            uint32_t tails = 0, t = 0, n_own = 0;
            bool ok = true;
            auto load_own = [&](const BwdItem& item) {  // (rows behind the end of the queries stay in their own rows of dQ, which are not stored)
                for (int i = 0; ok && i < 2; ++i)
                    ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->own_free[i], (n_own & 1u) ^ 1u, abort_flag, p.status, 0x10022)) &&
                         bwd_load_tile<HDIM>(i ? sDO : sQ, i ? &map_do : &map_q, &ctrl->own_full[i], &ctrl->tail, tails, item.h, item.q0 + item.row0,
                                             128, lane, abort_flag, p.status);
                ++n_own;
            };
            // An item is handed out, and its Q and dO are fetched, while the copies of the one before it are still to come: its D is
            // then there in time.
            BwdItem ahead{};
            bool more = schedule.next(ctrl, p, lane, ahead);
            if (more && bwd_key_tiles(p, ahead).count > 0) load_own(ahead);
            while (ok && more) {
                it = ahead;
                more = schedule.next(ctrl, p, lane, ahead);
                const bool fetch = more && bwd_key_tiles(p, ahead).count > 0;
                const BwdRange range = bwd_key_tiles(p, it);
                const int kh = it.h / (p.hq / p.hkv);
                for (int j = 0; j < range.count; ++j, ++t) {
                    const int n0 = (range.begin + j) * 128, ks = t % KS, vs = t % VS;
                    if (!(ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->a_empty[ks], ((t / KS) & 1u) ^ 1u, abort_flag, p.status, 0x10020)))) break;
                    // (K rows behind the end meet dS = 0; those of V only make columns of dP that are masked by index)
                    if (!(ok = bwd_load_tile<HDIM>(sK + ks * TILE, &map_k, &ctrl->a_full[ks], &ctrl->tail, tails, kh, it.k0 + n0, it.sk - n0, lane,
                                                   abort_flag, p.status))) break;
                    if (!(ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->b_empty[vs], ((t / VS) & 1u) ^ 1u, abort_flag, p.status, 0x10021)))) break;
                    bwd_load_tile<HDIM>(sV + vs * TILE, &map_v, &ctrl->b_full[vs], &ctrl->tail, tails, kh, it.k0 + n0, 128, lane, abort_flag, p.status);
                    if (fetch && j == min(KS, range.count) - 1) load_own(ahead);
                    if (!ok) break;
                }
                if (ok && fetch && range.count == 0) load_own(ahead);
            }
        } else if (warp == 19) {
            // ================================ O of the coming item on its way to L2 ================================
            while (bwd_next_item(ctrl, p, k_item, lane, it)) {
                for (int r = lane; r < min(128, it.sq - it.row0); r += 32) {
                    const T* row = (const T*)p.o + ((int64_t)(it.q0 + it.row0 + r) * p.hq + it.h) * HDIM;
#pragma unroll
                    for (int c = 0; c < HDIM; c += 64) asm volatile("prefetch.global.L2 [%0];\n" ::"l"(row + c));
                }
            }
        } else {
            // ================================ MMA issuers: 16 S, 17 dP and dQ ================================
            // All lanes walk the loop, the elected one issues.
            const bool leader = elect_one_sync();
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
                return ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag, p.status, code)) != 0;
            };
            auto commit = [&](uint64_t* bar) { if (leader) umma_commit(bar); };
            auto at = [&](uint64_t d, uint32_t bytes) { return d + (uint64_t)(bytes >> 4); };
            constexpr uint32_t idesc_s = make_idesc<T>(false, 64), idesc_q = make_idesc<T>(true, HDIM);
            const uint64_t dK = make_smem_desc(smem_u32(sK), 0, 1024), dV = make_smem_desc(smem_u32(sV), 0, 1024);
            const uint64_t dKt = make_smem_desc(smem_u32(sK), HALF_BYTES, 1024);
            const uint64_t dQ = make_smem_desc(smem_u32(sQ), 0, 1024), dDO = make_smem_desc(smem_u32(sDO), 0, 1024);
            uint32_t t = 0, ks = 0, kph = 0, n_item = 0;  // steps so far, K slot and its phase, items with steps so far
            if (warp == 16) {
                while (ok && bwd_next_item(ctrl, p, k_item, lane, it)) {
                    const int N = bwd_key_tiles(p, it).count;
                    if (N > 0) {  // Q, over the last item's, whose last S is complete
                        if (!wait(&ctrl->own_full[0], n_item++ & 1u, 0x10030)) break;
                        if (t > 0 && !wait(&ctrl->s_full[1], (t - 1) & 1u, 0x10038)) break;
                        tc_fence_after();
                        if (leader) bwd_copy_to_tmem<HDIM>(tmem + cQ, dQ);
                        commit(&ctrl->own_free[0]);
                    }
                    for (int j = 0; j < N; ++j) {
                        if (!wait(&ctrl->a_full[ks], kph, 0x10031)) break;
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            if (t > 0 && !wait(&ctrl->s_free[half], (t - 1) & 1u, 0x10032)) break;
                            tc_fence_after();
                            if (leader) bwd_issue_ts<HDIM>(tmem + cS + half * 64, tmem + cQ, at(dK, ks * TILE + half * 8192), idesc_s);
                            commit(&ctrl->s_full[half]);
                        }
                        if (!ok) break;
                        ++t;
                        if (++ks == KS) { ks = 0; kph ^= 1u; }
                    }
                }
            } else {
                auto issue_dp = [&](uint32_t st, int half) -> bool {
                    const uint32_t vs = st & 1u;
                    if (half == 0 && !wait(&ctrl->b_full[vs], (st >> 1) & 1u, 0x10034)) return false;
                    tc_fence_after();
                    if (leader) bwd_issue_ts<HDIM>(tmem + cDP + half * 64, tmem + cDO, at(dV, vs * TILE + half * 8192), idesc_s);
                    commit(&ctrl->dp_full[half]);
                    if (half == 1) commit(&ctrl->b_empty[vs]);
                    return true;
                };
                while (ok && bwd_next_item(ctrl, p, k_item, lane, it)) {
                    const int N = bwd_key_tiles(p, it).count;
                    if (N == 0) continue;
                    // dO, over the last item's, whose last dP has been read
                    if (!wait(&ctrl->own_full[1], n_item & 1u, 0x10033)) break;
                    tc_fence_after();
                    if (leader) bwd_copy_to_tmem<HDIM>(tmem + cDO, dDO);
                    commit(&ctrl->own_free[1]);
                    if (!issue_dp(t, 0) || !issue_dp(t, 1)) break;
                    if (n_item > 0 && !wait(&ctrl->acc_free, (n_item - 1) & 1u, 0x10036)) break;
                    for (int j = 0; j < N; ++j) {
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            if (!wait(&ctrl->ds_full[half], t & 1u, 0x10037)) break;
                            tc_fence_after();
                            if (leader) bwd_issue_xb(tmem + cDQ, tmem + cDP, at(dKt, ks * TILE), idesc_q, half, j + half > 0);
                            if (half == 1) commit(&ctrl->a_empty[ks]);
                            if (j + 1 < N && !issue_dp(t + 1, half)) break;
                        }
                        if (!ok) break;
                        ++t;
                        if (++ks == KS) ks = 0;
                    }
                    if (!ok) break;
                    commit(&ctrl->acc_full);
                    ++n_item;
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 104;\n" ::);
        const int quarter = warp >> 2, half = quarter >> 1, r = (warp & 3) * 32 + lane;
        const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t tS = lane_addr + cS + quarter * 32, tDP = lane_addr + cDP + quarter * 32;
        uint32_t t = 0, n_item = 0;
        bool ok = true;
        constexpr int COLS = HDIM / 4;                                        // of dQ that a warp stores
        constexpr int L = HDIM / 8, ROWS = 32 / L, LOADS = 8 / ROWS;          // D: lanes a row, rows a load
        const int sub = lane / L, piece = lane % L;
        // What an item's D needs from memory: O of rows warp * 8 .. + 7 (8 columns a lane), the row's LSE.  It is requested in front of the
        // stores of the item before.
        uint4 y[LOADS];
        float lse2;
        auto request = [&]() {
            const int left = it.sq - it.row0;
            const T* at = (const T*)p.o + ((int64_t)(it.q0 + it.row0) * p.hq + it.h) * HDIM + piece * 8;
#pragma unroll
            for (int u = 0; u < LOADS; ++u) {
                const int row = warp * 8 + u * ROWS + sub;
                y[u] = row < left ? *reinterpret_cast<const uint4*>(at + row * ((int64_t)p.hq * HDIM)) : make_uint4(0u, 0u, 0u, 0u);
            }
            const int64_t lr = (p.seqstart_q ? (int64_t)it.h * p.seqlen_q + it.q0 : ((int64_t)it.b * p.hq + it.h) * p.seqlen_q) + it.row0;
            lse2 = r < left ? bwd_lse_base2(p.lse[lr + r]) : INFINITY;
        };
        bool more = bwd_next_item(ctrl, p, k_item, lane, it);
        if (more) request();
        while (ok && more) {
            const int i = it.row0 + r, shift = p.mask_type == 2 ? it.sk - it.sq : 0;
            const int rows = it.sq - it.row0 - (warp & 3) * 32;  // of this warp's 32 that exist
            const BwdRange range = bwd_key_tiles(p, it);
            T* dst = (T*)p.dq + ((int64_t)(it.q0 + it.row0 + (warp & 3) * 32) * p.hq + it.h) * HDIM + quarter * COLS;
            // D = sum dO O - dLSE, dO from its tile (or from memory, where the item has no products)
            const int slot = n_item & 1, left = it.sq - it.row0;
            {
                const int64_t lr = (p.seqstart_q ? (int64_t)it.h * p.seqlen_q + it.q0 : ((int64_t)it.b * p.hq + it.h) * p.seqlen_q) + it.row0;
                if (range.count > 0 && !(ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->own_full[1], n_item & 1u, abort_flag, p.status, 0x10040)))) break;
#pragma unroll
                for (int u = 0; u < LOADS; ++u) {
                    const int row = warp * 8 + u * ROWS + sub;
                    uint4 x = make_uint4(0u, 0u, 0u, 0u);
                    if (range.count > 0) x = *reinterpret_cast<const uint4*>(sDO + (piece / 8) * HALF_BYTES + row * 128 + (((piece & 7) ^ (row & 7)) << 4));
                    else if (row < left) x = *reinterpret_cast<const uint4*>((const T*)p.dout + ((int64_t)(it.q0 + it.row0 + row) * p.hq + it.h) * HDIM + piece * 8);
                    const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y[u].x, y[u].y, y[u].z, y[u].w};
                    float sum = 0.f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 a = bias_pair<T>(xw[e]), o2 = bias_pair<T>(yw[e]);
                        sum = fmaf(a.x, o2.x, fmaf(a.y, o2.y, sum));
                    }
#pragma unroll
                    for (int off = L / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
                    if (piece == 0) {
                        if (row < left) {
                            if (p.dlse) sum -= p.dlse[lr + row];
                            p.delta[lr + row] = sum;
                        }
                        sDelta[slot * 128 + row] = sum;
                    }
                }
            }
            uint4 out[COLS / 8];
            if (range.count == 0) {  // no row of the tile sees a key
#pragma unroll
                for (int v = 0; v < COLS / 8; ++v) out[v] = make_uint4(0u, 0u, 0u, 0u);
                bwd_store_rows<T>(dst, (int64_t)p.hq * HDIM, rows, out, lane);
                more = bwd_next_item(ctrl, p, k_item, lane, it);
                if (more) request();
                continue;
            }
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&ctrl->own_free[1]);
                mbar_arrive(&ctrl->row_full[slot]);
            }
            if (!(ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->row_full[slot], (n_item >> 1) & 1u, abort_flag, p.status, 0x10044)))) break;
            const float delta = sDelta[slot * 128 + r];
            const float slope = VAR == 1 && p.alibi ? p.alibi[(p.alibi_rank ? it.b * p.hq : 0) + it.h] * kLog2e : 0.f;
            // visible keys of this row; key tiles that every row of the tile sees whole
            const int k_lo = p.mask_type != 0 && p.wl >= 0 ? i + shift - p.wl : 0;
            const int k_hi = p.mask_type != 0 && p.wr >= 0 ? min(it.sk - 1, i + shift + p.wr) : it.sk - 1;
            int full_lo = 0, full_hi = it.sk - 1;
            if (p.mask_type != 0) {
                if (p.wl >= 0) full_lo = max(0, min(it.sq, it.row0 + 128) - 1 + shift - p.wl);
                if (p.wr >= 0) full_hi = min(full_hi, it.row0 + shift + p.wr);
            }
            const float2 neg_lse2 = make_float2(-lse2, -lse2), neg_delta = make_float2(-delta, -delta);
            for (int j = 0; j < range.count; ++j, ++t) {
                const int n0 = (range.begin + j) * 128, key0 = n0 + quarter * 32;
                [[maybe_unused]] uint4 bw[VAR == 2 ? 4 : 1];  // the row's 32 bias values, requested before the wait for S
                if constexpr (VAR == 2) {
                    const unsigned short* row = r < left ? (const unsigned short*)p.bias + bwd_bias_block(p, it.b, it.h, it.q0, it.k0) + i * p.bias_sk : nullptr;
#pragma unroll
                    for (int v = 0; v < 4; ++v) bw[v] = load_bias_piece(row, key0 + v * 8, it.sk - key0 - v * 8);
                }
                if (!(ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->s_full[half], t & 1u, abort_flag, p.status, 0x10041)))) break;
                tc_fence_after();
                uint32_t x[32];
                tmem_ld32(tS, x);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctrl->s_free[half]);
                if constexpr (VAR != 0) {
                    if (p.soft_cap > 0.f) soft_cap_scores<32>(x, p.cap);
                }
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    float2 f = make_float2(1.f, 1.f), away = f;
                    if constexpr (VAR == 1) {
                        away.x = (float)(i + it.sk - it.sq - (key0 + e));
                        away.y = away.x - 1.f;
                    } else if constexpr (VAR == 2) {
                        away = bias_pair<T>((&bw[e / 8].x)[e / 2 % 4]);
                    }
                    const float2 y = bwd_exponent<VAR>(p, make_float2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), slope, away, neg_lse2, f);
                    float2 pr = bwd_exp2<VAR == 2 ? 0 : kPolyDq>(y, e / 2);
                    if constexpr (VAR != 0) pr = __fmul2_rn(pr, f);
                    x[e] = __float_as_uint(pr.x);
                    x[e + 1] = __float_as_uint(pr.y);
                }
                if (!(ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->dp_full[half], t & 1u, abort_flag, p.status, 0x10042)))) break;
                tc_fence_after();
                uint32_t dp[32], w[16];
                tmem_ld32(tDP, dp);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    const float2 d = __fadd2_rn(make_float2(__uint_as_float(dp[e]), __uint_as_float(dp[e + 1])), neg_delta);
                    const float2 ds = __fmul2_rn(make_float2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), d);
                    w[e / 2] = Elem<T>::pack2(ds.x, ds.y);
                }
                if (n0 < full_lo || n0 + 127 > full_hi) bwd_hide(w, bwd_column_bits(k_lo - key0, k_hi - key0));
                tmem_st16(tDP, w);  // (over columns of dP that this warp has read)
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctrl->ds_full[half]);
            }
            if (!ok || !(ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->acc_full, n_item & 1u, abort_flag, p.status, 0x10043)))) break;
            ++n_item;
            tc_fence_after();
            bwd_load_rows<T, COLS>(lane_addr + cDQ + quarter * COLS, p.scale, out);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctrl->acc_free);
            more = bwd_next_item(ctrl, p, k_item, lane, it);
            if (more) request();
            bwd_store_rows<T>(dst, (int64_t)p.hq * HDIM, rows, out, lane);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 16) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem));
    }
}

// The same tokens: 422 us, 1300 TFLOP/s of its four products, the tensor pipe busy 70 %.  A step takes 2600 clocks beside the 2048 of
// shared memory and of the products: S(i+1) waits for dP(i) to be read, so the elementwise work of a step (S and dP from tensor
// memory, 32 exponentials and two conversions a thread, P and dS back) lies on the chain.
// ---- dK / dV --------------------------------------------------------------------------------------------------------------
template <typename T, int HDIM, int VAR>
__global__ void __launch_bounds__(kBwdThreads, 1)
bwd_dkdv_sm100_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                      const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const BwdSm100Dev p) {
    constexpr int TILE = 128 * HDIM * 2, QS = 3, OS = 2;
    constexpr uint32_t cDV = 256, cDK = 384;  // columns 0-127 and 128-255: the two regions
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* sK = smem_raw;  // (no room for slack: that it starts on a 1024-byte boundary is checked below)
    uint8_t* sV = sK + TILE;
    uint8_t* sQ = sV + TILE;
    uint8_t* sDO = sQ + QS * TILE;
    float* sRow = reinterpret_cast<float*>(sDO + OS * TILE);  // [2 steps][LSE 128 | D 128] of the query columns, negated
    BwdCtrl* ctrl = reinterpret_cast<BwdCtrl*>(sRow + 512);
    volatile int* abort_flag = &ctrl->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = p.hq / p.hkv;

    // What this kernel reads has been there since before the dQ kernel in front of it began (that one lets it start only after its
    // own wait), but for D: the warp that fetches D waits for that kernel's end, and every other one before it leaves.
    if ((smem_u32(smem_raw) & 1023u) != 0) {
        if (threadIdx.x == 0) atomicOr(p.status, 0x10100);
        pdl_wait();
        return;
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < kBwdItemRing; ++i) {
            mbar_init(&ctrl->item_full[i], 1);
            mbar_init(&ctrl->item_empty[i], kBwdConsumers);
        }
        for (int i = 0; i < QS; ++i) { mbar_init(&ctrl->a_full[i], 1); mbar_init(&ctrl->a_empty[i], 1); }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&ctrl->b_full[i], 1);
            mbar_init(&ctrl->b_empty[i], 1);
            mbar_init(&ctrl->own_full[i], 1);
            mbar_init(&ctrl->own_free[i], 1);
            mbar_init(&ctrl->row_full[i], 1);
            mbar_init(&ctrl->row_empty[i], 16);
            mbar_init(&ctrl->p_full[i], 16);
        }
        mbar_init(&ctrl->s_full[0], 1);
        mbar_init(&ctrl->s_free[0], 16);
        mbar_init(&ctrl->dp_full[0], 1);
        mbar_init(&ctrl->ds_full[0], 16);
        mbar_init(&ctrl->acc_full, 1);
        mbar_init(&ctrl->acc_free, 16);
        mbar_init(&ctrl->tail, 1);
        ctrl->abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_u32(&ctrl->tmem_base)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctrl->tmem_base;
    uint32_t k_item = 0;
    BwdItem it{};

    // Registers: as in the dQ kernel.
    if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;\n" ::);
        if (warp == 18) {
            // ================================ items and TMA copies ================================
            BwdSchedule<false> schedule;
            schedule.init(p, lane);
            uint32_t tails = 0, t = 0, n_item = 0;
            bool ok = true;
            auto own = [&](int which, uint8_t* dst, const CUtensorMap* map) -> bool {
                if (!__all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->own_free[which], (n_item & 1u) ^ 1u, abort_flag, p.status, 0x10120))) return false;
                // (rows behind the end of the keys stay in their own rows of the gradients, which are not stored)
                return bwd_load_tile<HDIM>(dst, map, &ctrl->own_full[which], &ctrl->tail, tails, it.h, it.k0 + it.row0, 128, lane, abort_flag, p.status);
            };
            // (an item is handed out while the copies of the one before it are still to come: its LSE and D are then there in time)
            BwdItem ahead{};
            for (bool more = schedule.next(ctrl, p, lane, ahead); ok && more;) {
                it = ahead;
                more = schedule.next(ctrl, p, lane, ahead);
                const BwdRange range = bwd_query_tiles(p, it);
                if (range.count == 0) continue;
                for (int g = 0; ok && g < G; ++g)
                    for (int m = 0; m < range.count; ++m, ++t) {
                        const int m0 = (range.begin + m) * 128, h = it.h * G + g, qs = t % QS, os = t % OS;
                        if (g + m == 0 && !(ok = own(0, sK, &map_k))) break;
                        if (!(ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->a_empty[qs], ((t / QS) & 1u) ^ 1u, abort_flag, p.status, 0x10121)))) break;
                        if (!(ok = bwd_load_tile<HDIM>(sQ + qs * TILE, &map_q, &ctrl->a_full[qs], &ctrl->tail, tails, h, it.q0 + m0, it.sq - m0, lane,
                                                       abort_flag, p.status))) break;
                        if (g + m == 0 && !(ok = own(1, sV, &map_v))) break;
                        if (!(ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->b_empty[os], ((t / OS) & 1u) ^ 1u, abort_flag, p.status, 0x10122)))) break;
                        if (!(ok = bwd_load_tile<HDIM>(sDO + os * TILE, &map_do, &ctrl->b_full[os], &ctrl->tail, tails, h, it.q0 + m0, it.sq - m0, lane,
                                                       abort_flag, p.status))) break;
                    }
                ++n_item;
            }
        } else if (warp == 19) {
            // ================================ LSE and D of the query columns ================================
            pdl_wait();
            uint32_t t = 0;
            bool ok = true;
            while (ok && bwd_next_item(ctrl, p, k_item, lane, it)) {
                const BwdRange range = bwd_query_tiles(p, it);
                for (int g = 0; ok && g < G; ++g) {
                    const int64_t lr = p.seqstart_q ? (int64_t)(it.h * G + g) * p.seqlen_q + it.q0 : ((int64_t)it.b * p.hq + it.h * G + g) * p.seqlen_q;
                    for (int m = 0; m < range.count; ++m, ++t) {
                        const int m0 = (range.begin + m) * 128, slot = t & 1;
                        float l[4], d[4];
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            const int i = m0 + u * 32 + lane;
                            l[u] = i < it.sq ? -bwd_lse_base2(p.lse[lr + i]) : -INFINITY;
                            d[u] = i < it.sq ? -p.delta[lr + i] : 0.f;
                        }
                        if (!(ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->row_empty[slot], ((t >> 1) & 1u) ^ 1u, abort_flag, p.status, 0x10123)))) break;
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            sRow[slot * 256 + u * 32 + lane] = l[u];
                            sRow[slot * 256 + 128 + u * 32 + lane] = d[u];
                        }
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&ctrl->row_full[slot]);
                    }
                }
            }
        } else {
            // ================================ MMA issuers: 16 S, 17 dP, dV and dK ================================
            const bool leader = elect_one_sync();
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
                return ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag, p.status, code)) != 0;
            };
            auto commit = [&](uint64_t* bar) { if (leader) umma_commit(bar); };
            auto at = [&](uint64_t d, uint32_t bytes) { return d + (uint64_t)(bytes >> 4); };
            constexpr uint32_t idesc_s = make_idesc<T>(false), idesc_o = make_idesc<T>(true, HDIM);
            const uint64_t dK = make_smem_desc(smem_u32(sK), 0, 1024), dV = make_smem_desc(smem_u32(sV), 0, 1024);
            const uint64_t dQ = make_smem_desc(smem_u32(sQ), 0, 1024), dDO = make_smem_desc(smem_u32(sDO), 0, 1024);
            const uint64_t dQt = make_smem_desc(smem_u32(sQ), HALF_BYTES, 1024), dDOt = make_smem_desc(smem_u32(sDO), HALF_BYTES, 1024);
            uint32_t t = 0, qs = 0, qph = 0, n_item = 0;  // steps so far, Q slot and its phase, items with steps so far
            if (warp == 16) {
                while (ok && bwd_next_item(ctrl, p, k_item, lane, it)) {
                    const int N = bwd_query_tiles(p, it).count * G;
                    if (N > 0 && !wait(&ctrl->own_full[0], n_item & 1u, 0x10130)) break;
                    for (int j = 0; j < N; ++j) {
                        if (!wait(&ctrl->a_full[qs], qph, 0x10131)) break;
                        if (t > 0 && !wait(&ctrl->s_free[0], (t - 1) & 1u, 0x10132)) break;  // dP(t - 1) has been read from the region
                        tc_fence_after();
                        if (leader) bwd_issue_ss<HDIM>(tmem + (t & 1u) * 128, dK, at(dQ, qs * TILE), idesc_s);
                        commit(&ctrl->s_full[0]);
                        ++t;
                        if (++qs == QS) { qs = 0; qph ^= 1u; }
                    }
                    if (!ok) break;
                    if (N > 0) { commit(&ctrl->own_free[0]); ++n_item; }
                }
            } else {
                auto issue_dp = [&](uint32_t st) -> bool {  // to the region that P and dS of the step before have been read from
                    if (!wait(&ctrl->b_full[st & 1u], (st >> 1) & 1u, 0x10134)) return false;
                    tc_fence_after();
                    if (leader) bwd_issue_ss<HDIM>(tmem + ((st + 1) & 1u) * 128, dV, at(dDO, (st & 1u) * TILE), idesc_s);
                    commit(&ctrl->dp_full[0]);
                    return true;
                };
                while (ok && bwd_next_item(ctrl, p, k_item, lane, it)) {
                    const int N = bwd_query_tiles(p, it).count * G;
                    if (N == 0) continue;
                    if (!wait(&ctrl->own_full[1], n_item & 1u, 0x10133) || !issue_dp(t)) break;
                    if (n_item > 0 && !wait(&ctrl->acc_free, (n_item - 1) & 1u, 0x10136)) break;
                    for (int j = 0; j < N; ++j) {
                        const uint32_t region = tmem + (t & 1u) * 128;  // of every 32 columns P has the first 16, dS the others
                        const uint32_t os = t & 1u;
                        if (!wait(&ctrl->p_full[os], (t >> 1) & 1u, 0x10137)) break;
                        tc_fence_after();
                        if (leader) {
                            bwd_issue_xb(tmem + cDV, region, at(dDOt, os * TILE), idesc_o, 0, j > 0);
                            bwd_issue_xb(tmem + cDV, region, at(dDOt, os * TILE), idesc_o, 1, true);
                        }
                        commit(&ctrl->b_empty[os]);
                        if (!wait(&ctrl->ds_full[0], t & 1u, 0x10138)) break;
                        tc_fence_after();
                        if (leader) {
                            bwd_issue_xb(tmem + cDK, region + 16, at(dQt, qs * TILE), idesc_o, 0, j > 0);
                            bwd_issue_xb(tmem + cDK, region + 16, at(dQt, qs * TILE), idesc_o, 1, true);
                        }
                        commit(&ctrl->a_empty[qs]);
                        if (j + 1 < N && !issue_dp(t + 1)) break;
                        ++t;
                        if (++qs == QS) qs = 0;
                    }
                    if (!ok) break;
                    commit(&ctrl->own_free[1]);
                    commit(&ctrl->acc_full);
                    ++n_item;
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 104;\n" ::);
        const int quarter = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        uint32_t t = 0, n_item = 0;
        bool ok = true;
        while (ok && bwd_next_item(ctrl, p, k_item, lane, it)) {
            constexpr int COLS = HDIM / 2;  // of dV (warps 0-7) or dK (8-15) that this warp stores
            const bool is_dk = quarter >= 2;
            const int key = it.row0 + r, shift = p.mask_type == 2 ? it.sk - it.sq : 0;
            const int first = it.row0 + (warp & 3) * 32;  // of this warp's rows
            const BwdRange range = bwd_query_tiles(p, it);
            T* dst = (T*)(is_dk ? p.dk : p.dv) + ((int64_t)(it.k0 + first) * p.hkv + it.h) * HDIM + (quarter & 1) * COLS;
            uint4 out[COLS / 8];
            if (range.count == 0) {  // nobody sees these keys
#pragma unroll
                for (int v = 0; v < COLS / 8; ++v) out[v] = make_uint4(0u, 0u, 0u, 0u);
                bwd_store_rows<T>(dst, (int64_t)p.hkv * HDIM, it.sk - first, out, lane);
                continue;
            }
            // query rows that see all of the tile's keys
            int full_lo = 0, full_hi = it.sq - 1;
            if (p.mask_type != 0) {
                if (p.wr >= 0) full_lo = it.row0 + 127 - shift - p.wr;
                if (p.wl >= 0) full_hi = min(full_hi, it.row0 - shift + p.wl);
            }
            for (int g = 0, m = 0; g < G; ++t) {
                const int m0 = (range.begin + m) * 128, i0 = m0 + quarter * 32;
                const bool masked = m0 < full_lo || m0 + 127 > full_hi;
                const float slope = VAR == 1 && p.alibi ? p.alibi[(p.alibi_rank ? it.b * p.hq : 0) + it.h * G + g] * kLog2e : 0.f;
                [[maybe_unused]] const int head = g;  // of the group
                if (++m == range.count) { m = 0; ++g; }
                // columns of this quarter that see the key: i >= key - shift - wr, i <= key - shift + wl.  (Columns behind the last query are
                // zeros, but a key that nobody sees may hold a NaN.)
                uint32_t seen = 0xffffffffu;
                if (masked) {
                    const bool bounded = p.mask_type != 0;
                    seen = bwd_column_bits(bounded && p.wr >= 0 ? key - shift - p.wr - i0 : 0,
                                           (bounded && p.wl >= 0 ? min(it.sq - 1, key - shift + p.wl) : it.sq - 1) - i0);
                }
                [[maybe_unused]] uint32_t bw[VAR == 2 ? 16 : 1];  // the key's bias values in the 32 query columns
                if constexpr (VAR == 2) {
                    // A row of the tensor at a time: the warp's 32 keys lie side by side.  Every address is inside the block, so that no load
                    // waits for a test and all of them are in flight together; what lies outside is zeroed afterwards.
                    // (dK/dV of 2 x 1024 tokens of 16 heads: 134 us with a test in front of each load, 73 so; the next step's loads
                    // under the end of this one 93, with registers spilled.)
                    const unsigned short* at = (const unsigned short*)p.bias + bwd_bias_block(p, it.b, it.h * G + head, it.q0, it.k0) + min(key, it.sk - 1);
                    unsigned short raw[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) raw[e] = __ldg(at + min(i0 + e, it.sq - 1) * p.bias_sk);
#pragma unroll
                    for (int e = 0; e < 32; e += 2) bw[e / 2] = raw[e] | (uint32_t)raw[e + 1] << 16;
                    if (key >= it.sk || i0 + 32 > it.sq) bwd_hide(bw, key < it.sk ? bwd_column_bits(0, it.sq - 1 - i0) : 0u);
                }
                const float* rows = sRow + (t & 1) * 256 + quarter * 32;
                const uint32_t tS = lane_addr + (t & 1u) * 128 + quarter * 32, tDP = lane_addr + ((t + 1) & 1u) * 128 + quarter * 32;
                if (!(ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->row_full[t & 1], (t >> 1) & 1u, abort_flag, p.status, 0x10140)))) break;
                if (!(ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->s_full[0], t & 1u, abort_flag, p.status, 0x10141)))) break;
                tc_fence_after();
                uint32_t x[32], w[16];
                tmem_ld32(tS, x);
                tmem_wait_ld();
                if constexpr (VAR != 0) {
                    if (p.soft_cap > 0.f) soft_cap_scores<32>(x, p.cap);
                }
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    const float4 l4 = *reinterpret_cast<const float4*>(rows + e);
#pragma unroll
                    for (int u = 0; u < 4; u += 2) {
                        float2 f = make_float2(1.f, 1.f), away = f;
                        if constexpr (VAR == 1) {
                            away.x = (float)(i0 + e + u + it.sk - it.sq - key);
                            away.y = away.x + 1.f;
                        } else if constexpr (VAR == 2) {
                            away = bias_pair<T>(bw[(e + u) / 2]);
                        }
                        const float2 y = bwd_exponent<VAR>(p, make_float2(__uint_as_float(x[e + u]), __uint_as_float(x[e + u + 1])), slope, away,
                                                             u ? make_float2(l4.z, l4.w) : make_float2(l4.x, l4.y), f);
                        float2 pr = bwd_exp2<VAR == 2 ? 0 : kPolyDkdv>(y, (e + u) / 2);
                        w[(e + u) / 2] = Elem<T>::pack2(pr.x, pr.y);
                        if constexpr (VAR != 0) pr = __fmul2_rn(pr, f);  // (from here on P serves dS alone)
                        x[e + u] = __float_as_uint(pr.x);
                        x[e + u + 1] = __float_as_uint(pr.y);
                    }
                }
                if (masked) bwd_hide(w, seen);
                tmem_st16(tS, w);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctrl->p_full[t & 1u]);
                if (!(ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->dp_full[0], t & 1u, abort_flag, p.status, 0x10142)))) break;
                tc_fence_after();
                uint32_t dp[32];
                tmem_ld32(tDP, dp);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctrl->s_free[0]);
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    const float4 d4 = *reinterpret_cast<const float4*>(rows + 128 + e);
#pragma unroll
                    for (int u = 0; u < 4; u += 2) {
                        const float2 d = __fadd2_rn(make_float2(__uint_as_float(dp[e + u]), __uint_as_float(dp[e + u + 1])),
                                                    u ? make_float2(d4.z, d4.w) : make_float2(d4.x, d4.y));
                        const float2 ds = __fmul2_rn(make_float2(__uint_as_float(x[e + u]), __uint_as_float(x[e + u + 1])), d);
                        w[(e + u) / 2] = Elem<T>::pack2(ds.x, ds.y);
                    }
                }
                if (masked) bwd_hide(w, seen);
                tmem_st16(tS + 16, w);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&ctrl->ds_full[0]);
                    mbar_arrive(&ctrl->row_empty[t & 1]);
                }
            }
            if (!ok || !(ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->acc_full, n_item & 1u, abort_flag, p.status, 0x10143)))) break;
            ++n_item;
            tc_fence_after();
            bwd_load_rows<T, COLS>(lane_addr + (is_dk ? cDK : cDV) + (quarter & 1) * COLS, is_dk ? p.scale : 1.f, out);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctrl->acc_free);
            bwd_store_rows<T>(dst, (int64_t)p.hkv * HDIM, it.sk - first, out, lane);
        }
    }
    pdl_wait();
    tc_fence_before();
    __syncthreads();
    if (warp == 16) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem));
    }
}

// ---- the gradient of a bias tensor --------------------------------------------------------------------------------------------
// dbias = dT = P (dP - D), summed over the heads and sequences that share a plane.  A work item is a 128 x 128 tile of one plane (group
// mode: of one sequence's block): its CTA walks the sharers in order, S = Q K^T and dP = dO V^T into two buffers each, and
// adds up in registers.  Four tiles are copied for two products, so shared memory (2048 clocks a step) and L2 bound it: 56 us for
// 2 x 1024 tokens of 16 heads of 128 with a plane per head.  With a bias tensor, dQ takes 64 us there and dK/dV 73: transposed, a
// thread reads its 32 bias values a step two bytes at a time.
__device__ __forceinline__ void bwd_tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}
struct BwdBiasItem {
    int row0, key0, b_begin, b_end, h_begin, h_end, steps;
    BwdSeq s;  // of the first sharer (the sharers' lengths are equal)
};
// The items of a CTA: those tiles of plane after plane that lie inside the plane's sequence (planes: heads, or none, inside sequences,
// or none), dealt in turn.  Every role walks them for itself.
struct BwdBiasWalk {
    int pb, ph, tiles_k;
    int at, tiles;  // the next item of this CTA, and the tiles, of the plane (a plane that memory holds has fewer than 2^25)

    __device__ __forceinline__ void plane(const BwdSm100Dev& p) {
        const BwdSeq s = bwd_sequence(p, pb);
        tiles_k = (s.sk + 127) / 128;
        tiles = (s.sq + 127) / 128 * tiles_k;
    }
    __device__ __forceinline__ void init(const BwdSm100Dev& p) {
        pb = ph = 0;
        at = blockIdx.x;
        plane(p);
    }
    __device__ __forceinline__ bool next(const BwdSm100Dev& p, BwdBiasItem& it);
};
__device__ __forceinline__ BwdBiasItem bwd_bias_item(const BwdSm100Dev& p, int pb, int ph, int tile_q, int tile_k) {
    BwdBiasItem it;
    it.key0 = tile_k * 128;
    it.row0 = tile_q * 128;
    const bool own_b = p.bias_rank == 2 || p.seqstart_q;
    it.b_begin = own_b ? pb : 0;
    it.b_end = own_b ? pb + 1 : p.batch;
    it.h_begin = p.bias_rank >= 1 ? ph : 0;
    it.h_end = p.bias_rank >= 1 ? ph + 1 : p.hq;
    it.s = bwd_sequence(p, it.b_begin);
    bool seen = true;  // by some row: the first key of the last row's window, the last key of the last row
    if (p.mask_type != 0) {
        const int last = min(it.s.sq, it.row0 + 128) - 1;
        if (p.wr >= 0 && it.key0 > last + it.s.shift + p.wr) seen = false;
        if (p.wl >= 0 && min(it.s.sk, it.key0 + 128) - 1 < it.row0 + it.s.shift - p.wl) seen = false;
    }
    it.steps = seen ? (it.b_end - it.b_begin) * (it.h_end - it.h_begin) : 0;
    return it;
}
__device__ __forceinline__ bool BwdBiasWalk::next(const BwdSm100Dev& p, BwdBiasItem& it) {
    const int planes_h = p.bias_rank >= 1 ? p.hq : 1, planes_b = p.bias_rank == 2 || p.seqstart_q ? p.batch : 1;
    while (at >= tiles) {
        at -= tiles;
        if (++ph == planes_h) {
            ph = 0;
            if (++pb >= planes_b) return false;
            plane(p);
        }
    }
    const int tile_q = at / tiles_k;
    it = bwd_bias_item(p, pb, ph, tile_q, at - tile_q * tiles_k);
    at += gridDim.x;
    return true;
}

constexpr int kBwdBiasThreads = 576;  // warps 0-15 elementwise, 16 products, 17 copies

template <typename T, int HDIM>
__global__ void __launch_bounds__(kBwdBiasThreads, 1)
bwd_dbias_sm100_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                       const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const BwdSm100Dev p) {
    constexpr int TILE = 128 * HDIM * 2;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sQ = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));  // 2 x (Q, K)
    uint8_t* sDO = sQ + 4 * TILE;                                                             // dO, V
    BwdCtrl* ctrl = reinterpret_cast<BwdCtrl*>(sDO + 2 * TILE);
    volatile int* abort_flag = &ctrl->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&ctrl->a_full[i], 1);
            mbar_init(&ctrl->a_empty[i], 1);
            mbar_init(&ctrl->s_full[i], 1);
            mbar_init(&ctrl->dp_full[i], 1);
            mbar_init(&ctrl->s_free[i], 16);
        }
        mbar_init(&ctrl->b_full[0], 1);
        mbar_init(&ctrl->b_empty[0], 1);
        ctrl->abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_u32(&ctrl->tmem_base)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    }
    pdl_wait();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctrl->tmem_base;  // S in columns 0-127 and 128-255, dP in 256-383 and 384-511
    const int G = p.hq / p.hkv;
    bool ok = true;
    uint32_t t = 0;
    BwdBiasWalk walk;
    BwdBiasItem it;
    walk.init(p);
    auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
        return ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag, p.status, code)) != 0;
    };
    if (warp == 17) {
        // ================================ TMA producer ================================
        // (Rows behind a sequence's end make rows and columns of dT that are not stored.)
        auto load = [&](uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int head, int row) {
#pragma unroll
            for (int hb = 0; hb < HDIM / 64; ++hb) tma_load_3d(dst + hb * HALF_BYTES, map, bar, hb * 64, head, row);
        };
        while (ok && walk.next(p, it)) {
            int b = it.b_begin, h = it.h_begin;
            for (int j = 0; j < it.steps; ++j, ++t) {
                const BwdSeq s = bwd_sequence(p, b);
                const int kh = h / G, slot = t & 1;
                if (!wait(&ctrl->a_empty[slot], ((t >> 1) & 1u) ^ 1u, 0x10201)) break;
                if (lane == 0) {
                    mbar_expect_tx(&ctrl->a_full[slot], 2 * TILE);
                    load(sQ + slot * 2 * TILE, &map_q, &ctrl->a_full[slot], h, s.q0 + it.row0);
                    load(sQ + slot * 2 * TILE + TILE, &map_k, &ctrl->a_full[slot], kh, s.k0 + it.key0);
                }
                if (!wait(&ctrl->b_empty[0], (t & 1u) ^ 1u, 0x10202)) break;
                if (lane == 0) {
                    mbar_expect_tx(&ctrl->b_full[0], 2 * TILE);
                    load(sDO, &map_do, &ctrl->b_full[0], h, s.q0 + it.row0);
                    load(sDO + TILE, &map_v, &ctrl->b_full[0], kh, s.k0 + it.key0);
                }
                if (++h == it.h_end) { h = it.h_begin; ++b; }
            }
        }
    } else if (warp == 16) {
        // ================================ MMA issuer ================================
        constexpr uint32_t idesc = make_idesc<T>(false);
        const bool leader = elect_one_sync();
        auto commit = [&](uint64_t* bar) { if (leader) umma_commit(bar); };
        const uint64_t dQ = make_smem_desc(smem_u32(sQ), 0, 1024), dDO = make_smem_desc(smem_u32(sDO), 0, 1024);
        while (ok && walk.next(p, it)) {
            for (int j = 0; j < it.steps; ++j, ++t) {
                const uint32_t buf = t & 1u, par = (t >> 1) & 1u;
                if (!wait(&ctrl->a_full[buf], par, 0x10211) || !wait(&ctrl->s_free[buf], par ^ 1u, 0x10212)) break;
                tc_fence_after();
                if (leader) bwd_issue_ss<HDIM>(tmem + buf * 128, dQ + ((buf * 2 * TILE) >> 4), dQ + ((buf * 2 * TILE + TILE) >> 4), idesc);
                commit(&ctrl->s_full[buf]);
                commit(&ctrl->a_empty[buf]);
                if (!wait(&ctrl->b_full[0], t & 1u, 0x10213)) break;
                tc_fence_after();
                if (leader) bwd_issue_ss<HDIM>(tmem + 256 + buf * 128, dDO, dDO + (TILE >> 4), idesc);
                commit(&ctrl->dp_full[buf]);
                commit(&ctrl->b_empty[0]);
            }
        }
    } else if (warp < 16) {
        const int quarter = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16) + quarter * 32;
        while (ok && walk.next(p, it)) {
            const int i = it.row0 + r, key0 = it.key0 + quarter * 32, left = it.s.sq - it.row0;
            const int64_t block = bwd_bias_block(p, it.b_begin, it.h_begin, it.s.q0, it.s.k0);
            uint32_t bw[16];
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const uint4 x = load_bias_piece(r < left ? (const unsigned short*)p.bias + block + i * p.bias_sk : nullptr, key0 + v * 8, it.s.sk - key0 - v * 8);
                bw[4 * v] = x.x; bw[4 * v + 1] = x.y; bw[4 * v + 2] = x.z; bw[4 * v + 3] = x.w;
            }
            const int k_lo = p.mask_type != 0 && p.wl >= 0 ? i + it.s.shift - p.wl : 0;
            const int k_hi = p.mask_type != 0 && p.wr >= 0 ? min(it.s.sk - 1, i + it.s.shift + p.wr) : it.s.sk - 1;
            const uint32_t seen = bwd_column_bits(k_lo - key0, k_hi - key0);
            float2 acc[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[e] = make_float2(0.f, 0.f);
            int b = it.b_begin, h = it.h_begin;
            for (int j = 0; j < it.steps; ++j, ++t) {
                const BwdSeq s = bwd_sequence(p, b);
                const int64_t lr = (p.seqstart_q ? (int64_t)h * p.seqlen_q + s.q0 : ((int64_t)b * p.hq + h) * p.seqlen_q) + i;
                const float lse2 = r < left ? bwd_lse_base2(p.lse[lr]) : INFINITY, delta = r < left ? p.delta[lr] : 0.f;
                if (++h == it.h_end) { h = it.h_begin; ++b; }
                const uint32_t buf = t & 1u, par = (t >> 1) & 1u;
                if (!wait(&ctrl->s_full[buf], par, 0x10221) || !wait(&ctrl->dp_full[buf], par, 0x10222)) break;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < 32; c += 8) {
                    uint32_t x[8], dp[8];
                    bwd_tmem_ld8(lane_addr + buf * 128 + c, x);
                    bwd_tmem_ld8(lane_addr + 256 + buf * 128 + c, dp);
                    tmem_wait_ld();
                    if (p.soft_cap > 0.f) soft_cap_scores<8>(x, p.cap);
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        float2 f;
                        const float2 y = bwd_exponent<2>(p, make_float2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), 0.f, bias_pair<T>(bw[(c + e) / 2]),
                                                         make_float2(-lse2, -lse2), f);
                        const float2 dt = __fadd2_rn(make_float2(__uint_as_float(dp[e]), __uint_as_float(dp[e + 1])), make_float2(-delta, -delta));
                        float2& a = acc[(c + e) / 2];
                        if (seen >> (c + e) & 1u) a.x = fmaf(ex2_fast(y.x), dt.x, a.x);
                        if (seen >> (c + e + 1) & 1u) a.y = fmaf(ex2_fast(y.y), dt.y, a.y);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctrl->s_free[buf]);
            }
            if (!ok) break;
            uint4 out[4];
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                out[v].x = Elem<T>::pack2(acc[4 * v].x, acc[4 * v].y);
                out[v].y = Elem<T>::pack2(acc[4 * v + 1].x, acc[4 * v + 1].y);
                out[v].z = Elem<T>::pack2(acc[4 * v + 2].x, acc[4 * v + 2].y);
                out[v].w = Elem<T>::pack2(acc[4 * v + 3].x, acc[4 * v + 3].y);
            }
            bwd_exchange<4>(out, lane);
            const int first = (warp & 3) * 32 + (lane & ~3), col = key0 + (lane & 3) * 8;  // this lane: 8 elements of rows first .. + 3
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (first + j >= left) continue;
                unsigned short* dst = (unsigned short*)p.dbias + block + (int64_t)(it.row0 + first + j) * p.bias_sk + col;
                if (col + 8 <= it.s.sk && (reinterpret_cast<uintptr_t>(dst) & 15u) == 0) {
                    *reinterpret_cast<uint4*>(dst) = out[j];
                } else {
                    const uint32_t w[4] = {out[j].x, out[j].y, out[j].z, out[j].w};
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (col + e < it.s.sk) dst[e] = (unsigned short)(w[e / 2] >> (16 * (e & 1)));
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 16) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem));
    }
}

}  // namespace sm100

}  // namespace fck
