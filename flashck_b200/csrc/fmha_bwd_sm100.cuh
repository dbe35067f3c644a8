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
// The kernels are persistent (one CTA per SM).  Roles: warps 0-7 the elementwise work (thread = tensor memory lane = row; warps
// 0-3 take columns 0-63 of a tile, 4-7 columns 64-127), warp 8 issues S and dP, another warp the products that P and dS enter (a
// single issuer spends as long on its waits and commits as the products take, and the tensor pipe takes instructions only
// about one ahead: 16 % slower), warp 9 the TMA copies, warp 11 finds the work items and hands them to the others through a ring.
// dQ: warps 12-15 bring Q and dO to tensor memory and compute D.  dK/dV: warp 10 fetches LSE and D of the query columns.
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
    int listed;                    // items are found in order of cost by a persistent grid; 0: one per CTA, by its index
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
// D += X B over 64 of 128 rows (half 0 / 1): X in tensor memory, 32 columns from a + 64 half; B MN-major.
__device__ __forceinline__ void bwd_issue_xb(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, int half, bool accumulate) {
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
        umma_ts(d, a + half * 64 + ks * 8, b + (uint64_t)(((half * 4 + ks) * 2048) >> 4), idesc, (accumulate || ks > 0) ? 1u : 0u);
}

// 2^x on the FMA pipe for two values: x = n + f, f in [-0.5, 0.5], 2^f by the polynomial of degree 4 of least relative error
// (2.7e-6 with its fp32 rounding), n added to the exponent.  x above -126 (2^-126 stands for everything below).
__device__ __forceinline__ float2 bwd_exp2_poly(float2 x) {
    x.x = fmaxf(x.x, -126.f);
    x.y = fmaxf(x.y, -126.f);
    const float2 t = __fadd2_rn(x, make_float2(12582912.f, 12582912.f));  // 1.5 * 2^23: n lands in the low mantissa bits
    const float2 f = __fadd2_rn(x, __fadd2_rn(make_float2(12582912.f, 12582912.f), make_float2(-t.x, -t.y)));
    float2 q = __ffma2_rn(make_float2(0.009570076f, 0.009570076f), f, make_float2(0.05591789f, 0.05591789f));
    q = __ffma2_rn(q, f, make_float2(0.24024746f, 0.24024746f));
    q = __ffma2_rn(q, f, make_float2(0.6931218f, 0.6931218f));
    q = __ffma2_rn(q, f, make_float2(0.9999993f, 0.9999993f));
    return make_float2(__int_as_float(__float_as_int(q.x) + (__float_as_int(t.x) << 23)),
                       __int_as_float(__float_as_int(q.y) + (__float_as_int(t.y) << 23)));
}
// The exponentials of a pair: pairs `i` of every 8 below kPolyPairs go to the FMA pipe, the others to the exp2 unit, which alone would
// take 1024 clocks per tile.
constexpr int kPolyPairs = 3;
__device__ __forceinline__ float2 bwd_exp2(float2 y, int i) {
    return (i & 7) < kPolyPairs ? bwd_exp2_poly(y) : make_float2(ex2_fast(y.x), ex2_fast(y.y));
}

// Base-2 exponent of a pair of scores (raw, or with EXTRA what soft_cap_scores left of them), LSE subtracted; with a soft cap
// f is what dS gets from it, 1 - tanh^2.
template <bool EXTRA>
__device__ __forceinline__ float2 bwd_exponent(const BwdSm100Dev& p, float2 x, float slope_log2, float2 away, float2 neg_lse2, float2& f) {
    if constexpr (!EXTRA) return __ffma2_rn(x, make_float2(p.scale_log2, p.scale_log2), neg_lse2);
    float2 y = x;
    if (p.soft_cap > 0.f) {
        const float2 t = __fmul2_rn(x, make_float2(p.inv_cap_log2, p.inv_cap_log2));
        f = __ffma2_rn(make_float2(-t.x, -t.y), t, make_float2(1.f, 1.f));
    } else {
        y = __fmul2_rn(x, make_float2(p.scale_log2, p.scale_log2));
    }
    y = __ffma2_rn(make_float2(-slope_log2, -slope_log2), make_float2(fabsf(away.x), fabsf(away.y)), y);
    return __fadd2_rn(y, neg_lse2);
}

// 32 fp32 columns of one row, times f, as 64 bytes of the element type.
template <typename T>
__device__ __forceinline__ void bwd_store32(T* dst, const uint32_t (&t)[32], float f) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        uint4 w;
        w.x = Elem<T>::pack2(__uint_as_float(t[8 * v]) * f, __uint_as_float(t[8 * v + 1]) * f);
        w.y = Elem<T>::pack2(__uint_as_float(t[8 * v + 2]) * f, __uint_as_float(t[8 * v + 3]) * f);
        w.z = Elem<T>::pack2(__uint_as_float(t[8 * v + 4]) * f, __uint_as_float(t[8 * v + 5]) * f);
        w.w = Elem<T>::pack2(__uint_as_float(t[8 * v + 6]) * f, __uint_as_float(t[8 * v + 7]) * f);
        reinterpret_cast<uint4*>(dst)[v] = w;
    }
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
    uint64_t own_full[2], own_free[2];  // what an item owns: dQ Q / dO in tensor memory, dK/dV the K / V tile
    uint64_t s_full[2], s_free[2], dp_full[2], ds_full[2];  // dQ: by half; dK/dV: [0] (s_free[0]: dP has been read)
    uint64_t x_done[2];         // the product that reads dS is complete (dQ: by half)
    uint64_t p_full[2];         // dK/dV, by step: the elementwise warps can be one step ahead of the products that read P
    uint64_t acc_full, acc_free, tail;
    uint64_t row_full[2], row_empty[2];
    uint32_t tmem_base;
    int abort_flag;
};

// The scheduling warp.  Items of a level cost the same under a causal mask: level l is the row tile l of dQ (the last tiles see the
// most keys), the tile l places in front of the last one of dK/dV (the first tiles are seen by the most queries).  Levels come
// in decreasing order, a level's sequences in order, their heads side by side (they share tiles through L2); rounds of the grid
// take the items in alternate directions.  Tile counts are held eight sequences a lane.
template <bool DQ>
__device__ __forceinline__ void bwd_schedule(BwdCtrl* ctrl, const BwdSm100Dev& p, int lane) {
    const int heads = DQ ? p.hq : p.hkv;
    uint32_t k = 0;
    auto publish = [&](int valid, int b, int h, int row0) -> bool {
        const int slot = k % kBwdItemRing;
        const bool ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->item_empty[slot], ((k / kBwdItemRing) & 1u) ^ 1u, &ctrl->abort_flag, p.status, 0x10001));
        ++k;
        if (ok && lane == 0) {
            BwdItem it{valid, b, h, row0, 0, 0, 0, 0};
            if (valid) {
                const BwdSeq s = bwd_sequence(p, b);
                it.q0 = s.q0; it.k0 = s.k0; it.sq = s.sq; it.sk = s.sk;
            }
            ctrl->items[slot] = it;
            mbar_arrive(&ctrl->item_full[slot]);
        }
        __syncwarp();
        return ok;
    };
    if (!p.listed) {  // one item per CTA
        const int per_tile = heads * p.batch, t = (int)blockIdx.x / per_tile, rest = (int)blockIdx.x - t * per_tile;
        const int b = rest / heads, h = rest - b * heads, row0 = (DQ ? (int)gridDim.x / per_tile - 1 - t : t) * 128;
        const BwdSeq s = bwd_sequence(p, b);
        if (row0 < (DQ ? s.sq : s.sk) && !publish(1, b, h, row0)) return;
        publish(0, 0, 0, 0);
        return;
    }
    int cnt[kBwdMaxBatch / 32], most = 0;
#pragma unroll
    for (int u = 0; u < kBwdMaxBatch / 32; ++u) {
        cnt[u] = 0;
        if (u * 32 + lane < p.batch) {
            const BwdSeq s = bwd_sequence(p, u * 32 + lane);
            cnt[u] = min(((DQ ? s.sq : s.sk) + 127) / 128, p.max_tiles);
        }
        most = max(most, cnt[u]);
    }
    int level = (int)__reduce_max_sync(0xffffffffu, (unsigned)most) - 1;
    int64_t base = 0;  // first item of the level
    for (int r = 0;; ++r) {
        const int64_t w = (int64_t)r * gridDim.x + ((r & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        for (; level >= 0; --level) {
            int n = 0;
#pragma unroll
            for (int u = 0; u < kBwdMaxBatch / 32; ++u) n += __popc(__ballot_sync(0xffffffffu, cnt[u] > level));
            if (w < base + (int64_t)n * heads) break;
            base += (int64_t)n * heads;
        }
        if (level < 0) break;
        int rank = (int)((w - base) / heads), b = 0, tiles = 0;
        const int h = (int)(w - base) - rank * heads;
        bool found = false;
#pragma unroll
        for (int u = 0; u < kBwdMaxBatch / 32; ++u) {
            const uint32_t m = __ballot_sync(0xffffffffu, cnt[u] > level);
            const int c = __popc(m);
            if (!found && rank < c) {
                const int l = __fns(m, 0, rank + 1);
                b = u * 32 + l;
                tiles = __shfl_sync(0xffffffffu, cnt[u], l);
                found = true;
            }
            if (!found) rank -= c;
        }
        if (!publish(1, b, h, (DQ ? level : tiles - 1 - level) * 128)) return;
    }
    publish(0, 0, 0, 0);
}
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


// ---- dQ -----------------------------------------------------------------------------------------------------------------
constexpr int kBwdDqThreads = 512;

template <typename T, int HDIM, bool EXTRA>
__global__ void __launch_bounds__(kBwdDqThreads, 1)
bwd_dq_sm100_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const BwdSm100Dev p) {
    constexpr int TILE = 128 * HDIM * 2, KS = 3, VS = 2;
    constexpr uint32_t cS = 0, cDP = 128, cDQ = 256, cQ = 384, cDO = 448;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
    uint8_t* sK = base;
    uint8_t* sV = sK + KS * TILE;
    float* sRow = reinterpret_cast<float*>(sV + VS * TILE);  // [2 items][LSE 128 | D 128] of the rows
    BwdCtrl* ctrl = reinterpret_cast<BwdCtrl*>(sRow + 512);
    volatile int* abort_flag = &ctrl->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kBwdItemRing; ++i) {
            mbar_init(&ctrl->item_full[i], 1);
            mbar_init(&ctrl->item_empty[i], 15);  // every warp but the scheduling one
        }
        for (int i = 0; i < KS; ++i) { mbar_init(&ctrl->a_full[i], 1); mbar_init(&ctrl->a_empty[i], 1); }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&ctrl->b_full[i], 1);
            mbar_init(&ctrl->b_empty[i], 1);
            mbar_init(&ctrl->own_full[i], 4);
            mbar_init(&ctrl->own_free[i], 1);
            mbar_init(&ctrl->s_full[i], 1);
            mbar_init(&ctrl->s_free[i], 4);
            mbar_init(&ctrl->dp_full[i], 1);
            mbar_init(&ctrl->ds_full[i], 4);
            mbar_init(&ctrl->x_done[i], 1);
            mbar_init(&ctrl->row_full[i], 4);
            mbar_init(&ctrl->row_empty[i], 8);
        }
        mbar_init(&ctrl->acc_full, 1);
        mbar_init(&ctrl->acc_free, 8);
        mbar_init(&ctrl->tail, 1);
        ctrl->abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 8) {
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

    // Registers: launched with 512 x 128; 256 x 168 + 128 x 72 + 128 x 104 = the same 65536.
    if (warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;\n" ::);
        // ================ Q and dO to tensor memory, row by row; D = sum dO O - dLSE on the way ================
        const int r = (warp & 3) * 32 + lane;
        const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        uint32_t n_item = 0;  // items with products so far
        while (bwd_next_item(ctrl, p, k_item, lane, it)) {
            const int i = it.row0 + r, N = bwd_key_tiles(p, it).count;
            const bool row_ok = i < it.sq;
            const int64_t at = ((int64_t)(it.q0 + i) * p.hq + it.h) * HDIM;
            const int64_t lr = (p.seqstart_q ? (int64_t)it.h * p.seqlen_q + it.q0 : ((int64_t)it.b * p.hq + it.h) * p.seqlen_q) + i;
            uint32_t w[HDIM / 64][32];
            auto fetch = [&](const void* src) {
                const uint4* s4 = reinterpret_cast<const uint4*>((const T*)src + at);
#pragma unroll
                for (int v = 0; v < HDIM / 8; ++v) {
                    const uint4 x = row_ok ? s4[v] : make_uint4(0u, 0u, 0u, 0u);
                    w[v / 8][4 * (v % 8)] = x.x; w[v / 8][4 * (v % 8) + 1] = x.y; w[v / 8][4 * (v % 8) + 2] = x.z; w[v / 8][4 * (v % 8) + 3] = x.w;
                }
            };
            auto put = [&](int which, uint32_t col) -> bool {
                if (!__all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->own_free[which], (n_item & 1u) ^ 1u, abort_flag, p.status, 0x10010))) return false;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < HDIM / 64; ++c) tmem_st32(lane_addr + col + c * 32, w[c]);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctrl->own_full[which]);
                return true;
            };
            float lse2 = INFINITY, dlse = 0.f;
            if (N > 0) {
                fetch(p.q);
                if (row_ok) lse2 = bwd_lse_base2(p.lse[lr]);
                if (!put(0, cQ)) break;
            }
            fetch(p.dout);
            if (row_ok && p.dlse) dlse = p.dlse[lr];
            float delta = 0.f;
            const uint4* osrc = reinterpret_cast<const uint4*>((const T*)p.o + at);
#pragma unroll
            for (int v = 0; v < HDIM / 8; ++v) {
                const uint4 y = row_ok ? osrc[v] : make_uint4(0u, 0u, 0u, 0u);
                const uint32_t yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 a = bias_pair<T>(w[v / 8][4 * (v % 8) + e]), o2 = bias_pair<T>(yw[e]);
                    delta = fmaf(a.x, o2.x, fmaf(a.y, o2.y, delta));
                }
            }
            delta -= dlse;
            if (row_ok) p.delta[lr] = delta;
            if (N == 0) continue;
            const int slot = n_item & 1;
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->row_empty[slot], ((n_item >> 1) & 1u) ^ 1u, abort_flag, p.status, 0x10011))) break;
            sRow[slot * 256 + r] = lse2;
            sRow[slot * 256 + 128 + r] = delta;
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctrl->row_full[slot]);
            if (!put(1, cDO)) break;
            ++n_item;
        }
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n" ::);
        if (warp == 11) {
            bwd_schedule<true>(ctrl, p, lane);
        } else if (warp == 9) {
            // ================================ TMA producer ================================
            uint32_t tails = 0, t = 0;
            bool ok = true;
            while (ok && bwd_next_item(ctrl, p, k_item, lane, it)) {
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
                }
            }
        } else {
            // ================================ MMA issuers: 8 S and dP, 10 dQ ================================
            // All lanes walk the loop, the elected one issues.
            const bool leader = elect_one_sync();
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
                return ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag, p.status, code)) != 0;
            };
            auto commit = [&](uint64_t* bar) { if (leader) umma_commit(bar); };
            auto at = [&](uint64_t d, uint32_t bytes) { return d + (uint64_t)(bytes >> 4); };
            uint32_t t = 0, ks = 0, kph = 0, n_item = 0;  // steps so far, K slot and its phase, items with steps so far
            if (warp == 8) {
                constexpr uint32_t idesc_s = make_idesc<T>(false, 64);
                const uint64_t dK = make_smem_desc(smem_u32(sK), 0, 1024), dV = make_smem_desc(smem_u32(sV), 0, 1024);
                while (ok && bwd_next_item(ctrl, p, k_item, lane, it)) {
                    const int N = bwd_key_tiles(p, it).count;
                    for (int j = 0; j < N; ++j) {
                        const uint32_t vs = t & 1u;
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            if (half == 0) {
                                if (j == 0 && !wait(&ctrl->own_full[0], n_item & 1u, 0x10030)) break;
                                if (!wait(&ctrl->a_full[ks], kph, 0x10031)) break;
                            }
                            if (t > 0 && !wait(&ctrl->s_free[half], (t - 1) & 1u, 0x10032)) break;
                            tc_fence_after();
                            if (leader) bwd_issue_ts<HDIM>(tmem + cS + half * 64, tmem + cQ, at(dK, ks * TILE + half * 8192), idesc_s);
                            commit(&ctrl->s_full[half]);
                            if (half == 1 && j + 1 == N) commit(&ctrl->own_free[0]);
                            if (half == 0) {
                                if (j == 0 && !wait(&ctrl->own_full[1], n_item & 1u, 0x10033)) break;
                                if (!wait(&ctrl->b_full[vs], (t >> 1) & 1u, 0x10034)) break;
                            }
                            if (t > 0 && !wait(&ctrl->x_done[half], (t - 1) & 1u, 0x10035)) break;
                            tc_fence_after();
                            if (leader) bwd_issue_ts<HDIM>(tmem + cDP + half * 64, tmem + cDO, at(dV, vs * TILE + half * 8192), idesc_s);
                            commit(&ctrl->dp_full[half]);
                        }
                        if (!ok) break;
                        commit(&ctrl->b_empty[vs]);
                        if (j + 1 == N) commit(&ctrl->own_free[1]);
                        ++t;
                        if (++ks == KS) { ks = 0; kph ^= 1u; }
                    }
                    if (N > 0) ++n_item;
                }
            } else {
                constexpr uint32_t idesc_q = make_idesc<T>(true, HDIM);
                const uint64_t dKt = make_smem_desc(smem_u32(sK), HALF_BYTES, 1024);
                while (ok && bwd_next_item(ctrl, p, k_item, lane, it)) {
                    const int N = bwd_key_tiles(p, it).count;
                    if (N > 0 && n_item > 0 && !wait(&ctrl->acc_free, (n_item - 1) & 1u, 0x10036)) break;
                    for (int j = 0; j < N; ++j) {
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            if (!wait(&ctrl->ds_full[half], t & 1u, 0x10037)) break;
                            tc_fence_after();
                            if (leader) bwd_issue_xb(tmem + cDQ, tmem + cDP, at(dKt, ks * TILE), idesc_q, half, j + half > 0);
                            commit(&ctrl->x_done[half]);
                        }
                        if (!ok) break;
                        commit(&ctrl->a_empty[ks]);
                        ++t;
                        if (++ks == KS) ks = 0;
                    }
                    if (!ok) break;
                    if (N > 0) { commit(&ctrl->acc_full); ++n_item; }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 168;\n" ::);
        const int half = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t tS = lane_addr + cS + half * 64, tDP = lane_addr + cDP + half * 64;
        uint32_t t = 0, n_item = 0;
        bool ok = true;
        while (ok && bwd_next_item(ctrl, p, k_item, lane, it)) {
            const int i = it.row0 + r, shift = p.mask_type == 2 ? it.sk - it.sq : 0;
            const BwdRange range = bwd_key_tiles(p, it);
            const bool row_ok = i < it.sq;
            T* dst = (T*)p.dq + ((int64_t)(it.q0 + i) * p.hq + it.h) * HDIM + half * (HDIM / 2);
            if (range.count == 0) {  // no row of the tile sees a key
                if (row_ok)
#pragma unroll
                    for (int v = 0; v < HDIM / 16; ++v) reinterpret_cast<uint4*>(dst)[v] = make_uint4(0u, 0u, 0u, 0u);
                continue;
            }
            const int slot = n_item & 1;
            if (!(ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->row_full[slot], (n_item >> 1) & 1u, abort_flag, p.status, 0x10040)))) break;
            const float lse2 = sRow[slot * 256 + r], delta = sRow[slot * 256 + 128 + r];
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctrl->row_empty[slot]);
            const float slope = EXTRA && p.alibi ? p.alibi[(p.alibi_rank ? it.b * p.hq : 0) + it.h] * kLog2e : 0.f;
            // visible keys of this row; key tiles that every row of the tile sees whole
            const int k_lo = p.mask_type != 0 && p.wl >= 0 ? i + shift - p.wl : 0;
            const int k_hi = p.mask_type != 0 && p.wr >= 0 ? min(it.sk - 1, i + shift + p.wr) : it.sk - 1;
            int full_lo = 0, full_hi = it.sk - 1;
            if (p.mask_type != 0) {
                if (p.wl >= 0) full_lo = max(0, min(it.sq, it.row0 + 128) - 1 + shift - p.wl);
                if (p.wr >= 0) full_hi = min(full_hi, it.row0 + shift + p.wr);
            }
            const float2 neg_lse2 = make_float2(-lse2, -lse2), neg_delta = make_float2(-delta, -delta);
            auto step = [&](int j, auto masked) -> bool {
                const int key0 = (range.begin + j) * 128 + half * 64;
                if (!__all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->s_full[half], t & 1u, abort_flag, p.status, 0x10041))) return false;
                tc_fence_after();
                uint32_t x[2][32];
                tmem_ld32(tS, x[0]);
                tmem_ld32(tS + 32, x[1]);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctrl->s_free[half]);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    if constexpr (EXTRA) {
                        if (p.soft_cap > 0.f) soft_cap_scores<32>(x[c], p.cap);
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        float2 f = make_float2(1.f, 1.f), away = f;
                        if constexpr (EXTRA) {
                            away.x = (float)(i + it.sk - it.sq - (key0 + c * 32 + e));
                            away.y = away.x - 1.f;
                        }
                        const float2 y = bwd_exponent<EXTRA>(p, make_float2(__uint_as_float(x[c][e]), __uint_as_float(x[c][e + 1])), slope, away, neg_lse2, f);
                        float2 pr = bwd_exp2(y, e / 2);
                        if constexpr (EXTRA) pr = __fmul2_rn(pr, f);
                        x[c][e] = __float_as_uint(pr.x);
                        x[c][e + 1] = __float_as_uint(pr.y);
                    }
                }
                if (!__all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->dp_full[half], t & 1u, abort_flag, p.status, 0x10042))) return false;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t dp[32], w[16];
                    tmem_ld32(tDP + c * 32, dp);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const float2 d = __fadd2_rn(make_float2(__uint_as_float(dp[e]), __uint_as_float(dp[e + 1])), neg_delta);
                        float2 ds = __fmul2_rn(make_float2(__uint_as_float(x[c][e]), __uint_as_float(x[c][e + 1])), d);
                        if constexpr (decltype(masked)::value) {
                            const int key = key0 + c * 32 + e;
                            if (key < k_lo || key > k_hi) ds.x = 0.f;
                            if (key + 1 < k_lo || key + 1 > k_hi) ds.y = 0.f;
                        }
                        w[e / 2] = Elem<T>::pack2(ds.x, ds.y);
                    }
                    tmem_st16(tDP + c * 16, w);  // (over columns of dP that this warp has read)
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctrl->ds_full[half]);
                ++t;
                return true;
            };
            for (int j = 0; ok && j < range.count; ++j) {
                const int n0 = (range.begin + j) * 128;
                ok = n0 < full_lo || n0 + 127 > full_hi ? step(j, std::true_type{}) : step(j, std::false_type{});
            }
            if (!ok || !(ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->acc_full, n_item & 1u, abort_flag, p.status, 0x10043)))) break;
            ++n_item;
            tc_fence_after();
            uint32_t acc[HDIM / 64][32];
#pragma unroll
            for (int c = 0; c < HDIM / 64; ++c) tmem_ld32(lane_addr + cDQ + half * (HDIM / 2) + c * 32, acc[c]);
            tmem_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctrl->acc_free);
            if (row_ok)
#pragma unroll
                for (int c = 0; c < HDIM / 64; ++c) bwd_store32<T>(dst + c * 32, acc[c], p.scale);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem));
    }
}

// ---- dK / dV --------------------------------------------------------------------------------------------------------------
constexpr int kBwdDkdvThreads = 512;

template <typename T, int HDIM, bool EXTRA>
__global__ void __launch_bounds__(kBwdDkdvThreads, 1)
bwd_dkdv_sm100_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                      const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const BwdSm100Dev p) {
    constexpr int TILE = 128 * HDIM * 2, QS = 3, OS = 2;
    constexpr uint32_t cDV = 256, cDK = 384;  // columns 0-127 and 128-255: the two regions
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* sK = smem_raw;  // (no room for slack: that it starts on a 1024-byte boundary is checked below)
    uint8_t* sV = sK + TILE;
    uint8_t* sQ = sV + TILE;
    uint8_t* sDO = sQ + QS * TILE;
    float* sRow = reinterpret_cast<float*>(sDO + OS * TILE);  // [2 steps][LSE 128 | D 128] of the query columns
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
            mbar_init(&ctrl->item_empty[i], 12);  // every warp but the scheduling and the idle ones
        }
        for (int i = 0; i < QS; ++i) { mbar_init(&ctrl->a_full[i], 1); mbar_init(&ctrl->a_empty[i], 1); }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&ctrl->b_full[i], 1);
            mbar_init(&ctrl->b_empty[i], 2);  // both products that read dO
            mbar_init(&ctrl->own_full[i], 1);
            mbar_init(&ctrl->own_free[i], 1);
            mbar_init(&ctrl->row_full[i], 1);
            mbar_init(&ctrl->row_empty[i], 8);
            mbar_init(&ctrl->p_full[i], 8);
        }
        mbar_init(&ctrl->s_full[0], 1);
        mbar_init(&ctrl->s_free[0], 8);
        mbar_init(&ctrl->dp_full[0], 1);
        mbar_init(&ctrl->ds_full[0], 8);
        mbar_init(&ctrl->x_done[0], 1);
        mbar_init(&ctrl->acc_full, 1);
        mbar_init(&ctrl->acc_free, 8);
        mbar_init(&ctrl->tail, 1);
        ctrl->abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_u32(&ctrl->tmem_base)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctrl->tmem_base;
    uint32_t k_item = 0;
    BwdItem it{};

    // Registers: launched with 512 x 128 = 256 x 192 + 256 x 64.
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;\n" ::);
        if (warp == 11) {
            bwd_schedule<false>(ctrl, p, lane);
        } else if (warp == 9) {
            // ================================ TMA producer ================================
            uint32_t tails = 0, t = 0, n_item = 0;
            bool ok = true;
            auto own = [&](int which, uint8_t* dst, const CUtensorMap* map) -> bool {
                if (!__all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->own_free[which], (n_item & 1u) ^ 1u, abort_flag, p.status, 0x10120))) return false;
                // (rows behind the end of the keys stay in their own rows of the gradients, which are not stored)
                return bwd_load_tile<HDIM>(dst, map, &ctrl->own_full[which], &ctrl->tail, tails, it.h, it.k0 + it.row0, 128, lane, abort_flag, p.status);
            };
            while (ok && bwd_next_item(ctrl, p, k_item, lane, it)) {
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
        } else if (warp == 10) {
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
        } else if (warp == 8 || warp == 12) {
            // ================================ MMA issuers: 8 S and dP, 12 dV and dK ================================
            const bool leader = elect_one_sync();
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
                return ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag, p.status, code)) != 0;
            };
            auto commit = [&](uint64_t* bar) { if (leader) umma_commit(bar); };
            auto at = [&](uint64_t d, uint32_t bytes) { return d + (uint64_t)(bytes >> 4); };
            uint32_t t = 0, qs = 0, qph = 0, n_item = 0;  // steps so far, Q slot and its phase, items with steps so far
            if (warp == 8) {
                constexpr uint32_t idesc_s = make_idesc<T>(false);
                const uint64_t dK = make_smem_desc(smem_u32(sK), 0, 1024), dV = make_smem_desc(smem_u32(sV), 0, 1024);
                const uint64_t dQ = make_smem_desc(smem_u32(sQ), 0, 1024), dDO = make_smem_desc(smem_u32(sDO), 0, 1024);
                while (ok && bwd_next_item(ctrl, p, k_item, lane, it)) {
                    const int N = bwd_query_tiles(p, it).count * G;
                    for (int j = 0; j < N; ++j) {
                        const uint32_t os = t & 1u;
                        if (j == 0 && !wait(&ctrl->own_full[0], n_item & 1u, 0x10130)) break;
                        if (!wait(&ctrl->a_full[qs], qph, 0x10131)) break;
                        if (t > 0 && !wait(&ctrl->s_free[0], (t - 1) & 1u, 0x10132)) break;  // dP(t - 1) has been read from the region
                        tc_fence_after();
                        if (leader) bwd_issue_ss<HDIM>(tmem + (t & 1u) * 128, dK, at(dQ, qs * TILE), idesc_s);
                        commit(&ctrl->s_full[0]);
                        if (j + 1 == N) commit(&ctrl->own_free[0]);
                        if (j == 0 && !wait(&ctrl->own_full[1], n_item & 1u, 0x10133)) break;
                        if (!wait(&ctrl->b_full[os], (t >> 1) & 1u, 0x10134)) break;
                        if (t > 0 && !wait(&ctrl->x_done[0], (t - 1) & 1u, 0x10135)) break;  // P(t - 1) and dS(t - 1) have been used
                        tc_fence_after();
                        if (leader) bwd_issue_ss<HDIM>(tmem + ((t + 1) & 1u) * 128, dV, at(dDO, os * TILE), idesc_s);
                        commit(&ctrl->dp_full[0]);
                        commit(&ctrl->b_empty[os]);
                        if (j + 1 == N) commit(&ctrl->own_free[1]);
                        ++t;
                        if (++qs == QS) { qs = 0; qph ^= 1u; }
                    }
                    if (N > 0) ++n_item;
                }
            } else {
                constexpr uint32_t idesc_o = make_idesc<T>(true, HDIM);
                const uint64_t dQt = make_smem_desc(smem_u32(sQ), HALF_BYTES, 1024), dDOt = make_smem_desc(smem_u32(sDO), HALF_BYTES, 1024);
                while (ok && bwd_next_item(ctrl, p, k_item, lane, it)) {
                    const int N = bwd_query_tiles(p, it).count * G;
                    if (N > 0 && n_item > 0 && !wait(&ctrl->acc_free, (n_item - 1) & 1u, 0x10136)) break;
                    for (int j = 0; j < N; ++j) {
                        const uint32_t region = tmem + (t & 1u) * 128;  // P in its columns 0-31 and 64-95, dS in 32-63 and 96-127
                        const uint32_t os = t & 1u;
                        if (!wait(&ctrl->b_full[os], (t >> 1) & 1u, 0x10139)) break;  // (dP may still be waiting for this dO)
                        if (!wait(&ctrl->p_full[t & 1u], (t >> 1) & 1u, 0x10137)) break;
                        tc_fence_after();
                        if (leader) {
                            bwd_issue_xb(tmem + cDV, region, at(dDOt, os * TILE), idesc_o, 0, j > 0);
                            bwd_issue_xb(tmem + cDV, region, at(dDOt, os * TILE), idesc_o, 1, true);
                        }
                        commit(&ctrl->b_empty[os]);
                        if (!wait(&ctrl->ds_full[0], t & 1u, 0x10138)) break;
                        tc_fence_after();
                        if (leader) {
                            bwd_issue_xb(tmem + cDK, region + 32, at(dQt, qs * TILE), idesc_o, 0, j > 0);
                            bwd_issue_xb(tmem + cDK, region + 32, at(dQt, qs * TILE), idesc_o, 1, true);
                        }
                        commit(&ctrl->x_done[0]);
                        commit(&ctrl->a_empty[qs]);
                        ++t;
                        if (++qs == QS) qs = 0;
                    }
                    if (!ok) break;
                    if (N > 0) { commit(&ctrl->acc_full); ++n_item; }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 192;\n" ::);
        const int half = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16) + half * 64;
        uint32_t t = 0, n_item = 0;
        bool ok = true;
        while (ok && bwd_next_item(ctrl, p, k_item, lane, it)) {
            const int key = it.row0 + r, shift = p.mask_type == 2 ? it.sk - it.sq : 0;
            const BwdRange range = bwd_query_tiles(p, it);
            T* dst = (T*)(half ? p.dk : p.dv) + ((int64_t)(it.k0 + key) * p.hkv + it.h) * HDIM;  // warps 0-3 store dV, 4-7 dK
            if (range.count == 0) {  // nobody sees these keys
                if (key < it.sk)
#pragma unroll
                    for (int v = 0; v < HDIM / 8; ++v) reinterpret_cast<uint4*>(dst)[v] = make_uint4(0u, 0u, 0u, 0u);
                continue;
            }
            // query rows that see all of the tile's keys
            int full_lo = 0, full_hi = 0x3fffffff;
            if (p.mask_type != 0) {
                if (p.wr >= 0) full_lo = it.row0 + 127 - shift - p.wr;
                if (p.wl >= 0) full_hi = it.row0 - shift + p.wl;
            }
            auto step = [&](int m0, float slope, auto masked) -> bool {
                // columns of this half that see the key: i >= key - shift - wr, i <= key - shift + wl
                int c_lo = 0, c_hi = 0x3fffffff;
                if constexpr (decltype(masked)::value) {
                    const int i0 = m0 + half * 64;
                    c_lo = p.wr >= 0 ? key - shift - p.wr - i0 : 0;
                    c_hi = p.wl >= 0 ? key - shift + p.wl - i0 : 0x3fffffff;
                }
                const float* rows = sRow + (t & 1) * 256 + half * 64;
                const uint32_t tS = lane_addr + (t & 1u) * 128, tDP = lane_addr + ((t + 1) & 1u) * 128;
                if (!__all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->row_full[t & 1], (t >> 1) & 1u, abort_flag, p.status, 0x10140))) return false;
                if (!__all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->s_full[0], t & 1u, abort_flag, p.status, 0x10141))) return false;
                tc_fence_after();
                uint32_t x[2][32];
                tmem_ld32(tS, x[0]);
                tmem_ld32(tS + 32, x[1]);
                tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t w[16];
                    if constexpr (EXTRA) {
                        if (p.soft_cap > 0.f) soft_cap_scores<32>(x[c], p.cap);
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const float4 l4 = *reinterpret_cast<const float4*>(rows + c * 32 + e);
#pragma unroll
                        for (int u = 0; u < 4; u += 2) {
                            const int col = c * 32 + e + u;
                            float2 f = make_float2(1.f, 1.f), away = f;
                            if constexpr (EXTRA) {
                                away.x = (float)(m0 + half * 64 + col + it.sk - it.sq - key);
                                away.y = away.x + 1.f;
                            }
                            const float2 y = bwd_exponent<EXTRA>(p, make_float2(__uint_as_float(x[c][e + u]), __uint_as_float(x[c][e + u + 1])), slope,
                                                                 away, u ? make_float2(l4.z, l4.w) : make_float2(l4.x, l4.y), f);
                            float2 pr = bwd_exp2(y, (e + u) / 2);
                            if constexpr (decltype(masked)::value) {
                                if (col < c_lo || col > c_hi) pr.x = 0.f;
                                if (col + 1 < c_lo || col + 1 > c_hi) pr.y = 0.f;
                            }
                            w[(e + u) / 2] = Elem<T>::pack2(pr.x, pr.y);
                            if constexpr (EXTRA) pr = __fmul2_rn(pr, f);  // (from here on P serves dS alone)
                            x[c][e + u] = __float_as_uint(pr.x);
                            x[c][e + u + 1] = __float_as_uint(pr.y);
                        }
                    }
                    tmem_st16(tS + c * 16, w);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctrl->p_full[t & 1u]);
                if (!__all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->dp_full[0], t & 1u, abort_flag, p.status, 0x10142))) return false;
                tc_fence_after();
                uint32_t dp[2][32];
                tmem_ld32(tDP, dp[0]);
                tmem_ld32(tDP + 32, dp[1]);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctrl->s_free[0]);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t w[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const float4 d4 = *reinterpret_cast<const float4*>(rows + 128 + c * 32 + e);
#pragma unroll
                        for (int u = 0; u < 4; u += 2) {
                            const float2 d = __fadd2_rn(make_float2(__uint_as_float(dp[c][e + u]), __uint_as_float(dp[c][e + u + 1])),
                                                        u ? make_float2(d4.z, d4.w) : make_float2(d4.x, d4.y));
                            const float2 ds = __fmul2_rn(make_float2(__uint_as_float(x[c][e + u]), __uint_as_float(x[c][e + u + 1])), d);
                            w[(e + u) / 2] = Elem<T>::pack2(ds.x, ds.y);
                        }
                    }
                    tmem_st16(tS + 32 + c * 16, w);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&ctrl->ds_full[0]);
                    mbar_arrive(&ctrl->row_empty[t & 1]);
                }
                ++t;
                return true;
            };
            for (int g = 0; ok && g < G; ++g) {
                const float slope = EXTRA && p.alibi ? p.alibi[(p.alibi_rank ? it.b * p.hq : 0) + it.h * G + g] * kLog2e : 0.f;
                for (int m = 0; ok && m < range.count; ++m) {
                    const int m0 = (range.begin + m) * 128;
                    ok = m0 < full_lo || m0 + 127 > full_hi ? step(m0, slope, std::true_type{}) : step(m0, slope, std::false_type{});
                }
            }
            if (!ok || !(ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->acc_full, n_item & 1u, abort_flag, p.status, 0x10143)))) break;
            ++n_item;
            tc_fence_after();
            uint32_t acc[HDIM / 32][32];
#pragma unroll
            for (int c = 0; c < HDIM / 32; ++c) tmem_ld32(lane_addr - half * 64 + (half ? cDK : cDV) + c * 32, acc[c]);
            tmem_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctrl->acc_free);
            if (key < it.sk)
#pragma unroll
                for (int c = 0; c < HDIM / 32; ++c) bwd_store32<T>(dst + c * 32, acc[c], half ? p.scale : 1.f);
        }
    }
    pdl_wait();
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem));
    }
}

}  // namespace sm100

}  // namespace fck
