// Backward of fmha_fwd on tcgen05 (formulas and the ownership of the sums: fmha_bwd_generic.cu).  hdim 128 / 64, every mask, batch
// and group mode, GQA, ALiBi, soft cap.  Two kernels, each with one 128-row tile per CTA whose gradient stays in tensor memory:
//
//   dQ   (bwd_dq_sm100_kernel):    128 queries of one head walk the key tiles:    S = Q K^T, dP = dO V^T, dQ += dS K
//   dK/dV (bwd_dkdv_sm100_kernel): 128 keys of one kv head walk the query tiles of the group's heads, transposed:
//                                  S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q
//
// Seven products where one pass with a shared sum for dQ has five; but that pass pays 64 KB of fp32 reductions per tile pair and
// order-dependent results.  Counted in the 128 bytes a clock of shared memory, which feeds both operands of an SS product and
// one of a TS product (128 x 128 x 128: 512 clocks of the tensor pipe, 512 or 256 of shared memory): dQ 3 x 256 + K/V copies 512
// = 1280 clocks beside 1536 of products (Q and dO live in tensor memory, so all three products are TS); dK/dV 2 x 512 + 2 x 256 +
// 512 = 2048 beside 2048.  P and dS go from registers to tensor memory as A operands and never through shared memory.
//
// Roles: warps 0-7 the elementwise work (thread = tensor memory lane = row; warps 0-3 take columns 0-63 of a tile, 4-7 64-127),
// warp 8 issues the products, warp 9 the TMA copies, warp 10 (dK/dV) fetches LSE and D of the query columns.  The products are
// ordered so that the pipe always has one to run while the elementwise warps work on another's result:
//   dQ:     S(j+1) | dQ(j) | dP(j+1)            dK/dV:  dV(i) | S(i+1) | dK(i) | dP(i+1)
// P^T lies over the columns of S^T, dS over those of dP, each warp's 64 columns in its own half.
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
    float cap, cap_log2, two_inv_cap_log2;  // soft cap c: c, c log2(e), 2 log2(e) / c times the scale
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
__device__ __forceinline__ int64_t bwd_lse_row(const BwdSm100Dev& p, const BwdSeq& s, int b, int h) {
    return p.seqstart_q ? (int64_t)h * p.seqlen_q + s.q0 : ((int64_t)b * p.hq + h) * p.seqlen_q;
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
// D += X B over 128 rows: X in tensor memory, its first 64 K elements from column a, the others from a + 64; B MN-major.
__device__ __forceinline__ void bwd_issue_xb(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
#pragma unroll
    for (int ks = 0; ks < 8; ++ks)
        umma_ts(d, a + (ks / 4) * 64 + (ks % 4) * 8, b + (uint64_t)((ks * 2048) >> 4), idesc, (accumulate || ks > 0) ? 1u : 0u);
}

// x (raw scores) -> exponents in base 2 without the LSE; with a soft cap, f is what dS gets from it (1 - tanh^2).
template <bool EXTRA>
__device__ __forceinline__ float2 bwd_exponent(const BwdSm100Dev& p, float2 x, float slope_log2, float2 away, float2 lse2, float2& f) {
    if constexpr (!EXTRA) return __ffma2_rn(x, make_float2(p.scale_log2, p.scale_log2), make_float2(-lse2.x, -lse2.y));
    float2 y;
    if (p.cap > 0.f) {  // tanh(z) = 1 - 2 / (1 + e^2z), from the side on which nothing cancels
        const float2 z = __fmul2_rn(x, make_float2(p.two_inv_cap_log2, p.two_inv_cap_log2));
        auto tanh_of = [](float w) {
            const float e = ex2_fast(-fabsf(w));
            return copysignf(__fdividef(1.f - e, 1.f + e), w);
        };
        const float2 t = make_float2(tanh_of(z.x), tanh_of(z.y));
        y = __fmul2_rn(t, make_float2(p.cap_log2, p.cap_log2));
        f = __ffma2_rn(make_float2(-t.x, -t.y), t, make_float2(1.f, 1.f));
    } else {
        y = __fmul2_rn(x, make_float2(p.scale_log2, p.scale_log2));
    }
    y = __ffma2_rn(make_float2(-slope_log2, -slope_log2), make_float2(fabsf(away.x), fabsf(away.y)), y);
    return __fadd2_rn(y, make_float2(-lse2.x, -lse2.y));
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

struct BwdCtrl {
    uint64_t a_full[3], a_empty[3], b_full[2], b_empty[2];  // rings: dQ K / V; dK/dV Q / dO
    uint64_t own_full;          // dK/dV: the CTA's K and V tiles; dQ: Q and dO are in tensor memory
    uint64_t s_full, s_free, p_full, dp_full, ds_full, acc_full, tail;
    uint64_t row_full[2], row_empty[2];
    uint32_t tmem_base;
    int abort_flag;
};

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

constexpr int kBwdThreads = 384;

// ---- dQ -----------------------------------------------------------------------------------------------------------------
template <typename T, int HDIM, bool EXTRA>
__global__ void __launch_bounds__(kBwdThreads, 1)
bwd_dq_sm100_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const BwdSm100Dev p) {
    constexpr int TILE = 128 * HDIM * 2, KS = 3, VS = 2;
    constexpr uint32_t cS = 0, cDP = 128, cDQ = 256, cQ = 384, cDO = 448;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
    uint8_t* sK = base;
    uint8_t* sV = sK + KS * TILE;
    float* sDelta = reinterpret_cast<float*>(sV + VS * TILE);
    BwdCtrl* ctrl = reinterpret_cast<BwdCtrl*>(sDelta + 128);
    volatile int* abort_flag = &ctrl->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // work item: heads of a (sequence, row tile) side by side (they share K/V through L2), the last row tiles first
    const int per_tile = p.hq * p.batch, mt = gridDim.x / per_tile;
    const int tile = mt - 1 - (int)blockIdx.x / per_tile, rest = (int)blockIdx.x % per_tile, b = rest / p.hq, h = rest % p.hq;
    const int kh = h / (p.hq / p.hkv), m0 = tile * 128;

    pdl_wait();
    pdl_launch_dependents();
    bwd_zero_outside<HDIM>(p);
    const BwdSeq s = bwd_sequence(p, b);
    if (m0 >= s.sq) return;
    if (threadIdx.x == 0) {
        for (int i = 0; i < KS; ++i) { mbar_init(&ctrl->a_full[i], 1); mbar_init(&ctrl->a_empty[i], 1); }
        for (int i = 0; i < VS; ++i) { mbar_init(&ctrl->b_full[i], 1); mbar_init(&ctrl->b_empty[i], 1); }
        mbar_init(&ctrl->own_full, 8);
        mbar_init(&ctrl->s_full, 1);
        mbar_init(&ctrl->s_free, 8);
        mbar_init(&ctrl->dp_full, 1);
        mbar_init(&ctrl->ds_full, 8);
        mbar_init(&ctrl->acc_full, 1);
        mbar_init(&ctrl->tail, 1);
        ctrl->abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_u32(&ctrl->tmem_base)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    }
    int n_begin = 0, N = 0;  // key tiles that some row sees
    {
        int lo = 0, hi = s.sk - 1;
        if (p.mask_type != 0) {
            if (p.wl >= 0) lo = max(lo, m0 + s.shift - p.wl);
            if (p.wr >= 0) hi = min(hi, min(s.sq, m0 + 128) - 1 + s.shift + p.wr);
        }
        if (hi >= lo) {
            n_begin = lo / 128;
            N = hi / 128 + 1 - n_begin;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctrl->tmem_base;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;\n" ::);
        if (warp == 9) {
            // ================================ TMA producer ================================
            uint32_t tails = 0;
            for (int j = 0; j < N; ++j) {
                const int n0 = (n_begin + j) * 128, ks = j % KS, vs = j % VS;
                if (!__all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->a_empty[ks], ((j / KS) & 1u) ^ 1u, abort_flag, p.status, 0x10001))) break;
                // (K rows behind the end meet dS = 0; those of V only make columns of dP that are masked by index)
                if (!bwd_load_tile<HDIM>(sK + ks * TILE, &map_k, &ctrl->a_full[ks], &ctrl->tail, tails, kh, s.k0 + n0, s.sk - n0, lane,
                                         abort_flag, p.status)) break;
                if (!__all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->b_empty[vs], ((j / VS) & 1u) ^ 1u, abort_flag, p.status, 0x10002))) break;
                bwd_load_tile<HDIM>(sV + vs * TILE, &map_v, &ctrl->b_full[vs], &ctrl->tail, tails, kh, s.k0 + n0, 128, lane, abort_flag, p.status);
            }
        } else if (warp == 8 && N > 0) {
            // ================================ MMA issuer ================================
            constexpr uint32_t idesc_s = make_idesc<T>(false), idesc_q = make_idesc<T>(true, HDIM);
            const bool leader = elect_one_sync();
            auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
                return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag, p.status, code)) != 0;
            };
            auto commit = [&](uint64_t* bar) { if (leader) umma_commit(bar); };
            const uint64_t dK = make_smem_desc(smem_u32(sK), 0, 1024), dV = make_smem_desc(smem_u32(sV), 0, 1024);
            const uint64_t dKt = make_smem_desc(smem_u32(sK), HALF_BYTES, 1024);
            auto at = [&](uint64_t d, int slot) { return d + (uint64_t)((slot * TILE) >> 4); };
            bool ok = wait(&ctrl->own_full, 0, 0x10010) && wait(&ctrl->a_full[0], 0, 0x10011);
            if (ok) {
                tc_fence_after();
                if (leader) bwd_issue_ts<HDIM>(tmem + cS, tmem + cQ, at(dK, 0), idesc_s);
                commit(&ctrl->s_full);
                ok = wait(&ctrl->b_full[0], 0, 0x10012);
            }
            if (ok) {
                if (leader) bwd_issue_ts<HDIM>(tmem + cDP, tmem + cDO, at(dV, 0), idesc_s);
                commit(&ctrl->dp_full);
                commit(&ctrl->b_empty[0]);
            }
            for (int j = 0; ok && j < N; ++j) {
                const int ks1 = (j + 1) % KS, vs1 = (j + 1) % VS;
                if (j + 1 < N) {
                    if (!(ok = wait(&ctrl->a_full[ks1], ((j + 1) / KS) & 1u, 0x10011))) break;
                    if (!(ok = wait(&ctrl->s_free, j & 1u, 0x10013))) break;
                    tc_fence_after();
                    if (leader) bwd_issue_ts<HDIM>(tmem + cS, tmem + cQ, at(dK, ks1), idesc_s);
                    commit(&ctrl->s_full);
                    if (!(ok = wait(&ctrl->b_full[vs1], ((j + 1) / VS) & 1u, 0x10012))) break;
                }
                if (!(ok = wait(&ctrl->ds_full, j & 1u, 0x10014))) break;
                tc_fence_after();
                if (leader) bwd_issue_xb(tmem + cDQ, tmem + cDP, at(dKt, j % KS), idesc_q, j > 0);
                commit(&ctrl->a_empty[j % KS]);
                if (j + 1 < N) {
                    if (leader) bwd_issue_ts<HDIM>(tmem + cDP, tmem + cDO, at(dV, vs1), idesc_s);
                    commit(&ctrl->dp_full);
                    commit(&ctrl->b_empty[vs1]);
                } else {
                    commit(&ctrl->acc_full);
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;\n" ::);
        const int half = warp >> 2, r = (warp & 3) * 32 + lane, i = m0 + r;
        const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const bool row_ok = i < s.sq;
        const int64_t at = ((int64_t)(s.q0 + i) * p.hq + h) * HDIM;
        // Q (warps 0-3) and dO (warps 4-7) to tensor memory, row by row; D from dO and O on the way
        float delta = 0.f;
#pragma unroll
        for (int c = 0; c < HDIM / 64; ++c) {
            uint32_t w[32];
            const uint4* src = reinterpret_cast<const uint4*>((const T*)(half ? p.dout : p.q) + at) + c * 8;
#pragma unroll
            for (int v = 0; v < 8; ++v) {
                const uint4 x = row_ok ? src[v] : make_uint4(0u, 0u, 0u, 0u);
                w[4 * v] = x.x; w[4 * v + 1] = x.y; w[4 * v + 2] = x.z; w[4 * v + 3] = x.w;
            }
            tmem_st32(lane_addr + (half ? cDO : cQ) + c * 32, w);
            if (half && row_ok) {
                const uint4* osrc = reinterpret_cast<const uint4*>((const T*)p.o + at) + c * 8;
#pragma unroll
                for (int v = 0; v < 8; ++v) {
                    const uint4 y = osrc[v];
                    const uint32_t yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 a = bias_pair<T>(w[4 * v + e]), o2 = bias_pair<T>(yw[e]);
                        delta = fmaf(a.x, o2.x, fmaf(a.y, o2.y, delta));
                    }
                }
            }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctrl->own_full);
        const int64_t lr = bwd_lse_row(p, s, b, h) + i;
        const float lse2 = row_ok ? bwd_lse_base2(p.lse[lr]) : INFINITY;
        if (half) {
            if (row_ok) {
                if (p.dlse) delta -= p.dlse[lr];
                p.delta[lr] = delta;
            }
            sDelta[r] = delta;
        }
        asm volatile("bar.sync 1, 256;\n" ::: "memory");
        delta = sDelta[r];
        const float slope = EXTRA && p.alibi ? p.alibi[(p.alibi_rank ? b * p.hq : 0) + h] * kLog2e : 0.f;
        // visible keys of this row
        const int k_lo = p.mask_type != 0 && p.wl >= 0 ? i + s.shift - p.wl : 0;
        const int k_hi = p.mask_type != 0 && p.wr >= 0 ? min(s.sk - 1, i + s.shift + p.wr) : s.sk - 1;
        const float2 lse22 = make_float2(lse2, lse2);
        bool ok = true;
        auto step = [&](int j, auto masked) -> bool {
            const int key0 = (n_begin + j) * 128 + half * 64;
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->s_full, j & 1u, abort_flag, p.status, 0x10020))) return false;
            tc_fence_after();
            uint32_t x[2][32];
            tmem_ld32(lane_addr + cS + half * 64, x[0]);
            tmem_ld32(lane_addr + cS + half * 64 + 32, x[1]);
            tmem_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctrl->s_free);
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    float2 f = make_float2(1.f, 1.f), away = f;
                    if constexpr (EXTRA) {
                        away.x = (float)(i + s.sk - s.sq - (key0 + c * 32 + e));
                        away.y = away.x - 1.f;
                    }
                    const float2 y = bwd_exponent<EXTRA>(p, make_float2(__uint_as_float(x[c][e]), __uint_as_float(x[c][e + 1])), slope, away, lse22, f);
                    float2 pr = make_float2(ex2_fast(y.x), ex2_fast(y.y));
                    if constexpr (EXTRA) pr = __fmul2_rn(pr, f);
                    x[c][e] = __float_as_uint(pr.x);
                    x[c][e + 1] = __float_as_uint(pr.y);
                }
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->dp_full, j & 1u, abort_flag, p.status, 0x10021))) return false;
            tc_fence_after();
            uint32_t dp[2][32], w[32];
            tmem_ld32(lane_addr + cDP + half * 64, dp[0]);
            tmem_ld32(lane_addr + cDP + half * 64 + 32, dp[1]);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    const float2 t = __fadd2_rn(make_float2(__uint_as_float(dp[c][e]), __uint_as_float(dp[c][e + 1])), make_float2(-delta, -delta));
                    float2 ds = __fmul2_rn(make_float2(__uint_as_float(x[c][e]), __uint_as_float(x[c][e + 1])), t);
                    if constexpr (decltype(masked)::value) {
                        const int key = key0 + c * 32 + e;
                        if (key < k_lo || key > k_hi) ds.x = 0.f;
                        if (key + 1 < k_lo || key + 1 > k_hi) ds.y = 0.f;
                    }
                    w[c * 16 + e / 2] = Elem<T>::pack2(ds.x, ds.y);
                }
            tmem_st32(lane_addr + cDP + half * 64, w);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctrl->ds_full);
            return true;
        };
        // key tiles that every row of the tile sees whole
        int full_lo = 0, full_hi = s.sk - 1;
        if (p.mask_type != 0) {
            if (p.wl >= 0) full_lo = max(0, min(s.sq, m0 + 128) - 1 + s.shift - p.wl);
            if (p.wr >= 0) full_hi = min(full_hi, m0 + s.shift + p.wr);
        }
        for (int j = 0; ok && j < N; ++j) {
            const int n0 = (n_begin + j) * 128;
            ok = n0 < full_lo || n0 + 127 > full_hi ? step(j, std::true_type{}) : step(j, std::false_type{});
        }
        if (ok && N > 0) {
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->acc_full, 0, abort_flag, p.status, 0x10022));
            tc_fence_after();
        }
        if (ok) {
            T* dst = (T*)p.dq + at + half * (HDIM / 2);
#pragma unroll
            for (int c = 0; c < HDIM / 64; ++c) {
                uint32_t t[32];
                if (N > 0) {
                    tmem_ld32(lane_addr + cDQ + half * (HDIM / 2) + c * 32, t);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) t[e] = 0u;
                }
                if (row_ok) bwd_store32<T>(dst + c * 32, t, p.scale);
            }
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
template <typename T, int HDIM, bool EXTRA>
__global__ void __launch_bounds__(kBwdThreads, 1)
bwd_dkdv_sm100_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                      const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const BwdSm100Dev p) {
    constexpr int TILE = 128 * HDIM * 2, QS = 3, OS = 2;
    constexpr uint32_t cS = 0, cDP = 128, cDV = 256, cDK = 384;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* sK = smem_raw;  // (no room for slack: that it starts on a 1024-byte boundary is checked below)
    uint8_t* sV = sK + TILE;
    uint8_t* sQ = sV + TILE;
    uint8_t* sDO = sQ + QS * TILE;
    float* sRow = reinterpret_cast<float*>(sDO + OS * TILE);  // [2 slots][LSE 128 | D 128]
    BwdCtrl* ctrl = reinterpret_cast<BwdCtrl*>(sRow + 2 * 256);
    volatile int* abort_flag = &ctrl->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // work item: the kv heads of a (sequence, key tile) side by side, the first key tiles (the longest under a causal mask) first
    const int per_tile = p.hkv * p.batch, G = p.hq / p.hkv;
    const int n0 = ((int)blockIdx.x / per_tile) * 128, rest = (int)blockIdx.x % per_tile, b = rest / p.hkv, kh = rest % p.hkv;

    // What this kernel reads has been there since before the dQ kernel in front of it began (that one lets it start only after its
    // own wait), but for D: the warp that fetches D waits for that kernel's end, and every other one before it leaves.
    const BwdSeq s = bwd_sequence(p, b);
    const bool aligned = (smem_u32(smem_raw) & 1023u) == 0;
    if (n0 >= s.sk || !aligned) {
        if (!aligned && threadIdx.x == 0) atomicOr(p.status, 0x10130);
        pdl_wait();
        return;
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < QS; ++i) { mbar_init(&ctrl->a_full[i], 1); mbar_init(&ctrl->a_empty[i], 1); }
        for (int i = 0; i < OS; ++i) {
            mbar_init(&ctrl->b_full[i], 1);
            mbar_init(&ctrl->b_empty[i], 1);
            mbar_init(&ctrl->row_full[i], 1);
            mbar_init(&ctrl->row_empty[i], 8);
        }
        mbar_init(&ctrl->own_full, 1);
        mbar_init(&ctrl->s_full, 1);
        mbar_init(&ctrl->p_full, 8);
        mbar_init(&ctrl->dp_full, 1);
        mbar_init(&ctrl->ds_full, 8);
        mbar_init(&ctrl->acc_full, 1);
        mbar_init(&ctrl->tail, 1);
        ctrl->abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_u32(&ctrl->tmem_base)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    }
    int m_begin = 0, tiles = 0;  // query tiles with a row that sees one of these keys: i + shift - wl <= j <= i + shift + wr
    {
        int lo = 0, hi = s.sq - 1;
        if (p.mask_type != 0) {
            if (p.wr >= 0) lo = max(lo, n0 - s.shift - p.wr);
            if (p.wl >= 0) hi = min(hi, min(s.sk, n0 + 128) - 1 - s.shift + p.wl);
        }
        if (hi >= lo) {
            m_begin = lo / 128;
            tiles = hi / 128 + 1 - m_begin;
        }
    }
    const int N = tiles * G;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctrl->tmem_base;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;\n" ::);
        if (warp == 9) {
            // ================================ TMA producer ================================
            uint32_t tails = 0;
            if (N > 0 && lane == 0) {
                mbar_expect_tx(&ctrl->own_full, 2 * TILE);
#pragma unroll
                for (int hb = 0; hb < HDIM / 64; ++hb) {
                    tma_load_3d(sK + hb * HALF_BYTES, &map_k, &ctrl->own_full, hb * 64, kh, s.k0 + n0);
                    tma_load_3d(sV + hb * HALF_BYTES, &map_v, &ctrl->own_full, hb * 64, kh, s.k0 + n0);
                }
            }
            __syncwarp();
            int g = 0, m = 0;
            for (int it = 0; it < N; ++it) {
                const int m0 = (m_begin + m) * 128, h = kh * G + g, qs = it % QS, os = it % OS;
                if (++m == tiles) { m = 0; ++g; }
                if (!__all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->a_empty[qs], ((it / QS) & 1u) ^ 1u, abort_flag, p.status, 0x10101))) break;
                if (!bwd_load_tile<HDIM>(sQ + qs * TILE, &map_q, &ctrl->a_full[qs], &ctrl->tail, tails, h, s.q0 + m0, s.sq - m0, lane, abort_flag,
                                         p.status)) break;
                if (!__all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->b_empty[os], ((it / OS) & 1u) ^ 1u, abort_flag, p.status, 0x10102))) break;
                if (!bwd_load_tile<HDIM>(sDO + os * TILE, &map_do, &ctrl->b_full[os], &ctrl->tail, tails, h, s.q0 + m0, s.sq - m0, lane, abort_flag,
                                         p.status)) break;
            }
        } else if (warp == 10) {
            // ================================ LSE and D of the query columns ================================
            pdl_wait();
            int g = 0, m = 0;
            for (int it = 0; it < N; ++it) {
                const int m0 = (m_begin + m) * 128, slot = it & 1;
                const int64_t lr = bwd_lse_row(p, s, b, kh * G + g) + m0;
                if (++m == tiles) { m = 0; ++g; }
                float l[4], d[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int c = u * 32 + lane;
                    l[u] = m0 + c < s.sq ? bwd_lse_base2(p.lse[lr + c]) : INFINITY;
                    d[u] = m0 + c < s.sq ? p.delta[lr + c] : 0.f;
                }
                if (!__all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->row_empty[slot], ((it >> 1) & 1u) ^ 1u, abort_flag, p.status, 0x10103))) break;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    sRow[slot * 256 + u * 32 + lane] = l[u];
                    sRow[slot * 256 + 128 + u * 32 + lane] = d[u];
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctrl->row_full[slot]);
            }
        } else if (warp == 8 && N > 0) {
            // ================================ MMA issuer ================================
            constexpr uint32_t idesc_s = make_idesc<T>(false), idesc_o = make_idesc<T>(true, HDIM);
            const bool leader = elect_one_sync();
            auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
                return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag, p.status, code)) != 0;
            };
            auto commit = [&](uint64_t* bar) { if (leader) umma_commit(bar); };
            auto at = [&](uint64_t d, int slot) { return d + (uint64_t)((slot * TILE) >> 4); };
            const uint64_t dK = make_smem_desc(smem_u32(sK), 0, 1024), dV = make_smem_desc(smem_u32(sV), 0, 1024);
            const uint64_t dQ = make_smem_desc(smem_u32(sQ), 0, 1024), dDO = make_smem_desc(smem_u32(sDO), 0, 1024);
            const uint64_t dQt = make_smem_desc(smem_u32(sQ), HALF_BYTES, 1024), dDOt = make_smem_desc(smem_u32(sDO), HALF_BYTES, 1024);
            bool ok = wait(&ctrl->own_full, 0, 0x10110) && wait(&ctrl->a_full[0], 0, 0x10111);
            if (ok) {
                tc_fence_after();
                if (leader) bwd_issue_ss<HDIM>(tmem + cS, dK, at(dQ, 0), idesc_s);
                commit(&ctrl->s_full);
                ok = wait(&ctrl->b_full[0], 0, 0x10112);
            }
            if (ok) {
                if (leader) bwd_issue_ss<HDIM>(tmem + cDP, dV, at(dDO, 0), idesc_s);
                commit(&ctrl->dp_full);
            }
            for (int it = 0; ok && it < N; ++it) {
                const int qs1 = (it + 1) % QS, os1 = (it + 1) % OS;
                if (it + 1 < N) {
                    if (!(ok = wait(&ctrl->a_full[qs1], ((it + 1) / QS) & 1u, 0x10111))) break;
                }
                if (!(ok = wait(&ctrl->p_full, it & 1u, 0x10113))) break;
                tc_fence_after();
                if (leader) bwd_issue_xb(tmem + cDV, tmem + cS, at(dDOt, it % OS), idesc_o, it > 0);
                commit(&ctrl->b_empty[it % OS]);
                if (it + 1 < N) {
                    if (leader) bwd_issue_ss<HDIM>(tmem + cS, dK, at(dQ, qs1), idesc_s);
                    commit(&ctrl->s_full);
                    if (!(ok = wait(&ctrl->b_full[os1], ((it + 1) / OS) & 1u, 0x10112))) break;
                }
                if (!(ok = wait(&ctrl->ds_full, it & 1u, 0x10114))) break;
                tc_fence_after();
                if (leader) bwd_issue_xb(tmem + cDK, tmem + cDP, at(dQt, it % QS), idesc_o, it > 0);
                commit(&ctrl->a_empty[it % QS]);
                if (it + 1 < N) {
                    if (leader) bwd_issue_ss<HDIM>(tmem + cDP, dV, at(dDO, os1), idesc_s);
                    commit(&ctrl->dp_full);
                } else {
                    commit(&ctrl->acc_full);
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;\n" ::);
        const int half = warp >> 2, r = (warp & 3) * 32 + lane, key = n0 + r;
        const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        bool ok = true;
        auto step = [&](int it, int m0, float slope, auto masked) -> bool {
            // columns of this half that see the key: i >= key - shift - wr, i <= key - shift + wl
            int c_lo = 0, c_hi = 0x3fffffff;
            if constexpr (decltype(masked)::value) {
                const int i0 = m0 + half * 64;
                c_lo = p.wr >= 0 ? key - s.shift - p.wr - i0 : 0;
                c_hi = p.wl >= 0 ? key - s.shift + p.wl - i0 : 0x3fffffff;
            }
            const float* rows = sRow + (it & 1) * 256 + half * 64;
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->row_full[it & 1], (it >> 1) & 1u, abort_flag, p.status, 0x10120))) return false;
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->s_full, it & 1u, abort_flag, p.status, 0x10121))) return false;
            tc_fence_after();
            uint32_t x[2][32], w[32];
            tmem_ld32(lane_addr + cS + half * 64, x[0]);
            tmem_ld32(lane_addr + cS + half * 64 + 32, x[1]);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    const float4 l4 = *reinterpret_cast<const float4*>(rows + c * 32 + e);
#pragma unroll
                    for (int u = 0; u < 4; u += 2) {
                        const int col = c * 32 + e + u;
                        float2 f = make_float2(1.f, 1.f), away = f;
                        if constexpr (EXTRA) {
                            away.x = (float)(m0 + half * 64 + col + s.sk - s.sq - key);
                            away.y = away.x + 1.f;
                        }
                        const float2 lse2 = u ? make_float2(l4.z, l4.w) : make_float2(l4.x, l4.y);
                        const float2 y = bwd_exponent<EXTRA>(p, make_float2(__uint_as_float(x[c][e + u]), __uint_as_float(x[c][e + u + 1])), slope,
                                                             away, lse2, f);
                        float2 pr = make_float2(ex2_fast(y.x), ex2_fast(y.y));
                        if constexpr (decltype(masked)::value) {
                            if (col < c_lo || col > c_hi) pr.x = 0.f;
                            if (col + 1 < c_lo || col + 1 > c_hi) pr.y = 0.f;
                        }
                        w[col / 2] = Elem<T>::pack2(pr.x, pr.y);
                        if constexpr (EXTRA) pr = __fmul2_rn(pr, f);  // (from here on P serves dS alone)
                        x[c][e + u] = __float_as_uint(pr.x);
                        x[c][e + u + 1] = __float_as_uint(pr.y);
                    }
                }
            tmem_st32(lane_addr + cS + half * 64, w);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctrl->p_full);
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->dp_full, it & 1u, abort_flag, p.status, 0x10122))) return false;
            tc_fence_after();
            uint32_t dp[2][32];
            tmem_ld32(lane_addr + cDP + half * 64, dp[0]);
            tmem_ld32(lane_addr + cDP + half * 64 + 32, dp[1]);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    const float4 d4 = *reinterpret_cast<const float4*>(rows + 128 + c * 32 + e);
#pragma unroll
                    for (int u = 0; u < 4; u += 2) {
                        const float2 d2 = u ? make_float2(-d4.z, -d4.w) : make_float2(-d4.x, -d4.y);
                        const float2 t = __fadd2_rn(make_float2(__uint_as_float(dp[c][e + u]), __uint_as_float(dp[c][e + u + 1])), d2);
                        const float2 ds = __fmul2_rn(make_float2(__uint_as_float(x[c][e + u]), __uint_as_float(x[c][e + u + 1])), t);
                        w[c * 16 + (e + u) / 2] = Elem<T>::pack2(ds.x, ds.y);
                    }
                }
            tmem_st32(lane_addr + cDP + half * 64, w);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&ctrl->ds_full);
                mbar_arrive(&ctrl->row_empty[it & 1]);
            }
            return true;
        };
        // query rows that see all of the tile's keys
        int full_lo = 0, full_hi = 0x3fffffff;
        if (p.mask_type != 0) {
            if (p.wr >= 0) full_lo = n0 + 127 - s.shift - p.wr;
            if (p.wl >= 0) full_hi = n0 - s.shift + p.wl;
        }
        int it = 0;
        for (int g = 0; ok && g < (tiles > 0 ? G : 0); ++g) {
            const float slope = EXTRA && p.alibi ? p.alibi[(p.alibi_rank ? b * p.hq : 0) + kh * G + g] * kLog2e : 0.f;
            for (int m = 0; ok && m < tiles; ++m, ++it) {
                const int m0 = (m_begin + m) * 128;
                ok = m0 < full_lo || m0 + 127 > full_hi ? step(it, m0, slope, std::true_type{}) : step(it, m0, slope, std::false_type{});
            }
        }
        if (ok && N > 0) {
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ctrl->acc_full, 0, abort_flag, p.status, 0x10123));
            tc_fence_after();
        }
        if (ok) {  // warps 0-3 dV, 4-7 dK
            T* dst = (T*)(half ? p.dk : p.dv) + ((int64_t)(s.k0 + key) * p.hkv + kh) * HDIM;
#pragma unroll
            for (int c = 0; c < HDIM / 32; ++c) {
                uint32_t t[32];
                if (N > 0) {
                    tmem_ld32(lane_addr + (half ? cDK : cDV) + c * 32, t);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) t[e] = 0u;
                }
                if (key < s.sk) bwd_store32<T>(dst + c * 32, t, half ? p.scale : 1.f);
            }
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
