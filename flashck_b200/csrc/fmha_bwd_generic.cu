// Backward of fmha_fwd -- the general instance: every call that the forward takes on contiguous K/V (hdim 64 / 128, fp16 / bf16,
// batch and group mode, GQA, the four masks, elementwise bias with its gradient, ALiBi, soft cap).  It serves what the tcgen05
// kernels leave (no keys or no queries at all: zeros) and is the second instance that "use_sm100_bwd" = 0
// selects, against which the other can be checked: 6155 us on 2 x 4096 causal tokens of 32 / 8 heads of 128, where the tcgen05
// kernels take 770.
//
// With S = scale Q K^T, S' = cap tanh(S / cap), T = S' + bias, P = exp(T - LSE) (recomputed, 0 where masked),
//     D_i = sum_c dO_ic O_ic - dLSE_i      dP = dO V^T      dT = P (dP - D)      dS = dT (1 - (S' / cap)^2)
//     dV = P^T dO      dK = scale dS^T Q      dQ = scale dS K      dbias = dT, summed over what the bias is shared by.
// Each output element has one owner that sums its terms in a fixed order in fp32 -- no atomics, equal bits on every run.  The
// price is that S and dP are computed once for dQ (a CTA per 64 queries of a head) and once for dK / dV (a CTA per 64 keys
// of a kv head, which walks the group's heads one after the other): seven products where one pass with shared sums has five.
//
// All products are mma.sync m16n8k16 on 64 x 64 tiles, 4 warps x 16 rows, operands by cp.async into an XOR-swizzled double
// buffer.  P and dS enter their second product rounded to the element type, as P does in the forward; rows behind a sequence's
// end come as zeros, so that what lies there (another sequence, a NaN) does not count.
#include "kernels.h"

#include <algorithm>

namespace fck {

namespace {

constexpr int BT = 64, NWARP = 4;  // rows of a tile on either side

struct BwdDev {
    const void* dout;
    const void* q;
    const void* k;
    const void* v;
    const void* o;
    const float* lse;
    const float* dlse;
    float* delta;
    void* dq;
    void* dk;
    void* dv;
    void* dbias;
    const int64_t* seqstart_q;
    const int64_t* seqstart_k;
    int batch, seqlen_q, seqlen_k, hq, hkv;
    int mask_type, wl, wr;
    float scale, scale_log2;
    const void* bias;
    int bias_type, bias_rank;
    int64_t bias_sq, bias_sk;
    float cap, inv_cap;
};

// Row-major [rows][D] 16-bit tile; 16-byte chunk index XORed with (row & 7).
template <int D>
__device__ __forceinline__ uint32_t swz(int row, int chunk) {
    return (uint32_t)(row * (D * 2) + (((chunk & ~7) | ((chunk ^ row) & 7)) << 4));
}

struct Seq {  // where a sequence's rows are
    int64_t q0, k0;
    int sq, sk, shift;
};
__device__ __forceinline__ Seq sequence(const BwdDev& p, int b) {
    Seq s;
    s.q0 = p.seqstart_q ? p.seqstart_q[b] : (int64_t)b * p.seqlen_q;
    s.k0 = p.seqstart_k ? p.seqstart_k[b] : (int64_t)b * p.seqlen_k;
    s.sq = p.seqstart_q ? (int)max((int64_t)0, p.seqstart_q[b + 1] - s.q0) : p.seqlen_q;
    s.sk = p.seqstart_k ? (int)max((int64_t)0, p.seqstart_k[b + 1] - s.k0) : p.seqlen_k;
    s.shift = p.mask_type == 2 ? s.sk - s.sq : 0;
    return s;
}
// index of (row 0 of sequence b, head h) in the LSE layout
__device__ __forceinline__ int64_t lse_row(const BwdDev& p, const Seq& s, int b, int h) {
    return p.seqstart_q ? (int64_t)h * p.seqlen_q + s.q0 : ((int64_t)b * p.hq + h) * p.seqlen_q;
}
__device__ __forceinline__ bool sees(const BwdDev& p, const Seq& s, int i, int j) {
    if (i >= s.sq || j >= s.sk) return false;
    if (p.mask_type == 0) return true;
    return (p.wl < 0 || j >= i + s.shift - p.wl) && (p.wr < 0 || j <= i + s.shift + p.wr);
}
// LSE in base-2 units; a row without keys gets +inf, which makes every P of it 0
__device__ __forceinline__ float lse_base2(float lse) { return lse == -INFINITY ? INFINITY : lse * kLog2e; }

struct Additions {  // of one (sequence, head)
    const void* bias;  // element (0, 0) of the sequence's block, or nullptr
    float slope;       // ALiBi
};
template <typename T>
__device__ __forceinline__ Additions additions(const BwdDev& p, const Seq& s, int b, int h) {
    Additions a{nullptr, 0.f};
    if (p.bias_type == 1) {
        const int64_t plane = p.bias_sq * p.bias_sk;
        const int64_t at = (p.bias_rank >= 1 ? (int64_t)h * plane : 0) + (p.bias_rank == 2 ? (int64_t)b * p.hq * plane : 0) +
                           (p.seqstart_q ? s.q0 * p.bias_sk + s.k0 : 0);
        a.bias = (const T*)p.bias + at;
    } else if (p.bias_type == 2) {
        a.slope = ((const float*)p.bias)[(p.bias_rank >= 1 ? (int64_t)b * p.hq : 0) + h];
    }
    return a;
}
// P of a visible pair, and the derivative of the soft cap at its score.
template <typename T, bool EXTRA>
__device__ __forceinline__ float probability(const BwdDev& p, const Seq& s, const Additions& a, float raw, int i, int j, float lse2,
                                             float& dcap) {
    dcap = 1.f;
    if constexpr (!EXTRA) return fast_exp2(raw * p.scale_log2 - lse2);
    float y = raw * p.scale;
    if (p.cap > 0.f) {
        const float t = tanh_inline(y * p.inv_cap);
        y = p.cap * t;
        dcap = 1.f - t * t;
    }
    if (a.bias) y += Elem<T>::to_f32(((const T*)a.bias)[(int64_t)i * p.bias_sk + j]);
    else y -= a.slope * fabsf((float)(i + s.sk - s.sq - j));
    return fast_exp2(y * kLog2e - lse2);
}

// 64 rows of head h (row stride `heads` * D) to a swizzled tile; rows at and behind `n` become zeros.
template <typename T, int D>
__device__ __forceinline__ void load_tile(uint32_t dst, const T* src, int heads, int h, int row0, int n, int tid) {
    constexpr int CH = D / 8;
    const int c = tid % CH;
#pragma unroll
    for (int r = tid / CH; r < BT; r += (NWARP * 32) / CH) {
        const bool ok = row0 + r < n;
        cp_async_16(dst + swz<D>(r, c), src + ((int64_t)(ok ? row0 + r : 0) * heads + h) * D + c * 8, ok);
    }
}

// acc (16 x 64 of this warp) += A[16 rows of the warp][D] B[64][D]^T, both tiles row-major
template <typename T, int D>
__device__ __forceinline__ void product_abt(float (&acc)[BT / 8][4], uint32_t a_tile, uint32_t b_tile, int warp, int lane) {
    const int lm = lane >> 3, lr = lane & 7;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t a[4];
        ldmatrix_x4(a, a_tile + swz<D>(warp * 16 + (lm & 1) * 8 + lr, 2 * ks + (lm >> 1)));
#pragma unroll
        for (int jp = 0; jp < BT / 16; ++jp) {
            uint32_t bfr[4];
            ldmatrix_x4(bfr, b_tile + swz<D>(jp * 16 + (lm >> 1) * 8 + lr, 2 * ks + (lm & 1)));
            mma_16816<T>(acc[2 * jp], a, bfr[0], bfr[1]);
            mma_16816<T>(acc[2 * jp + 1], a, bfr[2], bfr[3]);
        }
    }
}
// acc (16 x D of this warp) += X (16 x 64, accumulator layout, rounded to T) B[64][D]
template <typename T, int D>
__device__ __forceinline__ void product_xb(float (&acc)[D / 8][4], const float (&x)[BT / 8][4], uint32_t b_tile, int lane) {
    const int lm = lane >> 3, lr = lane & 7;
#pragma unroll
    for (int kk = 0; kk < BT / 16; ++kk) {
        uint32_t a[4];
        a[0] = Elem<T>::pack2(x[2 * kk][0], x[2 * kk][1]);
        a[1] = Elem<T>::pack2(x[2 * kk][2], x[2 * kk][3]);
        a[2] = Elem<T>::pack2(x[2 * kk + 1][0], x[2 * kk + 1][1]);
        a[3] = Elem<T>::pack2(x[2 * kk + 1][2], x[2 * kk + 1][3]);
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
            uint32_t bfr[4];
            ldmatrix_x4_trans(bfr, b_tile + swz<D>(kk * 16 + (lm & 1) * 8 + lr, 2 * j + (lm >> 1)));
            mma_16816<T>(acc[2 * j], a, bfr[0], bfr[1]);
            mma_16816<T>(acc[2 * j + 1], a, bfr[2], bfr[3]);
        }
    }
}
template <int N>
__device__ __forceinline__ void clear(float (&x)[N][4]) {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j][0] = x[j][1] = x[j][2] = x[j][3] = 0.f;
}
// The warp's 16 x D accumulator times f to rows row0 .. of a [rows, heads, D] tensor, as far as they exist.
template <typename T, int D>
__device__ __forceinline__ void store_rows(T* dst, const float (&acc)[D / 8][4], float f, int heads, int h, int row0, int n, int lane) {
    const int quad = lane >> 2, ql = lane & 3;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int r = row0 + quad + 8 * half;
        if (r >= n) continue;
        T* row = dst + ((int64_t)r * heads + h) * D + ql * 2;
#pragma unroll
        for (int j = 0; j < D / 8; ++j)
            *reinterpret_cast<uint32_t*>(row + j * 8) = Elem<T>::pack2(acc[j][2 * half] * f, acc[j][2 * half + 1] * f);
    }
}

// D_i = sum_c dO_ic O_ic - dLSE_i, half a warp per row, summed in fp32; and zeros to the rows of dQ, dK, dV that belong to no
// sequence (in front of the first, behind the last one).  It reads dO and O once: 4 d bytes per row and head.
template <typename T, int D>
__global__ void __launch_bounds__(256) bwd_prepare_kernel(const BwdDev p) {
    pdl_wait();
    const int sub = threadIdx.x & 15;
    const uint32_t half = 0xffffu << (threadIdx.x & 16);  // the row's lanes
    const int64_t rows = (p.seqstart_q ? 1 : p.batch) * (int64_t)p.seqlen_q;
    for (int64_t w = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 4; w < rows * p.hq; w += ((int64_t)gridDim.x * blockDim.x) >> 4) {
        const int64_t row = w / p.hq;
        const int h = (int)(w - row * p.hq);
        const T* a = (const T*)p.dout + w * D;
        const T* b = (const T*)p.o + w * D;
        float sum = 0.f;
        if (sub * 8 < D) {
            const uint4 x = *reinterpret_cast<const uint4*>(a + sub * 8), y = *reinterpret_cast<const uint4*>(b + sub * 8);
            const T* xe = reinterpret_cast<const T*>(&x);
            const T* ye = reinterpret_cast<const T*>(&y);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += Elem<T>::to_f32(xe[e]) * Elem<T>::to_f32(ye[e]);
        }
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) sum += __shfl_xor_sync(half, sum, off);
        if (sub == 0) {
            const int64_t at = p.seqstart_q ? (int64_t)h * p.seqlen_q + row
                                            : ((row / p.seqlen_q) * p.hq + h) * p.seqlen_q + row % p.seqlen_q;
            p.delta[at] = sum - (p.dlse ? p.dlse[at] : 0.f);
        }
    }
    if (p.seqstart_q) {
        const int64_t tid = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, threads = (int64_t)gridDim.x * blockDim.x;
        auto zero = [&](void* t, int64_t from, int64_t to, int heads) {  // 16-byte pieces of the rows [from, to)
            const int64_t per_row = (int64_t)heads * D / 8;
            for (int64_t i = from * per_row + tid; i < to * per_row; i += threads) reinterpret_cast<uint4*>(t)[i] = make_uint4(0u, 0u, 0u, 0u);
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
}

// dQ: 64 queries of one head against the key tiles that the mask leaves them.
template <typename T, int D, bool EXTRA>
__global__ void __launch_bounds__(NWARP * 32) bwd_dq_kernel(const BwdDev p) {
    constexpr int TILE = BT * D * 2;
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t sQ = smem_u32(smem), sDO = sQ + TILE, sK = sDO + TILE, sV = sK + 2 * TILE;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = lane >> 2, ql = lane & 3;
    const int b = blockIdx.z, h = blockIdx.y, kh = h / (p.hq / p.hkv), m0 = (gridDim.x - 1 - blockIdx.x) * BT;
    const Seq s = sequence(p, b);
    if (m0 >= s.sq) return;
    int lo_first, hi_first, lo_last, hi_last;
    visible_range(m0, s.sq, s.sk, p.mask_type, p.wl, p.wr, lo_first, hi_first);
    visible_range(min(s.sq, m0 + BT) - 1, s.sq, s.sk, p.mask_type, p.wl, p.wr, lo_last, hi_last);
    const int n_begin = max(0, lo_first) / BT, n_end = hi_last < 0 ? 0 : hi_last / BT + 1;
    const T* kbase = (const T*)p.k + s.k0 * p.hkv * D;
    const T* vbase = (const T*)p.v + s.k0 * p.hkv * D;
    auto load_kv = [&](int n, int buf) {
        load_tile<T, D>(sK + buf * TILE, kbase, p.hkv, kh, n * BT, s.sk, tid);
        load_tile<T, D>(sV + buf * TILE, vbase, p.hkv, kh, n * BT, s.sk, tid);
    };
    if (n_begin < n_end) {
        load_tile<T, D>(sQ, (const T*)p.q + s.q0 * p.hq * D, p.hq, h, m0, s.sq, tid);
        load_tile<T, D>(sDO, (const T*)p.dout + s.q0 * p.hq * D, p.hq, h, m0, s.sq, tid);
        load_kv(n_begin, 0);
    }
    cp_async_commit();
    const Additions add = additions<T>(p, s, b, h);
    const int64_t lr = lse_row(p, s, b, h);
    float lse2[2], delta[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int i = m0 + warp * 16 + quad + 8 * half;
        lse2[half] = i < s.sq ? lse_base2(p.lse[lr + i]) : INFINITY;
        delta[half] = i < s.sq ? p.delta[lr + i] : 0.f;
    }
    float dq[D / 8][4];
    clear(dq);
    for (int n = n_begin; n < n_end; ++n) {
        const int buf = (n - n_begin) & 1;
        __syncthreads();  // everyone is done with the buffer the next load overwrites
        if (n + 1 < n_end) load_kv(n + 1, buf ^ 1);
        cp_async_commit();
        cp_async_wait<1>();
        __syncthreads();
        float x[BT / 8][4], dp[BT / 8][4];
        clear(x);
        clear(dp);
        product_abt<T, D>(x, sQ, sK + buf * TILE, warp, lane);
        product_abt<T, D>(dp, sDO, sV + buf * TILE, warp, lane);
#pragma unroll
        for (int j = 0; j < BT / 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = m0 + warp * 16 + quad + 8 * (e >> 1), key = n * BT + j * 8 + ql * 2 + (e & 1);
                float ds = 0.f, dcap;
                if (sees(p, s, i, key)) {
                    const float pr = probability<T, EXTRA>(p, s, add, x[j][e], i, key, lse2[e >> 1], dcap);
                    ds = pr * (dp[j][e] - delta[e >> 1]) * dcap;
                }
                x[j][e] = ds;
            }
        product_xb<T, D>(dq, x, sK + buf * TILE, lane);
    }
    store_rows<T, D>((T*)p.dq + s.q0 * p.hq * D, dq, p.scale, p.hq, h, m0 + warp * 16, s.sq, lane);
}

// dK and dV: 64 keys of one kv head against the query tiles that see them, head after head of the group.  The transposed
// products (rows = keys) leave P^T and dS^T in the layout that the second products take them in.
template <typename T, int D, bool EXTRA>
__global__ void __launch_bounds__(NWARP * 32) bwd_dkdv_kernel(const BwdDev p) {
    constexpr int TILE = BT * D * 2;
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t sK = smem_u32(smem), sV = sK + TILE, sQ = sV + TILE, sDO = sQ + 2 * TILE;
    float* sRow = reinterpret_cast<float*>(smem + 6 * TILE);  // [2][64] LSE, [2][64] D
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = lane >> 2, ql = lane & 3;
    const int b = blockIdx.z, kh = blockIdx.y, n0 = blockIdx.x * BT, G = p.hq / p.hkv;
    const Seq s = sequence(p, b);
    if (n0 >= s.sk) return;
    // queries that see any of these keys: i + shift - wl <= j <= i + shift + wr
    int i_lo = 0, i_hi = s.sq - 1;
    if (p.mask_type != 0) {
        if (p.wr >= 0) i_lo = max(i_lo, n0 - s.shift - p.wr);
        if (p.wl >= 0) i_hi = min(i_hi, min(s.sk, n0 + BT) - 1 - s.shift + p.wl);
    }
    const int m_begin = i_lo / BT, tiles = i_hi >= i_lo ? i_hi / BT + 1 - m_begin : 0;
    const T* qbase = (const T*)p.q + s.q0 * p.hq * D;
    const T* dobase = (const T*)p.dout + s.q0 * p.hq * D;
    auto load_q = [&](int it, int buf) {
        const int h = kh * G + it / tiles, m0 = (m_begin + it % tiles) * BT;
        load_tile<T, D>(sQ + buf * TILE, qbase, p.hq, h, m0, s.sq, tid);
        load_tile<T, D>(sDO + buf * TILE, dobase, p.hq, h, m0, s.sq, tid);
        const int i = m0 + (tid & 63);
        const int64_t at = lse_row(p, s, b, h) + i;
        sRow[(tid >> 6) * 128 + buf * 64 + (tid & 63)] =
            tid < 64 ? (i < s.sq ? lse_base2(p.lse[at]) : INFINITY) : (i < s.sq ? p.delta[at] : 0.f);
    };
    float dk[D / 8][4], dv[D / 8][4];
    clear(dk);
    clear(dv);
    const int steps = tiles * G;
    if (steps > 0) {
        load_tile<T, D>(sK, (const T*)p.k + s.k0 * p.hkv * D, p.hkv, kh, n0, s.sk, tid);
        load_tile<T, D>(sV, (const T*)p.v + s.k0 * p.hkv * D, p.hkv, kh, n0, s.sk, tid);
        load_q(0, 0);
    }
    cp_async_commit();
    for (int it = 0; it < steps; ++it) {
        const int buf = it & 1, h = kh * G + it / tiles, m0 = (m_begin + it % tiles) * BT;
        __syncthreads();
        if (it + 1 < steps) load_q(it + 1, buf ^ 1);
        cp_async_commit();
        cp_async_wait<1>();
        __syncthreads();
        const Additions add = additions<T>(p, s, b, h);
        const float* lse2 = sRow + buf * 64;
        const float* delta = sRow + 128 + buf * 64;
        float x[BT / 8][4], dcap[EXTRA ? BT / 8 : 1][4];
        clear(x);
        product_abt<T, D>(x, sK, sQ + buf * TILE, warp, lane);
#pragma unroll
        for (int j = 0; j < BT / 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int key = n0 + warp * 16 + quad + 8 * (e >> 1), c = j * 8 + ql * 2 + (e & 1);
                float dc = 1.f, pr = 0.f;
                if (sees(p, s, m0 + c, key)) pr = probability<T, EXTRA>(p, s, add, x[j][e], m0 + c, key, lse2[c], dc);
                x[j][e] = pr;
                if constexpr (EXTRA) dcap[j][e] = dc;
            }
        product_xb<T, D>(dv, x, sDO + buf * TILE, lane);
        float dp[BT / 8][4];
        clear(dp);
        product_abt<T, D>(dp, sV, sDO + buf * TILE, warp, lane);
#pragma unroll
        for (int j = 0; j < BT / 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = j * 8 + ql * 2 + (e & 1);
                // (a hidden pair: P is 0, but what stands beside it may be a NaN of a key behind the end)
                const bool vis = sees(p, s, m0 + c, n0 + warp * 16 + quad + 8 * (e >> 1));
                float ds = vis ? x[j][e] * (dp[j][e] - delta[c]) : 0.f;
                if constexpr (EXTRA) ds *= dcap[j][e];
                x[j][e] = ds;
            }
        product_xb<T, D>(dk, x, sQ + buf * TILE, lane);
    }
    store_rows<T, D>((T*)p.dk + s.k0 * p.hkv * D, dk, p.scale, p.hkv, kh, n0 + warp * 16, s.sk, lane);
    store_rows<T, D>((T*)p.dv + s.k0 * p.hkv * D, dv, 1.f, p.hkv, kh, n0 + warp * 16, s.sk, lane);
}

// dbias: a 64 x 64 tile of one plane; the CTA sums dT over the heads and sequences that share the plane, in order.
template <typename T, int D>
__global__ void __launch_bounds__(NWARP * 32) bwd_dbias_kernel(const BwdDev p) {
    constexpr int TILE = BT * D * 2;
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t sQ = smem_u32(smem), sDO = sQ + TILE, sK = sDO + TILE, sV = sK + TILE;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = lane >> 2, ql = lane & 3;
    const int n0 = blockIdx.x * BT, m0 = blockIdx.y * BT;
    // plane index: rank 0 none, 1 head, 2 (sequence, head); group mode: and the sequence, whose block it is
    const int planes_h = p.bias_rank >= 1 ? p.hq : 1, ph = blockIdx.z % planes_h, pb = blockIdx.z / planes_h;
    const bool own_b = p.bias_rank == 2 || p.seqstart_q;
    const int b_begin = own_b ? pb : 0, b_end = own_b ? pb + 1 : p.batch;
    const int h_begin = p.bias_rank >= 1 ? ph : 0, h_end = p.bias_rank >= 1 ? ph + 1 : p.hq;
    const Seq s0 = sequence(p, b_begin);
    if (m0 >= s0.sq || n0 >= s0.sk) return;
    float acc[BT / 8][4];
    clear(acc);
    for (int b = b_begin; b < b_end; ++b) {
        const Seq s = sequence(p, b);
        for (int h = h_begin; h < h_end; ++h) {
            const int kh = h / (p.hq / p.hkv);
            load_tile<T, D>(sQ, (const T*)p.q + s.q0 * p.hq * D, p.hq, h, m0, s.sq, tid);
            load_tile<T, D>(sDO, (const T*)p.dout + s.q0 * p.hq * D, p.hq, h, m0, s.sq, tid);
            load_tile<T, D>(sK, (const T*)p.k + s.k0 * p.hkv * D, p.hkv, kh, n0, s.sk, tid);
            load_tile<T, D>(sV, (const T*)p.v + s.k0 * p.hkv * D, p.hkv, kh, n0, s.sk, tid);
            cp_async_commit();
            const Additions add = additions<T>(p, s, b, h);
            const int64_t lr = lse_row(p, s, b, h);
            float lse2[2], delta[2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int i = m0 + warp * 16 + quad + 8 * half;
                lse2[half] = i < s.sq ? lse_base2(p.lse[lr + i]) : INFINITY;
                delta[half] = i < s.sq ? p.delta[lr + i] : 0.f;
            }
            cp_async_wait<0>();
            __syncthreads();
            float x[BT / 8][4], dp[BT / 8][4];
            clear(x);
            clear(dp);
            product_abt<T, D>(x, sQ, sK, warp, lane);
            product_abt<T, D>(dp, sDO, sV, warp, lane);
#pragma unroll
            for (int j = 0; j < BT / 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = m0 + warp * 16 + quad + 8 * (e >> 1), key = n0 + j * 8 + ql * 2 + (e & 1);
                    float dcap;
                    if (sees(p, s, i, key))
                        acc[j][e] += probability<T, true>(p, s, add, x[j][e], i, key, lse2[e >> 1], dcap) * (dp[j][e] - delta[e >> 1]);
                }
            __syncthreads();  // the tiles are read before the next ones land
        }
    }
    const int64_t plane = p.bias_sq * p.bias_sk;
    T* dst = (T*)p.dbias + (int64_t)(p.bias_rank == 2 ? pb * p.hq + ph : ph) * plane + (p.seqstart_q ? s0.q0 * p.bias_sk + s0.k0 : 0);
#pragma unroll
    for (int j = 0; j < BT / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = m0 + warp * 16 + quad + 8 * (e >> 1), key = n0 + j * 8 + ql * 2 + (e & 1);
            if (i < s0.sq && key < s0.sk) dst[(int64_t)i * p.bias_sk + key] = Elem<T>::from_f32(acc[j][e]);
        }
}

template <typename K>
int allow_smem(K kern, size_t bytes) {
    FCK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    return FLASHCK_OK;
}

template <typename T, int D>
int launch_prepare(const BwdDev& dev, int64_t rows, cudaStream_t stream) {
    const int64_t want = (rows * dev.hq + 15) / 16;  // 16 rows per block and pass
    const unsigned grid = (unsigned)std::min<int64_t>(std::max<int64_t>(want, 1), (int64_t)sm_count() * 8);
    FCK_CUDA(launch_dependent(bwd_prepare_kernel<T, D>, dim3(grid), dim3(256), 0, stream, dev));
    return FLASHCK_OK;
}

template <typename T, int D, bool EXTRA>
int launch_t(const BwdParams& p, const BwdDev& dev, cudaStream_t stream) {
    constexpr size_t TILE = BT * D * 2;
    const int64_t rows = (p.seqstart_q ? 1 : p.batch) * p.seqlen_q;
    if (int rc = launch_prepare<T, D>(dev, rows, stream)) return rc;
    const unsigned mt = (unsigned)((p.max_seqlen_q + BT - 1) / BT), nt = (unsigned)((p.max_seqlen_k + BT - 1) / BT);
    if (mt > 0) {
        auto kern = bwd_dq_kernel<T, D, EXTRA>;
        if (int rc = allow_smem(kern, 6 * TILE)) return rc;
        kern<<<dim3(mt, (unsigned)p.hq, (unsigned)p.batch), NWARP * 32, 6 * TILE, stream>>>(dev);
        FCK_CUDA(cudaGetLastError());
    }
    if (nt > 0) {
        auto kern = bwd_dkdv_kernel<T, D, EXTRA>;
        constexpr size_t bytes = 6 * TILE + 4 * BT * sizeof(float);
        if (int rc = allow_smem(kern, bytes)) return rc;
        kern<<<dim3(nt, (unsigned)p.hkv, (unsigned)p.batch), NWARP * 32, bytes, stream>>>(dev);
        FCK_CUDA(cudaGetLastError());
    }
    if constexpr (EXTRA) {
        if (p.dbias && mt > 0 && nt > 0) {
            const int64_t planes = (p.bias_rank >= 1 ? p.hq : 1) * (p.bias_rank == 2 || p.seqstart_q ? p.batch : 1);
            FCK_REQUIRE(planes <= 65535 && mt <= 65535, FLASHCK_ERR_UNSUPPORTED,
                        "fmha_bwd: a bias gradient of %lld planes and %u row tiles (at most 65535 of each)", (long long)planes, mt);
            auto kern = bwd_dbias_kernel<T, D>;
            if (int rc = allow_smem(kern, 4 * TILE)) return rc;
            kern<<<dim3(nt, mt, (unsigned)planes), NWARP * 32, 4 * TILE, stream>>>(dev);
            FCK_CUDA(cudaGetLastError());
        }
    }
    return FLASHCK_OK;
}

template <typename T>
int launch_d(const BwdParams& p, const BwdDev& dev, cudaStream_t stream) {
    const bool extra = p.bias_type != 0 || p.logits_soft_cap > 0.f;
    if (p.d == 128) return extra ? launch_t<T, 128, true>(p, dev, stream) : launch_t<T, 128, false>(p, dev, stream);
    return extra ? launch_t<T, 64, true>(p, dev, stream) : launch_t<T, 64, false>(p, dev, stream);
}

}  // namespace

int launch_bwd_generic(const BwdParams& p, cudaStream_t stream) {
    FCK_REQUIRE(p.batch <= 65535 && p.hq <= 65535, FLASHCK_ERR_UNSUPPORTED, "fmha_bwd: nhead_q and batch must be <= 65535");
    BwdDev dev{};
    dev.dout = p.dout; dev.q = p.q; dev.k = p.k; dev.v = p.v; dev.o = p.o; dev.lse = p.lse; dev.dlse = p.dlse; dev.delta = p.delta;
    dev.dq = p.dq; dev.dk = p.dk; dev.dv = p.dv; dev.dbias = p.dbias;
    dev.seqstart_q = p.seqstart_q; dev.seqstart_k = p.seqstart_k;
    dev.batch = (int)p.batch; dev.seqlen_q = (int)p.seqlen_q; dev.seqlen_k = (int)p.seqlen_k; dev.hq = (int)p.hq; dev.hkv = (int)p.hkv;
    dev.mask_type = p.mask_type;
    dev.wl = p.wl < 0 ? -1 : (int)p.wl;
    dev.wr = p.wr < 0 ? -1 : (int)p.wr;
    dev.scale = p.scale; dev.scale_log2 = p.scale * kLog2e;
    dev.bias = p.bias; dev.bias_type = p.bias_type; dev.bias_rank = p.bias_rank;
    dev.bias_sq = p.seqlen_q; dev.bias_sk = p.seqlen_k;
    dev.cap = p.logits_soft_cap; dev.inv_cap = p.logits_soft_cap > 0.f ? 1.f / p.logits_soft_cap : 0.f;
    return p.dtype == FLASHCK_DTYPE_BFLOAT16 ? launch_d<__nv_bfloat16>(p, dev, stream) : launch_d<__half>(p, dev, stream);
}

}  // namespace fck
