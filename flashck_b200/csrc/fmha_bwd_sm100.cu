// Backward of fmha_fwd on the tcgen05 kernels: which calls they take, the device parameters of a call, and the launches.
#include <algorithm>

#include "fmha_bwd_sm100.cuh"

namespace fck {

using namespace sm100;

namespace {

// 128 x 128 tiles of all planes (group mode: of every sequence's block in them, as if all were as long as the longest)
int64_t bias_items(const BwdParams& p) {
    const int64_t planes = (p.bias_rank >= 1 ? p.hq : 1) * (p.bias_rank == 2 || p.seqstart_q ? p.batch : 1);
    return (p.max_seqlen_q + 127) / 128 * ((p.max_seqlen_k + 127) / 128) * planes;
}

template <typename T, int HDIM, int VAR>
int launch_bwd_t(const BwdParams& p, const BwdSm100Dev& dev, cudaStream_t stream) {
    constexpr size_t TILE = 128 * HDIM * 2;
    const int64_t rows_q = p.seqstart_q ? p.seqlen_q : p.batch * p.seqlen_q, rows_k = p.seqstart_k ? p.seqlen_k : p.batch * p.seqlen_k;
    CUtensorMap mq, mdo, mk, mv;
    int rc;
    if ((rc = make_map_3d(&mq, p.q, p.dtype, rows_q, p.hq, 128, HDIM))) return rc;
    if ((rc = make_map_3d(&mdo, p.dout, p.dtype, rows_q, p.hq, 128, HDIM))) return rc;
    if ((rc = make_map_3d(&mk, p.k, p.dtype, rows_k, p.hkv, 128, HDIM))) return rc;
    if ((rc = make_map_3d(&mv, p.v, p.dtype, rows_k, p.hkv, 128, HDIM))) return rc;
    auto dq = bwd_dq_sm100_kernel<T, HDIM, VAR>;
    auto dkdv = bwd_dkdv_sm100_kernel<T, HDIM, VAR>;
    constexpr size_t smem_dq = 7 * TILE + 256 * sizeof(float) + sizeof(BwdCtrl);
    constexpr size_t smem_dkdv = 7 * TILE + 512 * sizeof(float) + sizeof(BwdCtrl);
    static_assert(smem_dq <= 227 * 1024 && smem_dkdv <= 227 * 1024, "tiles and the control block must fit the 227 KB a CTA can have");
    static thread_local int configured_device = -1;  // per instantiation
    int devid = 0;
    FCK_CUDA(cudaGetDevice(&devid));
    if (configured_device != devid) {
        FCK_CUDA(cudaFuncSetAttribute(dq, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_dq));
        FCK_CUDA(cudaFuncSetAttribute(dkdv, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_dkdv));
        configured_device = devid;
    }
    for (int i = 0; i < 2; ++i) {
        BwdSm100Dev d = dev;
        const int64_t tiles = ((i ? p.max_seqlen_k : p.max_seqlen_q) + 127) / 128, items = tiles * (i ? p.hkv : p.hq) * p.batch;
        // One item per CTA where they all fit at once, else a persistent grid.  (One per CTA for more sequences than the schedule by cost
        // holds, tiles of the longest one times sequences of them: us beside sequence after sequence, 512 causal ones of 128 tokens, 32 / 8
        // heads of 128, 1396 and 959; 600 of 1-400 tokens 4749 and 3013; 300 of 128 tokens, 2 / 1 heads of 64, 85 and 63; and with the
        // longest one not stated 512 x 512 x heads CTAs in the first case, nearly all without work.)
        d.listed = items <= sm_count() ? 0 : p.batch <= kBwdMaxBatch ? 1 : 2;
        d.max_tiles = (int)tiles;
        const dim3 grid((unsigned)(d.listed ? sm_count() : items));
        if (i == 0) FCK_CUDA(launch_dependent(dq, grid, dim3(kBwdThreads), smem_dq, stream, mk, mv, mq, mdo, d));
        else FCK_CUDA(launch_dependent(dkdv, grid, dim3(kBwdThreads), smem_dkdv, stream, mq, mdo, mk, mv, d));
    }
    if constexpr (VAR == 2) {
        if (p.dbias) {
            auto dbias = bwd_dbias_sm100_kernel<T, HDIM>;
            constexpr size_t smem = 1024 + 6 * TILE + sizeof(BwdCtrl);
            FCK_CUDA(cudaFuncSetAttribute(dbias, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
            FCK_CUDA(launch_dependent(dbias, dim3((unsigned)std::min<int64_t>(bias_items(p), sm_count())), dim3(kBwdBiasThreads), smem, stream, mq, mdo,
                                      mk, mv, dev));
        }
    }
    return FLASHCK_OK;
}

template <typename T>
int launch_bwd_d(const BwdParams& p, const BwdSm100Dev& dev, cudaStream_t stream) {
    const int var = p.bias_type == 1 ? 2 : p.bias_type == 2 || p.logits_soft_cap > 0.f ? 1 : 0;
    if (p.d == 128)
        return var == 2 ? launch_bwd_t<T, 128, 2>(p, dev, stream) : var ? launch_bwd_t<T, 128, 1>(p, dev, stream) : launch_bwd_t<T, 128, 0>(p, dev, stream);
    return var == 2 ? launch_bwd_t<T, 64, 2>(p, dev, stream) : var ? launch_bwd_t<T, 64, 1>(p, dev, stream) : launch_bwd_t<T, 64, 0>(p, dev, stream);
}

// (a batch without padding costs its launch: 2 us)
__global__ void __launch_bounds__(256) zero_outside_kernel(uint4* o, float* lse, const int64_t* seqstart, int64_t batch, int64_t total, int64_t hq,
                                                           int64_t row_vecs) {
    pdl_wait();
    const int64_t tid = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, threads = (int64_t)gridDim.x * blockDim.x;
    const int64_t first = min(max(seqstart[0], (int64_t)0), total), end = min(max(seqstart[batch], first), total), n = total - end + first;
    auto outside = [&](int64_t i) { return i < first ? i : i - first + end; };  // i-th row that belongs to no sequence
    for (int64_t e = tid; e < n * row_vecs; e += threads) o[outside(e / row_vecs) * row_vecs + e % row_vecs] = make_uint4(0u, 0u, 0u, 0u);
    if (lse)
        for (int64_t e = tid; e < n * hq; e += threads) lse[e / n * total + outside(e % n)] = 0.f;
}

}  // namespace

int launch_zero_outside(void* o, float* lse, const int64_t* seqstart, int64_t batch, int64_t total, int64_t hq, int64_t row_bytes, cudaStream_t stream) {
    FCK_CUDA(launch_dependent(zero_outside_kernel, dim3((unsigned)sm_count()), dim3(256), 0, stream, (uint4*)o, lse, seqstart, batch, total, hq,
                              row_bytes / 16));
    return FLASHCK_OK;
}

bool bwd_sm100_supported(const BwdParams& p) {
    return p.max_seqlen_q > 0 && p.max_seqlen_k > 0 && p.batch > 0;  // (something to multiply)
}

int launch_bwd_sm100(const BwdParams& p, cudaStream_t stream) {
    int* status = device_status_ptr();
    if (!status) return FLASHCK_ERR_CUDA;
    BwdSm100Dev dev{};
    dev.dout = p.dout; dev.q = p.q; dev.o = p.o; dev.lse = p.lse; dev.dlse = p.dlse; dev.delta = p.delta;
    dev.dq = p.dq; dev.dk = p.dk; dev.dv = p.dv; dev.seqstart_q = p.seqstart_q; dev.seqstart_k = p.seqstart_k; dev.status = status;
    dev.batch = (int)p.batch; dev.seqlen_q = (int)p.seqlen_q; dev.seqlen_k = (int)p.seqlen_k; dev.hq = (int)p.hq; dev.hkv = (int)p.hkv;
    dev.mask_type = p.mask_type; dev.wl = p.wl < 0 ? -1 : (int)p.wl; dev.wr = p.wr < 0 ? -1 : (int)p.wr;
    dev.scale = p.scale; dev.scale_log2 = p.scale * kLog2e;
    dev.bias = p.bias_type == 1 ? p.bias : nullptr; dev.dbias = p.dbias; dev.bias_rank = p.bias_rank;
    dev.bias_sq = p.seqlen_q; dev.bias_sk = p.seqlen_k;
    dev.alibi = p.bias_type == 2 ? (const float*)p.bias : nullptr; dev.alibi_rank = p.bias_rank;
    dev.soft_cap = p.logits_soft_cap;
    if (p.logits_soft_cap > 0.f) {
        dev.cap = soft_cap_constants(p.scale, p.logits_soft_cap);
        dev.inv_cap_log2 = 1.f / (p.logits_soft_cap * kLog2e);
    }
    return p.dtype == FLASHCK_DTYPE_BFLOAT16 ? launch_bwd_d<__nv_bfloat16>(p, dev, stream) : launch_bwd_d<__half>(p, dev, stream);
}

}  // namespace fck
