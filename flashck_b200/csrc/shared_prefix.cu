// fmha_fwd_shared_prefix: decode for a batch whose sequences share a long prefix, in three kernels.
//
//     O = sum_s w_s O_s,   w_s = exp(LSE_s - LSE),   LSE = log sum_s exp(LSE_s)
//
// over the partials s of the prefix and of the sequence's own cache.  1. The prefix: the query rows of all sequences as those of
// one sequence (rows x group per kv head fill whole tiles, so the split kernels read the prefix once per 128 or 256 rows instead
// of once per sequence; the tcgen05 split mode takes 16 tiles of rows in one launch, so more rows go in runs).  2. The own caches,
// as any split-KV call.  3. The merge of both sets of partials, here.
// 131072 keys under 32 sequences of 64 / 8 heads with 1-4096 keys of their own: 217 us a call; by themselves the prefix 125 (537 MB at
// 4.3 TB/s, 1100 TFLOP/s: bound by the steps, as the prefill forms are), the own caches 59 (5.2 TB/s), the merge 13.  8192 keys under
// 64 sequences of 32 / 8 heads with 64-2048 keys of their own: 103 us; 24, 58 and 12.
#include <algorithm>

#include "kernels.h"

namespace fck {

namespace {

// Shortest run of 128-key tiles that a CTA takes of the prefix.  2, 3, 4, 6 or 8 tiles, us in a graph: 1000 keys under 8 sequences of 4
// heads a kv head 28.3, 29.1, 29.2, 31.4, 31.4; 4000 keys under 48 sequences of 1-4 tokens, hdim 64, 44.0, 44.1, 44.2, 45.3, 47.3;
// 2000 keys under 256 sequences 87.5, 87.5, 87.6, 87.5, 89.3; 8192 under 64 103.1, 103.5, 103.0, 102.1, 101.8.
constexpr int64_t kMinPieceTiles = 2;

struct MergeDev {
    const float* lse1;  // prefix: runs of `chunk` rows one behind the other, each [hq, S1, rows of the run]
    const float* o1;
    const float* lse2;  // own caches: [b, hq, S2, sq], group mode [hq, S2, total]
    const float* o2;
    void* o;
    float* lse;
    const int64_t* seqstart_q;
    int batch, rows, sq, hq, s1, s2, chunk;  // rows: all query rows; sq: of a sequence (group mode: all of them)
};

// One CTA = W warps = one (row, head); warp w takes partials w, w + W, ...; O passes through registers once.  What bounds it is
// the round trips of the partials (LSEs, then the rows), of which every warp keeps kAhead in flight.
template <typename T, int D, int W>
__global__ void __launch_bounds__(W * 32) shared_prefix_merge_kernel(const MergeDev p) {
    constexpr int kAhead = 4, V = D / 4;  // float4 of a row
    __shared__ float4 part[W][V];
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = (int)(blockIdx.x / p.hq), h = (int)(blockIdx.x % p.hq);
    if (p.seqstart_q && (row < p.seqstart_q[0] || row >= p.seqstart_q[p.batch])) return;  // (belongs to no sequence: left as it was)
    const int c0 = row / p.chunk * p.chunk, crows = min(p.chunk, p.rows - c0);
    const int64_t at1 = ((int64_t)c0 * p.hq + (int64_t)h * crows) * p.s1 + (row - c0);  // partial s: + s * crows
    const int64_t at2 = ((int64_t)(row / p.sq) * p.hq + h) * p.s2 * p.sq + row % p.sq;  // + s * sq
    const int S = p.s1 + p.s2;
    auto slot = [&](int s) { return s < p.s1 ? at1 + (int64_t)s * crows : at2 + (int64_t)(s - p.s1) * p.sq; };
    auto lse_of = [&](int s) { return s < p.s1 ? p.lse1[slot(s)] : p.lse2[slot(s)]; };
    float m = -INFINITY;
    for (int s = lane; s < S; s += 32) m = fmaxf(m, lse_of(s));
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    float sum = 0.f;
    for (int s = lane; s < S; s += 32) {
        const float l = lse_of(s);
        sum += l == -INFINITY ? 0.f : expf(l - m);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    const float inv = m == -INFINITY ? 0.f : 1.f / sum;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    const bool mine = lane < V;
    for (int j0 = warp; j0 < S; j0 += W * kAhead) {
        float w[kAhead];
        float4 x[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int s = j0 + u * W;
            const float l = s < S ? lse_of(s) : -INFINITY;
            w[u] = l == -INFINITY ? 0.f : expf(l - m) * inv;  // (an unused partial's row may hold anything: it is not read)
            x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (w[u] != 0.f && mine) x[u] = reinterpret_cast<const float4*>((s < p.s1 ? p.o1 : p.o2) + slot(s) * D)[lane];
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            acc.x += w[u] * x[u].x; acc.y += w[u] * x[u].y; acc.z += w[u] * x[u].z; acc.w += w[u] * x[u].w;
        }
    }
    if constexpr (W > 1) {
        if (mine) part[warp][lane] = acc;
        __syncthreads();
        if (warp > 0) return;
        if (mine) {
#pragma unroll
            for (int w = 1; w < W; ++w) {
                const float4 y = part[w][lane];
                acc.x += y.x; acc.y += y.y; acc.z += y.z; acc.w += y.w;
            }
        }
    }
    if (mine)
        reinterpret_cast<uint2*>((T*)p.o + ((int64_t)row * p.hq + h) * D)[lane] =
            make_uint2(Elem<T>::pack2(acc.x, acc.y), Elem<T>::pack2(acc.z, acc.w));
    if (p.lse && lane == 0)
        p.lse[((int64_t)(row / p.sq) * p.hq + h) * p.sq + row % p.sq] = m == -INFINITY ? -INFINITY : m + logf(sum);
}

template <typename T, int D>
int launch_merge(const MergeDev& d, cudaStream_t stream) {
    const int64_t items = (int64_t)d.rows * d.hq;
    const int S = d.s1 + d.s2;
    const dim3 grid((unsigned)items);
    if (S > 32 && items <= (int64_t)sm_count() * 16) FCK_CUDA(launch_dependent(shared_prefix_merge_kernel<T, D, 8>, grid, dim3(256), 0, stream, d));
    else if (S > 8) FCK_CUDA(launch_dependent(shared_prefix_merge_kernel<T, D, 4>, grid, dim3(128), 0, stream, d));
    else FCK_CUDA(launch_dependent(shared_prefix_merge_kernel<T, D, 1>, grid, dim3(32), 0, stream, d));
    return FLASHCK_OK;
}

SplitKVParams prefix_pass(const SharedPrefixParams& p, int64_t row0, int64_t rows) {
    SplitKVParams s{};
    s.q = (const uint8_t*)p.q + row0 * p.hq * p.d * 2;
    s.k = p.k_prefix; s.v = p.v_prefix;
    s.block_table = p.prefix_table;
    s.batch = 1; s.seqlen_q = s.max_seqlen_q = s.total_q = rows;
    s.seqlen_k_cap = p.prefix_len; s.shared_prefix = true; s.min_piece_tiles = kMinPieceTiles;
    s.hq = p.hq; s.hkv = p.hkv; s.d = s.dv = p.d;
    s.num_pages = p.prefix_table ? p.prefix_pool_pages : 1;
    s.bt_stride = p.prefix_table ? (p.prefix_len + p.prefix_page - 1) / p.prefix_page : 0;
    s.page = p.prefix_page;
    s.scale = p.scale; s.wl = s.wr = -1; s.dtype = p.dtype;
    return s;
}

// Nothing in it may depend on what can change between the sizing of the workspace and the call (the instance parameters do).
struct Plan {
    int64_t rows, chunk, s1, s2, floats1, floats2;  // workspace: LSEs and rows of the prefix's partials, then of the others
};

Plan plan(const SharedPrefixParams& p) {
    Plan r{};
    const int64_t group = p.hq / p.hkv;
    r.rows = p.seqstart_q ? p.seqlen_q : p.batch * p.seqlen_q;
    r.chunk = r.rows;
    if (p.prefix_len > 0 && r.rows > 0) {
        const int64_t rpt = group <= 128 ? 128 / group * group : group;  // rows of a tile: whole tokens
        r.chunk = std::min(r.rows, std::max<int64_t>(1, 16 * rpt / group));
        SplitKVParams s = prefix_pass(p, 0, r.chunk);
        s.num_splits = 2;
        s.lse_acc = reinterpret_cast<float*>(16);  // (only asked whether there is one)
        if (splitkv_sm100_supported(s)) {
            r.s1 = splitkv_sm100_prefix_splits(s);
        } else {
            r.chunk = r.rows;
            r.s1 = std::min<int64_t>(128, (p.prefix_len + 31) / 32 + 1);  // the decode kernel: a piece per SM, of two tiles of 16 keys or more
        }
        r.s1 = std::min<int64_t>(std::max<int64_t>(r.s1, 2), 128);
    }
    r.s2 = p.max_seqlen_q * group > 16 ? 16
                                       : std::max<int64_t>(2, std::min<int64_t>(128, (2 * sm_count() + p.batch - 1) / std::max<int64_t>(p.batch, 1) + 1));
    r.floats1 = r.rows * p.hq * r.s1;
    r.floats2 = r.rows * p.hq * r.s2;
    return r;
}

}  // namespace

int64_t shared_prefix_workspace(const SharedPrefixParams& p) {
    Plan r = plan(p);
    if (p.prefix_table) {  // a page size is all that is known here: the call is paged if it has a table
        SharedPrefixParams q = p;
        q.prefix_table = nullptr;
        q.prefix_page = 0;
        r.floats1 = std::max(r.floats1, plan(q).floats1);
    }
    // rows of 16 bytes first, LSEs behind them
    return (r.floats1 + r.floats2) * (p.d + 1) * (int64_t)sizeof(float);
}

int launch_shared_prefix(const SharedPrefixParams& p, cudaStream_t stream) {
    Plan r = plan(p);
    if (r.rows == 0) return FLASHCK_OK;
    FCK_REQUIRE(r.rows * p.hq < (1ll << 31), FLASHCK_ERR_UNSUPPORTED, "FmhaFwdSharedPrefix: %lld rows of %lld heads (fewer than 2^31)",
                (long long)r.rows, (long long)p.hq);
    // (no more partials than pieces of two 16-key tiles in the room that a sequence has: short caches leave fewer slots to mark and merge)
    const int64_t room = p.block_table ? p.bt_stride * p.page : p.seqlen_k_cap;
    r.s2 = std::min(r.s2, std::max<int64_t>(2, (room + 31) / 32 + 1));
    float* o1 = (float*)p.workspace;
    float* o2 = o1 + r.floats1 * p.d;
    float* lse1 = o2 + r.floats2 * p.d;
    float* lse2 = lse1 + r.floats1;
    for (int64_t row0 = 0; r.s1 > 0 && row0 < r.rows; row0 += r.chunk) {
        SplitKVParams s = prefix_pass(p, row0, std::min(r.chunk, r.rows - row0));
        s.num_splits = r.s1;
        s.o_acc = o1 + row0 * p.hq * r.s1 * p.d;
        s.lse_acc = lse1 + row0 * p.hq * r.s1;
        if (int rc = splitkv_sm100_supported(s) ? launch_splitkv_sm100(s, stream) : launch_splitkv_decode(s, stream)) return rc;
    }
    SplitKVParams s{};
    s.q = p.q; s.k = p.k; s.v = p.v; s.o_acc = o2; s.lse_acc = lse2;
    s.seqstart_q = p.seqstart_q; s.seqlen_k = p.seqlen_k; s.block_table = p.block_table;
    s.batch = p.batch; s.seqlen_q = p.seqlen_q; s.max_seqlen_q = p.max_seqlen_q; s.total_q = r.rows;
    s.seqlen_k_cap = p.seqlen_k_cap; s.hq = p.hq; s.hkv = p.hkv; s.d = s.dv = p.d; s.num_splits = r.s2;
    s.num_pages = p.block_table ? p.pool_pages : p.batch;
    s.bt_stride = p.bt_stride; s.page = p.page; s.scale = p.scale;
    s.mask_type = p.causal ? 2 : 0; s.wl = -1; s.wr = p.causal ? 0 : -1; s.dtype = p.dtype;
    if (room == 0) r.s2 = 0;  // caches without room: no sequence has own keys
    else if (int rc = splitkv_sm100_supported(s) ? launch_splitkv_sm100(s, stream) : launch_splitkv_decode(s, stream)) return rc;
    MergeDev m{};
    m.lse1 = lse1; m.o1 = o1; m.lse2 = lse2; m.o2 = o2; m.o = p.o; m.lse = p.lse; m.seqstart_q = p.seqstart_q;
    m.batch = (int)p.batch; m.rows = (int)r.rows; m.sq = (int)p.seqlen_q; m.hq = (int)p.hq;
    m.s1 = (int)r.s1; m.s2 = (int)r.s2; m.chunk = (int)r.chunk;
    if (p.dtype == FLASHCK_DTYPE_BFLOAT16)
        return p.d == 128 ? launch_merge<__nv_bfloat16, 128>(m, stream) : launch_merge<__nv_bfloat16, 64>(m, stream);
    return p.d == 128 ? launch_merge<__half, 128>(m, stream) : launch_merge<__half, 64>(m, stream);
}

}  // namespace fck
