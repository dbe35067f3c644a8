// fmha_fwd_splitkv over a 4-bit cache: partial attention of a few query rows per kv head, one partial (O_s, LSE_s) per split.
//
// A token of a kv head is d codes u (4 bits) and, for each group of channels, (scale s, least value m):  k_c = m + s u_c.  So
//     q . k = sum_g ( s_g sum_{c in g} q_c u_c  +  m_g sum_{c in g} q_c ),
//     O_c   = sum_j p_j (m_j + s_j u_jc) = sum_j (p_j s_j) (u_jc - 8)  +  sum_j p_j (m_j + 8 s_j),
// and no key or value is ever written out: the products run over the codes themselves, scales and least values come in once per key.
// The second sum of O is one number per row and group; with 8 taken off, what the rounding of p s to 16 bits costs is in proportion to
// the values' spread, not to their distance from the least one.
//
// Codes become MMA operands in a few instructions: a 4-bit field in the low mantissa bits of a half IS u * 2^-24 (a subnormal, which the tensor
// cores multiply exactly), a byte of two fields u0 + 16 u1.  ldmatrix hands a warp the K rows as they lie, and, transposed, the 16-bit pieces (4
// channels) of the V rows of two keys side by side.  A mask or a byte permutation makes each operand; the powers of two go to Q, or to O at the
// end, and so does the lower field that a byte brings along: V's bytes are freed of it by one subtraction of sums, K's by a subtraction of halves
// (8 rows) or by a second column of Q (4 rows).
// Both products are taken transposed (S^T = K Q^T, O^T = V^T P^T): m16n8k16 then has 16 keys or channels against 8 query columns, which a group of
// 8 heads fills (or 4 with two columns each), instead of 16 rows half empty.  P^T's fragments come from S^T's by movmatrix.
//
// Halves have no range for arbitrary Q and scales.  A row of Q is scaled by a power of two.  The weights p s are kept in range by the row's
// reference R (p' = exp2(x - R)): it follows the largest x + log2 s seen, moves when a weight passes 2^13, and then everything the row
// has summed is rescaled.  Moves are rare, and what decides one is a maximum over packed halves and a vote, without a shuffle.
// Each group of channels follows its own largest x + log2 s, by a power of two (its lift) that its weights are multiplied by on top: with R
// alone a group whose scales are 2^-20 of another's would keep 9 of its weights' 11 bits, and none at 2^-30; and R keeps p' within 2^-96 and 2^60, which
// scales outside 2^-60 and 2^100 need more than.
//
// A CTA per SM: four producer warps and 16 consumer warps.  A stage is 256 (head, token) pairs -- 32 tokens of 8 heads, 256 of one -- of K and V
// codes, by TMA (boxes of up to 256 tokens of a page, rows of 128 bytes, swizzled: a warp's reads meet no bank twice), and their scales, by 4- to
// 16-byte asynchronous copies.  A consumer warp takes 32 tokens of one head; the warps form two teams of 8, which take stages in turn (up to 8
// rows per kv head), or all stages with a tile of 8 rows each (more).  The warps of a head meet once per segment, in shared memory.  The work
// is cut as in splitkv_decode.cu, by what it costs: a tile of more than 8 rows is 3 units where one of fewer is 2 (see cost()), a sequence's
// beginning kBegin units.
//
// What bounds it (B200, bf16, hdim 128, 8 kv heads): the floor is the cache's bytes in HBM, 136 a token and head with one group.  64 sequences of
// 1-32k keys under 32 heads: 202-204 us and 5 for the merge, floor 171 at 6.54 TB/s; with the arithmetic left out of a copy the loads alone take
// 178-181, with the codes' loads left out the arithmetic 193-195: about 380 instructions a warp and 32 keys, at 0.6 a cycle and scheduler.  4 x 524288
// keys under 64 heads with two groups: 540-545 us, floor 370: eight rows and two groups have more sums than registers, and 30 loads and stores of
// spilled ones per 32 keys.
#include <algorithm>
#include <type_traits>

#include "kernels.h"

namespace fck {

namespace {

constexpr int kPairs = 256;  // (head, token) pairs of a stage
constexpr int kUnit = 32;    // tokens a warp takes of it
constexpr int kCentre = 8;   // units between two centrings
constexpr int kMeetWarps = 4;  // warps that hand their sums over at a time
// Units of the schedule that a sequence costs beside its tiles, for its queries and the meeting of the warps: 4 x 524288 keys 560 -> 550 us, 32 sequences
// of 1-32k keys and 64 / 8 heads 165 -> 159; 3 and 10 gave about the same.
constexpr int kBegin = 6;
constexpr uint32_t kCode = 0x000f000fu;
// Least lift of a group, as a power of two, up or down.  (Below it the largest weights are within 2^-2 and 2^10, and a half's numbers are normal down to
// 2^-14; groups whose scales are of a kind, the usual ones, then take no lift at all.)
constexpr float kLeastLift = 6.f;
constexpr float kNoKey = -1e30f;  // (any score is so far above it that the reference moves)

struct Int4Dev {
    const void* q;
    float* o_acc;
    float* lse_acc;
    const int64_t* seqstart_q;
    const int32_t* seqlen_k;
    const int32_t* block_table;
    const int64_t* cache_batch_idx;
    const uint8_t* k_params;
    const uint8_t* v_params;
    int* status;
    int batch, seqlen_q, hq, hkv, num_splits, total_q, bt_stride, page, pool, room;  // room: tokens that a sequence's part of the cache has
    int mask_type, wl, wr;
    int heads_log2, chunk_log2, stages;  // kv heads of a CTA; tokens of a box
    int dual;                            // sequences may have a second tile of 8 rows, which the second team of warps takes: both go through all stages
    int line_log2;                       // bytes of a box's innermost rows: 128, or what the CTA's heads have
    float scale_log2;
};

__device__ __forceinline__ int len_q(const Int4Dev& p, int b) {
    return p.seqstart_q ? (int)(p.seqstart_q[b + 1] - p.seqstart_q[b]) : p.seqlen_q;
}
__device__ __forceinline__ int len_k(const Int4Dev& p, int b) { return min(p.seqlen_k[b], p.room); }
// What a tile of a sequence costs, in units of the schedule: with more than 8 rows both teams go through all tiles, else each through every other one.  (A CTA
// alone took 3200 and 2000 cycles a tile at hdim 64; 32 sequences of 1-4 tokens, 32 / 8 heads, hdim 128, with one cost for both: groups of 128 210 -> 191 us,
// of 64 282 -> 251, of 32 486 -> 433.  2 : 1 was worse than one cost: 48 short ones at hdim 64 85 -> 97.)
__device__ __forceinline__ int cost(const Int4Dev& p, int b) { return !p.dual ? 1 : len_q(p, b) * (p.hq / p.hkv) > 8 ? 3 : 2; }
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}
template <bool TRANS, int OFFSET>
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t addr) {
    if constexpr (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4+%5];\n"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr), "n"(OFFSET));
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4+%5];\n"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr), "n"(OFFSET));
}
// c = a b, or with SUM c += a b
template <bool SUM>
__device__ __forceinline__ void product(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (SUM) {
        mma_16816<__half>(c, a, b0, b1);
    } else {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
    }
}
template <int N>
__device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(N)); }
// The four fields of a word whose halves hold four codes each, as halves over 2^24: first the lowest, then 16 times the next one (from the
// byte that both make up, less the lowest: that subtraction runs beside the masks, which have half of its rate), the same of the upper bytes.
__device__ __forceinline__ uint32_t less(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ void fields(uint32_t w, uint32_t (&f)[4]) {
    const uint32_t lower = w & 0x00ff00ffu, upper = __byte_perm(w, 0, 0x4341);
    f[0] = w & kCode;
    f[1] = less(lower, f[0]);
    f[2] = upper & kCode;
    f[3] = less(upper, f[2]);
}
// For values: the lowest field, and the byte, 16 times the next one plus the lowest, which the sums are freed from at the end.
__device__ __forceinline__ void bytes(uint32_t w, uint32_t (&f)[4]) {
    f[1] = w & 0x00ff00ffu;
    f[3] = __byte_perm(w, 0, 0x4341);
    f[0] = w & kCode;
    f[2] = f[3] & kCode;
}
__device__ __forceinline__ uint32_t max_halves(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.f16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// s[0] and s[1] plus the halves of a word
__device__ __forceinline__ void add_halves(float (&s)[2], uint32_t w) {
    asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %2;\nadd.f32.f16 %0, lo, %0;\nadd.f32.f16 %1, hi, %1;\n}\n" : "+f"(s[0]), "+f"(s[1]) : "r"(w));
}
__device__ __forceinline__ void add_halves(float (&s)[1], uint32_t w) {
    asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %1;\nadd.f32.f16 %0, lo, %0;\n}\n" : "+f"(s[0]) : "r"(w));
}
__device__ __forceinline__ bool elected() {
    uint32_t yes;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(yes));
    return yes != 0;
}
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;\n" ::"r"(dst), "l"(src), "n"(BYTES), "r"(there ? BYTES : 0) : "memory");
}
__device__ __forceinline__ void arrive_after_copies(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ uint32_t halves(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Shared memory of a stage: K codes, V codes [chunk][128-byte column][token] rows, K params, V params [token] rows of the CTA's heads, with
// 16 bytes between two where they are 64 bytes and more: a warp reads one of 8 tokens at a time, which then lie in different banks.  (With E = 2 it
// costs more than it gives: 32 sequences of 64 / 8 heads, groups of 64, 167 -> 185 us; with E = 1 and 32 / 8 heads 159 -> 135, groups of 32
// 275 -> 209.)
template <int D, int NG, int E>
struct Stage {
    static constexpr int kCodes = kPairs * (D / 2);
    static constexpr int kParams = kPairs * NG * 4 + (E == 2 || NG == 1 ? 0 : 256 * NG);
    static constexpr int kBytes = (2 * kCodes + 2 * kParams + 1023) / 1024 * 1024;
};

// 16 consumer warps and 4 producer warps share the registers that the block is launched with: kLaunch a thread (what the launch bounds leave:
// 65536 / threads, down to a multiple of 8).
constexpr int kConsumers = 16, kThreads = (kConsumers + 4) * 32, kLaunch = 65536 / kThreads / 8 * 8, kProducerRegs = 32, kConsumerRegs = 112;
static_assert((kConsumers * kConsumerRegs + 4 * kProducerRegs) * 32 <= kThreads * kLaunch, "an increase would wait for good");

// What one warp has summed over its keys (weights w = p' s times the group's lift, a power of two in shared memory), for the lane's E rows: 2t and 2t + 1 of 8 (E = 2, t = lane % 4), or t of 4 (E = 1; what belongs to odd
// columns then stays zero).
template <int D, int NG, int E>
struct Sums {
    float o[D / 32][2][4];  // sum w u over 2^24 ([0]: channels 4g, 4g + 2 of 32; [1]: 16 times 4g + 1, 4g + 3 plus those)
    float ones[NG][E];      // sum w (as rounded) over the lane's keys since the last centring
    float mid[NG][E];       // sum p' (m + 8 s) over the lane's keys
    float l[E];             // sum p' over the lane's keys
    float ref[E];           // R; kNoKey before the first key
};

template <typename T, int D, int NG, int E>
__global__ void __launch_bounds__(kThreads, 1)
splitkv_int4_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Int4Dev p) {
    constexpr int ROW = D / 2, GR = D / 32, PER = GR / NG;  // bytes of a row; 16-byte pieces (32 channels) of it; of them per group
    using St = Stage<D, NG, E>;
    extern __shared__ uint8_t smem_raw[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = p.hq / p.hkv, stages = p.stages;
    const int heads = 1 << p.heads_log2, tok_log2 = 8 - p.heads_log2, toks = 1 << tok_log2;

    uint8_t* ring = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    float4* meet = reinterpret_cast<float4*>(ring + (size_t)stages * St::kBytes);  // [kMeetWarps][rows and columns of a lane][lane]: warps' sums
    constexpr int kMeetFloat4 = E * GR;  // float4 per lane
    float* meet_stats = reinterpret_cast<float*>(meet + kMeetWarps * kMeetFloat4 * 32);  // [warp][4 E rows][ref, l]
    uint64_t* bars = reinterpret_cast<uint64_t*>(meet_stats + kMeetWarps * 4 * E * 2);
    uint64_t* full = bars;
    uint64_t* empty = bars + stages;
    int* prefix = reinterpret_cast<int*>(bars + 2 * stages);  // [batch + 1] cost of the tiles before each sequence
    int* tile0 = prefix + p.batch + 1;
    volatile int* abort_flag = tile0 + p.batch;
    int* longest = const_cast<int*>(abort_flag) + 1;
    int* begin = longest + 1;  // what the first tile of a sequence costs more
    float* lifts = reinterpret_cast<float*>(begin + 1) + ((warp & (kConsumers - 1)) * NG * 4 + (lane & 3)) * E;  // [warp][NG][rows]: see Sums; of this lane's first row

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(&full[s], 33);  // the lanes' copies of scales, and the byte count of the boxes
            mbar_init(&empty[s], p.dual ? 16 : 8);
        }
        *abort_flag = 0;
        mbar_fence_init();
    }
    const bool per_sequence = p.num_splits <= 1;
    pdl_launch_dependents();
    pdl_wait();
    // ---- schedule: what the tiles (stages) of each sequence cost, and the prefix sums ----
    if (warp == 0) {
        int run = 0, mx = 0, sequences = 0;
        for (int base = 0; base < p.batch; base += 32) {
            const int b = base + lane;
            int n = 0, t0 = 0;
            if (b < p.batch) {
                const int len = len_k(p, b);
                if (len > 0) {
                    int first = 0;
                    if (p.mask_type != 0 && p.wl >= 0) first = max(0, min(len - 1, (p.mask_type == 2 ? len - len_q(p, b) : 0) - p.wl));
                    t0 = first >> tok_log2;
                    n = (((len - 1) >> tok_log2) + 1 - t0) * cost(p, b);
                }
                tile0[b] = t0;
            }
            int incl = n;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, incl, off);
                if (lane >= off) incl += y;
            }
            if (b < p.batch) prefix[b] = run + incl - n;
            run += __shfl_sync(0xffffffffu, incl, 31);
            sequences += __popc(__ballot_sync(0xffffffffu, n > 0));
            mx = max(mx, __reduce_max_sync(0xffffffffu, n));
        }
        // (where the CTAs have kBegin units each and more; a piece, which has to have a tile of a sequence that it cuts, would else be longer than the
        // share of a CTA.  Below: one sequence of 3000 keys 18.5 -> 22.5 us.  Above: 256 of 10-200 keys, 6.4 units a CTA, 47 -> 41, 16 of 500-8000,
        // 16 a CTA, 41 -> 39.)
        const int extra = !per_sequence && run / kBegin >= (int)gridDim.x ? kBegin : 0;
        if (extra) {
            __syncwarp();
            int before = 0;  // sequences with tiles
            for (int base = 0; base < p.batch; base += 32) {
                const int b = base + lane, from = b < p.batch ? prefix[b] : run, to = b + 1 < p.batch ? prefix[b + 1] : run;
                const uint32_t have = __ballot_sync(0xffffffffu, to > from);  // (and all have read)
                if (b < p.batch) prefix[b] = from + extra * (before + __popc(have & ((1u << lane) - 1u)));
                before += __popc(have);
            }
            run += extra * sequences;
        }
        if (lane == 0) {
            prefix[p.batch] = run;
            *longest = mx + extra;
            *begin = extra;
        }
    }
    __syncthreads();

    const int total = prefix[p.batch];
    const int even = (total + (int)gridDim.x - 1) / (int)gridDim.x;
    const int cap = per_sequence ? 0 : (*longest + p.num_splits - 2) / (p.num_splits - 1);
    const int piece_len = max((p.dual ? 3 : 1) + *begin, max(even, cap));  // (a piece amid a sequence has a tile of it)
    const int pieces = per_sequence ? p.batch : (total + piece_len - 1) / piece_len;
    auto begin_piece = [&](int piece, int& lo, int& hi) {  // its units, and the sequence it starts in
        if (per_sequence) {
            lo = prefix[piece];
            hi = prefix[piece + 1];
            return piece;
        }
        lo = piece * piece_len;
        hi = min(total, lo + piece_len);
        int a = 0, z = p.batch - 1;
        while (a < z) {
            const int mid = (a + z + 1) >> 1;
            if (prefix[mid] <= lo) a = mid; else z = mid - 1;
        }
        return a;
    };
    auto tiles = [&](int b, int lo, int hi, int& ta, int& tb) {  // a piece's tiles of a sequence: those whose first unit it has
        const int w = cost(p, b), from = max(lo, prefix[b]) - prefix[b], to = min(hi, prefix[b + 1]) - prefix[b];
        const auto before = [&](int x) {  // tiles whose first unit is below x: the first one's is 0, the others' begin + w, begin + 2 w, ..
            if (x <= *begin) return x > 0 ? 1 : 0;
            x += w - 1 - *begin;
            return w == 1 ? x : w == 2 ? x / 2 : x / 3;
        };
        ta = before(from);
        tb = before(to);
    };
    const int head0 = blockIdx.z << p.heads_log2;
    const int row0 = blockIdx.y * (p.dual ? 16 : 4 * E);  // first (token, group head) row of this CTA

    if (warp >= kConsumers) {
        // ============ producer warps: two fetch codes and two scales, each pair every other stage (their number is even, so a stage always falls
        // to the same two; one warp for all of it was what bound the kernel, at 1700 cycles a stage) ============
        registers_down<kProducerRegs>();
        const int mine = warp & 1, kind = (warp >> 1) & 1;  // stages mine, mine + 2, ..; 0: codes, 1: scales and least values
        if (kind == 0 && lane == 0) {
            tma_prefetch_desc(&map_k);
            tma_prefetch_desc(&map_v);
        }
        const int chunk = 1 << p.chunk_log2, box = heads * chunk * ROW, column0 = (head0 * ROW) >> p.line_log2;
        // scales and least values: a lane copies a piece of 4 to 16 bytes of a token's, for K and V
        const int width = heads * NG * 4, pitch = width + (E == 1 && width >= 64 ? 16 : 0);
        const int piece_log2 = min(4, 31 - __clz(width)), pieces_log2 = 31 - __clz(width) - piece_log2;
        const int copies = toks << pieces_log2;
        const int per_tile_log2 = tok_log2 - p.chunk_log2;
        int tile_count = 0, next = mine, stage = mine;  // (as the consumers count them)
        uint32_t phase = 0;
        bool ok = true;
        for (int piece = blockIdx.x; piece < pieces && ok; piece += gridDim.x) {
            int lo, hi, b = begin_piece(piece, lo, hi);
            for (; b < p.batch && prefix[b] < hi && ok; ++b) {
                int ta, tb;
                tiles(b, lo, hi, ta, tb);
                if (tb <= ta || row0 >= len_q(p, b) * G) continue;  // (the consumers skip the same segments)
                const int len = len_k(p, b);
                const int64_t bphys = p.cache_batch_idx ? p.cache_batch_idx[b] : b;
                // pages of 32 chunks (a few tiles) per round, a lane each, loaded one round ahead; a page that is not there is one behind the pool
                const int first_chunk = (tile0[b] + ta) << per_tile_log2, all_chunks = (tb - ta) << per_tile_log2;
                auto entry = [&](int c, int& pg, int& tok) {
                    const int64_t token = (int64_t)(first_chunk + c) << p.chunk_log2;
                    pg = p.pool;
                    tok = 0;
                    if (token >= len || c >= all_chunks) return;
                    if (p.block_table) {
                        const int slot = (int)token / p.page;
                        tok = (int)token - slot * p.page;
                        const int id = slot < p.bt_stride ? p.block_table[bphys * p.bt_stride + slot] : -1;
                        if ((uint32_t)id < (uint32_t)p.pool) pg = id;
                    } else {
                        tok = (int)token;
                        if ((uint64_t)bphys < (uint64_t)p.pool) pg = (int)bphys;
                    }
                };
                int pg_cur = 0, tok_cur = 0, pg_next, tok_next, round = -1;
                entry(lane, pg_next, tok_next);
                for (int t = ta + next - tile_count; t < tb; t += 2) {
                    const int s = stage, c0 = (t - ta) << per_tile_log2;  // the tile's first chunk
                    const uint32_t parity = phase ^ 1u;
                    next += 2;
                    stage += 2;
                    if (stage >= stages) {
                        stage -= stages;
                        phase ^= 1u;
                    }
                    if ((c0 >> 5) != round) {  // (a round has 2 tiles or more, so none is passed over)
                        round = c0 >> 5;
                        pg_cur = pg_next;
                        tok_cur = tok_next;
                        entry((round + 1) * 32 + lane, pg_next, tok_next);
                    }
                    const int from = (c0 & 31) + (lane & ((1 << per_tile_log2) - 1));
                    const int pg = __shfl_sync(0xffffffffu, pg_cur, from), tok = __shfl_sync(0xffffffffu, tok_cur, from);
                    const int token0 = (tile0[b] + t) << tok_log2;
                    // (stages ahead of the consumers there is no hurry: looking seldom leaves them the issue slots)
                    for (int k = 0; k < 64 && !mbar_try_wait(&empty[s], parity); ++k) __nanosleep(200);
                    // (all lanes leave a wait with one outcome, here and in the consumers: shuffles and arrivals of whole warps follow)
                    if (!(ok = __all_sync(0xffffffffu, mbar_wait_bounded(&empty[s], parity, abort_flag, p.status, 0x100)))) break;
                    uint8_t* st = ring + (size_t)s * St::kBytes;
                    if (kind == 0) {
                        const int chunks = min(1 << per_tile_log2, (len - token0 + chunk - 1) >> p.chunk_log2);
                        if (lane == 0) mbar_expect_tx(&full[s], 2 * chunks * box);
                        __syncwarp();
                        if (lane < chunks) {
                            tma_load_4d(st + lane * box, &map_k, &full[s], 0, tok, column0, pg);
                            tma_load_4d(st + St::kCodes + lane * box, &map_v, &full[s], 0, tok, column0, pg);
                        }
                        continue;
                    }
                    const int64_t at = pg < p.pool ? ((int64_t)pg * p.page + tok) * p.hkv + head0 : -1;  // the chunk's first (token, head)
                    const uint32_t dst = smem_u32(st + 2 * St::kCodes);
                    for (int e = lane; e < copies; e += 32) {
                        const int k = e >> pieces_log2, part = (e & ((1 << pieces_log2) - 1)) << piece_log2;  // token of the tile, byte of its row
                        const int64_t first = __shfl_sync(0xffffffffu, at, k >> p.chunk_log2);
                        const bool there = first >= 0 && token0 + k < len;  // (the rest of a tile has scales of zero)
                        const int64_t off = there ? (first + (int64_t)(k & (chunk - 1)) * p.hkv) * (4 * NG) + part : 0;
                        const uint32_t to = dst + k * pitch + part;
                        if (piece_log2 == 4) {
                            copy_async<16>(to, p.k_params + off, there);
                            copy_async<16>(to + St::kParams, p.v_params + off, there);
                        } else if (piece_log2 == 3) {
                            copy_async<8>(to, p.k_params + off, there);
                            copy_async<8>(to + St::kParams, p.v_params + off, there);
                        } else {
                            copy_async<4>(to, p.k_params + off, there);
                            copy_async<4>(to + St::kParams, p.v_params + off, there);
                        }
                    }
                    arrive_after_copies(&full[s]);
                }
                tile_count += tb - ta;
            }
        }
        // ---- unused splits get LSE = -inf (see splitkv_decode.cu: shared out over gridDim.x / batch CTAs) ----
        if (ok && warp == kConsumers && blockIdx.y == 0 && blockIdx.z == 0) {
            const int parts = max(1, (int)gridDim.x / p.batch), part = parts > 1 ? (int)blockIdx.x / p.batch : 0;
            for (int b = parts > 1 ? (int)blockIdx.x % p.batch : (int)blockIdx.x; b < p.batch && part < parts; b += gridDim.x) {
                const int n = prefix[b + 1] - prefix[b];
                const int w = cost(p, b), last = n == *begin + w ? prefix[b] : prefix[b + 1] - w;  // the last tile's first unit
                const int used = n == 0 ? 0 : per_sequence ? 1 : last / piece_len - prefix[b] / piece_len + 1;
                const int sq = len_q(p, b);
                const int64_t rows = p.seqstart_q ? p.total_q : p.seqlen_q, head = p.num_splits * rows;  // LSEs of a split, of a head
                float* first = p.lse_acc + (p.seqstart_q ? p.seqstart_q[b] : (int64_t)b * p.hq * head) + used * rows;
                for (int e = lane; e < (p.num_splits - used) * sq; e += 32) {
                    const int s = e / sq;
                    float* at = first + s * rows + (e - s * sq);
                    for (int h = part; h < p.hq; h += parts) at[h * head] = -INFINITY;
                }
            }
        }
        // Copies of its own end before the warp does: of the small ones always, and after a wait that ran out, when no consumer may have
        // waited for them, of the boxes too.
        asm volatile("cp.async.wait_all;\n" ::: "memory");
        if (*abort_flag) {
            // (the last use of each of this warp's stages; one that it did not fill, or not wholly, costs the limit)
            for (int u = next - 2; u >= 0 && u >= next - stages; u -= 2)
                for (int k = 0; k < 10000 && !mbar_try_wait_hint(&full[u % stages], (uint32_t)(u / stages) & 1u, 2000u); ++k) {}
        }
        return;
    }

    // =============================== consumer warps =============================================
    registers_up<kConsumerRegs>();
    const int team = warp >> 3, wi = warp & 7;
    const int hw = wi & (heads - 1), unit = wi >> p.heads_log2;  // head of the CTA; which 32 tokens of a tile
    const int kh = head0 + hw;
    const int g = lane >> 2, t4 = lane & 3;
    // ldmatrix: this lane's row of the four 8 x 16-byte matrices of 16 keys and two 16-byte pieces (32 channels each): matrix m holds keys
    // 8 (m & 1) .. + 7 and piece m >> 1.  Swizzled as the boxes are, the 8 rows of a matrix lie in different banks.
    const int mrow = (lane & 7) + 8 * ((lane >> 3) & 1);
    const int mswz = p.line_log2 == 7 ? lane & 7 : p.line_log2 == 6 ? (lane >> 1) & 3 : (lane >> 2) & 1;
    const int per_line_log2 = p.line_log2 - (D == 128 ? 6 : 5);  // heads of a line
    uint32_t off[2][GR / 2];  // in the ring: of the warp's two blocks of 16 keys and two pairs of pieces of a stage
    {
        const int k = unit * kUnit, c = k >> p.chunk_log2;
        const int column = (c << (p.heads_log2 - per_line_log2)) + (hw >> per_line_log2);
        const int row = (column << p.chunk_log2) + (k & ((1 << p.chunk_log2) - 1)) + mrow;
        const int piece = (hw & ((1 << per_line_log2) - 1)) * GR + (lane >> 4);
        const int block_step = p.chunk_log2 == 4 ? heads * 16 * ROW : 16 << p.line_log2;  // (the next chunk, or further down this one)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < GR / 2; ++i) off[u][i] = smem_u32(ring) + u * block_step + (row << p.line_log2) + (((piece + 2 * i) ^ mswz) << 4);
    }
    const int width = heads * NG * 4, pitch = width + (E == 1 && width >= 64 ? 16 : 0);
    const uint32_t param_off = 2 * St::kCodes + (unit * kUnit + g) * pitch + hw * (4 * NG);
    bool failed = false;
    // Tiles are counted over all segments; a team takes every other one, or (dual) goes through all.  tile_count: before this segment; next: this team's next
    // one, its stage and the parity of its use.
    const int step = p.dual ? 1 : 2;
    int tile_count = 0, next = p.dual ? 0 : team, stage = next;
    uint32_t phase = 0;

    for (int piece = blockIdx.x; piece < pieces; piece += gridDim.x) {
        int lo, hi, b = begin_piece(piece, lo, hi);
        for (; b < p.batch && prefix[b] < hi; ++b) {
            int ta, tb;
            tiles(b, lo, hi, ta, tb);
            const int sq = len_q(p, b), rows = sq * G;
            if (tb <= ta || row0 >= rows) continue;
            const int len = len_k(p, b);
            const int split = per_sequence ? 0 : piece - prefix[b] / piece_len;
            const int64_t q0 = p.seqstart_q ? p.seqstart_q[b] : (int64_t)b * p.seqlen_q;
            const bool two_tiles = p.dual && rows - row0 > 8;  // a team's own rows; else the teams share one tile, and take stages in turn
            const int first_row = row0 + (two_tiles ? 8 * team : 0);

            // ---- Q^T fragments: this lane has channels 32 i + 8 t .. + 7 of a row, as halves scaled by a power of two.  E = 2: of row g.  K's
            // operands are fields (channels 0, 4 of 8), and 16 times the next ones (1, 5), and so on.  E = 1: columns 2r and 2r + 1 belong to row r,
            // whose score is the sum of both.  K's operands are fields n0 and whole bytes n0 + 16 n1; q0 n0 + q1 n1 = q0 n0 + q1/16 (n0 + 16 n1) -
            // q1/16 n0, of which the odd column holds the last term: no subtraction to free the bytes of their lower fields. ----
            uint32_t qf[GR][4];
            float ka[E], kb[NG][E];  // x = ka * (s . a) + kb . m
            {
                const int r = first_row + (E == 2 ? g : g >> 1), i = r / G;
                float x[GR][8], amax = 0.f;
                const T* src = (const T*)p.q + ((q0 + i) * p.hq + kh * G + (r - i * G)) * D + 8 * t4;
#pragma unroll
                for (int c = 0; c < GR; ++c) {
                    uint4 w = make_uint4(0, 0, 0, 0);
                    if (r < rows) w = *reinterpret_cast<const uint4*>(src + 32 * c);
                    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        x[c][k] = Elem<T>::to_f32(e[k]);
                        amax = fmaxf(amax, fabsf(x[c][k]));
                    }
                }
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                // largest magnitude into [2^13, 2^14): with it the /16 of half of the channels and 2^-24 of the rest stay exact
                // (as far as 32 bits hold ka = scale 2^(ex + 11): ex up to 118 for scales of 2^-3, and halves up to 2^16 take rows up to 2^121)
                const int most = min(120, 115 - ((int)((__float_as_uint(p.scale_log2) >> 23) & 255) - 127));
                const int ex = amax > 0.f ? max(-100, min(most, (int)((__float_as_uint(amax) >> 23) & 255) - 127)) : 13;
                const float up = __uint_as_float((uint32_t)(127 + 13 - ex) << 23), down = __uint_as_float((uint32_t)(127 - 13 + ex) << 23);
                float sum[NG];
#pragma unroll
                for (int k = 0; k < NG; ++k) sum[k] = 0.f;
#pragma unroll
                for (int c = 0; c < GR; ++c) {
                    __half h[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        h[k] = __float2half_rn(x[c][k] * up);
                        sum[c / PER] += __half2float(h[k]);
                    }
#pragma unroll
                    for (int k = 0; k < 4; k += 2) {
                        const __half2 own = __halves2half2(h[k], h[k + 4]);
                        const __half2 odd = __hmul2(__halves2half2(h[k + 1], h[k + 5]), __float2half2_rn(0.0625f)), minus = __hneg2(odd);
                        qf[c][k] = *reinterpret_cast<const uint32_t*>(&own);
                        qf[c][k + 1] = *reinterpret_cast<const uint32_t*>(&odd);
                        if (E == 1 && (g & 1)) {
                            qf[c][k] = *reinterpret_cast<const uint32_t*>(&minus);
                            qf[c][k + 1] = 0u;
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < NG; ++k) {
                    sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 1);
                    sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 2);
                }
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int from = (2 * t4 + e) * 4;  // a lane of the row
                    const float scale = p.scale_log2 * __shfl_sync(0xffffffffu, down, from);
                    ka[e] = scale * 16777216.f;
#pragma unroll
                    for (int k = 0; k < NG; ++k) kb[k][e] = scale * __shfl_sync(0xffffffffu, sum[k], from);
                }
            }
            int mask_from = len;  // first key that some row may not see
            int mask_below = 0;     // and the first one that no row's left bound hides
            if (p.mask_type != 0) {
                const int shift = p.mask_type == 2 ? len - sq : 0;
                if (p.wr >= 0) mask_from = min(mask_from, shift + p.wr + 1);
                if (p.wl >= 0) mask_below = shift + sq - 1 - p.wl;
            }

            Sums<D, NG, E> z;
#pragma unroll
            for (int c = 0; c < GR; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) z.o[c][j >> 2][j & 3] = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) {
#pragma unroll
                for (int k = 0; k < NG; ++k) z.ones[k][e] = z.mid[k][e] = 0.f;
                z.l[e] = 0.f;
                z.ref[e] = kNoKey;
            }

            bool lifted = false;  // some lift is not 1

            // 8 times the weights' sum taken off the sums of codes.  Tensor cores cut the sums of their products off instead of rounding them;
            // codes are never negative, so uncentred sums grow with the keys and lose on one side (4 x 524288 keys: O 0.9 % off), which
            // centring every 256 keys of the warp's own prevents.
            auto centre = [&]() {
#pragma unroll
                for (int k = 0; k < NG; ++k)
#pragma unroll
                    for (int e = 0; e < E; ++e)
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) z.ones[k][e] += __shfl_xor_sync(0xffffffffu, z.ones[k][e], d);
#pragma unroll
                for (int c = 0; c < GR; ++c)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if ((j & 1) >= E) continue;
                        z.o[c][0][j] = fmaf(-8.f / 16777216.f, z.ones[c / PER][j & (E - 1)], z.o[c][0][j]);
                        z.o[c][1][j] = fmaf(-136.f / 16777216.f, z.ones[c / PER][j & (E - 1)], z.o[c][1][j]);
                    }
#pragma unroll
                for (int k = 0; k < NG; ++k)
#pragma unroll
                    for (int e = 0; e < E; ++e) z.ones[k][e] = 0.f;
            };
            // a team that takes every other tile has those of one parity: its own count is half of the tile's number
            const int own_log2 = tok_log2 + (two_tiles ? 0 : 1);
            int key0 = ((tile0[b] + ta + next - tile_count) << tok_log2) + unit * kUnit - step * toks;
            for (int t = ta + next - tile_count; t < tb; t += step) {
                key0 += step * toks;
                const int now = stage;
                const uint32_t parity = phase;
                next += step;
                stage += step;
                if (stage >= stages) {
                    stage -= stages;
                    phase ^= 1u;
                }
                if (failed || !__all_sync(0xffffffffu, mbar_wait_bounded(&full[now], parity, abort_flag, p.status, 0x200))) { failed = true; continue; }
                // (dual, one tile: the other team's stages are only given back)
                if (key0 < len && (!p.dual || two_tiles || ((next ^ team) & 1))) {
                    uint32_t at[2][GR / 2];
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int i = 0; i < GR / 2; ++i) at[u][i] = off[u][i] + now * St::kBytes;
                    const uint32_t pk = smem_u32(ring) + now * St::kBytes + param_off;
                    const bool masked = key0 + kUnit > mask_from || key0 < mask_below;
                    // scale and least value of the lane's key g + 8 i of the unit
                    auto param = [&](uint32_t base, int i, int k, float& sc, float& least) {
                        uint32_t w;
                        asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(w) : "r"(base + 8 * i * pitch + 4 * k));
                        sc = Elem<T>::to_f32(reinterpret_cast<const T*>(&w)[0]);
                        least = Elem<T>::to_f32(reinterpret_cast<const T*>(&w)[1]);
                    };
                    float x[4][E];       // scores of the lane's 4 keys, then weights p'
                    uint32_t wt[NG][4];  // p' s as halves
                    constexpr bool kKeepMids = NG == 1 || D == 64;  // (else they would take too many registers, and are worked out again)
                    float mid[4][NG];    // m + 8 s of the keys
                    bool careful = false;  // a hidden key's scale or least value is not finite: its weight of 0 must not meet it
                    // Usually one round.  A second one (that starts from the scores again) moves the reference of rows that need it.
#pragma unroll 1
                    for (int round = 0;; ++round) {
                        // ---- x = log2(e) scale q . k - R ----
                        {
                            float a[2][NG][4];
#pragma unroll
                            for (int i = 0; i < GR / 2; ++i)
#pragma unroll
                                for (int u = 0; u < 2; ++u) {
                                    uint32_t w[4];  // keys g, g + 8 of piece 2 i, of piece 2 i + 1: the lane's 8 channels
                                    load_matrices<false, 0>(w, at[u][i]);
#pragma unroll
                                    for (int h = 0; h < 2; ++h) {
                                        const int c = 2 * i + h;
                                        uint32_t f0[4], f1[4];
                                        if constexpr (E == 2) {
                                            fields(w[2 * h], f0);
                                            fields(w[2 * h + 1], f1);
                                        } else {
                                            bytes(w[2 * h], f0);
                                            bytes(w[2 * h + 1], f1);
                                        }
                                        const uint32_t a0[4] = {f0[0], f1[0], f0[1], f1[1]}, a1[4] = {f0[2], f1[2], f0[3], f1[3]};
                                        if (c % PER == 0) product<false>(a[u][c / PER], a0, qf[c][0], qf[c][1]);
                                        else product<true>(a[u][c / PER], a0, qf[c][0], qf[c][1]);
                                        product<true>(a[u][c / PER], a1, qf[c][2], qf[c][3]);
                                    }
                                }
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                float sc[NG], least[NG];
#pragma unroll
                                for (int k = 0; k < NG; ++k) param(pk, i, k, sc[k], least[k]);
#pragma unroll
                                for (int e = 0; e < E; ++e) {
                                    float y = 0.f, v = round ? 0.f : -z.ref[e];
#pragma unroll
                                    for (int k = 0; k < NG; ++k) {
                                        const float(&both)[4] = a[i >> 1][k];
                                        const float dot = E == 2 ? both[2 * (i & 1) + e] : both[2 * (i & 1)] + both[2 * (i & 1) + 1];
                                        y = k == 0 ? sc[k] * dot : fmaf(sc[k], dot, y);
                                        v = fmaf(least[k], kb[k][e], v);
                                    }
                                    x[i][e] = fmaf(y, ka[e], v);
                                }
                            }
                        }
                        float vs[4][NG];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int k = 0; k < NG; ++k) {
                                float least;
                                param(pk + St::kParams, i, k, vs[i][k], least);
                                if (kKeepMids) mid[i][k] = fmaf(8.f, vs[i][k], least);
                            }
                        if (masked) {
#pragma unroll
                            for (int e = 0; e < E; ++e) {
                                const int r = first_row + E * t4 + e;
                                int first_key = 0, last_key = len - 1;
                                if (r < rows) visible_range(r / G, sq, len, p.mask_type, p.wl, p.wr, first_key, last_key);
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const int key = key0 + g + 8 * i;
                                    if (key < first_key || key > last_key) x[i][e] = -INFINITY;
                                }
                            }
                            bool finite = true;
#pragma unroll
                            for (int i = 0; i < 4; ++i)
#pragma unroll
                                for (int k = 0; k < NG; ++k) {
                                    float sc, least;
                                    param(pk + St::kParams, i, k, sc, least);
                                    finite &= fabsf(sc) < INFINITY && fabsf(least) < INFINITY;
                                }
                            careful = __any_sync(0xffffffffu, !finite);
                        }
                        if (round == 1) {
                            float lift[NG][E];
                            float top[4][NG];  // log2 of a key's scales
#pragma unroll
                            for (int i = 0; i < 4; ++i)
#pragma unroll
                                for (int k = 0; k < NG; ++k) top[i][k] = vs[i][k] > 0.f ? __log2f(vs[i][k]) : -INFINITY;
#pragma unroll
                            for (int e = 0; e < E; ++e) {
                                float mx = -INFINITY, jx = -INFINITY, jk[NG];  // jk: of a group, jx: of all
#pragma unroll
                                for (int i = 0; i < 4; ++i) mx = fmaxf(mx, x[i][e]);
#pragma unroll
                                for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
#pragma unroll
                                for (int k = 0; k < NG; ++k) {
                                    jk[k] = -INFINITY;
#pragma unroll
                                    for (int i = 0; i < 4; ++i) jk[k] = fmaxf(jk[k], x[i][e] == -INFINITY ? -INFINITY : x[i][e] + top[i][k]);
#pragma unroll
                                    for (int d = 4; d < 32; d <<= 1) jk[k] = fmaxf(jk[k], __shfl_xor_sync(0xffffffffu, jk[k], d));
                                    jx = fmaxf(jx, jk[k]);
                                }
                                // weights up to 2^4 after a move; p' of the largest x within 2^-96 and 2^60, whatever the scales are
                                const float ref = fmaxf(z.ref[e], fminf(fmaxf(jx - 4.f, mx - 60.f), mx + 96.f));
                                const float f = fast_exp2(z.ref[e] - ref);  // (0 where nothing is summed yet)
                                z.l[e] *= f;
#pragma unroll
                                for (int k = 0; k < NG; ++k) {
                                    // weights up to 2^4 in each group, and no more against what the group has summed than the new reference takes off
                                    const int was = lifted ? (int)(__float_as_uint(lifts[k * 4 * E + e]) >> 23) : 127;
                                    const float most = floorf(fminf((float)(was - 127) + (ref - z.ref[e]), 4.f - (jk[k] - ref)));
                                    const int is = fabsf(most) < kLeastLift ? 127 : 127 + (int)fminf(fmaxf(most, -100.f), 100.f);
                                    lift[k][e] = __uint_as_float((uint32_t)is << 23);
                                    const float fo = f * __uint_as_float((uint32_t)max(0, min(254, 127 + is - was)) << 23);  // for sums of weights
                                    z.mid[k][e] *= f;
                                    z.ones[k][e] *= fo;
#pragma unroll
                                    for (int c = k * PER; c < (k + 1) * PER; ++c) {
                                        z.o[c][0][e] *= fo;
                                        z.o[c][0][2 + e] *= fo;
                                        z.o[c][1][e] *= fo;
                                        z.o[c][1][2 + e] *= fo;
                                    }
                                }
                                z.ref[e] = ref;
#pragma unroll
                                for (int i = 0; i < 4; ++i) x[i][e] -= ref;
                            }
                            bool any = false;
                            __syncwarp();  // (8 lanes have a row: all have read what it was lifted by)
#pragma unroll
                            for (int k = 0; k < NG; ++k)
#pragma unroll
                                for (int e = 0; e < E; ++e) {
                                    lifts[k * 4 * E + e] = lift[k][e];
                                    any |= lift[k][e] != 1.f;
                                }
                            lifted = __any_sync(0xffffffffu, any);
                        }
                        // ---- weights ----
                        float sum[E];
#pragma unroll
                        for (int e = 0; e < E; ++e) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) x[i][e] = fast_exp2(x[i][e]);
                            sum[e] = (x[0][e] + x[1][e]) + (x[2][e] + x[3][e]);
                        }
#pragma unroll
                        for (int k = 0; k < NG; ++k)
#pragma unroll
                            for (int i = 0; i < 4; ++i) wt[k][i] = halves(x[i][0] * vs[i][k], E == 2 ? x[i][E - 1] * vs[i][k] : 0.f);
                        // (the weights again: a lift multiplied into every weight took 8 rows and two groups 551 -> 585 us)
                        if (careful || lifted) {
                            auto weight = [&](int i, int k, int e) {
                                const float w = x[i][e] == 0.f ? 0.f : x[i][e] * vs[i][k];
                                return lifted ? w * lifts[k * 4 * E + e] : w;
                            };
#pragma unroll
                            for (int k = 0; k < NG; ++k)
#pragma unroll
                                for (int i = 0; i < 4; ++i) wt[k][i] = halves(weight(i, k, 0), E == 2 ? weight(i, k, E - 1) : 0.f);
                        }
                        uint32_t most = 0;
#pragma unroll
                        for (int k = 0; k < NG; ++k)
#pragma unroll
                            for (int i = 0; i < 4; ++i) most = max_halves(most, wt[k][i]);
                        const bool moves = fmaxf(sum[0], sum[E - 1]) > 1e27f || ((most + 0x10001000u) & 0x80008000u) != 0u;  // (2^13 and more)
                        if (round == 1 || !__any_sync(0xffffffffu, moves)) {
#pragma unroll
                            for (int e = 0; e < E; ++e) z.l[e] += sum[e];
                            break;
                        }
                    }
                    // ---- what each weight adds ----
                    if (careful) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int k = 0; k < NG; ++k) {
                                float sc, least;
                                param(pk + St::kParams, i, k, sc, least);
#pragma unroll
                                for (int e = 0; e < E; ++e)
                                    if (x[i][e] != 0.f) z.mid[k][e] = fmaf(x[i][e], fmaf(8.f, sc, least), z.mid[k][e]);
                            }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int k = 0; k < NG; ++k) {
                                float centre_of = mid[i][k];
                                if (!kKeepMids) {
                                    float sc, least;
                                    param(pk + St::kParams, i, k, sc, least);
                                    centre_of = fmaf(8.f, sc, least);
                                }
#pragma unroll
                                for (int e = 0; e < E; ++e) z.mid[k][e] = fmaf(x[i][e], centre_of, z.mid[k][e]);
                            }
                    }
#pragma unroll
                    for (int k = 0; k < NG; ++k)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            add_halves(z.ones[k], wt[k][i]);
                            wt[k][i] = transpose8x8(wt[k][i]);
                        }
#pragma unroll
                    for (int i = 0; i < GR / 2; ++i)
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            uint32_t y[4];  // transposed: codes 4 g .. + 3 of piece 2 i, keys 2 t, 2 t + 1 and the same + 8; of piece 2 i + 1
                            load_matrices<true, St::kCodes>(y, at[u][i]);
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const int c = 2 * i + h;
                                uint32_t f0[4], f1[4];
                                bytes(y[2 * h], f0);
                                bytes(y[2 * h + 1], f1);
                                const uint32_t even_ch[4] = {f0[0], f0[2], f1[0], f1[2]}, odd_ch[4] = {f0[1], f0[3], f1[1], f1[3]};
                                mma_16816<__half>(z.o[c][0], even_ch, wt[c / PER][2 * u], wt[c / PER][2 * u + 1]);
                                mma_16816<__half>(z.o[c][1], odd_ch, wt[c / PER][2 * u], wt[c / PER][2 * u + 1]);
                            }
                        }
                    if (((key0 >> own_log2) & (kCentre - 1)) == 0) centre();
                }
                // the last reads of the stage have to have come back before it is given back (see splitkv_decode.cu)
                __threadfence_block();
                __syncwarp();
                if (elected()) mbar_arrive(&empty[now]);
            }
            tile_count += tb - ta;

            // ---- this warp's sums: o[e][c] = channels 32 c + 4 g .. + 3 of the lane's row e, in its reference ----
            centre();
            float4 o[E][GR];
            float l[E];
            bool has[E];  // any key (the largest score's p' is at least 2^-96; a NaN counts)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                float rest[NG];
                l[e] = z.l[e];
#pragma unroll
                for (int k = 0; k < NG; ++k) rest[k] = z.mid[k][e];
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    l[e] += __shfl_xor_sync(0xffffffffu, l[e], d);
#pragma unroll
                    for (int k = 0; k < NG; ++k) rest[k] += __shfl_xor_sync(0xffffffffu, rest[k], d);
                }
                has[e] = !(l[e] <= 0.f);
#pragma unroll
                for (int c = 0; c < GR; ++c) {
                    const float add = rest[c / PER], even0 = z.o[c][0][e], even2 = z.o[c][0][2 + e];
                    // 2^24 and 2^20 over the group's lift
                    const float whole = !lifted ? 16777216.f : __uint_as_float((278u << 23) - __float_as_uint(lifts[(c / PER) * 4 * E + e]));
                    const float byte = whole * 0.0625f;
                    o[e][c] = make_float4(fmaf(whole, even0, add), fmaf(byte, z.o[c][1][e] - even0, add), fmaf(whole, even2, add),
                                          fmaf(byte, z.o[c][1][2 + e] - even2, add));
                }
            }
            // ---- the warps of a head (and team, if these have rows of their own) meet: the upper half hands its sums to the lower one until one
            // warp is left, kMeetWarps at a time ----
            for (int half = two_tiles ? 4 : 8; half >= heads; half >>= 1) {
                const int parts = two_tiles ? 2 : max(1, half / kMeetWarps), many = min(kMeetWarps, half);
                for (int part = 0; part < parts; ++part) {
                    const int gives = (two_tiles ? (team == part ? wi : -1) : warp - kMeetWarps * part) - half;
                    const int takes = two_tiles ? (team == part ? wi : -1) : warp - kMeetWarps * part;
                    if (gives >= 0 && gives < many) {
#pragma unroll
                        for (int e = 0; e < E; ++e) {
#pragma unroll
                            for (int c = 0; c < GR; ++c) meet[(gives * kMeetFloat4 + e * GR + c) * 32 + lane] = o[e][c];
                            if (g == 0) {
                                float* stats = meet_stats + (gives * 4 * E + E * t4 + e) * 2;
                                stats[0] = z.ref[e];
                                stats[1] = has[e] ? l[e] : -1.f;  // (-1: no key)
                            }
                        }
                    }
                    asm volatile("bar.sync 1, %0;\n" ::"n"(kConsumers * 32) : "memory");
                    if (takes >= 0 && takes < many) {
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            const float* stats = meet_stats + (takes * 4 * E + E * t4 + e) * 2;
                            const float ref = stats[0], other = stats[1];
                            if (other != -1.f) {
                                const float both = has[e] ? fmaxf(ref, z.ref[e]) : ref;
                                const float fa = has[e] ? fast_exp2(z.ref[e] - both) : 0.f, fb = fast_exp2(ref - both);
                                z.ref[e] = both;
                                has[e] = true;
                                l[e] = l[e] * fa + other * fb;
#pragma unroll
                                for (int c = 0; c < GR; ++c) {
                                    const float4 y = meet[(takes * kMeetFloat4 + e * GR + c) * 32 + lane];
                                    float4& v = o[e][c];
                                    v = make_float4(v.x * fa + y.x * fb, v.y * fa + y.y * fb, v.z * fa + y.z * fb, v.w * fa + y.w * fb);
                                }
                            }
                        }
                    }
                    asm volatile("bar.sync 1, %0;\n" ::"n"(kConsumers * 32) : "memory");
                }
            }
            if ((two_tiles ? wi : warp) >= heads || failed) continue;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int r = first_row + E * t4 + e, i = r / G, h = kh * G + (r - i * G);
                if (r >= rows) continue;
                const int64_t idx = p.seqstart_q ? ((int64_t)h * p.num_splits + split) * p.total_q + (q0 + i)
                                                 : (((int64_t)b * p.hq + h) * p.num_splits + split) * p.seqlen_q + i;
                const float inv = has[e] ? 1.f / l[e] : 0.f;
#pragma unroll
                for (int c = 0; c < GR; ++c) {
                    const float4 v = o[e][c];
                    *reinterpret_cast<float4*>(p.o_acc + idx * D + 32 * c + 4 * g) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
                }
                if (g == 0) p.lse_acc[idx] = !has[e] ? -INFINITY : l[e] != l[e] ? INFINITY  // (the merge makes NaN of it)
                                                                 : (z.ref[e] + log2f(l[e])) * 0.6931471805599453f;
            }
        }
    }
}

// Codes of a pool as (bytes of a line, token of the page, line of the token, page); a box lands as [line][token][bytes].  (TMA takes a few
// cycles for an innermost row: with 64-byte rows, a head each, it fetched 4.0 TB/s.)
int make_codes_map(CUtensorMap* map, const void* base, int64_t pool, int64_t page, int64_t token_bytes, int line, int box_lines, int chunk) {
    PFN_encodeTiled enc = get_encode_tiled();
    FCK_REQUIRE(enc != nullptr, FLASHCK_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[4] = {(cuuint64_t)line, (cuuint64_t)page, (cuuint64_t)(token_bytes / line), (cuuint64_t)pool};
    const cuuint64_t strides[3] = {(cuuint64_t)token_bytes, (cuuint64_t)line, (cuuint64_t)(page * token_bytes)};
    const cuuint32_t box[4] = {(cuuint32_t)line, (cuuint32_t)chunk, (cuuint32_t)box_lines, 1};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUtensorMapSwizzle swizzle = line == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : line == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    FCK_REQUIRE(r == CUDA_SUCCESS, FLASHCK_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) for pool pages=%lld page=%lld bytes of a token=%lld", (int)r,
                (long long)pool, (long long)page, (long long)token_bytes);
    return FLASHCK_OK;
}

template <typename T, int D, int NG, int E>
int launch(const SplitKVInt4Params& p, Int4Dev dev, cudaStream_t stream) {
    using St = Stage<D, NG, E>;
    const Int4Cache& c = p.cache;
    while (dev.heads_log2 < 3 && c.hkv % (2ll << dev.heads_log2) == 0) ++dev.heads_log2;
    const int heads = 1 << dev.heads_log2, toks = kPairs / heads;
    FCK_REQUIRE((int64_t)c.batch * (dev.room / toks + 8) * (dev.dual ? 3 : 1) < (1ll << 30), FLASHCK_ERR_UNSUPPORTED,
                "FmhaFwdSplitKVInt4: %lld sequences of up to %d keys are more than the schedule counts", (long long)c.batch, dev.room);
    int chunk = 16;
    dev.chunk_log2 = 4;
    while (2 * chunk <= toks && (!c.block_table || c.page % (2 * chunk) == 0)) { chunk *= 2; ++dev.chunk_log2; }
    const size_t meet = (size_t)kMeetWarps * E * ((D / 32) * 32 * 16 + 32);
    const size_t lifts = (size_t)kConsumers * NG * 4 * E * sizeof(float);
    const size_t fixed = 1024 + meet + lifts + (size_t)(2 * c.batch + 6) * sizeof(int);
    const size_t room = 227 * 1024;
    FCK_REQUIRE(fixed + 2 * (St::kBytes + 16) <= room, FLASHCK_ERR_UNSUPPORTED, "FmhaFwdSplitKVInt4: batch %lld leaves no room for two stages",
                (long long)c.batch);
    // An even number, so that a stage always falls to the same team and the same producers.  (A parity tells two neighbouring uses apart: a warp that
    // came to a stage for every other use could take another's, not yet filled, for the one before its own.)
    dev.stages = (int)std::min<size_t>(8, (room - fixed) / (St::kBytes + 16)) & ~1;
    const size_t smem = fixed + (size_t)dev.stages * (St::kBytes + 16);
    CUtensorMap mk, mv;
    const int line = std::min(128, heads * (D / 2)), lines = heads * (D / 2) / line;
    dev.line_log2 = line == 128 ? 7 : line == 64 ? 6 : 5;
    if (int rc = make_codes_map(&mk, c.k_codes, c.pool, c.page, c.hkv * (D / 2), line, lines, chunk)) return rc;
    if (int rc = make_codes_map(&mv, c.v_codes, c.pool, c.page, c.hkv * (D / 2), line, lines, chunk)) return rc;
    auto kern = splitkv_int4_kernel<T, D, NG, E>;
    static thread_local int configured_device = -1;  // per instantiation
    int devid = 0;
    FCK_CUDA(cudaGetDevice(&devid));
    if (configured_device != devid) {
        FCK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)room));
        cudaFuncAttributes attr;
        FCK_CUDA(cudaFuncGetAttributes(&attr, kern));
        FCK_REQUIRE(attr.numRegs == kLaunch, FLASHCK_ERR_UNSUPPORTED, "FmhaFwdSplitKVInt4: built with %d registers a thread instead of %d",
                    attr.numRegs, kLaunch);  // (the warps' shares would not add up; the package's build checks it, so this is for other builds)
        configured_device = devid;
    }
    const int64_t rows = p.max_seqlen_q * (p.hq / c.hkv), rows_per_cta = dev.dual ? 16 : 4 * E;
    const int64_t gy = (rows + rows_per_cta - 1) / rows_per_cta, gz = c.hkv / heads;
    FCK_REQUIRE(gy <= 65535, FLASHCK_ERR_UNSUPPORTED, "FmhaFwdSplitKVInt4: too many query rows per kv head");
    const int64_t gx = std::max<int64_t>(1, sm_count() / (gy * gz));  // one wave, where the heads and rows leave one
    FCK_CUDA(launch_dependent(kern, dim3((unsigned)gx, (unsigned)gy, (unsigned)gz), dim3(kThreads), smem, stream, mk, mv, dev));
    return FLASHCK_OK;
}

template <typename T, int D, int NG>
int launch_rows(const SplitKVInt4Params& p, const Int4Dev& dev, cudaStream_t stream) {
    // Rows per kv head.  Up to 4: two columns a row.  Up to 8: one tile.  More: two tiles, a team of 8 warps each, per pass over the cache.
    Int4Dev d = dev;
    const int64_t rows = p.max_seqlen_q * (p.hq / p.cache.hkv);
    d.dual = rows > 8;
    return rows <= 4 ? launch<T, D, NG, 1>(p, d, stream) : launch<T, D, NG, 2>(p, d, stream);
}

template <typename T>
int launch_type(const SplitKVInt4Params& p, const Int4Dev& dev, cudaStream_t stream) {
    const int64_t groups = p.cache.d / p.cache.group;
    if (p.cache.d == 128) {
        if (groups == 1) return launch_rows<T, 128, 1>(p, dev, stream);
        return groups == 2 ? launch_rows<T, 128, 2>(p, dev, stream) : launch_rows<T, 128, 4>(p, dev, stream);
    }
    return groups == 1 ? launch_rows<T, 64, 1>(p, dev, stream) : launch_rows<T, 64, 2>(p, dev, stream);
}

}  // namespace

int launch_splitkv_int4(const SplitKVInt4Params& p, cudaStream_t stream) {
    const Int4Cache& c = p.cache;
    FCK_REQUIRE(c.d == 64 || c.d == 128, FLASHCK_ERR_UNSUPPORTED, "FmhaFwdSplitKVInt4: hdim 64 or 128 (got %lld)", (long long)c.d);
    FCK_REQUIRE((c.group == 32 || c.group == 64 || c.group == 128) && c.group <= c.d, FLASHCK_ERR_UNSUPPORTED,
                "FmhaFwdSplitKVInt4: groups of 32, 64 or 128 channels of a head (got %lld of %lld)", (long long)c.group, (long long)c.d);
    FCK_REQUIRE(c.batch >= 1 && c.batch <= 8192, FLASHCK_ERR_UNSUPPORTED, "FmhaFwdSplitKVInt4: batch must be in [1,8192]");
    FCK_REQUIRE(!c.block_table || c.page % 16 == 0, FLASHCK_ERR_UNSUPPORTED,
                "FmhaFwdSplitKVInt4: page_block_size must be a positive multiple of 16 (got %lld)", (long long)c.page);
    FCK_REQUIRE(c.page > 0 && c.page < (1ll << 31) && c.pool > 0 && c.pool < (1ll << 31) - 1, FLASHCK_ERR_INVALID_ARGUMENT,
                "FmhaFwdSplitKVInt4: bad page or pool size");
    FCK_REQUIRE(p.total_q < (1ll << 31), FLASHCK_ERR_UNSUPPORTED, "FmhaFwdSplitKVInt4: too many query rows");
    Int4Dev dev{};
    dev.status = device_status_ptr();
    if (!dev.status) return FLASHCK_ERR_CUDA;
    dev.q = p.q; dev.o_acc = p.o_acc; dev.lse_acc = p.lse_acc; dev.seqstart_q = p.seqstart_q;
    dev.seqlen_k = c.seqlen; dev.block_table = c.block_table; dev.cache_batch_idx = c.cache_batch_idx;
    dev.k_params = (const uint8_t*)c.k_params; dev.v_params = (const uint8_t*)c.v_params;
    dev.batch = (int)c.batch; dev.seqlen_q = (int)p.seqlen_q; dev.hq = (int)p.hq; dev.hkv = (int)c.hkv;
    dev.num_splits = (int)p.num_splits; dev.total_q = (int)p.total_q; dev.bt_stride = (int)c.bt_stride;
    dev.page = (int)c.page; dev.pool = (int)c.pool;
    dev.room = (int)std::min<int64_t>(c.block_table ? c.bt_stride * c.page : c.page, 0x7fffff00);
    dev.mask_type = p.mask_type;
    dev.wl = (int)(p.wl < 0 ? -1 : std::min<int64_t>(p.wl, 0x3fffffff));
    dev.wr = (int)(p.wr < 0 ? -1 : std::min<int64_t>(p.wr, 0x3fffffff));
    dev.scale_log2 = p.scale * 1.4426950408889634f;
    return c.dtype == FLASHCK_DTYPE_BFLOAT16 ? launch_type<__nv_bfloat16>(p, dev, stream) : launch_type<__half>(p, dev, stream);
}

}  // namespace fck
