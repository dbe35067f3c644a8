// The write of a 4-bit key/value cache, and its way back to 16-bit keys and values.
//
// Append: the queries and the new keys are turned (int4.cuh), the turned keys and the values quantised group by group and written
// through the block table.  One pass: a lane holds twice 8 channels of a head, so that both halves of its half-rotated pairs are its own; 4 to 8
// lanes have a group, whose least and greatest value take a shuffle a level.  A token's first rows are requested before its sequence is looked up.
// Read: 4 bytes of codes in and 16 bytes of values out a lane, four tokens of a run in flight.
//
// A job is one token's keys, values and queries (queries that are not the new tokens are jobs of their own); 1 to 8 warps share it.  What bounds
// the append of a decode step (32 tokens: 7 us) is a chain of memory round trips -- sequence starts, lengths, pages, angles -- and what bounds a
// long one its traffic and the issue slots about equally: 43178 tokens of 32 / 8 heads with the held values returned, 1.12 GB, 197-203 us, floor 172 at
// 6.54 TB/s.  Reading 48855 tokens of 8 heads back, 253 MB: 44 us, floor 39.
#include <algorithm>
#include <type_traits>

#include "int4.cuh"

namespace fck {

int fill_rotary(const char* fn, RotaryDev& r, const void* cosr, const void* sinr, int64_t rows, int64_t rotary_dim, int64_t d, int rope_type,
                const uint8_t* pair_axis, int64_t axes, bool rows_aligned) {
    r = RotaryDev{};
    r.type = rope_type;
    r.vec = rows_aligned;
    if (rope_type == 0) return FLASHCK_OK;
    FCK_REQUIRE(rope_type == 1 || rope_type == 2, FLASHCK_ERR_INVALID_ARGUMENT, "%s: rope_type must be 0..2", fn);
    FCK_REQUIRE(rotary_dim > 0 && rotary_dim <= d && rotary_dim % 2 == 0 && rotary_dim <= 2 * kMaxPairs, FLASHCK_ERR_INVALID_ARGUMENT,
                "%s: rotary_dim must be even and in (0, hdim], at most %d (got %lld)", fn, 2 * kMaxPairs, (long long)rotary_dim);
    FCK_REQUIRE(cosr && sinr, FLASHCK_ERR_INVALID_ARGUMENT, "%s: rotary tables must not be null when rope_type != 0", fn);
    FCK_REQUIRE(rows >= 0 && rows < (1ll << 31), FLASHCK_ERR_INVALID_ARGUMENT, "%s: bad number of rows of the rotary tables", fn);
    FCK_REQUIRE(axes >= 1 && axes <= kMaxAxes, FLASHCK_ERR_UNSUPPORTED, "%s: 1 to %d axes of positions (got %lld)", fn, kMaxAxes, (long long)axes);
    r.cosr = cosr; r.sinr = sinr;
    r.rows = (int)rows; r.half = (int)(rotary_dim / 2); r.axes = (int)axes;
    const auto aligned = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15u) == 0; };
    r.vec = rows_aligned && aligned(cosr) && aligned(sinr) && rotary_dim % (rope_type == 1 ? 8 : 16) == 0;
    for (int i = 0; pair_axis && i < r.half; ++i) {
        FCK_REQUIRE(pair_axis[i] < axes, FLASHCK_ERR_INVALID_ARGUMENT, "%s: pair %d turns with axis %d of %lld", fn, i, (int)pair_axis[i],
                    (long long)axes);
        r.axis[i >> 4] |= (uint32_t)pair_axis[i] << (2 * (i & 15));
    }
    return FLASHCK_OK;
}

namespace {

struct CacheDev {
    uint8_t* codes[2];   // K, V
    uint32_t* params[2];
    const int32_t* seqlen;
    const int32_t* block_table;
    const int64_t* cache_batch_idx;
    int batch, hkv, d, group, bt_stride, page, pool;
};

// The cache row of token `pos` of sequence b, or -1: behind the cache's end, or on a page that the pool does not have.
__device__ __forceinline__ int64_t cache_row(const CacheDev& c, int b, int64_t pos) {
    const int64_t bphys = c.cache_batch_idx ? c.cache_batch_idx[b] : b;
    if (pos < 0) return -1;
    if (!c.block_table) return pos < c.page && (uint64_t)bphys < (uint64_t)c.pool ? bphys * c.page + pos : -1;
    if (pos > 0x7fffffff) return -1;
    const uint32_t slot = (uint32_t)pos / (uint32_t)c.page;
    if (slot >= (uint32_t)c.bt_stride) return -1;
    const int32_t pg = c.block_table[bphys * c.bt_stride + slot];
    return (uint32_t)pg < (uint32_t)c.pool ? (int64_t)pg * c.page + ((uint32_t)pos - slot * c.page) : -1;
}

// The sequence of packed row t, by the whole warp: the number of starts 1 .. batch - 1 at or below t.
__device__ __forceinline__ int sequence_of(const int64_t* seqstart, int batch, int64_t t, int lane) {
    int n = 0;
    for (int i = 1 + lane; i < batch; i += 32) n += seqstart[i] <= t;
    return __reduce_add_sync(0xffffffffu, n);
}

// Least of two pairs of T; NaN where either is.
template <typename T>
__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t min2_nan<__half>(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <>
__device__ __forceinline__ uint32_t min2_nan<__nv_bfloat16>(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// What 8 codes stand for: lo + scale * code, one rounding.  A code set into the low mantissa bits of 128 (bf16) or 1024 (fp16) is that number
// plus the code; two at a time are four channels apart in the word.
template <typename T>
__device__ __forceinline__ Vec8<T> values_of(uint32_t word, T scale, T lo) {
    using T2 = typename Elem<T>::T2;
    constexpr bool kHalf = std::is_same<T, __half>::value;
    constexpr uint32_t kBase = kHalf ? 0x64006400u : 0x43004300u;
    const T2 base = Elem<T>::bcast2(kHalf ? -1024.f : -128.f);
    T2 s2, l2;
    s2.x = s2.y = scale;
    l2.x = l2.y = lo;
    uint32_t f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t u = ((word >> (4 * i)) & 0x000f000fu) | kBase;
        const T2 v = __hfma2(__hadd2(*reinterpret_cast<const T2*>(&u), base), s2, l2);
        f[i] = *reinterpret_cast<const uint32_t*>(&v);  // channels i and i + 4
    }
    Vec8<T> x;
    x.w[0] = __byte_perm(f[0], f[1], 0x5410);
    x.w[1] = __byte_perm(f[2], f[3], 0x5410);
    x.w[2] = __byte_perm(f[0], f[1], 0x7632);
    x.w[3] = __byte_perm(f[2], f[3], 0x7632);
    return x;
}

// r / scale to the nearest code, ties to even, without rounding a quotient: a multiple of one half, times the scale, is compared with r by the
// sign of one FMA, which is exact.
__device__ __noinline__ uint32_t exact_code(float r, float s) {
    uint32_t k = 0;
    if (!(s > 0.f)) return 0;
#pragma unroll 1
    for (int i = 0; i < 15; ++i) {
        const float e = fmaf(-(i + 0.5f), s, r);
        k += e > 0.f || (e == 0.f && (i & 1));
    }
    return k;
}

// Least and (negated) greatest of 8 values, together in a word, so that a level of a reduction takes one shuffle.
template <typename T>
__device__ __forceinline__ uint32_t range_of(const Vec8<T>& x) {
    constexpr uint32_t kSigns = 0x80008000u;
    const uint32_t least = min2_nan<T>(min2_nan<T>(x.w[0], x.w[1]), min2_nan<T>(x.w[2], x.w[3]));
    const uint32_t most = min2_nan<T>(min2_nan<T>(x.w[0] ^ kSigns, x.w[1] ^ kSigns), min2_nan<T>(x.w[2] ^ kSigns, x.w[3] ^ kSigns));
    return min2_nan<T>(__byte_perm(least, most, 0x5410), __byte_perm(least, most, 0x7632));
}

// The codes of 8 channels of a group with range `both`, and the group's scale and least value.
template <typename T>
__device__ __forceinline__ uint32_t quantise(const Vec8<T>& x, uint32_t both, T& scale_t, T& lo_t) {
    lo_t = reinterpret_cast<const T*>(&both)[0];
    const float lo = Elem<T>::to_f32(lo_t), hi = -Elem<T>::to_f32(reinterpret_cast<const T*>(&both)[1]);
    // A quotient is rounded correctly by a product with the reciprocal, and once more with its exact remainder (Markstein's correction).
    const float range = hi - lo;
    constexpr float kFifteenth = 1.f / 15.f;
    float step = range * kFifteenth;
    step = fmaf(fmaf(-step, 15.f, range), kFifteenth, step);
    scale_t = Elem<T>::from_f32(range < INFINITY ? step : NAN);  // (a group that is not finite is NaN as a whole)
    const float s = Elem<T>::to_f32(scale_t);
    // The codes: such a quotient, to an integer by the addition of 1.5 * 2^23, ties to even.  Rounding twice does no harm: (k + 1/2) scale
    // has at most 16 bits, so a difference x - lo that is not equal to it is at least a step of 32 bits away, relatively more than the half
    // step at k + 1/2 to which its quotient is rounded.  (Half way between two codes is common: a difference of two 8-bit significands meets
    // a multiple of another one in a few per thousand.)
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
    if (s == 0.f) inv = 0.f;  // (all codes 0; a lane without a head comes here too)
    const uint64_t inv2 = two(inv, inv), minus_s = two(-s, -s), minus_lo = two(-lo, -lo), round2 = two(12582912.f, 12582912.f);
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint64_t r = add2(widen<T>(x.w[i]), minus_lo), q = mul2(r, inv2);
        float k0, k1;
        apart(add2(fma2(fma2(q, minus_s, r), inv2, q), round2), k0, k1);
        u[2 * i] = __float_as_uint(k0);
        u[2 * i + 1] = __float_as_uint(k1);
    }
    // scales that T holds with few digits (a code may pass 15), and those whose reciprocal or remainder fp32 may not hold
    constexpr bool kHalf = std::is_same<T, __half>::value;
    if (!(s == 0.f || (s >= (kHalf ? 6.103515625e-5f : 1e-25f) && s <= 1e25f))) {
        scale_t = Elem<T>::from_f32(range < INFINITY ? __fdiv_rn(range, 15.f) : NAN);
        const float exact = Elem<T>::to_f32(scale_t);
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = exact_code(Elem<T>::to_f32(x.e[i]) - lo, exact);
    }
    // lowest bytes: even channels and odd ones
    const uint32_t even = __byte_perm(__byte_perm(u[0], u[2], 0x0040), __byte_perm(u[4], u[6], 0x0040), 0x5410);
    const uint32_t odd = __byte_perm(__byte_perm(u[1], u[3], 0x0040), __byte_perm(u[5], u[7], 0x0040), 0x5410);
    return (even & 0x0f0f0f0fu) | ((odd & 0x0f0f0f0fu) << 4);
}

struct AppendInt4Dev {
    CacheDev cache;
    RotaryDev rot;
    const void* q;
    void* q_out;
    const void* knew;
    const void* vnew;
    void* k_held;
    void* v_held;
    const int64_t* seqstart_q;
    const int64_t* seqstart_knew;
    const int32_t* positions;
    int* status;
    int seqlen_q, seqlen_knew, hq, warps_log2;  // warps of a job
    bool joined;  // the queries are the new tokens: one job for both
    int64_t total_new, total_q;
};

template <typename T>
__device__ __forceinline__ Vec8<T> load8(const T* p, bool vec) {
    Vec8<T> x;
    if (vec) {
        x.v = *reinterpret_cast<const uint4*>(p);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x.e[i] = p[i];
    }
    return x;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const Vec8<T>& x, bool vec) {
    if (vec) {
        *reinterpret_cast<uint4*>(p) = x.v;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = x.e[i];
    }
}

// A token's place: its sequence b, and its place j among the rows of the sequence in its tensor, of which there are n.
struct Token {
    int b;
    int64_t j, n, first;  // first: packed row of the sequence's first new token
};
__device__ __forceinline__ Token find_token(const AppendInt4Dev& a, bool queries, int64_t t, int lane) {
    const int64_t* starts = queries ? a.seqstart_q : a.seqstart_knew;
    const int64_t each = queries ? a.seqlen_q : a.seqlen_knew;
    Token k;
    if (starts) {
        k.b = sequence_of(starts, a.cache.batch, t, lane);
        const int64_t s0 = starts[k.b];
        k.j = t - s0;
        k.n = starts[k.b + 1] - s0;
        k.first = queries ? a.seqstart_knew[k.b] : s0;
    } else {
        k.b = (int)((uint32_t)t / (uint32_t)each);
        k.j = t - k.b * each;
        k.n = each;
        k.first = (int64_t)k.b * a.seqlen_knew;
    }
    return k;
}

// ROPE as in Turn; 3: channel by channel, any width and alignment.
template <typename T, int ROPE>
__global__ void __launch_bounds__(256, 4) append_int4_kernel(const __grid_constant__ AppendInt4Dev a) {
    constexpr bool kVec = ROPE != 3;
    pdl_launch_dependents();
    pdl_wait();
    const CacheDev& c = a.cache;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t job = (int64_t)blockIdx.x << (3 - a.warps_log2) | (warp >> a.warps_log2);
    const int part = warp & ((1 << a.warps_log2) - 1);
    if (job >= a.total_new + a.total_q) return;  // (whole warps)
    // a job of queries, of keys and values, or (joined: the queries are the new tokens) of both
    const bool only_queries = job >= a.total_new;
    const int64_t t = only_queries ? job - a.total_new : job;
    const int lanes_log2 = c.d == 64 ? 2 : 3, lanes = 1 << lanes_log2, at_once = 32 >> lanes_log2;
    const int sub = lane >> lanes_log2, e0 = (lane & (lanes - 1)) << 3, step = at_once << a.warps_log2;
    if (part * at_once >= (only_queries || a.joined ? max(a.hq, only_queries ? 0 : c.hkv) : c.hkv)) return;
    Turn<T, kVec ? ROPE : 0> turn(a.rot, e0, c.d);

    Pieces<T> x, y, v;
    auto request = [&](bool queries, int h0) {
        const int heads = queries ? a.hq : c.hkv, h = h0 + sub;
        const T* src = (const T*)(queries ? a.q : a.knew) + (t * heads + h) * c.d;
        x.a.v = x.b.v = v.a.v = v.b.v = make_uint4(0, 0, 0, 0);
        if (kVec && h < heads) {
            x = turn.own(src);
            if (ROPE == 4) y = turn.other(src);
            if (!queries) v = turn.own((const T*)a.vnew + (t * heads + h) * c.d);
        }
    };
    request(only_queries, part * at_once);  // (a row is there whether it belongs to a sequence or not: its loads do not wait for what follows)

    const Token k = find_token(a, only_queries, t, lane);
    const bool real = k.j >= 0 && k.j < k.n;  // (a row that belongs to no sequence leaves as zeros)
    // the last new tokens are the queries'
    const int64_t j = k.j + (only_queries ? (a.seqstart_knew ? a.seqstart_knew[k.b + 1] - k.first : (int64_t)a.seqlen_knew) - k.n : 0);
    const int64_t at = real ? c.seqlen[k.b] + j : -1;  // place in the cache
    const int64_t token = k.first + j;
    Positions pos;
    if (ROPE != 0 && a.positions && j >= 0 && token < a.total_new) pos.load(a.positions, a.rot.axes, a.total_new, token);
    else pos.fill(a.positions ? -1 : at);
    if (real) turn.load(a.rot, pos);
    const int64_t row = !only_queries && real ? cache_row(c, k.b, at) : -1;
    if (!only_queries && real && row < 0 && lane == 0 && part == 0) atomicOr(a.status, FLASHCK_STATUS_APPEND_OVERFLOW);
    const bool joint = c.group == c.d;  // one group: both pieces
    const int group_lanes = joint ? lanes : c.group >> 3, group_log2 = 31 - __clz(c.group), groups = c.d >> group_log2;

    auto turned = [&](bool queries, int h) {
        const int heads = queries ? a.hq : c.hkv;
        if constexpr (!kVec) {
            if (h < heads && real) {
                const T* src = (const T*)(queries ? a.q : a.knew) + (t * heads + h) * c.d;
                turn_piece_any<T>(a.rot, e0, pos, src, x.a);
                turn_piece_any<T>(a.rot, e0 + (c.d >> 1), pos, src, x.b);
                if (!queries) {
                    const T* vsrc = (const T*)a.vnew + (t * heads + h) * c.d;
                    v.a = load8(vsrc + e0, false);
                    v.b = load8(vsrc + e0 + (c.d >> 1), false);
                }
            }
        } else {
            turn(x, y);
            if (!real) x.a.v = x.b.v = v.a.v = v.b.v = make_uint4(0, 0, 0, 0);
        }
    };
    if (!only_queries) {
        for (int h0 = part * at_once; h0 < c.hkv; h0 += step) {
            const int h = h0 + sub;
            const bool mine = h < c.hkv;
            if (h0 != part * at_once) request(false, h0);
            turned(false, h);
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                const Pieces<T>& z = kv ? v : x;
                uint32_t ra = range_of(z.a), rb = range_of(z.b);
                if (joint) ra = rb = min2_nan<T>(ra, rb);
                for (int off = 1; off < group_lanes; off <<= 1) {
                    ra = min2_nan<T>(ra, __shfl_xor_sync(0xffffffffu, ra, off));
                    if (!joint) rb = min2_nan<T>(rb, __shfl_xor_sync(0xffffffffu, rb, off));
                }
                if (joint) rb = ra;
                T scale[2], lo[2];
                const uint32_t wa = quantise<T>(z.a, ra, scale[0], lo[0]), wb = quantise<T>(z.b, rb, scale[1], lo[1]);
                if (!mine) continue;
                if (row >= 0) {
                    const int64_t place = row * c.hkv + h;
                    uint32_t* codes = reinterpret_cast<uint32_t*>(c.codes[kv]) + place * (c.d >> 3) + (e0 >> 3);
                    codes[0] = wa;
                    codes[lanes] = wb;
                    if ((e0 & (c.group - 1)) == 0) {
                        const T ta[2] = {scale[0], lo[0]}, tb[2] = {scale[1], lo[1]};
                        uint32_t* params = c.params[kv] + place * groups + (e0 >> group_log2);
                        params[0] = *reinterpret_cast<const uint32_t*>(ta);
                        if (!joint) params[groups >> 1] = *reinterpret_cast<const uint32_t*>(tb);
                    }
                }
                T* held = (T*)(kv ? a.v_held : a.k_held);
                if (held) {
                    held += (t * c.hkv + h) * c.d + e0;
                    store8(held, values_of<T>(wa, scale[0], lo[0]), kVec);
                    store8(held + (c.d >> 1), values_of<T>(wb, scale[1], lo[1]), kVec);
                }
            }
        }
    }
    if (only_queries || a.joined) {
        for (int h0 = part * at_once; h0 < a.hq; h0 += step) {
            const int h = h0 + sub;
            if (!only_queries || h0 != part * at_once) request(true, h0);
            turned(true, h);
            if (h < a.hq) {
                T* dst = (T*)a.q_out + (t * a.hq + h) * c.d + e0;
                store8(dst, x.a, kVec);
                store8(dst + (c.d >> 1), x.b, kVec);
            }
        }
    }
}

struct ReadInt4Dev {
    CacheDev cache;
    void* out[2];
    const int64_t* seqstart;
    int64_t tokens, total;
    int warps_log2;
};

// A job is R neighbouring tokens: a lane looks one of them up for all, and their loads are in flight together.
template <typename T, int R>
__global__ void __launch_bounds__(256) read_int4_kernel(const __grid_constant__ ReadInt4Dev a) {
    pdl_launch_dependents();
    pdl_wait();
    const CacheDev& c = a.cache;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t t0 = ((int64_t)blockIdx.x << (3 - a.warps_log2) | (warp >> a.warps_log2)) * R;
    const int part = warp & ((1 << a.warps_log2) - 1), w = 1 << a.warps_log2;
    if (t0 >= a.total) return;
    int64_t row = -1;  // of token t0 + lane (no such token: zeros)
    {
        const int64_t t = t0 + lane;
        int b;
        int64_t j, n;
        if (a.seqstart) {
            b = sequence_of(a.seqstart, c.batch, t0, lane);
            while (lane < R && b + 1 < c.batch && a.seqstart[b + 1] <= t) ++b;
            j = t - a.seqstart[b];
            n = min((int64_t)c.seqlen[b], a.seqstart[b + 1] - a.seqstart[b]);
        } else {
            b = (int)(t / a.tokens);
            j = t - b * a.tokens;
            n = b < c.batch ? c.seqlen[b] : 0;
        }
        if (lane < R && t < a.total && j >= 0 && j < n) row = cache_row(c, b, j);
    }
    int64_t rows[R];
#pragma unroll
    for (int r = 0; r < R; ++r) rows[r] = __shfl_sync(0xffffffffu, row, r);
    const int per_row = c.hkv * c.d >> 3, group_log2 = 31 - __clz(c.group >> 3);  // 8 channels each
    for (int i = part * 32 + lane; i < per_row; i += w * 32) {
        uint32_t word[2][R], two[2][R];
#pragma unroll
        for (int kv = 0; kv < 2; ++kv)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                word[kv][r] = two[kv][r] = 0;
                if (rows[r] >= 0) {
                    word[kv][r] = reinterpret_cast<const uint32_t*>(c.codes[kv])[rows[r] * per_row + i];
                    two[kv][r] = c.params[kv][rows[r] * (per_row >> group_log2) + (i >> group_log2)];
                }
            }
#pragma unroll
        for (int kv = 0; kv < 2; ++kv)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const T* p = reinterpret_cast<const T*>(&two[kv][r]);
                if (t0 + r < a.total)
                    *reinterpret_cast<uint4*>((T*)a.out[kv] + ((t0 + r) * per_row + i) * 8) = values_of<T>(word[kv][r], p[0], p[1]).v;
            }
    }
}

int fill_cache(const char* fn, const Int4Cache& p, CacheDev& c) {
    FCK_REQUIRE(p.d == 64 || p.d == 128, FLASHCK_ERR_UNSUPPORTED, "%s: hdim 64 or 128 (got %lld)", fn, (long long)p.d);
    FCK_REQUIRE((p.group == 32 || p.group == 64 || p.group == 128) && p.group <= p.d, FLASHCK_ERR_UNSUPPORTED,
                "%s: groups of 32, 64 or 128 channels of a head (got %lld of %lld)", fn, (long long)p.group, (long long)p.d);
    FCK_REQUIRE(p.page > 0 && p.page < (1ll << 31) && p.pool >= 0 && p.pool < (1ll << 31) && p.bt_stride < (1ll << 31), FLASHCK_ERR_INVALID_ARGUMENT,
                "%s: bad page, pool or block table size", fn);
    FCK_REQUIRE(p.hkv <= 1024, FLASHCK_ERR_UNSUPPORTED, "%s: at most 1024 kv heads", fn);
    c.codes[0] = (uint8_t*)p.k_codes; c.codes[1] = (uint8_t*)p.v_codes;
    c.params[0] = (uint32_t*)p.k_params; c.params[1] = (uint32_t*)p.v_params;
    c.seqlen = p.seqlen; c.block_table = p.block_table; c.cache_batch_idx = p.cache_batch_idx;
    c.batch = (int)p.batch; c.hkv = (int)p.hkv; c.d = (int)p.d; c.group = (int)p.group;
    c.bt_stride = (int)p.bt_stride; c.page = (int)p.page; c.pool = (int)p.pool;
    return FLASHCK_OK;
}

template <typename T>
cudaError_t launch_append_type(const AppendInt4Dev& a, dim3 grid, dim3 block, cudaStream_t stream) {
    switch (rope_form(a.rot, a.cache.d)) {
        case 0: return launch_dependent(append_int4_kernel<T, 0>, grid, block, 0, stream, a);
        case 1: return launch_dependent(append_int4_kernel<T, 1>, grid, block, 0, stream, a);
        case 2: return launch_dependent(append_int4_kernel<T, 2>, grid, block, 0, stream, a);
        case 4: return launch_dependent(append_int4_kernel<T, 4>, grid, block, 0, stream, a);
        default: return launch_dependent(append_int4_kernel<T, 3>, grid, block, 0, stream, a);
    }
}

template <typename T>
cudaError_t launch_read_type(const ReadInt4Dev& a, bool runs, unsigned blocks, cudaStream_t stream) {
    return runs ? launch_dependent(read_int4_kernel<T, 4>, dim3(blocks), dim3(256), 0, stream, a)
                : launch_dependent(read_int4_kernel<T, 1>, dim3(blocks), dim3(256), 0, stream, a);
}

}  // namespace

int launch_append_int4(const AppendInt4Params& p, cudaStream_t stream) {
    AppendInt4Dev a{};
    if (int rc = fill_cache("FmhaFwdAppendKVInt4", p.cache, a.cache)) return rc;
    const auto aligned = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15u) == 0; };
    const bool rows = aligned(p.q) && aligned(p.q_out) && aligned(p.knew) && aligned(p.vnew) && aligned(p.k_held) && aligned(p.v_held);
    if (int rc = fill_rotary("FmhaFwdAppendKVInt4", a.rot, p.rotary_cos, p.rotary_sin, p.rotary_rows, p.rotary_dim, p.cache.d, p.rope_type,
                             p.pair_axis, p.positions || p.pair_axis ? p.axes : 1, rows)) return rc;
    a.status = device_status_ptr();
    if (!a.status) return FLASHCK_ERR_CUDA;
    a.q = p.q; a.q_out = p.q_out; a.knew = p.knew; a.vnew = p.vnew; a.k_held = p.k_held; a.v_held = p.v_held;
    a.seqstart_q = p.seqstart_q; a.seqstart_knew = p.seqstart_knew; a.positions = p.positions;
    a.seqlen_q = (int)p.seqlen_q; a.seqlen_knew = (int)p.seqlen_knew; a.hq = (int)p.hq;
    a.total_new = p.seqstart_knew ? p.seqlen_knew : p.cache.batch * p.seqlen_knew;
    a.total_q = !p.q ? 0 : p.seqstart_q ? p.seqlen_q : p.cache.batch * p.seqlen_q;
    a.joined = p.q && p.seqstart_q == p.seqstart_knew && p.seqlen_q == p.seqlen_knew;
    if (a.joined) a.total_q = 0;
    const int64_t jobs = a.total_new + a.total_q;
    if (jobs == 0) return FLASHCK_OK;
    a.warps_log2 = warps_log2_for(jobs, std::max<int64_t>(1, std::max(p.hq, p.cache.hkv) * p.cache.d / 256));
    const int64_t blocks = ((jobs << a.warps_log2) + 7) / 8;
    FCK_REQUIRE(jobs < (1ll << 31), FLASHCK_ERR_UNSUPPORTED, "FmhaFwdAppendKVInt4: too many tokens");
    const dim3 grid((unsigned)blocks), block(256);
    if (p.cache.dtype == FLASHCK_DTYPE_BFLOAT16) FCK_CUDA(launch_append_type<__nv_bfloat16>(a, grid, block, stream));
    else FCK_CUDA(launch_append_type<__half>(a, grid, block, stream));
    return FLASHCK_OK;
}

int launch_read_int4(const ReadInt4Params& p, cudaStream_t stream) {
    ReadInt4Dev a{};
    if (int rc = fill_cache("FmhaReadKVInt4", p.cache, a.cache)) return rc;
    a.out[0] = p.k; a.out[1] = p.v; a.seqstart = p.seqstart; a.tokens = p.tokens;
    a.total = p.seqstart ? p.tokens : p.cache.batch * p.tokens;
    if (a.total == 0) return FLASHCK_OK;
    a.warps_log2 = warps_log2_for(a.total, std::max<int64_t>(1, p.cache.hkv * p.cache.d / 256));
    const bool runs = a.total >= (int64_t)sm_count() * 256;  // enough tokens to fill the SMs by fours
    const int64_t jobs = runs ? (a.total + 3) / 4 : a.total, blocks = ((jobs << a.warps_log2) + 7) / 8;
    FCK_REQUIRE(blocks < (1ll << 31), FLASHCK_ERR_UNSUPPORTED, "FmhaReadKVInt4: too many tokens");
    if (p.cache.dtype == FLASHCK_DTYPE_BFLOAT16) FCK_CUDA(launch_read_type<__nv_bfloat16>(a, runs, (unsigned)blocks, stream));
    else FCK_CUDA(launch_read_type<__half>(a, runs, (unsigned)blocks, stream));
    return FLASHCK_OK;
}

}  // namespace fck
