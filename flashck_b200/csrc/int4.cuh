// The 4-bit key/value cache: what its bytes mean, and the rotation of queries and keys that its write fuses.
//
// A group of 32, 64 or 128 neighbouring channels of one token's head is held as value = lo + scale * code, code 0..15:
//     lo = min x,   scale = T((max x - min x) / 15),   code = min(15, rne((x - lo) / scale)),   scale = 0: code 0
// with the difference and the quotient's dividend in fp32 and T the model's 16-bit type; lo is one of the x and therefore exact.
// Codes: uint8 [rows, hkv, d / 2], byte j with channel 2j in its low and 2j + 1 in its high half.  Params: T [rows, hkv, d / group, 2] =
// (scale, lo).  A group with a NaN or an infinity, or one whose range leaves fp32, reads back as NaN.
#pragma once

#include <type_traits>

#include "kernels.h"

namespace fck {

constexpr int kMaxPairs = 128, kMaxAxes = 4;

// What a rotation needs besides the row: cos / sin tables T [rows, half], and for each pair of a head the axis whose position turns it
// (2 bits a pair).
struct RotaryDev {
    const void* cosr;
    const void* sinr;
    int rows, half, axes, type;  // type: 0 none, 1 neighbouring pairs (2i, 2i + 1), 2 (i, i + half)
    bool vec;              // 16-byte form: tables and rows aligned, a piece of 8 channels holds whole runs of pairs
    bool back;             // turned the other way: the gradient of the rotation
    uint32_t axis[kMaxPairs / 16];
};

#ifdef __CUDACC__

__device__ __forceinline__ int axis_of(const RotaryDev& r, int pair) { return (r.axis[pair >> 4] >> (2 * (pair & 15))) & 3; }

template <typename T>
union Vec8 {
    uint4 v;
    uint32_t w[4];
    T e[8];
};

// A token's position along each axis, loaded together; -1 (outside the tables) for the axes that there are not.
struct Positions {
    int p[kMaxAxes];

    __device__ __forceinline__ void load(const int32_t* positions, int axes, int64_t tokens, int64_t t) {
#pragma unroll
        for (int i = 0; i < kMaxAxes; ++i) p[i] = i < axes ? positions[i * tokens + t] : -1;
    }
    __device__ __forceinline__ void fill(int64_t at) {
#pragma unroll
        for (int i = 0; i < kMaxAxes; ++i) p[i] = at < 0 || at > 0x7fffffff ? -1 : (int)at;
    }
    __device__ __forceinline__ int operator()(int axis) const { return axis < 2 ? (axis == 0 ? p[0] : p[1]) : (axis == 2 ? p[2] : p[3]); }
};

// cos and sin of pairs [first, first + N); a position outside the tables turns by NaN.  The vector form is taken where one axis turns all of
// them; in the other form too the loads do not wait for one another.
template <typename T, int N>
__device__ __forceinline__ void load_angles(const RotaryDev& r, int first, const Positions& pos, float (&c)[N], float (&s)[N]) {
    constexpr uint32_t kAll = (1u << (2 * N)) - 1u;
    const uint32_t axes = (r.axis[first >> 4] >> (2 * (first & 15))) & kAll, a0 = axes & 3u;
    if (axes == a0 * (0x5555u & kAll)) {
        const int p = pos(a0);
        if ((uint32_t)p < (uint32_t)r.rows) {
            using V = typename std::conditional<N == 8, uint4, uint2>::type;
            const V cv = *reinterpret_cast<const V*>((const T*)r.cosr + (int64_t)p * r.half + first);
            const V sv = *reinterpret_cast<const V*>((const T*)r.sinr + (int64_t)p * r.half + first);
            const T* ce = reinterpret_cast<const T*>(&cv);
            const T* se = reinterpret_cast<const T*>(&sv);
#pragma unroll
            for (int i = 0; i < N; ++i) { c[i] = Elem<T>::to_f32(ce[i]); s[i] = Elem<T>::to_f32(se[i]); }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) c[i] = s[i] = NAN;
        }
    } else if (r.rows > 0) {
        T ce[N], se[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int p = pos((axes >> (2 * i)) & 3);
            const int64_t at = (int64_t)((uint32_t)p < (uint32_t)r.rows ? p : 0) * r.half + first + i;
            ce[i] = ((const T*)r.cosr)[at];
            se[i] = ((const T*)r.sinr)[at];
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bool in = (uint32_t)pos((axes >> (2 * i)) & 3) < (uint32_t)r.rows;
            c[i] = in ? Elem<T>::to_f32(ce[i]) : NAN;
            s[i] = in ? Elem<T>::to_f32(se[i]) : NAN;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) c[i] = s[i] = NAN;
    }
}

// The 16-byte form of the rotation.  A lane has channels [e0, e0 + 8) and [e0 + d / 2, e0 + d / 2 + 8) of every head of a token, so that it holds
// both halves of its half-rotated pairs where all of a head turns (ROPE 2); the angles are loaded once per token.  ROPE 1: neighbouring pairs;
// 4: half-rotated pairs of which a head's front part consists, whose other half is read a second time (other()); 0: nothing turns.
// Each product and sum is rounded by itself, as in the append to a 16-bit cache.
template <typename T>
struct Pieces {
    Vec8<T> a, b;  // channels e0 .. and e0 + d / 2 ..
};

// two fp32 operations an instruction
__device__ __forceinline__ uint64_t two(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void apart(uint64_t x, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
template <typename T>
__device__ __forceinline__ uint64_t widen(uint32_t w) {
    if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        return two(f.x, f.y);
    } else {
        return two(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
}
template <typename T>
__device__ __forceinline__ uint32_t narrow(uint64_t x) {
    float lo, hi;
    apart(x, lo, hi);
    return Elem<T>::pack2(lo, hi);
}

template <typename T, int ROPE>
struct Turn {
    static constexpr int N = ROPE == 1 ? 4 : 8, SETS = ROPE == 0 ? 0 : ROPE == 2 ? 1 : 2;
    // for each word (two channels) of a piece what its own channels and their partners are multiplied by
    uint64_t c[SETS ? SETS : 1][4], s[SETS ? SETS : 1][4];
    int e[2], partner[2];
    bool turns[2];

    __device__ __forceinline__ Turn(const RotaryDev& r, int e0, int d) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            e[i] = e0 + i * (d >> 1);
            turns[i] = ROPE != 0 && e[i] < 2 * r.half;
            partner[i] = !turns[i] ? e[i] : e[i] < r.half ? e[i] + r.half : e[i] - r.half;
        }
    }
    __device__ __forceinline__ void load(const RotaryDev& r, const Positions& pos) {
#pragma unroll
        for (int i = 0; i < SETS; ++i) {
            if (!turns[i]) continue;
            float ca[N], sa[N];
            const bool low = ROPE == 4 && e[i] < r.half;
            load_angles<T, N>(r, ROPE == 1 ? e[i] / 2 : ROPE == 2 || low ? e[i] : e[i] - r.half, pos, ca, sa);
            if (low != r.back) {
#pragma unroll
                for (int k = 0; k < N; ++k) sa[k] = -sa[k];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                c[i][k] = ROPE == 1 ? two(ca[k], ca[k]) : two(ca[2 * k % N], ca[(2 * k + 1) % N]);
                s[i][k] = ROPE == 1 ? two(-sa[k], sa[k]) : two(sa[2 * k % N], sa[(2 * k + 1) % N]);
            }
        }
    }
    static __device__ __forceinline__ Pieces<T> read(const T* head, const int (&at)[2]) {
        Pieces<T> x;
        x.a.v = *reinterpret_cast<const uint4*>(head + at[0]);
        x.b.v = *reinterpret_cast<const uint4*>(head + at[1]);
        return x;
    }
    __device__ __forceinline__ Pieces<T> own(const T* head) const { return read(head, e); }
    __device__ __forceinline__ Pieces<T> other(const T* head) const { return read(head, partner); }
    __device__ __forceinline__ void write(T* head, const Pieces<T>& x) const {
        *reinterpret_cast<uint4*>(head + e[0]) = x.a.v;
        *reinterpret_cast<uint4*>(head + e[1]) = x.b.v;
    }
    __device__ __forceinline__ void one(Vec8<T>& x, const Vec8<T>& y, int i) const {
        if (!turns[i]) return;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint64_t own = widen<T>(x.w[k]);
            uint64_t partners = own;
            if constexpr (ROPE == 1) {
                float lo, hi;
                apart(own, lo, hi);
                partners = two(hi, lo);
            } else {
                partners = widen<T>(y.w[k]);
            }
            x.w[k] = narrow<T>(add2(mul2(own, c[i][k]), mul2(partners, s[i][k])));
        }
    }
    __device__ __forceinline__ void operator()(Pieces<T>& x, const Pieces<T>& y) const {
        if constexpr (ROPE == 2) {
            const uint64_t minus = two(-1.f, -1.f);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint64_t a = widen<T>(x.a.w[k]), b = widen<T>(x.b.w[k]);
                x.a.w[k] = narrow<T>(fma2(mul2(b, s[0][k]), minus, mul2(a, c[0][k])));
                x.b.w[k] = narrow<T>(add2(mul2(b, c[0][k]), mul2(a, s[0][k])));
            }
        } else if constexpr (ROPE != 0) {
            one(x.a, y.a, 0);
            one(x.b, y.b, 1);
        }
    }
};

// The form that a call takes: 3 is channel by channel.
inline int rope_form(const RotaryDev& r, int d) {
    if (!r.vec || d % 16 != 0 || d > 512 || 32 % (d / 16) != 0) return 3;
    return r.type != 2 ? r.type : 2 * r.half == d ? 2 : 4;
}

// The same channel by channel, for widths, tables and rows that the 16-byte form does not take.
template <typename T>
__device__ __forceinline__ void turn_piece_any(const RotaryDev& r, int e0, const Positions& pos, const T* row, Vec8<T>& out) {
    for (int i = 0; i < 8; ++i) {
        const int e = e0 + i;
        T y = row[e];
        if (r.type != 0 && e < 2 * r.half) {
            const int pair = r.type == 1 ? e >> 1 : e < r.half ? e : e - r.half;
            const bool low = r.type == 1 ? !(e & 1) : e < r.half;
            const T other = row[r.type == 1 ? e ^ 1 : low ? e + r.half : e - r.half];
            const int p = pos(axis_of(r, pair));
            const bool in = (uint32_t)p < (uint32_t)r.rows;
            const float c = in ? Elem<T>::to_f32(((const T*)r.cosr)[(int64_t)p * r.half + pair]) : NAN;
            float s = in ? Elem<T>::to_f32(((const T*)r.sinr)[(int64_t)p * r.half + pair]) : NAN;
            if (r.back) s = -s;
            const float other_s = __fmul_rn(Elem<T>::to_f32(other), s);
            y = Elem<T>::from_f32(__fadd_rn(__fmul_rn(Elem<T>::to_f32(y), c), low ? -other_s : other_s));
        }
        out.e[i] = y;
    }
}

#endif  // __CUDACC__

// Host side: the warps (log2) that share a token's work: enough to fill the SMs with few tokens, one with many (what they all work out is worked out
// fewer times).
inline int warps_log2_for(int64_t jobs, int64_t most) {
    int w = 3;
    while (w > 0 && ((1 << w) > most || jobs << w > (int64_t)sm_count() * 32)) --w;
    return w;
}

// Host side: `pair_axis` (one entry per pair, or nullptr: all turn with the first axis) into the bits of RotaryDev.
int fill_rotary(const char* fn, RotaryDev& r, const void* cosr, const void* sinr, int64_t rows, int64_t rotary_dim, int64_t d, int rope_type,
                const uint8_t* pair_axis, int64_t axes, bool rows_aligned);

}  // namespace fck
