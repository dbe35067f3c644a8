// The 4-bit key/value cache: what its bytes mean, and the rotation of queries and keys that its write fuses.
//
// A group of 32, 64 or 128 neighbouring channels of one token's head is held as value = lo + scale * code, code 0..15:
//     lo = min x,   scale = T((max x - min x) / 15),   code = min(15, rne((x - lo) / scale)),   scale = 0: code 0
// with the difference and the quotient's dividend in fp32 and T the model's 16-bit type; lo is one of the x and therefore exact.
// Codes: uint8 [rows, hkv, d / 2], byte j with channel 2j in its low and 2j + 1 in its high half.  Params: T [rows, hkv, d / group, 2] =
// (scale, lo).  A group with a NaN or an infinity, or one whose range leaves fp32, reads back as NaN.
#pragma once

#include "kernels.h"

namespace fck {

constexpr int kMaxPairs = 128, kMaxAxes = 4;

// What a rotation needs besides the row: cos / sin tables T [rows, half], and for each pair of a head the axis whose position turns it
// (2 bits a pair).
struct RotaryDev {
    const void* cosr;
    const void* sinr;
    int rows, half, type;  // type: 0 none, 1 neighbouring pairs (2i, 2i + 1), 2 (i, i + half)
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

// cos and sin of pairs [first, first + N) for positions pos(axis); a position outside the tables turns by NaN.  The vector form is taken
// where one axis turns all of them.
template <typename T, int N, typename Pos>
__device__ __forceinline__ void load_angles(const RotaryDev& r, int first, const Pos& pos, float (&c)[N], float (&s)[N]) {
    constexpr uint32_t kAll = (1u << (2 * N)) - 1u;
    const uint32_t axes = (r.axis[first >> 4] >> (2 * (first & 15))) & kAll, a0 = axes & 3u;
    if (axes == a0 * (0x5555u & kAll)) {
        const int64_t p = pos(a0);
        if ((uint64_t)p < (uint64_t)r.rows) {
            using V = typename std::conditional<N == 8, uint4, uint2>::type;
            const V cv = *reinterpret_cast<const V*>((const T*)r.cosr + p * r.half + first);
            const V sv = *reinterpret_cast<const V*>((const T*)r.sinr + p * r.half + first);
            const T* ce = reinterpret_cast<const T*>(&cv);
            const T* se = reinterpret_cast<const T*>(&sv);
#pragma unroll
            for (int i = 0; i < N; ++i) { c[i] = Elem<T>::to_f32(ce[i]); s[i] = Elem<T>::to_f32(se[i]); }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) c[i] = s[i] = NAN;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t p = pos(axis_of(r, first + i));
            const bool in = (uint64_t)p < (uint64_t)r.rows;
            c[i] = in ? Elem<T>::to_f32(((const T*)r.cosr)[p * r.half + first + i]) : NAN;
            s[i] = in ? Elem<T>::to_f32(((const T*)r.sinr)[p * r.half + first + i]) : NAN;
        }
    }
}

// The 16-byte form of the rotation: a lane's 8 channels [e0, e0 + 8) of every head of a token.  ROPE as RotaryDev::type.  The angles are
// loaded once per token; each product and sum is rounded by itself, as in the append to a 16-bit cache.
template <typename T, int ROPE>
struct Turn {
    static constexpr int N = ROPE == 1 ? 4 : 8;
    float c[N], s[N];  // (half-rotated: s with the sign that the partner channel comes with)
    int partner;       // where its partner channels are (itself where it needs none)
    bool turns;

    __device__ __forceinline__ Turn(const RotaryDev& r, int e0) {
        turns = ROPE != 0 && e0 < 2 * r.half;
        partner = ROPE != 2 || !turns ? e0 : e0 < r.half ? e0 + r.half : e0 - r.half;
    }
    template <typename Pos>
    __device__ __forceinline__ void load(const RotaryDev& r, int e0, const Pos& pos) {
        if (!turns) return;
        const bool low = ROPE == 2 && e0 < r.half;
        load_angles<T, N>(r, ROPE == 1 ? e0 / 2 : low ? e0 : e0 - r.half, pos, c, s);
        if (low != r.back) {
#pragma unroll
            for (int i = 0; i < N; ++i) s[i] = -s[i];
        }
    }
    __device__ __forceinline__ Vec8<T> operator()(const Vec8<T>& x, const Vec8<T>& y) const {
        if (!turns) return x;
        Vec8<T> out;
        if constexpr (ROPE == 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = Elem<T>::to_f32(x.e[2 * i]), b = Elem<T>::to_f32(x.e[2 * i + 1]);
                out.w[i] = Elem<T>::pack2(__fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i])), __fadd_rn(__fmul_rn(a, s[i]), __fmul_rn(b, c[i])));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                out.w[i] = Elem<T>::pack2(
                    __fadd_rn(__fmul_rn(Elem<T>::to_f32(x.e[2 * i]), c[2 * i]), __fmul_rn(Elem<T>::to_f32(y.e[2 * i]), s[2 * i])),
                    __fadd_rn(__fmul_rn(Elem<T>::to_f32(x.e[2 * i + 1]), c[2 * i + 1]), __fmul_rn(Elem<T>::to_f32(y.e[2 * i + 1]), s[2 * i + 1])));
        }
        return out;
    }
};

// The same channel by channel, for widths, tables and rows that the 16-byte form does not take.
template <typename T, typename Pos>
__device__ __forceinline__ void turn_piece_any(const RotaryDev& r, int e0, const Pos& pos, const T* row, Vec8<T>& out) {
    for (int i = 0; i < 8; ++i) {
        const int e = e0 + i;
        T y = row[e];
        if (r.type != 0 && e < 2 * r.half) {
            const int pair = r.type == 1 ? e >> 1 : e < r.half ? e : e - r.half;
            const bool low = r.type == 1 ? !(e & 1) : e < r.half;
            const T other = row[r.type == 1 ? e ^ 1 : low ? e + r.half : e - r.half];
            const int64_t p = pos(axis_of(r, pair));
            const bool in = (uint64_t)p < (uint64_t)r.rows;
            const float c = in ? Elem<T>::to_f32(((const T*)r.cosr)[p * r.half + pair]) : NAN;
            float s = in ? Elem<T>::to_f32(((const T*)r.sinr)[p * r.half + pair]) : NAN;
            if (r.back) s = -s;
            const float other_s = __fmul_rn(Elem<T>::to_f32(other), s);
            y = Elem<T>::from_f32(__fadd_rn(__fmul_rn(Elem<T>::to_f32(y), c), low ? -other_s : other_s));
        }
        out.e[i] = y;
    }
}

#endif  // __CUDACC__

// Host side: `pair_axis` (one entry per pair, or nullptr: all turn with the first axis) into the bits of RotaryDev.
int fill_rotary(const char* fn, RotaryDev& r, const void* cosr, const void* sinr, int64_t rows, int64_t rotary_dim, int64_t d, int rope_type,
                const uint8_t* pair_axis, int64_t axes, bool rows_aligned);

}  // namespace fck
