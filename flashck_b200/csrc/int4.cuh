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

// The 16-byte form of the rotation.  A lane has channels [e0, e0 + 8) and [e0 + d / 2, e0 + d / 2 + 8) of every head of a token, so that it holds
// both halves of its half-rotated pairs where all of a head turns (ROPE 2); the angles are loaded once per token.  ROPE 1: neighbouring pairs;
// 4: half-rotated pairs of which a head's front part consists, whose other half is read a second time (other()); 0: nothing turns.
// Each product and sum is rounded by itself, as in the append to a 16-bit cache.
template <typename T>
struct Pieces {
    Vec8<T> a, b;  // channels e0 .. and e0 + d / 2 ..
};

template <typename T, int ROPE>
struct Turn {
    static constexpr int N = ROPE == 1 ? 4 : 8, SETS = ROPE == 0 ? 0 : ROPE == 2 ? 1 : 2;
    float c[SETS ? SETS : 1][N], s[SETS ? SETS : 1][N];  // (ROPE 4: s with the sign that the partner channel comes with)
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
    template <typename Pos>
    __device__ __forceinline__ void load(const RotaryDev& r, const Pos& pos) {
#pragma unroll
        for (int i = 0; i < SETS; ++i) {
            if (!turns[i]) continue;
            const bool low = ROPE == 4 && e[i] < r.half;
            load_angles<T, N>(r, ROPE == 1 ? e[i] / 2 : ROPE == 2 || low ? e[i] : e[i] - r.half, pos, c[i], s[i]);
            if (low != r.back) {
#pragma unroll
                for (int k = 0; k < N; ++k) s[i][k] = -s[i][k];
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

    static __device__ __forceinline__ float f(T x) { return Elem<T>::to_f32(x); }
    static __device__ __forceinline__ float turned(T x, float cx, T y, float sy) { return __fadd_rn(__fmul_rn(f(x), cx), __fmul_rn(f(y), sy)); }
    __device__ __forceinline__ void one(Vec8<T>& x, const Vec8<T>& y, int i) const {
        if (!turns[i]) return;
        Vec8<T> out;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (ROPE == 1)
                out.w[k] = Elem<T>::pack2(turned(x.e[2 * k], c[i][k], x.e[2 * k + 1], -s[i][k]), turned(x.e[2 * k + 1], c[i][k], x.e[2 * k], s[i][k]));
            else
                out.w[k] = Elem<T>::pack2(turned(x.e[2 * k], c[i][2 * k], y.e[2 * k], s[i][2 * k]),
                                          turned(x.e[2 * k + 1], c[i][2 * k + 1], y.e[2 * k + 1], s[i][2 * k + 1]));
        }
        x = out;
    }
    __device__ __forceinline__ void operator()(Pieces<T>& x, const Pieces<T>& y) const {
        if constexpr (ROPE == 2) {
            Pieces<T> out;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                out.a.w[k] = Elem<T>::pack2(turned(x.a.e[2 * k], c[0][2 * k], x.b.e[2 * k], -s[0][2 * k]),
                                            turned(x.a.e[2 * k + 1], c[0][2 * k + 1], x.b.e[2 * k + 1], -s[0][2 * k + 1]));
                out.b.w[k] = Elem<T>::pack2(turned(x.b.e[2 * k], c[0][2 * k], x.a.e[2 * k], s[0][2 * k]),
                                            turned(x.b.e[2 * k + 1], c[0][2 * k + 1], x.a.e[2 * k + 1], s[0][2 * k + 1]));
            }
            x = out;
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
