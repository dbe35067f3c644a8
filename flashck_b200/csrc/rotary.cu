// Rotation of queries and keys by the positions of their tokens, along one or several axes (int4.cuh has the arithmetic).
//
// Bound by its traffic: each row read and written once.  A warp turns a token (a few warps, where tokens are few); a lane keeps the cosines
// and sines of its 16 channels for all heads.  16384 tokens of 32 + 8 heads of 128: 53 us among other calls, floor 51 at 6.54 TB/s (the copy rate).
// Widths whose 16-channel pieces do not divide a warp go channel by channel: heads of 96 174 us, floor 39.
#include <algorithm>
#include <type_traits>

#include "int4.cuh"

namespace fck {

namespace {

struct RotaryCall {
    RotaryDev rot;
    const void* src[2];  // q, k
    void* dst[2];
    const int32_t* positions;
    int64_t tokens;
    int heads[2], d, warps_log2;  // warps of a token
};

template <typename T, int ROPE>
__global__ void __launch_bounds__(256) rotary_kernel(const __grid_constant__ RotaryCall a) {
    constexpr int kAhead = ROPE == 4 ? 2 : 4;  // heads in flight
    pdl_launch_dependents();
    pdl_wait();
    const int w = 1 << a.warps_log2, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t t = (int64_t)blockIdx.x << (3 - a.warps_log2) | (warp >> a.warps_log2);
    const int part = warp & (w - 1);
    if (t >= a.tokens) return;
    const int lanes = a.d >> 4, sub = lane / lanes, e0 = (lane - sub * lanes) << 3, step = 32 / lanes * w;
    const int both = a.heads[0] + a.heads[1];  // the queries' heads, then the keys'
    auto src = [&](int h) { return h < a.heads[0] ? (const T*)a.src[0] + (t * a.heads[0] + h) * a.d : (const T*)a.src[1] + (t * a.heads[1] + h - a.heads[0]) * a.d; };
    auto dst = [&](int h) { return h < a.heads[0] ? (T*)a.dst[0] + (t * a.heads[0] + h) * a.d : (T*)a.dst[1] + (t * a.heads[1] + h - a.heads[0]) * a.d; };
    Positions pos;
    pos.load(a.positions, a.rot.axes, a.tokens, t);
    Turn<T, ROPE> turn(a.rot, e0, a.d);
    Pieces<T> x[kAhead], y[kAhead];
    auto request = [&](int h0) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int h = h0 + u * step;
            if (h < both) {
                x[u] = turn.own(src(h));
                if (ROPE == 4) y[u] = turn.other(src(h));
            }
        }
    };
    int h0 = part * (32 / lanes) + sub;
    request(h0);  // (in flight while positions and angles come)
    turn.load(a.rot, pos);
    for (; h0 < both; h0 += step * kAhead) {
        if (h0 >= step * kAhead) request(h0);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int h = h0 + u * step;
            if (h < both) {
                turn(x[u], y[u]);
                turn.write(dst(h), x[u]);
            }
        }
    }
}

// Any width, any alignment.
template <typename T>
__global__ void __launch_bounds__(256) rotary_any_kernel(const __grid_constant__ RotaryCall a) {
    pdl_launch_dependents();
    pdl_wait();
    const int w = 1 << a.warps_log2, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t t = (int64_t)blockIdx.x << (3 - a.warps_log2) | (warp >> a.warps_log2);
    const int part = warp & (w - 1);
    if (t >= a.tokens) return;
    Positions pos;
    pos.load(a.positions, a.rot.axes, a.tokens, t);
    const int pieces = a.d >> 3;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const T* src = (const T*)a.src[i] + t * a.heads[i] * a.d;
        T* dst = (T*)a.dst[i] + t * a.heads[i] * a.d;
        for (int p = part * 32 + lane; p < a.heads[i] * pieces; p += w * 32) {
            const int h = p / pieces, e0 = (p - h * pieces) << 3;
            Vec8<T> out;
            turn_piece_any<T>(a.rot, e0, pos, src + (int64_t)h * a.d, out);
            for (int k = 0; k < 8; ++k) dst[(int64_t)h * a.d + e0 + k] = out.e[k];
        }
    }
}

template <typename T>
cudaError_t launch_type(const RotaryCall& a, unsigned blocks, cudaStream_t stream) {
    const dim3 grid(blocks), block(256);
    switch (rope_form(a.rot, a.d)) {
        case 1: return launch_dependent(rotary_kernel<T, 1>, grid, block, 0, stream, a);
        case 2: return launch_dependent(rotary_kernel<T, 2>, grid, block, 0, stream, a);
        case 4: return launch_dependent(rotary_kernel<T, 4>, grid, block, 0, stream, a);
        default: return launch_dependent(rotary_any_kernel<T>, grid, block, 0, stream, a);
    }
}

}  // namespace

int launch_rotary(const RotaryParams& p, cudaStream_t stream) {
    FCK_REQUIRE(p.d > 0 && p.d % 8 == 0 && p.d <= 1024, FLASHCK_ERR_UNSUPPORTED, "FmhaRotary: hdim must be a multiple of 8, at most 1024 (got %lld)",
                (long long)p.d);
    FCK_REQUIRE(p.rope_type != 0, FLASHCK_ERR_INVALID_ARGUMENT, "FmhaRotary: rope_type must be 1 or 2");
    FCK_REQUIRE(p.hq <= 16384 && p.hkv <= 16384, FLASHCK_ERR_UNSUPPORTED, "FmhaRotary: at most 16384 heads");
    RotaryCall a{};
    const auto aligned = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15u) == 0; };
    if (int rc = fill_rotary("FmhaRotary", a.rot, p.rotary_cos, p.rotary_sin, p.rotary_rows, p.rotary_dim, p.d, p.rope_type, p.pair_axis, p.axes,
                             aligned(p.q) && aligned(p.q_out) && aligned(p.k) && aligned(p.k_out))) return rc;
    a.rot.back = p.inverse != 0;
    a.src[0] = p.q; a.src[1] = p.k; a.dst[0] = p.q_out; a.dst[1] = p.k_out;
    a.positions = p.positions; a.tokens = p.tokens; a.d = (int)p.d;
    a.heads[0] = (int)p.hq; a.heads[1] = p.k ? (int)p.hkv : 0;
    if (p.tokens == 0 || a.heads[0] + a.heads[1] == 0) return FLASHCK_OK;
    const int64_t most = std::max<int64_t>(1, (p.hq + a.heads[1]) * p.d / 256);
    a.warps_log2 = warps_log2_for(p.tokens, most);
    const int64_t blocks = ((p.tokens << a.warps_log2) + 7) / 8;
    FCK_REQUIRE(blocks < (1ll << 31), FLASHCK_ERR_UNSUPPORTED, "FmhaRotary: too many tokens");
    if (p.dtype == FLASHCK_DTYPE_BFLOAT16) FCK_CUDA(launch_type<__nv_bfloat16>(a, (unsigned)blocks, stream));
    else FCK_CUDA(launch_type<__half>(a, (unsigned)blocks, stream));
    return FLASHCK_OK;
}

}  // namespace fck
