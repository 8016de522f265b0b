// grouped.hpp — what the products by expert share: their operands, the rows of an
// expert, the row of x behind a row of y, and the epilogue.
#pragma once

#include <type_traits>

#include "common.hpp"
#include "grouped_args.h"

namespace pyc {

constexpr int kEpiBias = 1, kEpiRelu = 2, kEpiGate = 4;
constexpr int kMaxExperts = 1024;

typedef pyc_grouped Grouped;

// Inclusive scans over the wave's lanes: four steps in each row of 16, then the rows' last lanes.
template <int CTRL, int ROWS> __device__ inline int dpp_or(int old, int v) {
    return __builtin_amdgcn_update_dpp(old, v, CTRL, ROWS, 0xf, false);
}
__device__ inline int scan_add(int v) {
    v += dpp_or<0x111, 0xf>(0, v);  // row_shr 1, 2, 4, 8
    v += dpp_or<0x112, 0xf>(0, v);
    v += dpp_or<0x114, 0xf>(0, v);
    v += dpp_or<0x118, 0xf>(0, v);
    v += dpp_or<0x142, 0xa>(0, v);  // lane 15 of a row into the next, rows 1 and 3
    v += dpp_or<0x143, 0xc>(0, v);  // lane 31 into rows 2 and 3
    return v;
}
__device__ inline int scan_max(int v) {  // of numbers >= 0
    v = max(v, dpp_or<0x111, 0xf>(0, v));
    v = max(v, dpp_or<0x112, 0xf>(0, v));
    v = max(v, dpp_or<0x114, 0xf>(0, v));
    v = max(v, dpp_or<0x118, 0xf>(0, v));
    v = max(v, dpp_or<0x142, 0xa>(0, v));
    v = max(v, dpp_or<0x143, 0xc>(0, v));
    return v;
}

// Tile t of a grid whose tiles are `step` rows of one expert, expert after expert.
// offsets are held to 0 .. P and to what came before, so that no row has two experts
// whatever they say. Every wave finds its tile by itself, 64 experts at a time, lanes behind
// the last expert with none of its rows (no branch: see source_row).
struct ExpertTile {
    int e, begin, end;  // expert (-1: there is no tile t), the tile's first row, the expert's end
};
__device__ inline ExpertTile expert_tile(const Grouped& g, int t, int step, int lane) {
    if (g.offsets == nullptr) {
        const int b = t * step;
        return b < g.P ? ExpertTile{0, b, g.P} : ExpertTile{-1, 0, 0};
    }
    int held = 0, before = 0;  // the largest offset so far, tiles so far
    for (int e0 = 0; e0 < g.E; e0 += kWave) {
        const int e = e0 + lane;
        const int b = scan_max(max(held, min(g.offsets[min(e, g.E)], g.P)));
        const int end = max(b, min(g.offsets[min(e + 1, g.E)], g.P));
        const int n = (end - b + step - 1) / step;
        const int sum = scan_add(n);
        const uint64_t in = __ballot(t < before + sum);
        if (in) {
            const int l = __builtin_ctzll(in);
            const int first = __builtin_amdgcn_readlane(b, l), last = __builtin_amdgcn_readlane(end, l);
            const int tb = before + __builtin_amdgcn_readlane(sum - n, l);
            return ExpertTile{__builtin_amdgcn_readfirstlane(e0 + l), first + (t - tb) * step, last};
        }
        before += __builtin_amdgcn_readlane(sum, kWave - 1);
        held = __builtin_amdgcn_readlane(end, kWave - 1);
    }
    return ExpertTile{-1, 0, 0};
}

// Tiles there can be: every expert with rows begins one of its own.
inline int64_t expert_tiles_most(int E, int P, int step) {
    return (int64_t)P / step + (E < P ? E : P);
}

// `all` workgroups in as few launches as hold their threads: launch(the first one's place, grid).
template <typename F> inline int grouped_launches(int64_t all, int threads, F launch) {
    if (all > 0x7FFF0000) return -1;
    const int64_t most = kMostThreads / threads;
    for (int64_t at = 0; at < all; at += most) launch((uint32_t)at, dim3((unsigned)(all - at < most ? all - at : most)));
    return hipGetLastError() == hipSuccess ? 0 : -2;
}

// The row of x behind row p of y, -1 (zeros) where the index is outside x or p is not below end (the expert's, at least
// one). All lanes do the same, for some that there is no row for read another one's index: where lanes go apart among
// as many values as a tile's, the compiler has put copies of registers at the join before all of them were back.
__device__ inline int source_row(const Grouped& g, int p, int end) {
    int r = p;
    bool in = p < end;
    if (g.rows) {  // the same for all
        r = g.rows[min(p, end - 1)];
        in &= r >= 0;
        r = (int)((unsigned)max(r, 0) / (unsigned)g.fan);
    }
    return (in & (r < g.x_rows)) ? r : -1;
}

// Bias of row n of expert e's W, 0 for row -1 and without a bias: the range check of a descriptor takes the place of a
// branch that lanes take apart (an expert's biases are at most 2^26 bytes).
struct ExpertBias {
    __amdgpu_buffer_rsrc_t rsrc;
    bool there;  // the same for all lanes
    __device__ ExpertBias(const Grouped& g, int e)
        : rsrc(__builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(g.bias) + (int64_t)e * g.N, 0, (uint32_t)g.N * 4u, 0x00020000)),
          there(g.epi & kEpiBias) {}
    __device__ float operator[](int n) const {
        return there ? __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rsrc, (uint32_t)n * 4u, 0, 0)) : 0.f;
    }
};

// w[i] of lane group g becomes w[g] of lane group i.
__device__ inline void transpose4(u32x4& w) {
    auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
    auto b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    w = u32x4{c[0], c[1], d[0], d[1]};
}

// Eight codes as 16 + c, exact in either type, pairs k 0,1 2,3 4,5 6,7. A byte has two codes; the units of 16 are s
// bits up in its mantissa (bf16: 3, fp16: 6), so byte * (2^s + 2^(s + 12)) has one code in place in each half: a
// multiplication (which takes a byte of a register as it is) and an and-or for each pair. b: 16 twice, m: the codes' bits;
// both best in registers.
__device__ inline uint32_t codes16_mask(bf16_t) { return 0x00780078u; }
__device__ inline uint32_t codes16_mask(f16_t) { return 0x03c003c0u; }
template <typename T> __device__ inline u32x4 codes16(uint32_t w, uint32_t m, uint32_t b, T) {
    constexpr uint32_t f = std::is_same_v<T, bf16_t> ? 0x8008u : 0x40040u;
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (((w >> (8 * i)) & 255u) * f & m) | b;
    return r;
}

// v of the lane eight further on in each row of 16, around its end.
__device__ inline float row_half_turn(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xf, 0xf, false));
}

// max(v, 0), NaN of NaN (a maximum instruction would take 0).
__device__ inline float relu_of(float v) { return v < 0.f ? 0.f : v; }

// silu(g) * v = g v / (1 + e^-g), in fp32. All of it is taken in quarters: 1 + e^-g comes to 2^128 at g = -88.7,
// and the reciprocal instruction keeps no result below 2^-126. So it is off by at most one of its steps wherever
// e^-g is a number; below, silu(g) (under 3e-37 in size) counts as 0.
__device__ inline float silu_gate(float g, float v) {
    return 0.25f * g * __builtin_amdgcn_rcpf(fmaf(0.25f, __expf(-g), 0.25f)) * v;
}

}  // namespace pyc
