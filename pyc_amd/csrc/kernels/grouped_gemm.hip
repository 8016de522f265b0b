// grouped_gemm.hip — products grouped by expert: which kernel runs a call, and the one for any
// size and alignment.
//
//   y[p] = epi(x[src(p)] W[e]^T + bias[e])   for offsets[e] <= p < offsets[e + 1]
//
// with W 16-bit values, or 4-bit codes with a scale (and zero point) for each group
// along K. fp32 sums. The general kernel: a workgroup has 64 rows of one expert and 64 columns, four waves as
// 2 x 2, operands two steps ahead through registers into LDS (16-byte chunk c of row r at c ^ (r % 8)). The
// rows of x are the first operand of the matrix instruction, so a lane's four results are
// four rows of one column, and a column's scale is one value for each lane. Codes less
// their zero point are whole numbers of at most 8 bits, exact in 16-bit values: each
// 32 k of them (a group has 32, 64 or 128) are summed apart, then scaled into the sums
// in fp32. Gated: fragments of a wave alternate, 16 gates and the 16 values of the same
// columns, so that a lane has both. Rows at odd places are loaded as 16 unaligned bytes; what would
// cross the end of its row is loaded up to there and shifted. Bound by the L1, which 16 unaligned bytes cost more than one
// access: 2048 rows of 8 experts of 4096 x 4096 with x off 16 bytes take 447 thousand a CU in 444 thousand cycles,
// 194 us (aligned, in tiles, 112); 256 rows of 64 of 2048 x 2816 191 (in the ring 131).
#include "grouped.hpp"

namespace pyc {

constexpr int kGenTile = 64, kGenK = 64;

// Elements c .. c + 7 of a row of K, 0 behind its end. `edge` (uniform): some lane's reach past it.
__device__ inline u32x4 row_piece(const uint16_t* row, int c, int K, bool edge) {
    u32x4 v = u32x4{0, 0, 0, 0};
    if (!edge) {
        __builtin_memcpy(&v, row + c, 16);
    } else if (K >= 8) {
        const int from = min(c, K - 8), sh = c - from;  // elements of it that come before c
        __builtin_memcpy(&v, row + from, 16);
        uint64_t lo = (uint64_t)v[0] | ((uint64_t)v[1] << 32), hi = (uint64_t)v[2] | ((uint64_t)v[3] << 32);
        lo = sh >= 4 ? hi : lo;
        hi = sh >= 4 ? 0 : hi;
        const int b = 16 * (sh & 3);
        lo = (lo >> b) | ((hi << 1) << (63 - b));
        hi >>= b;
        if (sh >= 8) lo = hi = 0;
        v = u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
    } else {
        uint16_t e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = c + i < K ? row[c + i] : (uint16_t)0;
        __builtin_memcpy(&v, e, 16);
    }
    return v;
}

template <typename T, bool W4>
__global__ void __launch_bounds__(256) grouped_general_kernel(Grouped g, int tiles_n, uint32_t tile0) {
    __shared__ __attribute__((aligned(16))) uint16_t Xs[2][kGenTile * kGenK], Ws[2][kGenTile * kGenK];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave >> 1, wn = wave & 1, lrow = lane & 15, lgrp = lane >> 4;
    const uint32_t tile = tile0 + blockIdx.x;
    const int tn = tile % tiles_n;
    const ExpertTile t = expert_tile(g, tile / tiles_n, kGenTile, lane);
    if (t.e < 0) return;
    const bool gate = g.epi & kEpiGate;
    const int F = gate ? g.N / 2 : g.N;                    // columns of y
    const int cols = gate ? kGenTile / 2 : kGenTile;
    // the row of W behind tile row r (-1: none)
    auto weight_row = [&](int r) {
        if (!gate) return tn * cols + r < F ? tn * cols + r : -1;
        const int c = tn * cols + (r >> 5) * 16 + (r & 15);
        return c < F ? c + ((r >> 4) & 1) * F : -1;
    };
    // a thread's chunks: row tid / 8 and 32 rows on, 16-byte chunk tid % 8; codes: row tid / 4,
    // 16 of the 64 k
    const int row0 = tid >> 3, ch = tid & 7;
    const uint16_t* xr[2];
    const uint16_t* wr[2];
    bool xin[2];
    const int64_t ew = (int64_t)t.e * g.w_stride;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        // rows that there are not are read from the first one; x's count as zeros, W's reach no result
        const int p = t.begin + row0 + 32 * i;
        const int r = source_row(g, p, t.end);
        xin[i] = r >= 0;
        xr[i] = g.x + (int64_t)max(r, 0) * g.x_stride;
        wr[i] = static_cast<const uint16_t*>(g.w) + ew + (int64_t)max(weight_row(row0 + 32 * i), 0) * g.K;
    }
    const int crow = weight_row(tid >> 2);
    auto slot = [](int r, int c) { return r * kGenK + ((c ^ (r & 7)) << 3); };

    f32x4 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    int col[2];  // row of W of the lane's column in fragment j
#pragma unroll
    for (int j = 0; j < 2; ++j) col[j] = weight_row(wn * 32 + j * 16 + lrow);

    const int groups = W4 ? g.K / g.group : 0;
    // a step's chunks as loaded: two steps ahead of the one that is multiplied
    struct Step {
        u32x4 a[2], b[2];
        uint64_t q;
        int z;
    };
    const int xk = g.x_rows > 0 ? g.K : 0;  // without rows nothing of x is read
    auto load = [&](Step& s, int k0) {
        const bool edge = k0 + kGenK > g.K;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            s.a[i] = row_piece(xr[i], k0 + 8 * ch, xk, edge || xk == 0);
            if constexpr (!W4) s.b[i] = row_piece(wr[i], k0 + 8 * ch, g.K, edge);
        }
        if constexpr (W4) {
            const int k = k0 + 16 * (tid & 3);
            s.q = 0x8888888888888888ull;
            s.z = 8;
            if (crow >= 0 && k < g.K) {
                s.q = *reinterpret_cast<const uint64_t*>(static_cast<const uint8_t*>(g.w) + ew + (int64_t)crow * (g.K / 2) + k / 2);
                if (g.zeros) s.z = g.zeros[((int64_t)t.e * g.N + crow) * groups + k / g.group];
            }
        }
    };
    auto store = [&](Step& s, int buf) {
        if constexpr (W4) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int lo = (int)(s.q >> (32 * i + 8 * j)) & 15, hi = (int)(s.q >> (32 * i + 8 * j + 4)) & 15;
                    s.b[i][j] = elem<T>::from_f32((float)(lo - s.z)) | ((uint32_t)elem<T>::from_f32((float)(hi - s.z)) << 16);
                }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            *reinterpret_cast<u32x4*>(&Xs[buf][slot(row0 + 32 * i, ch)]) = xin[i] ? s.a[i] : u32x4{0, 0, 0, 0};
            if constexpr (W4) *reinterpret_cast<u32x4*>(&Ws[buf][slot(tid >> 2, 2 * (tid & 3) + i)]) = s.b[i];
            else *reinterpret_cast<u32x4*>(&Ws[buf][slot(row0 + 32 * i, ch)]) = s.b[i];
        }
    };
    auto multiply = [&](int k0, int buf) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            u32x4 fa[2], fb[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                fa[i] = *reinterpret_cast<const u32x4*>(&Xs[buf][slot(wm * 32 + i * 16 + lrow, kk * 4 + lgrp)]);
                fb[i] = *reinterpret_cast<const u32x4*>(&Ws[buf][slot(wn * 32 + i * 16 + lrow, kk * 4 + lgrp)]);
            }
            if constexpr (W4) {
                const int k = k0 + 32 * kk;
                if (k >= g.K) break;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float s = col[j] < 0 ? 0.f
                                               : elem<T>::to_f32(g.scale[((int64_t)t.e * g.N + col[j]) * groups + k / g.group]);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const f32x4 d = mfma16x16x32(fa[i], fb[j], f32x4{0.f, 0.f, 0.f, 0.f}, T{});
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[i][j][r] = fmaf(s, d[r], acc[i][j][r]);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[i][j] = mfma16x16x32(fa[i], fb[j], acc[i][j], T{});
            }
        }
    };
    Step s0, s1;
    load(s0, 0);
    load(s1, kGenK);
    for (int k0 = 0; k0 < g.K; k0 += 2 * kGenK) {  // k past K is zeros
        store(s0, 0);
        load(s0, k0 + 2 * kGenK);
        __syncthreads();
        multiply(k0, 0);
        store(s1, 1);
        load(s1, k0 + 3 * kGenK);
        __syncthreads();
        multiply(k0 + kGenK, 1);
    }

    const ExpertBias expert_bias(g, t.e);
    const float bias[2] = {expert_bias[col[0]], expert_bias[col[1]]};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int p = t.begin + wm * 32 + i * 16 + 4 * lgrp + r;
            if (p >= t.end) continue;
            uint16_t* y = g.y + (int64_t)p * g.y_stride;
            const float v0 = acc[i][0][r] + bias[0], v1 = acc[i][1][r] + bias[1];
            if (gate) {
                if (col[0] >= 0) y[col[0]] = elem<T>::from_f32(silu_gate(v0, v1));
            } else {
                const bool relu = g.epi & kEpiRelu;
                if (col[0] >= 0) y[col[0]] = elem<T>::from_f32(relu ? relu_of(v0) : v0);
                if (col[1] >= 0) y[col[1]] = elem<T>::from_f32(relu ? relu_of(v1) : v1);
            }
        }
}

}  // namespace pyc

extern "C" int pyc_hip_grouped_stream_takes(int w4, const pyc_grouped* g);
extern "C" int pyc_hip_grouped_stream_launch(int is_bf16, const pyc_grouped* g, void* stream);
extern "C" int pyc_hip_grouped_tile_takes(const pyc_grouped* g);
extern "C" int pyc_hip_grouped_tile_launch(int is_bf16, const pyc_grouped* g, void* stream);
extern "C" int pyc_hip_grouped_ring_launch(int is_bf16, const pyc_grouped* g, int fn, void* stream);
extern "C" int pyc_hip_grouped_w4_tile_launch(int is_bf16, const pyc_grouped* g, int form, void* stream);

// The kernel of a call, from what the host knows: rows in all, not whose they are. Measured on the MI355X
// over experts of K x N with P rows in all, in us (other side behind the stroke):
//  16-bit: the ring's tiles of 64 rows x 64 columns; of 128 columns where those fill the CUs twice (8 of
//    4096 x 4096: P = 256 62 / 74, 1024 87 / 98); 256 x 256 tiles from some 200 rows an expert on, or
//    100 in large calls (8 of 4096 x 4096: P = 2048 111 / 129, 1024 109 / 87; 64 of 2048 x 2816: P = 8192 207 / 292).
//  4-bit: streamed up to 6 rows an expert (32 of 4096 x 2816: P = 128 60 / 67 in tiles, 256 75 / 71), or where
//    columns are so few that only parts of K fill the CUs (11008 x 4096: P = 32 27 / 53, 64 48 / 57, 128 81 / 63), which
//    takes in wide products of up to 16 rows (4096 x 11008: P = 8 13.2 / 14.5, 12 14.8 / 14.6, 16 15.7 / 14.7, but 24
//    23.5 / 19.6); then the smallest tiles that are no more than 3 in two places (4096 x 11008: P = 48
//    25 / 29 in tiles of 16 rows, 128 33 / 54; 11008 x 4096: P = 128 63 / 80 in tiles of 64), and 128 x 256 from 96
//    rows an expert on where they fill half of the CUs (4096 x 11008: P = 256 66 / 53, 512 69 / 101; 32 of 4096 x
//    2816: P = 4096 189 / 263; 8 of 2048 x 2048: P = 2048 41 / 46).
// KIND: 0 the general kernel, 1 ring, 2 tiles, 3 stream, 4 4-bit tiles; arg: what its launch takes.
extern "C" int pyc_hip_grouped_form(int w4, const pyc_grouped* g, int* arg) {
    using namespace pyc;
    const int64_t P = g->P, E = g->offsets ? g->E : 1, N = g->N;
    *arg = 0;
    if (!pyc_hip_grouped_stream_takes(w4, g)) return 0;
    if (!w4) {
        if (pyc_hip_grouped_tile_takes(g) && ((P >= 192 * E && P * N >= 1 << 23) || (P >= 96 * E && P * N >= 1 << 24))) return 2;
        *arg = P * N >= 512 * 4096 ? 2 : 1;
        return 1;
    }
    auto tiles = [&](int rows) { return g->offsets ? expert_tiles_most((int)E, g->P, rows) : (P + rows - 1) / rows; };
    if (P <= 6 * E || tiles(16) * N <= 16384) return 3;
    if (P >= 96 * E && P * N >= 128 * 128 * 256) return 4;
    const int64_t blocks = (N + 63) / 64;
    *arg = tiles(16) * blocks <= 384 ? 1 : tiles(32) * blocks <= 384 ? 2 : 4;
    return 4;
}

extern "C" int pyc_hip_grouped_launch(int is_bf16, int w4, const pyc_grouped* gp, void* stream) {
    using namespace pyc;
    const Grouped& g = *gp;
    int arg;
    switch (pyc_hip_grouped_form(w4, gp, &arg)) {
        case 1: return pyc_hip_grouped_ring_launch(is_bf16, gp, arg, stream);
        case 2: return pyc_hip_grouped_tile_launch(is_bf16, gp, stream);
        case 3: return pyc_hip_grouped_stream_launch(is_bf16, gp, stream);
        case 4: return pyc_hip_grouped_w4_tile_launch(is_bf16, gp, arg, stream);
    }
    const int cols = g.epi & kEpiGate ? g.N / 2 : g.N, per = g.epi & kEpiGate ? kGenTile / 2 : kGenTile;
    const int tiles_n = (cols + per - 1) / per;
    const int64_t tiles = expert_tiles_most(g.offsets ? g.E : 1, g.P, kGenTile) * tiles_n;
    const hipStream_t s = (hipStream_t)stream;
    return grouped_launches(tiles, 256, [&](uint32_t tile0, dim3 grid) {
#define PYC_GENERAL(TY, W) hipLaunchKernelGGL((grouped_general_kernel<TY, W>), grid, dim3(256), 0, s, g, tiles_n, tile0)
        if (w4) {
            if (is_bf16) PYC_GENERAL(bf16_t, true);
            else PYC_GENERAL(f16_t, true);
        } else {
            if (is_bf16) PYC_GENERAL(bf16_t, false);
            else PYC_GENERAL(f16_t, false);
        }
#undef PYC_GENERAL
    });
}
