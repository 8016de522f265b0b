// grouped_gemm.hip — products grouped by expert, any size and alignment.
//
//   y[p] = epi(x[src(p)] W[e]^T + bias[e])   for offsets[e] <= p < offsets[e + 1]
//
// with W 16-bit values, or 4-bit codes with a scale (and zero point) for each group
// along K. fp32 sums. A workgroup has 64 rows of one expert and 64 columns, four waves as
// 2 x 2, operands through registers into LDS (16-byte chunk c of row r at c ^ (r % 8)). The
// rows of x are the first operand of the matrix instruction, so a lane's four results are
// four rows of one column, and a column's scale is one value for each lane. Codes less
// their zero point are whole numbers of at most 8 bits, exact in 16-bit values: each
// 32 k of them (a group has 32, 64 or 128) are summed apart, then scaled into the sums
// in fp32. Gated: fragments of a wave alternate, 16 gates and the 16 values of the same
// columns, so that a lane has both.
#include "grouped.hpp"

namespace pyc {

constexpr int kGenTile = 64, kGenK = 64;

// Eight elements from p, 0 behind `left` of them (p is not read there).
__device__ inline u32x4 load_guarded(const uint16_t* p, int left, bool wide) {
    if (wide && left >= 8) return *reinterpret_cast<const u32x4*>(p);
    uint16_t e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = i < left ? p[i] : (uint16_t)0;
    return u32x4{e[0] | ((uint32_t)e[1] << 16), e[2] | ((uint32_t)e[3] << 16), e[4] | ((uint32_t)e[5] << 16),
                 e[6] | ((uint32_t)e[7] << 16)};
}

template <typename T, bool W4>
__global__ void __launch_bounds__(256) grouped_general_kernel(Grouped g, int tiles_n, int wide) {
    __shared__ __attribute__((aligned(16))) uint16_t Xs[kGenTile * kGenK], Ws[kGenTile * kGenK];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave >> 1, wn = wave & 1, lrow = lane & 15, lgrp = lane >> 4;
    const int tn = blockIdx.x % tiles_n;
    const ExpertTile t = expert_tile(g, blockIdx.x / tiles_n, kGenTile, lane);
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
    int wr[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int p = t.begin + row0 + 32 * i;
        const int r = p < t.end ? source_row(g, p) : -1;
        xr[i] = r < 0 ? nullptr : g.x + (int64_t)r * g.x_stride;
        wr[i] = weight_row(row0 + 32 * i);
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

    const int64_t ew = (int64_t)t.e * g.w_stride;
    const int groups = W4 ? g.K / g.group : 0;
    for (int k0 = 0; k0 < g.K; k0 += kGenK) {
        u32x4 a[2], b[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int left = g.K - k0 - 8 * ch;
            a[i] = xr[i] ? load_guarded(xr[i] + k0 + 8 * ch, left, wide & 1) : u32x4{0, 0, 0, 0};
            if constexpr (!W4)
                b[i] = wr[i] >= 0 ? load_guarded(static_cast<const uint16_t*>(g.w) + ew + (int64_t)wr[i] * g.K + k0 + 8 * ch,
                                                 left, wide & 2)
                                  : u32x4{0, 0, 0, 0};
        }
        if constexpr (W4) {
            const int k = k0 + 16 * (tid & 3);
            uint64_t q = 0x8888888888888888ull;
            int z = 8;
            if (crow >= 0 && k < g.K) {
                q = *reinterpret_cast<const uint64_t*>(static_cast<const uint8_t*>(g.w) + ew + (int64_t)crow * (g.K / 2) + k / 2);
                if (g.zeros) z = g.zeros[((int64_t)t.e * g.N + crow) * groups + k / g.group];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int lo = (int)(q >> (32 * i + 8 * j)) & 15, hi = (int)(q >> (32 * i + 8 * j + 4)) & 15;
                    b[i][j] = elem<T>::from_f32((float)(lo - z)) | ((uint32_t)elem<T>::from_f32((float)(hi - z)) << 16);
                }
        }
        __syncthreads();  // the step before is read
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            *reinterpret_cast<u32x4*>(&Xs[slot(row0 + 32 * i, ch)]) = a[i];
            if constexpr (W4) *reinterpret_cast<u32x4*>(&Ws[slot(tid >> 2, 2 * (tid & 3) + i)]) = b[i];
            else *reinterpret_cast<u32x4*>(&Ws[slot(row0 + 32 * i, ch)]) = b[i];
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            u32x4 fa[2], fb[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                fa[i] = *reinterpret_cast<const u32x4*>(&Xs[slot(wm * 32 + i * 16 + lrow, kk * 4 + lgrp)]);
                fb[i] = *reinterpret_cast<const u32x4*>(&Ws[slot(wn * 32 + i * 16 + lrow, kk * 4 + lgrp)]);
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
    }

    float bias[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) bias[j] = (g.epi & kEpiBias) && col[j] >= 0 ? g.bias[(int64_t)t.e * g.N + col[j]] : 0.f;
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
                if (col[0] >= 0) y[col[0]] = elem<T>::from_f32(relu ? fmaxf(v0, 0.f) : v0);
                if (col[1] >= 0) y[col[1]] = elem<T>::from_f32(relu ? fmaxf(v1, 0.f) : v1);
            }
        }
}

}  // namespace pyc

extern "C" int pyc_hip_grouped_stream_takes(int w4, const pyc_grouped* g);
extern "C" int pyc_hip_grouped_stream_launch(int is_bf16, int w4, const pyc_grouped* g, void* stream);

extern "C" int pyc_hip_grouped_launch(int is_bf16, int w4, const pyc_grouped* gp, void* stream) {
    using namespace pyc;
    const Grouped& g = *gp;
    if ((int64_t)g.P <= 16 * (int64_t)g.E && pyc_hip_grouped_stream_takes(w4, gp)) return pyc_hip_grouped_stream_launch(is_bf16, w4, gp, stream);
    const int cols = g.epi & kEpiGate ? g.N / 2 : g.N, per = g.epi & kEpiGate ? kGenTile / 2 : kGenTile;
    const int tiles_n = (cols + per - 1) / per;
    const int64_t tiles = expert_tiles_most(g.offsets ? g.E : 1, g.P, kGenTile) * tiles_n;
    if (tiles > 0x7FFFFFFF) return -1;
    const int wide = (g.x_stride % 8 == 0 && ((uintptr_t)g.x & 15) == 0 ? 1 : 0) |
                     (g.K % 8 == 0 && g.w_stride % 8 == 0 && ((uintptr_t)g.w & 15) == 0 ? 2 : 0);
    const dim3 grid((unsigned)tiles), block(256);
    const hipStream_t s = (hipStream_t)stream;
#define PYC_GENERAL(TY, W) hipLaunchKernelGGL((grouped_general_kernel<TY, W>), grid, block, 0, s, g, tiles_n, wide)
    if (w4) {
        if (is_bf16) PYC_GENERAL(bf16_t, true);
        else PYC_GENERAL(f16_t, true);
    } else {
        if (is_bf16) PYC_GENERAL(bf16_t, false);
        else PYC_GENERAL(f16_t, false);
    }
#undef PYC_GENERAL
    return hipGetLastError() == hipSuccess ? 0 : -2;
}

extern "C" int pyc_hip_kinfo_grouped(int w4, int is_bf16, pyc_hip_kinfo* out) {
    using namespace pyc;
    if (!out) return -1;
    out->fn = w4 ? (is_bf16 ? reinterpret_cast<const void*>(&grouped_general_kernel<bf16_t, true>)
                            : reinterpret_cast<const void*>(&grouped_general_kernel<f16_t, true>))
                 : (is_bf16 ? reinterpret_cast<const void*>(&grouped_general_kernel<bf16_t, false>)
                            : reinterpret_cast<const void*>(&grouped_general_kernel<f16_t, false>));
    out->name = "grouped_general_kernel";
    out->lds_bytes = 2 * kGenTile * kGenK * 2;
    out->threads = 256;
    out->waves_per_simd = 8;
    return 0;
}
