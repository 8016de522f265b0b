// grouped_ring.hip — products by expert of some tens of rows, 16-bit weights: too many rows to
// stream W past them, too few tiles of 256 x 256 to fill the CUs.
//
// 64 rows of one expert x 64 FN rows of its W per workgroup, four waves side by side (64 rows x
// 16 FN columns each), K in stages of 64 through a ring in LDS that LDS-DMA fills, two workgroups
// to a CU. One barrier a stage: after it the stage is there for all waves, and the one before
// it is free for the loads that go out next. What bounds it is the stream of W where experts
// are many, else the stage: its barrier, fragment reads and loads (about 0.2 us). Tiles of up to 32
// and 16 rows multiply that many only. 32 tokens by 8 of 64 experts of 2048 x 2816: 133 us, 5.6 TB/s; 700 by 8 of
// 64 of 1408 x 2040: 93 us; one token by 4 of 32 of 2048 x 2048: 8.7 us. (Each XCD a contiguous eighth of the
// tiles, so that x is read into one L2 instead of eight: 130 and 100 us, not kept.) Gather, ends and the gate as in grouped_tile.hip.
#include <type_traits>

#include "grouped.hpp"
#include "lds_dma.hpp"

namespace pyc {

constexpr int kRingRows = 64, kRingK = 64;
constexpr uint32_t kRingPastEnd = 0xFFFFFFF0u;
constexpr int ring_stage_bytes(int fn) { return (kRingRows + 64 * fn) * kRingK * 2; }
constexpr int ring_stages(int fn) { return fn == 1 ? 5 : 3; }

template <typename T, int FN, bool GATE>
__global__ void __launch_bounds__(256, 2) grouped_ring_kernel(Grouped g, int tiles_n, int wide, uint32_t tile0) {
    constexpr int BN = 64 * FN, S = ring_stages(FN);
    constexpr uint32_t STAGE = ring_stage_bytes(FN), A_BYTES = kRingRows * kRingK * 2;
    constexpr int LA = 2, LB = 2 * FN, LOADS = LA + LB;  // 1 KB loads to a wave and stage
    constexpr int YC = GATE ? 8 * FN : 16 * FN;          // columns of y to a wave
    __shared__ __attribute__((aligned(1024))) uint8_t smem[S * STAGE];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lrow = lane & 15, lgrp = lane >> 4;
    const int F = GATE ? g.N / 2 : g.N;
    const uint32_t tile = tile0 + blockIdx.x;
    const ExpertTile t = expert_tile(g, tile / tiles_n, kRingRows, lane);
    if (t.e < 0) return;
    const int rows = min(t.end - t.begin, kRingRows);
    const int col0 = (int)(tile % tiles_n) * (GATE ? BN / 2 : BN);
    // the row of W in slot c of the tile (-1: none): a wave's 16 FN; gated, half gates and then their values
    auto weight_row = [&](int c) __attribute__((always_inline)) {
        if constexpr (GATE) {
            const int y = col0 + c / (2 * YC) * YC + c % YC;
            return y < F ? y + (c / YC & 1) * F : -1;
        } else {
            return col0 + c < F ? col0 + c : -1;
        }
    };
    const i32x4 a_rsrc = make_buf_rsrc(g.x, (uint32_t)(((int64_t)(g.x_rows - 1) * g.x_stride + g.K) * 2));
    const i32x4 b_rsrc = make_buf_rsrc(static_cast<const uint16_t*>(g.w) + (int64_t)t.e * g.w_stride, (uint32_t)g.N * (uint32_t)g.K * 2u);
    const uint32_t lds0 = (uint32_t)(uintptr_t)smem;
    const int steps = (g.K + kRingK - 1) / kRingK;
    // load q of a stage fills 8 LDS rows of 128 bytes: row 8 q + lane / 8, chunk lane % 8 holding (lane % 8) ^ (row % 8)
    const int lch = (lane & 7) ^ (lane >> 3);
    uint32_t voff[LOADS];
#pragma unroll
    for (int i = 0; i < LB; ++i) {
        const int n = weight_row(8 * (LB * wave + i) + lane / 8);
        voff[LA + i] = n < 0 ? kRingPastEnd : ((uint32_t)n * (uint32_t)g.K + 8 * lch) * 2u;
    }
#pragma unroll
    for (int i = 0; i < LA; ++i) {
        const int p = t.begin + 8 * (LA * wave + i) + lane / 8;
        // a wave without rows does not wait for an index
        const int r = t.begin + 8 * LA * wave < t.end ? source_row(g, p, t.end) : -1;
        voff[i] = r < 0 ? kRingPastEnd : (uint32_t)((int64_t)r * g.x_stride * 2) + 16 * lch;
    }
#pragma unroll
    for (int i = 0; i < LOADS; ++i) asm volatile("" : "+v"(voff[i]));  // complete before the first load goes out
    auto issue = [&](int s, int slot) __attribute__((always_inline)) {
        const bool in = s * kRingK + 8 * lch < g.K;  // stages behind the last read nothing
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const uint32_t lds = lds0 + (uint32_t)slot * STAGE + (i < LA ? (uint32_t)(LA * wave + i) * 1024 : A_BYTES + (uint32_t)(LB * wave + i - LA) * 1024);
            lds_dma_buf_b128_u(i < LA ? a_rsrc : b_rsrc, in ? voff[i] : kRingPastEnd, (uint32_t)s * (kRingK * 2), lds);
        }
    };
#pragma unroll
    for (int s = 0; s < S - 1; ++s) issue(s, s);

    auto run_tile = [&](auto fm) __attribute__((always_inline)) {
        constexpr int FM = decltype(fm)::value;
        f32x4 acc[FM][FN];
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        int slot = 0, into = S - 1;
#pragma unroll 1
        for (int s = 0; s < steps; ++s) {
            wait_vmem_le<(S - 2) * LOADS>();
            __syncthreads();  // stage s has landed for all, stage s - 1 has been read by all
            issue(s + S - 1, into);
            const uint16_t* const A = reinterpret_cast<const uint16_t*>(smem + slot * STAGE);
            const uint16_t* const B = A + A_BYTES / 2;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int pc = ((h * 4 + lgrp) ^ (lrow & 7)) * 8;
                u32x4 a[FM], b[FN];
#pragma unroll
                for (int i = 0; i < FM; ++i) a[i] = *reinterpret_cast<const u32x4*>(A + (16 * i + lrow) * kRingK + pc);
#pragma unroll
                for (int j = 0; j < FN; ++j) b[j] = *reinterpret_cast<const u32x4*>(B + (16 * (FN * wave + j) + lrow) * kRingK + pc);
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < FN; ++j) acc[i][j] = mfma16x16x32(a[i], b[j], acc[i][j], T{});
            }
            into = slot;
            slot = slot == S - 1 ? 0 : slot + 1;
        }
        wait_vmem_le<0>();
        __syncthreads();  // the ring is free: results go through it

        const ExpertBias expert_bias(g, t.e);
        float bias[FN];
#pragma unroll
        for (int j = 0; j < FN; ++j) bias[j] = expert_bias[weight_row(16 * (FN * wave + j) + lrow)];
        const bool relu = g.epi & kEpiRelu;
        constexpr int PITCH = 4 * YC + 8;  // all waves' columns of a row
        uint16_t* const out = reinterpret_cast<uint16_t*>(smem);
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < (GATE ? 1 : FN); ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float v = acc[i][j][r] + bias[j];
                    // gated: the value is in the other fragment, or eight lanes on
                    if constexpr (GATE) v = silu_gate(v, FN == 2 ? acc[i][FN - 1][r] + bias[FN - 1] : row_half_turn(v));
                    else if (relu) v = relu_of(v);
                    if (!GATE || FN == 2 || lrow < 8)
                        out[(16 * i + 4 * lgrp + r) * PITCH + wave * YC + 16 * j + lrow] = elem<T>::from_f32(v);
                }
        __syncthreads();
        constexpr int CH = 4 * YC / 8;
        for (int q = tid; q < rows * CH; q += 256) {
            const int r = q / CH, ch = q % CH, col = col0 + 8 * ch;
            if (col >= F) continue;
            const u32x4 v = *reinterpret_cast<const u32x4*>(out + r * PITCH + 8 * ch);
            uint16_t* const y = g.y + (int64_t)(t.begin + r) * g.y_stride + col;
            if (wide && col + 8 <= F) {
                *reinterpret_cast<u32x4*>(y) = v;
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (col + k < F) y[k] = (uint16_t)(v[k >> 1] >> (16 * (k & 1)));
            }
        }
    };
    if (rows > 32) run_tile(std::integral_constant<int, 4>{});
    else if (rows > 16) run_tile(std::integral_constant<int, 2>{});
    else run_tile(std::integral_constant<int, 1>{});
}

}  // namespace pyc

// fn: 1 or 2
extern "C" int pyc_hip_grouped_ring_launch(int is_bf16, const pyc_grouped* gp, int fn, void* stream) {
    using namespace pyc;
    const Grouped& g = *gp;
    const bool gate = g.epi & kEpiGate;
    const int cols = gate ? g.N / 2 : g.N, per = gate ? 32 * fn : 64 * fn;
    const int tiles_n = (cols + per - 1) / per;
    const int64_t tiles = expert_tiles_most(g.offsets ? g.E : 1, g.P, kRingRows) * tiles_n;
    const int wide = ((uintptr_t)g.y & 15) == 0 && (g.P == 1 || g.y_stride % 8 == 0);
    const hipStream_t s = (hipStream_t)stream;
    return grouped_launches(tiles, 256, [&](uint32_t tile0, dim3 grid) {
#define PYC_RING(TY, FN, GATE) hipLaunchKernelGGL((grouped_ring_kernel<TY, FN, GATE>), grid, dim3(256), 0, s, g, tiles_n, wide, tile0)
#define PYC_RING_TYPE(TY)                         \
    if (gate && fn == 2) PYC_RING(TY, 2, true);   \
    else if (gate) PYC_RING(TY, 1, true);         \
    else if (fn == 2) PYC_RING(TY, 2, false);     \
    else PYC_RING(TY, 1, false)
        if (is_bf16) PYC_RING_TYPE(bf16_t);
        else PYC_RING_TYPE(f16_t);
#undef PYC_RING_TYPE
#undef PYC_RING
    });
}

// The form of 64 columns.
extern "C" int pyc_hip_kinfo_grouped_ring(int is_bf16, pyc_hip_kinfo* out) {
    using namespace pyc;
    out->fn = is_bf16 ? reinterpret_cast<const void*>(&grouped_ring_kernel<bf16_t, 1, false>)
                      : reinterpret_cast<const void*>(&grouped_ring_kernel<f16_t, 1, false>);
    out->name = "grouped_ring_kernel";
    out->lds_bytes = (size_t)ring_stages(1) * ring_stage_bytes(1);
    out->threads = 256;
    out->waves_per_simd = 2;
    return 0;
}
