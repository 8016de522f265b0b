// grouped_w4_tile.hip — products of many rows with 4-bit weights, dense or by expert.
//
// 128 rows of one expert x 256 rows of its W per tile, eight waves of 64 x 64 (two to a SIMD: one
// unpacks or scales while the other multiplies), K in steps of 128. x, codes, scales and
// zero points of a step come by LDS-DMA into a ring of three, so that two steps are on their way
// while one is used, and no wait for one kind of load drains the others. The formula is the one of
// grouped_stream.hip: a code goes into the mantissa of 16, and the groups' sums are
//   sum_g scale_g (sum x (16 + code)) - sum_g scale_g (16 + zero_g) (sum x),
// with sum x from products by ones. The second part is a product itself, over groups: a matrix
// instruction in fp32 takes four groups of it, in place of a vector instruction for each result
// and group (groups of 32 690 -> 663 us, of 64 536 -> 514, of 128 448 -> 444; 2048 x 11008 x 8192). Weights are
// never rounded, which costs a second set of sums, a vector instruction for each result and group, and the sums of x,
// a fifth of the matrix instructions. What bounds it: both kinds of instructions, about half of the cycles each at the
// 2.0 GHz that the card holds under them, which overlap little (a barrier a step keeps the two waves of a SIMD in
// phase), and the ends of tiles, 10 us each, where all loads and stores are waited for.
// 1999 x 11008 x 4096 with groups of 128: 222 to 238 us over cards, 0.76 to 0.81 PFLOP/s (groups of 64 1.18 times that,
// of 32 1.55 times). Measured and not kept: scaling a group among the next one's products (239); the two waves of a SIMD half a
// step apart, which leaves loads one step instead of two (241); two workgroups of 64 rows a CU (267).
//
// Scales and zero points are 2-byte and 1-byte values at any alignment, LDS-DMA moves aligned
// dwords: the dwords that hold a row's values of the step are fetched (1 to 3, 1 or 2), and the
// values shifted out of them.
//
// The 128 x 256 form's registers are full: 8 to 26 values of a tile's start and end lie in scratch, none of the loop over K.
#include <type_traits>

#include "grouped.hpp"
#include "lds_dma.hpp"

namespace pyc {

constexpr int kW4K = 128;
constexpr uint32_t kW4PastEnd = 0xFFFFFFF0u;
constexpr int w4_scale_dwords(int g) { return g == 128 ? 1 : g == 64 ? 2 : 3; }
constexpr int w4_zero_dwords(int g) { return g == 128 ? 1 : 2; }
// A tile: 16 FM rows to a wave, WM waves of them; four waves of 16 FN columns. A step in LDS: x, codes, dwords
// of scales and zero points; as many steps as leave room for a second workgroup (of four waves)
constexpr uint32_t w4_x_bytes(int wm, int fm) { return (uint32_t)wm * fm * 16 * kW4K * 2; }
constexpr uint32_t w4_code_bytes(int fn) { return (uint32_t)64 * fn * kW4K / 2; }
constexpr uint32_t w4_step_bytes(int g, int wm, int fn, int fm) {
    return w4_x_bytes(wm, fm) + w4_code_bytes(fn) + (uint32_t)(w4_scale_dwords(g) + w4_zero_dwords(g)) * 64 * fn * 4;
}
constexpr int w4_steps(int g, int wm, int fn, int fm) {
    const int n = (int)((wm == 1 ? 80 : 160) * 1024 / w4_step_bytes(g, wm, fn, fm));
    return n < 8 ? n : 8;
}

// lane i's 4 bytes at offset voff land at lds_base + 4 * i
__device__ inline void lds_dma_buf_b32(i32x4 rsrc, uint32_t voff, uint32_t lds_base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
                 :
                 : "s"(lds_base), "v"(voff), "s"(rsrc)
                 : "memory", "m0");
}

template <typename T, int G, bool GATE, int WM, int FN, int FMX>
__global__ void __launch_bounds__(256 * WM, 2) grouped_w4_tile_kernel(Grouped g, int tiles_n, int wide) {
    constexpr int NW = 4 * WM, ROWS = 16 * WM * FMX, COLS = 64 * FN;
    constexpr int NG = kW4K / G;                                   // groups to a step
    constexpr int NS = w4_scale_dwords(G), NZ = w4_zero_dwords(G);
    constexpr int CL = FN / WM;                                    // loads of codes to a wave and step
    constexpr int DW = FN * (NS + NZ), SZ = (DW + NW - 1) / NW;    // loads of dwords in all, to a wave
    constexpr uint32_t X_BYTES = w4_x_bytes(WM, FMX), CODE_BYTES = w4_code_bytes(FN);
    constexpr uint32_t STEP = w4_step_bytes(G, WM, FN, FMX);
    constexpr int S = w4_steps(G, WM, FN, FMX);
    constexpr int YC = GATE ? 8 * FN : 16 * FN;                    // columns of y to a wave
    constexpr int PITCH = 4 * YC + 8;                              // results in LDS: a row of all waves' columns
    static_assert(CL * WM == FN && S >= 3 && (uint32_t)(ROWS * PITCH * 2) <= S * STEP, "tile shape");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[S * STEP];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 2, wn = wave & 3;
    const int lrow = lane & 15, lgrp = lane >> 4;
    const int F = GATE ? g.N / 2 : g.N, groups = g.K / G;
    const int steps = (g.K + kW4K - 1) / kW4K;
    const uint32_t lds0 = (uint32_t)(uintptr_t)smem;
    const i32x4 x_rsrc = make_buf_rsrc(g.x, (uint32_t)(((int64_t)(g.x_rows - 1) * g.x_stride + g.K) * 2));

    // row tiles there are
    int row_tiles = 0;
    if (g.offsets) {
        int held = 0;
        for (int e0 = 0; e0 < g.E; e0 += kWave) {
            const int e = e0 + lane;
            const int b = scan_max(max(held, min(g.offsets[min(e, g.E)], g.P)));
            const int end = max(b, min(g.offsets[min(e + 1, g.E)], g.P));
            row_tiles += __builtin_amdgcn_readlane(scan_add((end - b + ROWS - 1) / ROWS), kWave - 1);
            held = __builtin_amdgcn_readlane(end, kWave - 1);
        }
    } else {
        row_tiles = (g.P + ROWS - 1) / ROWS;
    }
    // XCD x (workgroups b with b % 8 == x) has the x-th eighth of the tiles
    const int64_t all = (int64_t)row_tiles * tiles_n;
    const int xcd = blockIdx.x & 7, per = gridDim.x >> 3;
    const int t_end = __builtin_amdgcn_readfirstlane((int)(all * (xcd + 1) / 8));
    int t = __builtin_amdgcn_readfirstlane((int)(all * xcd / 8) + (int)(blockIdx.x >> 3));

    for (; t < t_end; t += per) {
        const ExpertTile et = expert_tile(g, t / tiles_n, ROWS, lane);
        if (et.e < 0) break;
        const int e = __builtin_amdgcn_readfirstlane(et.e), row0 = __builtin_amdgcn_readfirstlane(et.begin);
        const int end = __builtin_amdgcn_readfirstlane(et.end);
        const int col0 = (t - t / tiles_n * tiles_n) * (GATE ? COLS / 2 : COLS);
        // the row of W in slot c of the tile, -1: none. A wave has 16 FN slots; gated, half gates and then the
        // values of the same columns.
        auto weight_row = [&](int c) __attribute__((always_inline)) {
            if constexpr (GATE) {
                const int y = col0 + c / (2 * YC) * YC + c % YC;
                return y < F ? y + (c / YC & 1) * F : -1;
            } else {
                return col0 + c < F ? col0 + c : -1;
            }
        };
        const char* const codes = static_cast<const char*>(g.w) + (int64_t)e * g.w_stride;
        const i32x4 w_rsrc = make_buf_rsrc(codes, (uint32_t)((int64_t)g.N * (g.K / 2)));
        const uintptr_t sa = (uintptr_t)(g.scale + (int64_t)e * g.N * groups);
        const uintptr_t za = (uintptr_t)(g.zeros ? g.zeros + (int64_t)e * g.N * groups : nullptr);
        const uint32_t s_mis = (uint32_t)(sa & 3) / 2, z_mis = (uint32_t)(za & 3);
        const i32x4 s_rsrc = make_buf_rsrc((const void*)(sa & ~(uintptr_t)3), ((uint32_t)(g.N * groups) * 2 + 2 * s_mis + 3) & ~3u);
        const i32x4 z_rsrc = make_buf_rsrc((const void*)(za & ~(uintptr_t)3), g.zeros ? ((uint32_t)(g.N * groups) + z_mis + 3) & ~3u : 0u);

        auto run_tile = [&](auto fm) __attribute__((always_inline)) {
            constexpr int FM = decltype(fm)::value;  // fragments of rows to a wave
            constexpr int LOADS = FM + CL + SZ;       // to a wave and step
            // x: load i of a wave has rows 4 (NW i + wave) + lane / 16, chunk lane % 16 holding logical chunk
            // (lane % 16) ^ (row % 16); codes: load i rows 16 (CL wave + i) + lane / 4, chunk lane % 4
            // holding (lane % 4) ^ (row / 4 % 4)
            uint32_t xo[FM], co[CL], so[SZ];
            const int xk = 8 * ((lane & 15) ^ ((4 * wave + lane / 16) & 15));  // first k of the lane's chunk
            const int ck = 32 * ((lane & 3) ^ ((lane >> 4) & 3));
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                const int p = row0 + 4 * (NW * i + wave) + lane / 16;
                const int s = source_row(g, p, end);
                xo[i] = s < 0 ? kW4PastEnd : (uint32_t)((int64_t)s * g.x_stride * 2) + 2 * xk;
            }
#pragma unroll
            for (int i = 0; i < CL; ++i) {
                const int n = weight_row(16 * (CL * wave + i) + lane / 4);
                co[i] = n < 0 ? kW4PastEnd : (uint32_t)n * (uint32_t)(g.K / 2) + ck / 2;
            }
            // dword load q: slots 64 (q % FN) + lane, dword q / FN, scales first; one too many is the last again
#pragma unroll
            for (int i = 0; i < SZ; ++i) {
                const int q = min(wave * SZ + i, DW - 1);
                const int n = weight_row(64 * (q % FN) + lane);
                so[i] = n < 0 ? kW4PastEnd : (uint32_t)n * (uint32_t)groups + (q < FN * NS ? s_mis : z_mis);
            }
#pragma unroll
            for (int i = 0; i < FM; ++i) asm volatile("" : "+v"(xo[i]));  // complete before the first load goes out
#pragma unroll
            for (int i = 0; i < CL; ++i) asm volatile("" : "+v"(co[i]));
#pragma unroll
            for (int i = 0; i < SZ; ++i) asm volatile("" : "+v"(so[i]));
            // load i of a wave for step s
            auto issue = [&](int i, int s, int slot) __attribute__((always_inline)) {
                const uint32_t base = lds0 + (uint32_t)slot * STEP;
                const int left = g.K - s * kW4K;  // k from this step on
                if (i < FM) {
                    lds_dma_buf_b128_u(x_rsrc, xk < left ? xo[i < FM ? i : 0] : kW4PastEnd, (uint32_t)s * (kW4K * 2),
                                       base + (uint32_t)(NW * i + wave) * 1024);
                } else if (i < FM + CL) {
                    const int j = i - FM;
                    lds_dma_buf_b128_u(w_rsrc, ck < left ? co[j < CL ? j : 0] : kW4PastEnd, (uint32_t)s * (kW4K / 2),
                                       base + X_BYTES + (uint32_t)(CL * wave + j) * 1024);
                } else {
                    const int j = i - FM - CL, q = min(wave * SZ + j, DW - 1);
                    const bool zero = q >= FN * NS;
                    const uint32_t o = so[j < SZ ? j : 0], a = o + (uint32_t)(s * NG);  // the first value's place
                    const uint32_t off = zero ? ((a >> 2) + (uint32_t)(q / FN - NS)) * 4 : ((a >> 1) + (uint32_t)(q / FN)) * 4;
                    lds_dma_buf_b32(zero ? z_rsrc : s_rsrc, o == kW4PastEnd ? kW4PastEnd : off,
                                    __builtin_amdgcn_readfirstlane(base + X_BYTES + CODE_BYTES + (uint32_t)q * 256));
                }
            };

            f32x4 acc[FM][FN], part[FM][FN], sum[FM];
            constexpr int NV = NG > 2 ? 2 : 1, HALVES = GATE && FN > 1 ? 2 : 1;
            u32x4 fa[2][FM], cw[FN];
            uint32_t sv[FN][NV], zv[FN];
            // how far into its dword a slot's first scale and zero point of step 0 stand, in bits (above the lowest five:
            // whole dwords). Slots 16 rows of W apart agree; gated, a wave's gates do and its values do.
            uint32_t sp[HALVES], zp[HALVES];
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
                const int n = max(weight_row(16 * FN * wn + YC * h + lrow), 0);
                sp[h] = ((uint32_t)n * (uint32_t)groups + s_mis) * 16;
                zp[h] = ((uint32_t)n * (uint32_t)groups + z_mis) * 8;
            }
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int i = 0; i < FM; ++i) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            auto read_x = [&](int b, int slot, int ks) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < FM; ++i)
                    fa[b][i] = *reinterpret_cast<const u32x4*>(smem + slot * STEP + ((wm * FM + i) * 16 + lrow) * 256 +
                                                               (((ks * 4 + lgrp) ^ lrow) << 4));
            };
            // a step's codes, scales and zero points, the latter as the step's values from the lowest bits on
            auto read_w = [&](int s, int slot) __attribute__((always_inline)) {
                const uint8_t* const c = smem + slot * STEP + X_BYTES + (16 * FN * wn + lrow) * 64 + ((lgrp ^ ((lrow >> 2) & 3)) << 4);
                const uint32_t* const d = reinterpret_cast<const uint32_t*>(smem + slot * STEP + X_BYTES + CODE_BYTES) + 16 * FN * wn + lrow;
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    cw[j] = *reinterpret_cast<const u32x4*>(c + j * 1024);
                    const int h = j * HALVES / FN;
                    const uint32_t ss = sp[h] + (uint32_t)(s * NG * 16), zs = zp[h] + (uint32_t)(s * NG * 8);  // alignbit takes five bits
                    const uint32_t d0 = d[16 * j], d1 = NS > 1 ? d[COLS + 16 * j] : 0;
                    sv[j][0] = __builtin_amdgcn_alignbit(d1, d0, ss);
                    if constexpr (NS > 2) sv[j][NV - 1] = __builtin_amdgcn_alignbit(d[2 * COLS + 16 * j], d1, ss);
                    const uint32_t z0 = d[NS * COLS + 16 * j], z1 = NZ > 1 ? d[(NS + 1) * COLS + 16 * j] : 0;
                    zv[j] = __builtin_amdgcn_alignbit(z1, z0, zs);
                }
            };

#pragma unroll
            for (int s = 0; s < S - 1; ++s)
#pragma unroll
                for (int i = 0; i < LOADS; ++i) issue(i, s, s);
            wait_vmem_le<(S - 2) * LOADS>();
            __syncthreads();
            read_x(0, 0, 0);
            read_w(0, 0);
            const u32x4 one = [] {
                const uint32_t o = elem<T>::from_f32(1.0f) * 0x10001u;
                return u32x4{o, o, o, o};
            }();
            uint32_t mask = codes16_mask(T{}), base = elem<T>::from_f32(16.0f) * 0x10001u;
            asm volatile("" : "+v"(mask), "+v"(base));  // in registers: and-or takes one constant at most
            // sums of x (lane: row lrow) and scales times -(16 + zero) of the last four groups, one to a lane group
            float sa[FM], sb[FN];
#pragma unroll
            for (int i = 0; i < FM; ++i) sa[i] = 0.f;
#pragma unroll
            for (int j = 0; j < FN; ++j) sb[j] = 0.f;
            auto zero_points = [&]() __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(sa[i], sb[j], acc[i][j], 0, 0, 0);
            };
            int slot = 0, into = S - 1;
#pragma unroll 1
            for (int s = 0; s < steps; ++s) {
                const int next = slot == S - 1 ? 0 : slot + 1;
#pragma unroll
                for (int j = 0; j < FN; ++j) transpose4(cw[j]);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) {
                    const bool first = ks % (G / 32) == 0, last = (ks + 1) % (G / 32) == 0;
                    float f[FN], fz[FN];
                    uint32_t c[FN];
#pragma unroll
                    for (int j = 0; j < FN; ++j) {
                        const int q = ks / (G / 32);
                        const bool there = NG == 1 || s * NG + q < groups;  // what lies behind the row is another's
                        f[j] = there ? elem<T>::to_f32((uint16_t)(sv[j][q < 2 ? 0 : NV - 1] >> (16 * (q & 1)))) : 0.f;
                        fz[j] = f[j] * (-16.0f - (g.zeros ? (float)((zv[j] >> (8 * q)) & 255u) : 8.0f));
                        c[j] = cw[j][ks];
                    }
                    if (ks < 3) {
                        read_x((ks + 1) & 1, slot, ks + 1);
                    } else {
                        // the next step has landed, and this one has been read by all
                        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                        wait_vmem_le<(S - 2) * LOADS>();
                        __syncthreads();
                        read_x(0, next, 0);
                        read_w(s + 1, next);
                    }
                    if (first) {
#pragma unroll
                        for (int i = 0; i < FM; ++i) {
                            sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                            for (int j = 0; j < FN; ++j) part[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
                        }
                    }
#pragma unroll
                    for (int i = 0; i < FM; ++i) sum[i] = mfma16x16x32(one, fa[ks & 1][i], sum[i], T{});
#pragma unroll
                    for (int j = 0; j < FN; ++j) {
                        const u32x4 w = codes16(c[j], mask, base, T{});
#pragma unroll
                        for (int i = 0; i < FM; ++i) part[i][j] = mfma16x16x32(fa[ks & 1][i], w, part[i][j], T{});
                        // the loads of the step that takes the place of the one before, a few between the products
                        if (ks < 3) {
                            constexpr int PLACES = 3 * FN;
                            const int q = ks * FN + j;
#pragma unroll
                            for (int i = q * LOADS / PLACES; i < (q + 1) * LOADS / PLACES; ++i) issue(i, s + S - 1, into);
                        }
                    }
                    if (last) {
                        const int turn = (s * NG + ks / (G / 32)) & 3;
#pragma unroll
                        for (int j = 0; j < FN; ++j) {
                            sb[j] = lgrp == turn ? fz[j] : sb[j];
#pragma unroll
                            for (int i = 0; i < FM; ++i)
#pragma unroll
                                for (int r = 0; r < 4; ++r) acc[i][j][r] = fmaf(f[j], part[i][j][r], acc[i][j][r]);
                        }
#pragma unroll
                        for (int i = 0; i < FM; ++i) sa[i] = lgrp == turn ? sum[i][0] : sa[i];
                        if (turn == 3) zero_points();
                    }
                }
                into = slot;
                slot = next;
            }
            if (const int rest = steps * NG & 3; rest) {
#pragma unroll
                for (int i = 0; i < FM; ++i) sa[i] = lgrp < rest ? sa[i] : 0.f;
#pragma unroll
                for (int j = 0; j < FN; ++j) sb[j] = lgrp < rest ? sb[j] : 0.f;
                zero_points();
            }
            wait_vmem_le<0>();
            __syncthreads();  // the ring is free: results go through it

            const ExpertBias expert_bias(g, e);
            float bias[FN];
#pragma unroll
            for (int j = 0; j < FN; ++j) bias[j] = expert_bias[weight_row(16 * (FN * wn + j) + lrow)];
            const bool relu = g.epi & kEpiRelu;
            uint16_t* const out = reinterpret_cast<uint16_t*>(smem);
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < (YC + 15) / 16; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float v = acc[i][j][r] + bias[j];
                        // gated: the value is FN / 2 fragments on, or eight lanes
                        if constexpr (GATE) v = silu_gate(v, FN > 1 ? acc[i][(j + FN / 2) % FN][r] + bias[(j + FN / 2) % FN] : row_half_turn(v));
                        else if (relu) v = relu_of(v);
                        if (!GATE || FN > 1 || lrow < 8)
                            out[(16 * (wm * FM + i) + 4 * lgrp + r) * PITCH + wn * YC + 16 * j + lrow] = elem<T>::from_f32(v);
                    }
            __syncthreads();
            constexpr int CH = 4 * YC / 8;
            for (int q = tid; q < min(end - row0, ROWS) * CH; q += 64 * NW) {
                const int r = q / CH, ch = q % CH, col = col0 + 8 * ch;
                if (col >= F) continue;
                const u32x4 v = *reinterpret_cast<const u32x4*>(out + r * PITCH + 8 * ch);
                uint16_t* const y = g.y + (int64_t)(row0 + r) * g.y_stride + col;
                if (wide && col + 8 <= F) {
                    *reinterpret_cast<u32x4*>(y) = v;
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (col + k < F) y[k] = (uint16_t)(v[k >> 1] >> (16 * (k & 1)));
                }
            }
            __syncthreads();  // the next tile's loads go into the ring
        };
        const int rows = end - row0;
        if (FMX > 2 && rows > 32 * WM) run_tile(std::integral_constant<int, FMX>{});
        else if (FMX > 1 && rows > 16 * WM) run_tile(std::integral_constant<int, (FMX > 1 ? 2 : 1)>{});
        else run_tile(std::integral_constant<int, 1>{});
    }
}

}  // namespace pyc

extern "C" int pyc_hip_grouped_stream_takes(int w4, const pyc_grouped* g);

// form 0: tiles of 128 rows and 256 columns; 1, 2 and 4: of 16, 32 and 64 rows and 64 columns
extern "C" int pyc_hip_grouped_w4_tile_launch(int is_bf16, const pyc_grouped* gp, int form, void* stream) {
    using namespace pyc;
    const Grouped& g = *gp;
    const bool gate = g.epi & kEpiGate;
    const int cols = gate ? g.N / 2 : g.N, per = (form ? 64 : 256) / (gate ? 2 : 1);
    const int tiles_n = (cols + per - 1) / per;
    if (expert_tiles_most(g.offsets ? g.E : 1, g.P, 16) * tiles_n > 0x7FFF0000) return -1;
    const int wide = ((uintptr_t)g.y & 15) == 0 && (g.P == 1 || g.y_stride % 8 == 0);
    const dim3 grid(form ? 512 : 256), block(form ? 256 : 512);
    const hipStream_t s = (hipStream_t)stream;
#define PYC_W4_FORM(TY, G, FORM, WM, FN, FMX)                                                                                   \
    if (form == FORM) {                                                                                                         \
        if (gate) hipLaunchKernelGGL((grouped_w4_tile_kernel<TY, G, true, WM, FN, FMX>), grid, block, 0, s, g, tiles_n, wide);  \
        else hipLaunchKernelGGL((grouped_w4_tile_kernel<TY, G, false, WM, FN, FMX>), grid, block, 0, s, g, tiles_n, wide);      \
    }
#define PYC_W4_TILE(TY, G)              \
    if (g.group == G) {                 \
        PYC_W4_FORM(TY, G, 0, 2, 4, 4)  \
        PYC_W4_FORM(TY, G, 1, 1, 1, 1)  \
        PYC_W4_FORM(TY, G, 2, 1, 1, 2)  \
        PYC_W4_FORM(TY, G, 4, 1, 1, 4)  \
    }
    if (is_bf16) {
        PYC_W4_TILE(bf16_t, 32)
        PYC_W4_TILE(bf16_t, 64)
        PYC_W4_TILE(bf16_t, 128)
    } else {
        PYC_W4_TILE(f16_t, 32)
        PYC_W4_TILE(f16_t, 64)
        PYC_W4_TILE(f16_t, 128)
    }
#undef PYC_W4_TILE
#undef PYC_W4_FORM
    return hipGetLastError() == hipSuccess ? 0 : -2;
}

// The form of 64 rows and columns, groups of 128.
extern "C" int pyc_hip_kinfo_grouped_w4(int is_bf16, pyc_hip_kinfo* out) {
    using namespace pyc;
    out->fn = is_bf16 ? reinterpret_cast<const void*>(&grouped_w4_tile_kernel<bf16_t, 128, false, 1, 1, 4>)
                      : reinterpret_cast<const void*>(&grouped_w4_tile_kernel<f16_t, 128, false, 1, 1, 4>);
    out->name = "grouped_w4_tile_kernel";
    out->lds_bytes = (size_t)w4_steps(128, 1, 1, 4) * w4_step_bytes(128, 1, 1, 4);
    out->threads = 256;
    out->waves_per_simd = 2;
    return 0;
}
