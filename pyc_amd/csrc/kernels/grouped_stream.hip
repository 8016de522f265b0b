// grouped_stream.hip — products by expert with 4-bit weights where an expert has few rows: single
// tokens and decoding batches. What bounds them is the stream of the weights, every byte of
// which is used once, and with it the waits of the two or three waves a SIMD has for it, between the vector
// instructions that unpack them (a third of the cycles of a token through 4096 x 11008, 40 % of 23 through 11008 x 4096).
//
// A wave has 32 rows of one expert's W (two fragments; gated: of gates, and of the same
// columns' values) and up to 16 rows of x. The eight waves of a workgroup take `ks` parts of
// K for 8 / ks such column blocks: parts of the same columns take every ks-th chunk of 128 k
// and are added up through LDS, in order, so that few columns still fill the CUs without a
// second launch. W goes from memory into registers as the operand it is, several chunks ahead,
// through buffer descriptors: rows and k past the end read zeros and cost no traffic.
//
// With x, scales and zero points loaded beside W a wave took 3700 cycles for a chunk and its 10 loads (one token
// through 4096 x 11008: 19 us). So a wave loads W alone: the rows of x
// and the scales and zero points of the workgroup's columns go through LDS, as much of K at a
// time as fits. Where x would take turns (each stops all waves), only the scales do, and x is
// loaded beside W (23 tokens, 11008 x 4096: 42 us in turns, 25 beside).
//
// One token through 4096 x 11008: 10.9 us (85 by the general kernel); 16 tokens by 4 of 32 experts of 4096 x 2816:
// 50 us, 3.9 TB/s (218). 23 tokens, 11008 x 4096, groups of 32: 25 us, 11 of them for each half of the depth (two
// workgroups read and unpack W for the two row tiles); 22 with groups of 128. Measured and not kept: x and scales
// loaded four pieces ahead of their way into LDS (12.6 and 56), 16 waves and parts of K (23 tokens, 11008 x 4096: 25 as
// with eight).
//
// The rows of x are the first operand: a lane's results are four rows of one column of y, so
// a column's scale is one value for each lane. A lane's 16 bytes of W are 32 k of a row, the
// four lanes of a row 128 k. A 4 x 4
// transposition between the lanes and their four words (four swaps) gives each product 32
// neighbouring k, so that groups of 32, 64 and 128 all work. A code c goes into the
// mantissa of 16, as 16 + c exactly, two to two instructions; a group's sum is then
//   scale (sum x (16 + c) - (16 + zero) sum x),
// all in fp32, with sum x from one more product by ones. (By conversion to whole numbers less
// zero a pair takes three to four times the instructions.)
#include "grouped.hpp"

namespace pyc {

constexpr int kStreamWaves = 8;
constexpr int kStreamThreads = kStreamWaves * kWave;
constexpr int kStreamK = 128;               // k of a chunk
// LDS: x, then scales and zero points as one word; the sums of the parts of K reuse x's. The smaller of each
// pair keeps two workgroups to a CU; where there are no more workgroups than CUs, one may have it all.
struct StreamLds {
    int x, scales;  // bytes for x, words
};
constexpr StreamLds kStreamLds[2][2] = {{{63 * 1024, 4096}, {111 * 1024, 12032}}, {{16 * 1024, 15872}, {16 * 1024, 36352}}};
constexpr size_t stream_lds_bytes(const StreamLds& l) { return l.x + 4 * l.scales; }
constexpr uint32_t kPastEnd = 0xFFFFFFF0u;  // not below any descriptor's byte count

// G: k of a group. XD: x is loaded beside W. wgs: workgroups that the column blocks take.
template <typename T, int G, bool XD>
__global__ void __launch_bounds__(kStreamThreads, 4)
grouped_stream_kernel(Grouped g, int wgs, int ks, int x_lds, int words, uint32_t wg0) {
    constexpr int CF = 2;
    constexpr int NG = kStreamK / G;       // groups to a chunk
    constexpr int AHEAD = XD ? 2 : 4;      // chunks in registers
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    __shared__ int64_t src[16];
    static_assert(kStreamWaves * CF * kWave * 16 <= kStreamLds[1][0].x, "sums through x's LDS");
    uint32_t* const sz = reinterpret_cast<uint32_t*>(smem + x_lds);  // [group][column of the workgroup]: scale, zero point << 16

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lrow = lane & 15, lgrp = lane >> 4;
    const int units = kStreamWaves / ks;                     // column blocks of the workgroup
    const int kp = wave & (ks - 1), unit = wave / ks;        // this wave's part of K and block
    const uint32_t wg = wg0 + blockIdx.x;
    const int tn0 = (int)(wg % wgs) * units, tn = tn0 + unit;
    const ExpertTile t = expert_tile(g, wg / wgs, 16, lane);
    if (t.e < 0) return;
    const int rows = min(t.end - t.begin, 16);
    const bool gate = g.epi & kEpiGate;
    const int F = gate ? g.N / 2 : g.N;
    // the row of W behind column c (0 .. 31) of block b, g.N: none
    auto weight_row = [&](int b, int c) __attribute__((always_inline)) {
        const int y = gate ? b * 16 + (c & 15) : b * 32 + c;
        return y < F ? (gate && c >= 16 ? y + F : y) : g.N;
    };
    const int chunks = (g.K + kStreamK - 1) / kStreamK;
    const int groups = g.K / G;

    // W: a chunk's place is the scalar part of a load's offset, which the descriptor's check leaves out. So k past
    // K, of the last chunk where K is no multiple of 128 and of all chunks behind it, have lane offsets past the end.
    const uint32_t row_bytes = (uint32_t)g.K / 2;
    void* const wbase = const_cast<char*>(static_cast<const char*>(g.w)) + (int64_t)t.e * g.w_stride;
    const auto wr = __builtin_amdgcn_make_buffer_rsrc(wbase, 0, (uint32_t)g.N * row_bytes, 0x00020000);
    uint32_t wo[CF];
#pragma unroll
    for (int f = 0; f < CF; ++f) {
        const int r = weight_row(tn, 16 * f + lrow);
        wo[f] = r < g.N ? (uint32_t)r * row_bytes + 16 * lgrp : kPastEnd;
    }
    struct Chunk {
        u32x4 w[CF], x[XD ? 4 : 1];
    };
    uint32_t xo = kPastEnd;  // XD: of the lane's row
    uint32_t xbytes = 0;
    if constexpr (XD) {
        const int r = source_row(g, t.begin + lrow, t.begin + rows);
        xo = r < 0 ? kPastEnd : (uint32_t)((int64_t)r * g.x_stride * 2) + 16 * lgrp;
        xbytes = (uint32_t)(((int64_t)(g.x_rows - 1) * g.x_stride + g.K) * 2);
    }
    auto load = [&](Chunk& c, int i) __attribute__((always_inline)) {
        const int end = g.K - i * kStreamK;  // k from this chunk on
#pragma unroll
        for (int f = 0; f < CF; ++f)
            c.w[f] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                   wr, 32 * lgrp < end ? wo[f] : kPastEnd, (uint32_t)i * (kStreamK / 2), 0));
        if constexpr (XD) {
            const auto xr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(g.x), 0, xbytes, 0x00020000);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                c.x[j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                       xr, 32 * j + 8 * lgrp < end ? xo : kPastEnd, (uint32_t)i * (kStreamK * 2) + 64 * j, 0));
        }
    };

    // the first chunks go before x and scales where a wave streams many, behind them where all is over soon (a
    // token through 4096 x 11008: 12.5 and 11.5 us; 16 by 4 of 32 experts, 4096 x 2816: 67 and 70 with 8 parts)
    Chunk c[AHEAD];
    auto load_first = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            __builtin_amdgcn_sched_barrier(0);  // the loop's waits count loads in this order
            load(c[a], kp + a * ks);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    if (ks < kStreamWaves) load_first();

    // As much of K at a time (a power of two of chunks to a wave) as x's rows and the scales leave room for;
    // one is in any case: 16 rows of 8 chunks, 8 chunks' scales of a column block
    int span = kStreamK * ks;
    while (span < g.K && (XD || rows * (2 * span * 2 + 16) <= x_lds) && 2 * span / G * 32 * units <= words) span *= 2;
    const int pitch = min(span, chunks * kStreamK) * 2 + 16;  // bytes of a row of x in LDS
    // element offset of the row of x behind each row of the tile, -1: zeros
    if (!XD && tid < rows) {
        const int r = source_row(g, t.begin + tid, t.end);
        src[tid] = r < 0 ? -1 : (int64_t)r * g.x_stride;
    }
    const uint16_t* const scale = g.scale + (int64_t)t.e * g.N * groups;
    const uint8_t* const zeros = g.zeros ? g.zeros + (int64_t)t.e * g.N * groups : nullptr;
    // four scales to a load where rows of them keep to 8 bytes
    const bool quads = (groups & 3) == 0 && ((uintptr_t)scale & 7) == 0 && ((uintptr_t)zeros & 3) == 0;
    const int columns = 32 * units;
    auto stage = [&](int k0) __attribute__((always_inline)) {
        if constexpr (!XD) {
            const int n = min(span, g.K - k0), padded = min(span, chunks * kStreamK - k0);
            const int shift = __builtin_ctz(span) - 3;  // pieces of 8 to a row
            for (int p = tid; p < rows << shift; p += kStreamThreads) {
                const int r = p >> shift, k = (p - (r << shift)) * 8;
                if (k >= padded) continue;
                const int64_t s = src[r];
                u32x4 v = u32x4{0, 0, 0, 0};
                if (k < n && s >= 0) v = *reinterpret_cast<const u32x4*>(g.x + s + k0 + k);
                *reinterpret_cast<u32x4*>(smem + r * pitch + 2 * k) = v;
            }
        }
        const int gshift = __builtin_ctz(span / G), q0 = k0 / G;
        if (quads) {
            const int qs = gshift > 2 ? gshift - 2 : 0;
            for (int p = tid; p < columns << qs; p += kStreamThreads) {
                const int c = p >> qs, q = (p - (c << qs)) * 4, r = weight_row(tn0 + (c >> 5), c & 31);
                if (q0 + q >= groups || r >= g.N) continue;
                const uint64_t v = *reinterpret_cast<const uint64_t*>(scale + (int64_t)r * groups + q0 + q);
                const uint32_t z = zeros ? *reinterpret_cast<const uint32_t*>(zeros + (int64_t)r * groups + q0 + q) : 0x08080808u;
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (u < 1 << gshift) sz[(q + u) * columns + c] = (uint32_t)(uint16_t)(v >> (16 * u)) | (z >> (8 * u) & 255u) << 16;
            }
        } else {
            for (int p = tid; p < columns << gshift; p += kStreamThreads) {
                const int c = p >> gshift, q = p - (c << gshift), r = weight_row(tn0 + (c >> 5), c & 31);
                if (q0 + q >= groups || r >= g.N) continue;
                const int64_t at = (int64_t)r * groups + q0 + q;
                sz[q * columns + c] = (uint32_t)scale[at] | (zeros ? (uint32_t)zeros[at] : 8u) << 16;
            }
        }
    };

    f32x4 acc[CF];
#pragma unroll
    for (int f = 0; f < CF; ++f) acc[f] = f32x4{0.f, 0.f, 0.f, 0.f};
    uint32_t mask = codes16_mask(T{}), base16 = elem<T>::from_f32(16.0f) * 0x10001u;
    asm volatile("" : "+v"(mask), "+v"(base16));  // in registers: and-or takes one constant at most
    const u32x4 one = [] {
        const uint32_t o = elem<T>::from_f32(1.0f) * 0x10001u;
        return u32x4{o, o, o, o};
    }();
    // chunk i, k0: the first k in LDS. Rows of x that are not there read as the last one's: their results are not stored
    auto multiply = [&](Chunk& c, int i, int k0) __attribute__((always_inline)) {
        const int at = i * kStreamK - k0;
        const uint8_t* const row = smem + min(lrow, rows - 1) * pitch + (at + 8 * lgrp) * 2;
#pragma unroll
        for (int f = 0; f < CF; ++f) transpose4(c.w[f]);
#pragma unroll
        for (int q = 0; q < NG; ++q) {
            f32x4 part[CF], sum = f32x4{0.f, 0.f, 0.f, 0.f};
            float s[CF], z[CF];
#pragma unroll
            for (int f = 0; f < CF; ++f) {
                part[f] = f32x4{0.f, 0.f, 0.f, 0.f};
                // what lies behind the last group was not brought
                const uint32_t v = i * NG + q < groups ? sz[(at / G + q) * columns + 32 * unit + 16 * f + lrow] : 0u;
                s[f] = elem<T>::to_f32((uint16_t)v);
                z[f] = -16.0f - (float)(v >> 16);
            }
#pragma unroll
            for (int j = q * (4 / NG); j < (q + 1) * (4 / NG); ++j) {
                const u32x4 x = XD ? c.x[XD ? j : 0] : *reinterpret_cast<const u32x4*>(row + 64 * j);
                sum = mfma16x16x32(x, one, sum, T{});
#pragma unroll
                for (int f = 0; f < CF; ++f) part[f] = mfma16x16x32(x, codes16(c.w[f][j], mask, base16, T{}), part[f], T{});
            }
#pragma unroll
            for (int f = 0; f < CF; ++f)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[f][r] = fmaf(s[f], fmaf(z[f], sum[r], part[f][r]), acc[f][r]);
        }
    };

    __syncthreads();  // src
    stage(0);
    if (ks == kStreamWaves) load_first();
    __syncthreads();
    // every wave has the same number of turns; chunks behind the last are not multiplied
    const int turns = (chunks + ks - 1) / ks, turns_here = span / (kStreamK * ks);
    int k0 = 0;
#pragma unroll 1
    for (int n = 0; n < turns; n += AHEAD) {
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            const int i = kp + (n + a) * ks;
            if (n + a > 0 && n + a < turns && ((n + a) & (turns_here - 1)) == 0) {
                k0 += span;
                __syncthreads();
                stage(k0);
                __syncthreads();
            }
            if (i < chunks) multiply(c[a], i, k0);
            __builtin_amdgcn_sched_barrier(0);
            load(c[a], i + AHEAD * ks);
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // the parts of K of the same columns, added up in order by the first of their waves
    if (ks > 1) {
        f32x4* const red = reinterpret_cast<f32x4*>(smem);
        __syncthreads();  // x has been read
#pragma unroll
        for (int f = 0; f < CF; ++f) red[(wave * CF + f) * kWave + lane] = acc[f];
        __syncthreads();
        if (kp) return;
        for (int w = 1; w < ks; ++w)
#pragma unroll
            for (int f = 0; f < CF; ++f) acc[f] += red[((wave + w) * CF + f) * kWave + lane];
    }
    if (g.epi & kEpiBias) {
#pragma unroll
        for (int f = 0; f < CF; ++f) acc[f] += g.bias[(int64_t)t.e * g.N + min(weight_row(tn, 16 * f + lrow), g.N - 1)];
    }
    const bool relu = g.epi & kEpiRelu;
#pragma unroll
    for (int f = 0; f < CF; ++f) {
        if (gate && f) break;
        const int col = gate ? tn * 16 + lrow : tn * 32 + 16 * f + lrow;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float v = gate ? silu_gate(acc[0][r], acc[1][r]) : relu ? relu_of(acc[f][r]) : acc[f][r];
            const int p = 4 * lgrp + r;
            if (p < rows && col < F) g.y[(int64_t)(t.begin + p) * g.y_stride + col] = elem<T>::from_f32(v);
        }
    }
}

}  // namespace pyc

// What the kernel needs: whole 16-byte pieces, and byte counts that a descriptor holds.
extern "C" int pyc_hip_grouped_stream_takes(int w4, const pyc_grouped* g) {
    const int64_t most = 0xFFFFFFF0ll;
    if (g->x_rows == 0 || ((uintptr_t)g->x & 15) || (g->x_rows > 1 && g->x_stride % 8) || ((uintptr_t)g->w & 15) ||
        g->K % 8 || (g->E > 1 && g->w_stride % (w4 ? 16 : 8)))
        return 0;
    return ((int64_t)(g->x_rows - 1) * g->x_stride + g->K) * 2 <= most &&
           (double)g->N * g->K * (w4 ? 0.5 : 2.0) <= (double)most;
}

extern "C" int pyc_hip_grouped_stream_launch(int is_bf16, const pyc_grouped* gp, void* stream) {
    using namespace pyc;
    const Grouped& g = *gp;
    const bool gate = g.epi & kEpiGate;
    const int cols = gate ? g.N / 2 : g.N, per = gate ? 16 : 32;
    const int tiles_n = (cols + per - 1) / per;
    const int64_t most = expert_tiles_most(g.offsets ? g.E : 1, g.P, 16);
    // K in as many parts as give a wave to every place there is (16 to a CU), two at least (16 tokens by 4 of 32
    // experts, 4096 x 2816: 8 parts 71 us, 4 58, 2 55)
    int ks = 8;
    while (ks > 2 && most * tiles_n * ks > 4096) ks /= 2;
    const int wgs = (tiles_n + kStreamWaves / ks - 1) / (kStreamWaves / ks);
    const hipStream_t s = (hipStream_t)stream;
    // x beside W where LDS would take it in turns; by expert, of about twice the mean of rows
    const int big = most * wgs <= 256;
    const int64_t rows = g.offsets ? 2 * (int64_t)g.P / g.E + 2 : g.P;
    const int xd = (rows < 16 ? rows : 16) * (2 * (int64_t)g.K + 16) > kStreamLds[0][big].x;
    const StreamLds lds = kStreamLds[xd][big];
    const size_t bytes = stream_lds_bytes(lds);
    return grouped_launches(most * wgs, kStreamThreads, [&](uint32_t wg0, dim3 grid) {
#define PYC_STREAM_X(TY, G, XD) \
    hipLaunchKernelGGL((grouped_stream_kernel<TY, G, XD>), grid, dim3(kStreamThreads), bytes, s, g, wgs, ks, lds.x, lds.scales, wg0)
#define PYC_STREAM(G)                                   \
    if (g.group == G) {                                 \
        if (is_bf16) {                                  \
            if (xd) PYC_STREAM_X(bf16_t, G, true);      \
            else PYC_STREAM_X(bf16_t, G, false);        \
        } else {                                        \
            if (xd) PYC_STREAM_X(f16_t, G, true);       \
            else PYC_STREAM_X(f16_t, G, false);         \
        }                                               \
    }
        PYC_STREAM(32)
        PYC_STREAM(64)
        PYC_STREAM(128)
#undef PYC_STREAM
#undef PYC_STREAM_X
    });
}
