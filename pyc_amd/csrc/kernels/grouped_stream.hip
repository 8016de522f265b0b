// grouped_stream.hip — products by expert where an expert has few rows: single tokens and
// decoding batches, with 16-bit weights or 4-bit ones. What bounds them is the stream of
// the weights, every byte of which is used once.
//
// A workgroup has 16 CF rows of one expert's W and up to 16 MT rows of x, over all of K: its
// eight waves take every eighth chunk of 128 k and are added up through LDS at the end, in
// a fixed order, so that a layer of a few thousand columns fills 256 CUs without a second
// launch. W goes from memory into registers as the operand it is (16 rows of 64 bytes to an
// instruction, two chunks in flight), through buffer descriptors: rows and k past the end,
// rows of x that are not there and chunks past the last read zeros and cost no traffic.
// The rows of x are the first operand: a lane's results are four rows of one column of y, so
// a column's scale is one value for each lane.
//
// 4-bit: a lane's 16 bytes are 32 k of a row, the four lanes of a row 128 k. A 4 x 4
// transposition between the lanes and their four words (four swaps) gives each product 32
// neighbouring k, so that groups of 32, 64 and 128 all work. A code c goes into the
// mantissa of 16, as 16 + c exactly, two to an instruction and nearly for free; a group's sum is then
//   scale (sum x (16 + c) - (16 + zero) sum x),
// all in fp32, with sum x from one more product by ones. (By conversion to whole numbers less
// zero a pair takes three to four times the instructions. 128 + c, which needs a shift less, has
// six times the cancellation.) Pairs come out as k 0,4 1,5 2,6 3,7, so x is put in that order.
#include "grouped.hpp"

namespace pyc {

constexpr int kStreamWaves = 8;
constexpr int kStreamK = 128;  // k of a chunk
constexpr uint32_t kPastEnd = 0xFFFFFFF0u;  // not below any descriptor's byte count

// w[i] of lane group g becomes w[g] of lane group i.
__device__ inline void transpose4(u32x4& w) {
    auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
    auto b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    w = u32x4{c[0], c[1], d[0], d[1]};
}

// Eight codes as 16 + c, pairs k 0,4 1,5 2,6 3,7.
__device__ inline u32x4 codes16(uint32_t w, bf16_t) {
    constexpr uint32_t m = 0x00780078u, b = 0x41804180u;  // 16.0, 3 bits below its units
    return u32x4{((w << 3) & m) | b, ((w >> 1) & m) | b, ((w >> 5) & m) | b, ((w >> 9) & m) | b};
}
__device__ inline u32x4 codes16(uint32_t w, f16_t) {
    constexpr uint32_t m = 0x03c003c0u, b = 0x4c004c00u;  // 16.0, 6 bits below its units
    return u32x4{((w << 6) & m) | b, ((w << 2) & m) | b, ((w >> 2) & m) | b, ((w >> 6) & m) | b};
}
__device__ inline u32x4 paired(const u32x4& x) {
    return u32x4{__builtin_amdgcn_perm(x[2], x[0], 0x05040100u), __builtin_amdgcn_perm(x[2], x[0], 0x07060302u),
                 __builtin_amdgcn_perm(x[3], x[1], 0x05040100u), __builtin_amdgcn_perm(x[3], x[1], 0x07060302u)};
}
template <typename T> __device__ inline u32x4 ones() {
    const uint32_t o = elem<T>::from_f32(1.0f) * 0x10001u;
    return u32x4{o, o, o, o};
}

// G: k of a group (0: 16-bit weights)
template <int G, int CF, int MT> struct Chunk {
    static constexpr int kGroups = G ? kStreamK / G : 1;
    u32x4 w[CF][G ? 1 : 4];
    u32x4 x[MT][4];
    uint64_t s[G ? CF : 1];  // the chunk's scales and zero points, the first ones lowest
    uint32_t z[G ? CF : 1];
};

// `n` values of type V from v[at], the first one lowest; what lies behind v[last] reads 0.
// One load at any alignment, moved back where it would pass the end (last >= n).
template <typename R, int n, typename V> __device__ inline R load_values(const V* v, uint32_t at, uint32_t last) {
    const uint32_t from = min(at, last - n);
    R r = 0;
    __builtin_memcpy(&r, v + from, n * sizeof(V));
    if constexpr (n > 1) {
        const uint32_t d = 8 * sizeof(V) * min(at - from, (uint32_t)(n - 1));
        r >>= d;
    }
    return r;
}

template <typename T, int G, int CF, int MT>
__global__ void __launch_bounds__(kStreamWaves * kWave, MT * CF <= 2 ? 4 : 2)
grouped_stream_kernel(Grouped g, int tiles_n, int wgs, int ks) {
    constexpr bool W4 = G != 0;
    typedef Chunk<G, CF, MT> C;
    __shared__ f32x4 red[kStreamWaves][MT][CF][kWave];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lrow = lane & 15, lgrp = lane >> 4;
    const int kp = wave & (ks - 1);                                     // this wave's part of K
    const int tn = (blockIdx.x % wgs) * (kStreamWaves / ks) + wave / ks;  // its columns
    const ExpertTile t = expert_tile(g, blockIdx.x / wgs, 16 * MT, lane);
    if (t.e < 0) return;
    const bool gate = g.epi & kEpiGate;
    const int F = gate ? g.N / 2 : g.N;
    const int half = gate ? CF / 2 : CF;  // fragments of columns of y
    // the row of W behind column lrow of fragment f (N: none)
    auto weight_row = [&](int f) {
        const int c = (tn * half + (f < half ? f : f - half)) * 16 + lrow;
        return c < F ? (f < half ? c : c + F) : g.N;
    };

    const uint32_t row_bytes = W4 ? (uint32_t)g.K / 2 : (uint32_t)g.K * 2;
    const int groups = W4 ? g.K / (W4 ? G : 1) : 0;
    const int chunks = (g.K + kStreamK - 1) / kStreamK;
    const int whole = g.K / kStreamK;
    // A chunk's place is the scalar part of a load's offset, which the descriptor's check leaves out. So the
    // last chunk, where K is no multiple of 128, has lane offsets of its own, past the end for k
    // past K, and chunks behind it a descriptor of no bytes.
    void* const wbase = const_cast<char*>(static_cast<const char*>(g.w)) + (int64_t)t.e * g.w_stride * (W4 ? 1 : 2);
    const uint32_t wbytes = tn < tiles_n ? (uint32_t)g.N * row_bytes : 0u;
    const uint32_t xbytes = (uint32_t)(((int64_t)(g.x_rows - 1) * g.x_stride + g.K) * 2);
    const int left = g.K - whole * kStreamK;
    uint32_t wo[CF], xo[MT], so[CF];
#pragma unroll
    for (int f = 0; f < CF; ++f) {
        const int r = weight_row(f);
        wo[f] = r < g.N ? (uint32_t)r * row_bytes + 16 * lgrp : kPastEnd;
        so[f] = (uint32_t)min(r, g.N - 1) * (uint32_t)groups;
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int p = t.begin + 16 * m + lrow;
        const int r = p < t.end ? source_row(g, p) : -1;
        xo[m] = r < 0 ? kPastEnd : (uint32_t)((int64_t)r * g.x_stride * 2) + 16 * lgrp;
    }
    const uint16_t* scale = W4 ? g.scale + (int64_t)t.e * g.N * groups : nullptr;
    // without zero points their loads take the scales' places, and what comes is not used: a branch
    // around loads would make every wait one for all of them
    const bool has_zeros = W4 && g.zeros != nullptr;
    const uint8_t* zeros = !W4 ? nullptr : has_zeros ? g.zeros + (int64_t)t.e * g.N * groups : reinterpret_cast<const uint8_t*>(scale);

    auto load = [&](C& c, int i) {
        const auto wr = __builtin_amdgcn_make_buffer_rsrc(wbase, 0, i < chunks ? wbytes : 0u, 0x00020000);
        const auto xr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(g.x), 0, i < chunks ? xbytes : 0u, 0x00020000);
        const int end = i == whole ? left : kStreamK;  // k of the chunk that there are
        const uint32_t at = (uint32_t)i * kStreamK;
        auto get = [&](const __amdgpu_buffer_rsrc_t& r, uint32_t off, uint32_t s) {
            return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, s, 0));
        };
#pragma unroll
        for (int f = 0; f < CF; ++f) {
            if constexpr (W4) {
                c.w[f][0] = get(wr, 32 * lgrp < end ? wo[f] : kPastEnd, at / 2);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) c.w[f][j] = get(wr, 32 * j + 8 * lgrp < end ? wo[f] : kPastEnd, at * 2 + 64 * j);
            }
        }
        if constexpr (W4) {
#pragma unroll
            for (int f = 0; f < CF; ++f) {
                const uint32_t q = so[f] + (uint32_t)min(i, chunks - 1) * C::kGroups, all = (uint32_t)(g.N * groups);
                c.s[f] = load_values<uint64_t, C::kGroups>(scale, q, all);
                const uint32_t z = load_values<uint32_t, C::kGroups>(zeros, has_zeros ? q : 2 * q, has_zeros ? all : 2 * all);
                c.z[f] = has_zeros ? z : 0x08080808u;
            }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) c.x[m][j] = get(xr, 32 * j + 8 * lgrp < end ? xo[m] : kPastEnd, at * 2 + 64 * j);
    };

    f32x4 acc[MT][CF];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int f = 0; f < CF; ++f) acc[m][f] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](C& c) {
        if constexpr (W4) {
            const u32x4 one = ones<T>();
            f32x4 part[MT][CF], sum[MT];
#pragma unroll
            for (int f = 0; f < CF; ++f) transpose4(c.w[f][0]);
#pragma unroll
            for (int q = 0; q < C::kGroups; ++q) {
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    sum[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int f = 0; f < CF; ++f) part[m][f] = f32x4{0.f, 0.f, 0.f, 0.f};
                }
#pragma unroll
                for (int j = q * (4 / C::kGroups); j < (q + 1) * (4 / C::kGroups); ++j) {
                    u32x4 x[MT];
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        x[m] = paired(c.x[m][j]);
                        sum[m] = mfma16x16x32(x[m], one, sum[m], T{});
                    }
#pragma unroll
                    for (int f = 0; f < CF; ++f) {
                        const u32x4 w = codes16(c.w[f][0][j], T{});
#pragma unroll
                        for (int m = 0; m < MT; ++m) part[m][f] = mfma16x16x32(x[m], w, part[m][f], T{});
                    }
                    __builtin_amdgcn_sched_barrier(0);  // a slice at a time: unpacked ahead, codes take four times the registers
                }
#pragma unroll
                for (int f = 0; f < CF; ++f) {
                    const float s = elem<T>::to_f32((uint16_t)(c.s[f] >> (16 * q)));
                    const float z = -16.0f - (float)((c.z[f] >> (8 * q)) & 255u);
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            acc[m][f][r] = fmaf(s, fmaf(z, sum[m][r], part[m][f][r]), acc[m][f][r]);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int f = 0; f < CF; ++f)
#pragma unroll
                    for (int m = 0; m < MT; ++m) acc[m][f] = mfma16x16x32(c.x[m][j], c.w[f][j], acc[m][f], T{});
        }
    };
    // two chunks in flight; each column block begins elsewhere in K
    const int rot = (int)((((uint32_t)(tn + 37 * t.e) * 0x9E37u & 0xFFFFu) * (uint32_t)chunks) >> 16);
    auto turned = [&](int i) { return i < chunks ? (i + rot < chunks ? i + rot : i + rot - chunks) : i; };
    C a, b;
    load(a, turned(kp));
    __builtin_amdgcn_sched_barrier(0);  // the loop's waits count loads in this order
    load(b, turned(kp + ks));
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll 1
    for (int i = kp; i < chunks; i += 2 * ks) {
        multiply(a);
        __builtin_amdgcn_sched_barrier(0);
        load(a, turned(i + 2 * ks));
        __builtin_amdgcn_sched_barrier(0);
        multiply(b);
        __builtin_amdgcn_sched_barrier(0);
        load(b, turned(i + 3 * ks));
        __builtin_amdgcn_sched_barrier(0);
    }

    // the parts of K of the same columns, added up in order by the first of their waves
    if (ks > 1) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int f = 0; f < CF; ++f) red[wave][m][f][lane] = acc[m][f];
        __syncthreads();
        if (kp) return;
        for (int w = 1; w < ks; ++w)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int f = 0; f < CF; ++f) acc[m][f] += red[wave + w][m][f][lane];
    }
    if (g.epi & kEpiBias) {
#pragma unroll
        for (int f = 0; f < CF; ++f) {
            const int r = weight_row(f);
            const float b = g.bias[(int64_t)t.e * g.N + min(r, g.N - 1)];
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[m][f] += b;
        }
    }
    auto put = [&](int m, int f, f32x4 v) {
        const int c = (tn * half + f) * 16 + lrow;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int p = t.begin + 16 * m + 4 * lgrp + r;
            if (p < t.end && c < F) g.y[(int64_t)p * g.y_stride + c] = elem<T>::from_f32(v[r]);
        }
    };
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        if (gate) {
#pragma unroll
            for (int f = 0; f < CF / 2; ++f) {
                f32x4 v;
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = silu_gate(acc[m][f][r], acc[m][f + CF / 2][r]);
                put(m, f, v);
            }
        } else {
#pragma unroll
            for (int f = 0; f < CF; ++f) {
                f32x4 v = acc[m][f];
                if (g.epi & kEpiRelu) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] = fmaxf(v[r], 0.f);
                }
                put(m, f, v);
            }
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
           (double)g->N * g->K * (w4 ? 0.5 : 2.0) <= (double)most && (!w4 || (int64_t)g->N * (g->K / g->group) >= 4);
}

extern "C" int pyc_hip_grouped_stream_launch(int is_bf16, int w4, const pyc_grouped* gp, void* stream) {
    using namespace pyc;
    const Grouped& g = *gp;
    const bool gate = g.epi & kEpiGate;
    const int cols = gate ? g.N / 2 : g.N, per = gate ? 16 : 32;
    const int tiles_n = (cols + per - 1) / per;
    const int64_t most = expert_tiles_most(g.offsets ? g.E : 1, g.P, 16);
    // K in as many parts as give a wave to every place there is (16 to a CU), two at least (32 tokens by
    // 8 of 64 experts, 2048 x 2816: 8 parts 158 us, 4 137, 2 139, 1 147)
    int ks = 8;
    while (ks > 2 && most * tiles_n * ks > 4096) ks /= 2;
    const int wgs = (tiles_n + kStreamWaves / ks - 1) / (kStreamWaves / ks);
    if (most * wgs > 0x7FFFFFFF) return -1;
    const hipStream_t s = (hipStream_t)stream;
    const dim3 grid((unsigned)(most * wgs)), block(kStreamWaves * kWave);
#define PYC_STREAM(G)                                                                                                  \
    if ((w4 ? g.group : 0) == G) {                                                                                     \
        if (is_bf16) hipLaunchKernelGGL((grouped_stream_kernel<bf16_t, G, 2, 1>), grid, block, 0, s, g, tiles_n, wgs, ks); \
        else hipLaunchKernelGGL((grouped_stream_kernel<f16_t, G, 2, 1>), grid, block, 0, s, g, tiles_n, wgs, ks);          \
        return hipGetLastError() == hipSuccess ? 0 : -2;                                                               \
    }
    PYC_STREAM(0)
    PYC_STREAM(32)
    PYC_STREAM(64)
    PYC_STREAM(128)
#undef PYC_STREAM
    return -1;
}
