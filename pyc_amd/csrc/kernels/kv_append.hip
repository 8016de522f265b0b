// kv_append.hip — a step's keys and values into the paged 8-bit cache.
//
// For a block with new tokens and one head, a = the largest finite |x| of its
// new rows and s_new = 2^e, the smallest power of two with a <= 448 * 2^e
// (e >= -100):
//   s = s_new                if the block's first slot is written (it starts anew),
//       max(s_old, s_new)    else;
//   code = e4m3(x * (1 / s)), round to nearest even; not finite -> NaN;
//   where s > s_old the codes already there become e4m3(code * (s_old / s)).
// Powers of two cost no precision in a floating-point code: x / s is exact, so
// there is one rounding, at one block scale the same for a token alone and in its prompt, and
// a block whose scale grows loses only what falls below the code's normal range.
//
// The tokens of one block stand together in the slot map; the workgroup that finds
// the first of them owns the block for its heads. A wave has one chunk of 16 slots
// of one head (a block of 128 slots is eight waves'), which it holds in registers from
// one read of the rows: maximum, across the block's waves through LDS, then the
// codes. Keys go out as they came, 8 codes a lane; values are transposed in
// LDS, so that a channel's 16 tokens leave as one 16-byte store, merged with the
// codes that are there when the chunk is not all new.
// HBM bounds it for prompts: 16000 tokens of 8 heads of 128 in bf16 take 21 us, 4.65 TB/s
// of rows read once and codes written once (a copy reaches 5.1); with every element checked
// and compared as a float they took 25, of them 18 vector instructions. Few tokens are
// latency: 32 of them, 32 blocks, 4.1 us on the device, of which loads that wait
// for each other (slots, scales, codes) are the most. A wave to a chunk, its rows held from
// one read: a workgroup to a block and head, which read them twice, took 241 us for the
// prompts (and 3.8 for the 32 tokens).
#include "kv_cache.hpp"

namespace pyc {

constexpr int kChunk = 16;

__device__ inline bool append_finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// The codes of a word times f (below 1: the block's scale grew).
__device__ inline uint32_t shrink_e4m3(uint32_t w, float f) {
    return pack_e4m3(__builtin_amdgcn_cvt_f32_fp8((int)w, 0) * f, __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * f,
                     __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * f, __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * f);
}

struct AppendArgs {
    KvCache c;
    int tokens, span;
    const uint16_t* k;
    const uint16_t* v;
    int64_t k_stride, v_stride;
    const int32_t* slots;
};

// Orders a wave's LDS accesses for its other lanes.
__device__ inline void lds_wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
typedef uint32_t __attribute__((may_alias)) word;
typedef uint16_t __attribute__((may_alias)) half_word;

// S: waves (chunks) of a block.
template <typename T, int D, int S>
__global__ void __launch_bounds__((S > 4 ? S : 4) * kWave) kv_append_kernel(AppendArgs a) {
    constexpr int WAVES = S > 4 ? S : 4;
    constexpr int HEADS = WAVES / S;        // heads of a workgroup
    constexpr int LANES = D / 8;            // lanes of a row, 8 channels each
    constexpr int RPL = kChunk * LANES / kWave;  // rows of a lane: slots RPL * (lane / LANES) ..
    constexpr int PITCH = kChunk + 4;       // bytes of a channel in the transposition, off the banks' stride
    __shared__ int where[WAVES][kChunk];    // row of x in each slot of the wave's chunk, -1: none
    __shared__ uint32_t tile[WAVES][D * PITCH / 4];
    __shared__ float most[WAVES];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int chunk = wave % S, h = blockIdx.y * HEADS + wave / S;
    const bool values = blockIdx.z != 0, live = h < a.c.heads;
    const int bs = kChunk * S;
    const int64_t last = (int64_t)a.c.blocks * bs;
    auto slot_of = [&](int i) { return i >= 0 && i < a.tokens ? a.slots[i] : -1; };
    auto block_of = [&](int s) { return s >= 0 && s < last ? s / bs : -1; };
    // Lane l looks at row t0 - 1 + l; the rows 1 .. span of these that begin a block are this workgroup's.
    const int t0 = blockIdx.x * a.span;
    const int my_slot = slot_of(t0 - 1 + lane), my_block = block_of(my_slot), before = __shfl_up(my_block, 1);
    uint64_t first = __ballot(lane >= 1 && lane <= a.span && my_block >= 0 && my_block != before);
    for (; first; first &= first - 1) {
        const int i = __builtin_ctzll(first), t = t0 - 1 + i;
        const int blk = __builtin_amdgcn_readlane(my_block, i);
        // The block's rows: lane l's (and, of long blocks, another 64 behind them).
        bool starts;
        {
            int x0 = lane - i, s0 = my_slot, s1 = -1;  // row t + x0
            if constexpr (S > 2) {                     // a span and a block do not fit 64 lanes
                x0 = lane;
                s0 = slot_of(t + lane);
                if constexpr (S > 4) s1 = slot_of(t + kWave + lane);
            }
            const uint64_t m0 = __ballot(block_of(s0) == blk) >> (S > 2 ? 0 : i), m1 = __ballot(block_of(s1) == blk);
            int n = ~m0 ? __builtin_ctzll(~m0) : kWave + (~m1 ? __builtin_ctzll(~m1) : kWave);
            n = min(n, bs);
            if (lane < kChunk) where[wave][lane] = -1;
            lds_wave_fence();
            const bool in0 = x0 >= 0 && x0 < n, in1 = S > 4 && kWave + lane < n;
            const int o0 = s0 % bs - kChunk * chunk, o1 = s1 % bs - kChunk * chunk;
            if (in0 && o0 >= 0 && o0 < kChunk) where[wave][o0] = t + x0;
            if (in1 && o1 >= 0 && o1 < kChunk) where[wave][o1] = t + kWave + lane;
            starts = __any((in0 && s0 % bs == 0) || (in1 && s1 % bs == 0));
        }
        lds_wave_fence();
        const int r = lane / LANES, c = lane % LANES;
        const uint16_t* x = values ? a.v : a.k;
        const int64_t stride = values ? a.v_stride : a.k_stride;
        int row[RPL];
        u32x4 w[RPL];
        bool all = true;
#pragma unroll
        for (int i = 0; i < RPL; ++i) {
            row[i] = live ? where[wave][RPL * r + i] : -1;
            all &= row[i] >= 0;
            w[i] = u32x4{0, 0, 0, 0};
            if (row[i] >= 0) w[i] = *reinterpret_cast<const u32x4*>(x + row[i] * stride + (int64_t)h * D + 8 * c);
        }
        const int64_t at = (int64_t)blk * a.c.heads + min(h, a.c.heads - 1);
        float* scale = (values ? a.c.v_scale : a.c.k_scale) + at;
        const float old = *scale;
        // The largest |x| by its bits, two at a time. Infinities and NaN lie above all others:
        // a wave that has any counts without them and makes them all NaN.
        typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
        constexpr uint32_t FINITE = __is_same(T, bf16_t) ? 0x7f80 : 0x7c00;  // below this
        u16x2 top{0, 0};
#pragma unroll
        for (int i = 0; i < RPL; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[i][j] & 0x7fff7fffu));
        uint32_t bits = max((uint32_t)top[0], (uint32_t)top[1]);
        if (__any(bits >= FINITE)) {
            bits = 0;
#pragma unroll
            for (int i = 0; i < RPL; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int y = 0; y < 32; y += 16) {
                        const uint32_t e = w[i][j] >> y & 0x7fffu;
                        if (e < FINITE) bits = max(bits, e);
                        else w[i][j] = (w[i][j] & ~(0xffffu << y)) | (0x7fffu << y);
                    }
        }
#pragma unroll
        for (int d = 1; d < kWave; d *= 2) bits = max(bits, (uint32_t)__shfl_xor((int)bits, d));
        float mx = half_at<T>(u32x4{bits, 0, 0, 0}, 0);
        if constexpr (S > 1) {
            asm volatile("" ::"v"(old));  // it is here before another wave may store the new scale
            __syncthreads();              // and the last block's maxima are read
            if (lane == 0) most[wave] = mx;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < S; ++i) mx = fmaxf(mx, most[wave - chunk + i]);
        }
        float s = e4m3_scale(mx);
        const bool had = old > 0.f && append_finite(old);  // a scale that means something
        if (!starts && had) s = fmaxf(s, old);
        const bool grow = !starts && had && s > old;
        const float f = grow ? old / s : 1.f, inv = 1.0f / s;
        if (!live) continue;
        if (chunk == 0 && lane == 0 && s != old) *scale = s;
        auto scaled = [&](int i, int j) { return half_at<T>(w[i], j) * inv; };
        if (!values) {
            uint8_t* dst = a.c.k + blk * a.c.k_stride + ((int64_t)h * bs + kChunk * chunk + RPL * r) * D + 8 * c;
#pragma unroll
            for (int i = 0; i < RPL; ++i) {
                u32x2 out;
                if (row[i] >= 0) {
                    out[0] = pack_e4m3(scaled(i, 0), scaled(i, 1), scaled(i, 2), scaled(i, 3));
                    out[1] = pack_e4m3(scaled(i, 4), scaled(i, 5), scaled(i, 6), scaled(i, 7));
                } else {
                    if (!grow) continue;
                    out = *reinterpret_cast<const u32x2*>(dst + i * D);
                    out[0] = shrink_e4m3(out[0], f);
                    out[1] = shrink_e4m3(out[1], f);
                }
                *reinterpret_cast<u32x2*>(dst + i * D) = out;
            }
        } else {
            // slots RPL r .. of channel 8 c + j, as one word (or half of one)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                uint8_t* to = (uint8_t*)tile[wave] + (8 * c + j) * PITCH + RPL * r;
                if constexpr (RPL == 4) {
                    *(word*)to = pack_e4m3(scaled(0, j), scaled(1, j), scaled(2, j), scaled(3, j));
                } else {
                    *(half_word*)to = (uint16_t)__builtin_amdgcn_cvt_pk_fp8_f32(scaled(0, j), scaled(1, j), 0, false);
                }
            }
            lds_wave_fence();
            const bool whole = __all(all);
            u32x4 keep{0, 0, 0, 0};  // bytes of a chunk that stay
            if (!whole) {
#pragma unroll
                for (int i = 0; i < kChunk; ++i)
                    if (where[wave][i] < 0) keep[i >> 2] |= 0xffu << (8 * (i & 3));
            }
            const bool none = (keep[0] & keep[1] & keep[2] & keep[3]) == 0xffffffffu;
            if (!none || grow) {
                uint8_t* dst = a.c.v + blk * a.c.v_stride + ((int64_t)h * D + lane) * bs + kChunk * chunk;
#pragma unroll
                for (int i = 0; i < D / kWave; ++i) {
                    u32x4* at16 = reinterpret_cast<u32x4*>(dst + (int64_t)kWave * i * bs);
                    const uint32_t* from = tile[wave] + (lane + kWave * i) * (PITCH / 4);
                    u32x4 out{from[0], from[1], from[2], from[3]};
                    if (!whole) {
                        u32x4 there = *at16;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (grow) there[e] = shrink_e4m3(there[e], f);
                            out[e] = (out[e] & ~keep[e]) | (there[e] & keep[e]);
                        }
                    }
                    *at16 = out;
                }
            }
        }
    }
}

template <typename T, int D> static const void* append_kernel_of(int bs) {
    return bs == 16   ? reinterpret_cast<const void*>(&kv_append_kernel<T, D, 1>)
           : bs == 32 ? reinterpret_cast<const void*>(&kv_append_kernel<T, D, 2>)
           : bs == 64 ? reinterpret_cast<const void*>(&kv_append_kernel<T, D, 4>)
                      : reinterpret_cast<const void*>(&kv_append_kernel<T, D, 8>);
}
static const void* append_kernel_of(int is_bf16, int d, int bs) {
    return d == 128 ? (is_bf16 ? append_kernel_of<bf16_t, 128>(bs) : append_kernel_of<f16_t, 128>(bs))
                    : (is_bf16 ? append_kernel_of<bf16_t, 64>(bs) : append_kernel_of<f16_t, 64>(bs));
}

}  // namespace pyc

extern "C" int pyc_hip_kv_append_launch(int is_bf16, const pyc_hip_kv_cache* cache, int tokens, const void* k,
                                        int64_t k_stride, const void* v, int64_t v_stride, const int32_t* slots,
                                        void* stream) {
    using namespace pyc;
    AppendArgs a{kv_cache_of(cache), tokens, 1, (const uint16_t*)k, (const uint16_t*)v, k_stride, v_stride, slots};
    // A workgroup for every row where that gives up to 16 k waves (most rows begin no
    // block and their waves end at once), else for up to 16 rows in a row. With blocks of 64 three
    // of four workgroups still find none, and the others read the slots a second time: 7 ragged
    // chunks of 12 heads of 64 in f16, 8.2 us.
    const int S = a.c.bs / kChunk, waves = S > 4 ? S : 4, per = waves / S;
    const unsigned hy = (unsigned)((a.c.heads + per - 1) / per);
    while (a.span < kChunk && (double)tokens / a.span * hy * 2 * waves > 16384.0) a.span *= 2;
    void* args[] = {&a};
    const hipError_t e = hipLaunchKernel(append_kernel_of(is_bf16, a.c.d, a.c.bs),
                                         dim3((unsigned)((tokens + a.span - 1) / a.span), hy, 2), dim3(waves * kWave),
                                         args, 0, (hipStream_t)stream);
    return e == hipSuccess && hipGetLastError() == hipSuccess ? 0 : -2;
}

extern "C" int pyc_hip_kinfo_kv_append(int is_bf16, pyc_hip_kinfo* out) {
    using namespace pyc;
    if (!out) return -1;
    out->fn = append_kernel_of(is_bf16, 128, 16);
    out->name = "kv_append_kernel<128, 1>";
    out->lds_bytes = 4 * (kChunk * sizeof(int) + 128 * (kChunk + 4));
    out->threads = 4 * kWave;
    out->waves_per_simd = 7;
    return 0;
}
