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
// there is one rounding, the same for a token alone and in its prompt, and a
// block whose scale grows loses only what falls below the code's normal range.
//
// The tokens of one block stand together in the slot map; the wave that finds
// the first of them owns the block for its head.
#include "kv_cache.hpp"

namespace pyc {

constexpr int kAppendWaves = 4;
constexpr int kMinExp = -100;

__device__ inline uint8_t to_e4m3(float x) {
    return (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(x, x, 0, false) & 0xff);
}
__device__ inline float from_e4m3(uint8_t c) { return __builtin_amdgcn_cvt_f32_fp8((int)c, 0); }

// The smallest power of two s >= 2^-100 with a <= 448 s (a finite, >= 0). a = m
// 2^x with 1 <= m < 2 and 448 = 1.75 * 2^8.
__device__ inline float append_scale(float a) {
    const uint32_t u = __float_as_uint(a);
    int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = max(e, kMinExp);
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

__device__ inline float append_finite(float x) {
    const float m = fabsf(x);
    return m <= 3.402823466e38f ? m : 0.f;
}

// One block of one head, keys (VALUES false) or values: rows t0 .. t0 + n - 1
// of x go to the offsets that slots[] says.
template <typename T, bool VALUES>
__device__ inline void append_block(const uint16_t* x, int64_t x_stride, const int32_t* slots, int t0, int n,
                                    uint8_t* codes, float* scale, int bs, int D) {
    const int lane = threadIdx.x & (kWave - 1);
    float a = 0.f;
    bool starts = false;
    for (int i = 0; i < n; ++i) {
        const uint16_t* row = x + (int64_t)(t0 + i) * x_stride;
        for (int d = lane; d < D; d += kWave) a = fmaxf(a, append_finite(elem<T>::to_f32(row[d])));
        starts |= slots[t0 + i] % bs == 0;
    }
#pragma unroll
    for (int w = 1; w < kWave; w *= 2) a = fmaxf(a, __shfl_xor(a, w));
    const float old = *scale;
    float s = append_scale(a);
    const bool had = old > 0.f && old <= 3.402823466e38f;  // a scale that means something
    if (!starts && had && old > s) s = old;
    if (!starts && had && s > old) {
        const float f = old / s;
        for (int i = lane; i < bs * D; i += kWave) codes[i] = to_e4m3(from_e4m3(codes[i]) * f);
        __threadfence_block();  // the new codes below go on top of these
    }
    const float inv = 1.0f / s;
    for (int i = 0; i < n; ++i) {
        const uint16_t* row = x + (int64_t)(t0 + i) * x_stride;
        const int off = slots[t0 + i] % bs;
        for (int d = lane; d < D; d += kWave) {
            const float v = elem<T>::to_f32(row[d]);
            const float y = fabsf(v) <= 3.402823466e38f ? v * inv : __builtin_nanf("");
            codes[VALUES ? d * bs + off : off * D + d] = to_e4m3(y);
        }
    }
    if (lane == 0 && s != old) *scale = s;
}

template <typename T>
__global__ void __launch_bounds__(kAppendWaves* kWave) kv_append_kernel(KvCache c, int tokens, const uint16_t* k,
                                                                       int64_t k_stride, const uint16_t* v,
                                                                       int64_t v_stride, const int32_t* slots) {
    const int t = blockIdx.x, h = blockIdx.y * kAppendWaves + threadIdx.x / kWave;
    if (h >= c.heads) return;
    const int64_t last = (int64_t)c.blocks * c.bs;
    auto block_of = [&](int i) {
        const int s = i >= 0 && i < tokens ? slots[i] : -1;
        return s >= 0 && s < last ? s / c.bs : -1;
    };
    const int blk = block_of(t);
    if (blk < 0 || block_of(t - 1) == blk) return;
    int n = 1;
    while (block_of(t + n) == blk) ++n;
    const int64_t at = (int64_t)blk * c.heads + h, hd = (int64_t)h * c.bs * c.d;
    if (blockIdx.z == 0)
        append_block<T, false>(k + (int64_t)h * c.d, k_stride, slots, t, n, c.k + blk * c.k_stride + hd, c.k_scale + at,
                               c.bs, c.d);
    else
        append_block<T, true>(v + (int64_t)h * c.d, v_stride, slots, t, n, c.v + blk * c.v_stride + hd, c.v_scale + at,
                              c.bs, c.d);
}

}  // namespace pyc

extern "C" int pyc_hip_kv_append_launch(int is_bf16, const pyc_hip_kv_cache* cache, int tokens, const void* k,
                                        int64_t k_stride, const void* v, int64_t v_stride, const int32_t* slots,
                                        void* stream) {
    using namespace pyc;
    const KvCache c = kv_cache_of(cache);
    const dim3 grid(tokens, (c.heads + kAppendWaves - 1) / kAppendWaves, 2), block(kAppendWaves * kWave);
    hipStream_t s = (hipStream_t)stream;
    if (is_bf16)
        hipLaunchKernelGGL(kv_append_kernel<bf16_t>, grid, block, 0, s, c, tokens, (const uint16_t*)k, k_stride,
                           (const uint16_t*)v, v_stride, slots);
    else
        hipLaunchKernelGGL(kv_append_kernel<f16_t>, grid, block, 0, s, c, tokens, (const uint16_t*)k, k_stride,
                           (const uint16_t*)v, v_stride, slots);
    return hipGetLastError() == hipSuccess ? 0 : -2;
}

extern "C" int pyc_hip_kinfo_kv_append(int is_bf16, pyc_hip_kinfo* out) {
    using namespace pyc;
    if (!out) return -1;
    out->fn = is_bf16 ? reinterpret_cast<const void*>(&kv_append_kernel<bf16_t>)
                      : reinterpret_cast<const void*>(&kv_append_kernel<f16_t>);
    out->name = "kv_append_kernel";
    out->lds_bytes = 0;
    out->threads = kAppendWaves * kWave;
    out->waves_per_simd = 8;
    return 0;
}
