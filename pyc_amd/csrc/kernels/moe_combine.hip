// moe_combine.hip — o[t] = base[t] + sum_j weights[t][j] y[places[t][j]]: the rows of a
// token's experts back onto the token. Sums in fp32, base first, then j in order, one
// rounding at the end. A place outside y counts as absent and is not read.
//
// Bound by memory: k rows read for one written. A thread has 16 bytes of a row (eight
// columns) and loads its k pieces before it adds any. Where a wave lies in one token (width
// a multiple of 512) its places and weights come by scalar loads. A call with 8200 tokens by
// 8 rows of 2048 columns: 63 us (74 with vector loads of them), 4.8 TB/s; a large copy reaches 5.1. Rows off 16
// bytes take a thread and 2-byte loads for each column: 225 us, of waiting for 128 bytes to a wave's load.
#include "common.hpp"

namespace pyc {

constexpr int kCombineThreads = 256;
constexpr int kCombineAhead = 8;  // pieces in flight

struct Combine {
    const uint16_t* y;
    int64_t y_stride;
    int P, T, k, H;
    const float* weights;
    const int32_t* places;
    const uint16_t* base;
    int64_t base_stride;
    uint16_t* out;
    int64_t out_stride;
};

// VEC columns to a thread: eight as 16-byte accesses, or one where rows do not keep to 16 bytes
template <typename T, int VEC, bool ONE>
__global__ void __launch_bounds__(kCombineThreads) moe_combine_kernel(Combine c, int chunks) {
    const int64_t at = (int64_t)blockIdx.x * kCombineThreads + threadIdx.x;
    int t = (int)(at / chunks);
    if constexpr (ONE) t = __builtin_amdgcn_readfirstlane(t);
    const int h = (int)(at - (int64_t)t * chunks) * VEC;
    if (t >= c.T) return;
    float sum[VEC];
    auto load = [&](const uint16_t* p, float (&v)[VEC]) {
        if constexpr (VEC == 8) {
            const u32x4 u = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = elem<T>::to_f32((uint16_t)(u[i >> 1] >> (16 * (i & 1))));
        } else {
            v[0] = elem<T>::to_f32(*p);
        }
    };
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[i] = 0.f;
    if (c.base) load(c.base + (int64_t)t * c.base_stride + h, sum);
    for (int j0 = 0; j0 < c.k; j0 += kCombineAhead) {
        float v[kCombineAhead][VEC], w[kCombineAhead];
        bool in[kCombineAhead];
#pragma unroll
        for (int j = 0; j < kCombineAhead; ++j) {
            const bool there = j0 + j < c.k;
            const int p = there ? c.places[(int64_t)t * c.k + j0 + j] : -1;
            in[j] = (unsigned)p < (unsigned)c.P;
            w[j] = there ? c.weights[(int64_t)t * c.k + j0 + j] : 0.f;
            if (in[j]) load(c.y + (int64_t)p * c.y_stride + h, v[j]);
        }
#pragma unroll
        for (int j = 0; j < kCombineAhead; ++j)
            if (in[j]) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) sum[i] = fmaf(w[j], v[j][i], sum[i]);
            }
    }
    uint16_t* o = c.out + (int64_t)t * c.out_stride + h;
    if constexpr (VEC == 8) {
        u32x4 u;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            u[i] = elem<T>::from_f32(sum[2 * i]) | ((uint32_t)elem<T>::from_f32(sum[2 * i + 1]) << 16);
        *reinterpret_cast<u32x4*>(o) = u;
    } else {
        *o = elem<T>::from_f32(sum[0]);
    }
}

}  // namespace pyc

extern "C" int pyc_hip_moe_combine_launch(int is_bf16, int P, int T, int k, int H, const void* y, int64_t y_stride,
                                          const float* weights, const int32_t* places, const void* base,
                                          int64_t base_stride, void* out, int64_t out_stride, void* stream) {
    using namespace pyc;
    const Combine c{(const uint16_t*)y, y_stride, P, T, k, H, weights, places, (const uint16_t*)base, base_stride,
                    (uint16_t*)out, out_stride};
    const bool wide = ((H | y_stride | out_stride | (base ? base_stride : 0)) & 7) == 0 &&
                      (((uintptr_t)y | (uintptr_t)out | (uintptr_t)base) & 15) == 0;
    const int chunks = wide ? H / 8 : H;
    const int64_t blocks = ((int64_t)T * chunks + kCombineThreads - 1) / kCombineThreads;
    if (blocks > kMostThreads / kCombineThreads) {  // more threads than a launch has: half of the tokens each (one alone never is)
        const int n = T / 2;
        const int rc = pyc_hip_moe_combine_launch(is_bf16, P, n, k, H, y, y_stride, weights, places, base, base_stride, out, out_stride, stream);
        return rc ? rc : pyc_hip_moe_combine_launch(is_bf16, P, T - n, k, H, y, y_stride, weights + (int64_t)n * k, places + (int64_t)n * k,
                                                    base ? c.base + n * base_stride : nullptr, base_stride, c.out + n * out_stride,
                                                    out_stride, stream);
    }
    const dim3 grid((unsigned)blocks);
    const hipStream_t s = (hipStream_t)stream;
    const bool one = chunks % kWave == 0;
#define PYC_COMBINE(TY)                                                                                                     \
    if (wide && one) hipLaunchKernelGGL((moe_combine_kernel<TY, 8, true>), grid, dim3(kCombineThreads), 0, s, c, chunks);   \
    else if (wide) hipLaunchKernelGGL((moe_combine_kernel<TY, 8, false>), grid, dim3(kCombineThreads), 0, s, c, chunks);    \
    else hipLaunchKernelGGL((moe_combine_kernel<TY, 1, false>), grid, dim3(kCombineThreads), 0, s, c, chunks)
    if (is_bf16) PYC_COMBINE(bf16_t);
    else PYC_COMBINE(f16_t);
#undef PYC_COMBINE
    return hipGetLastError() == hipSuccess ? 0 : -2;
}

extern "C" int pyc_hip_kinfo_moe_combine(int is_bf16, pyc_hip_kinfo* out) {
    using namespace pyc;
    if (!out) return -1;
    out->fn = is_bf16 ? reinterpret_cast<const void*>(&moe_combine_kernel<bf16_t, 8, true>)
                      : reinterpret_cast<const void*>(&moe_combine_kernel<f16_t, 8, true>);
    out->name = "moe_combine_kernel";
    out->lds_bytes = 0;
    out->threads = kCombineThreads;
    out->waves_per_simd = 6;
    return 0;
}
