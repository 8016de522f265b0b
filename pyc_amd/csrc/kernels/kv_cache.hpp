// kv_cache.hpp — the paged 8-bit key/value cache as its kernels see it.
//
// Keys   [blocks][kv heads][bs][D]  e4m3: a token's D codes run on.
// Values [blocks][kv heads][D][bs]  e4m3: a channel's tokens run on, so that 16
// tokens of one channel are one 16-byte load and, as they are, the operand
// of O^T = V^T P^T: the product over tokens needs no transposition anywhere.
// Scales [blocks][kv heads] fp32, one for keys and one for values.
#pragma once

#include "common.hpp"
#include "pyc/ir.h"
#include "pyc/hip_backend.h"

namespace pyc {

struct KvCache {
    uint8_t* k;
    uint8_t* v;
    float* k_scale;
    float* v_scale;
    int64_t k_stride, v_stride;  // bytes from a block to the next
    int blocks, heads, bs, d;
};

inline KvCache kv_cache_of(const pyc_hip_kv_cache* c) {
    return KvCache{(uint8_t*)c->k,    (uint8_t*)c->v,    c->k_scale,    c->v_scale,  c->k_block_stride,
                   c->v_block_stride, c->num_blocks, c->kv_heads, c->block_size, c->head_dim};
}

__device__ inline float read_lane(float x, int i) {
    return __uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(x), i));
}
__device__ inline int64_t read_lane(int64_t x, int i) {
    return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), i) << 32) |
                     (uint32_t)__builtin_amdgcn_readlane((int)x, i));
}

// Inclusive scan over the wave's lanes by DPP moves (a few cycles each where a
// shuffle through the LDS takes 60): rows of 16 lanes by shifts of 1, 2, 4 and
// 8, then lane 15 of the row before into rows 1 and 3, and lane 31 into rows 2 and 3.
// A move gives `none` where there is no lane to take from.
template <int CTRL, int ROWS> __device__ inline int dpp_move(int none, int x) {
    return __builtin_amdgcn_update_dpp(none, x, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS> __device__ inline float dpp_move(float none, float x) {
    return __int_as_float(dpp_move<CTRL, ROWS>(__float_as_int(none), __float_as_int(x)));
}
template <int CTRL, int ROWS> __device__ inline int64_t dpp_move(int64_t none, int64_t x) {
    return (int64_t)(((uint64_t)(uint32_t)dpp_move<CTRL, ROWS>((int)(none >> 32), (int)(x >> 32)) << 32) |
                     (uint32_t)dpp_move<CTRL, ROWS>((int)none, (int)x));
}
template <typename V, typename F> __device__ inline V wave_scan(V x, V none, F f) {
    x = f(x, dpp_move<0x111, 0xf>(none, x));
    x = f(x, dpp_move<0x112, 0xf>(none, x));
    x = f(x, dpp_move<0x114, 0xf>(none, x));
    x = f(x, dpp_move<0x118, 0xf>(none, x));
    x = f(x, dpp_move<0x142, 0xa>(none, x));
    x = f(x, dpp_move<0x143, 0xc>(none, x));
    return x;
}

constexpr int kMinExp = -100;
// The smallest power of two s >= 2^-100 with a <= 448 s (a finite, >= 0). a = m
// 2^x with 1 <= m < 2 and 448 = 1.75 * 2^8.
__device__ inline float e4m3_scale(float a) {
    const uint32_t u = __float_as_uint(a);
    int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = max(e, kMinExp);
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

// Four floats as codes, in one word.
__device__ inline uint32_t pack_e4m3(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
// Element j of 8 half-precision ones.
template <typename T> __device__ inline float half_at(const u32x4& w, int j) {
    return elem<T>::to_f32((uint16_t)(w[j >> 1] >> (16 * (j & 1))));
}

// e4m3 to bf16 or f16, two codes a conversion, both exact (4 significant bits,
// exponents -9 .. 8); 8 codes in two words.
__device__ inline u32x4 fp8x8_to_half8(uint32_t lo, uint32_t hi, bf16_t) {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true))};
}
__device__ inline u32x4 fp8x8_to_half8(uint32_t lo, uint32_t hi, f16_t) {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true))};
}

}  // namespace pyc
