// kv_attention.hip — attention of a step's tokens over the paged 8-bit cache.
//
//   o[t,h] = sum_j softmax_j(scale * q[t,h].k_j * sk(block of j)) v_j * sv(block of j),
// token i of the n that a request of `len` tokens brings sees keys j <= len - n + i;
// head h reads kv head h / G, G = q heads / kv heads. Without a key: zero.
//
// One wave works on 16 rows (row r of a request and kv head: token r / G, head
// r % G) and 64 keys at a time, on v_mfma_f32_16x16x32:
//   S^T = K Q^T: K's codes become 16-bit (exact) in registers, Q stays there.
//   Which key a row of the A operand is, is free: row 4g' + i of product t is
//   key 16 g' + 4 t + i, so that lane group g (lanes 16g .. 16g + 15) ends with
//   the scores of keys 16g .. 16g + 15, one chunk of one block: one pair of
//   scales per lane, and P is the B operand of the next product as it is.
//   O^T = V^T P^T: lane group g takes the 16 tokens of its chunk for one channel
//   from the transposed values with one 16-byte load.
// A block's value scale goes into P (p * sv), the sum of p stays without it.
// Statistics and sums are fp32. P is rounded to 16 bits for the product: for bf16
// output once (2^-8 of each p, below the output's own rounding once averaged);
// for f16 output P is split into two bf16 parts (2^-16 left), as bf16 holds any
// block's scale and f16 does not.
//
// Masked places never reach a sum: scores are selected away, tokens behind
// `len` (or of a block id outside the cache) have their value codes cleared, and
// where a row may not see a token that others see, a NaN code is taken out of the
// product and put back by a product of indicators.
#include "kv_cache.hpp"

namespace pyc {

struct AttnArgs {
    KvCache c;
    int B, tokens, hq, G, max_q, width;
    const uint16_t* q;
    int64_t q_stride;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* lens;
    const int32_t* q_offsets;
    uint16_t* o;
    int64_t o_stride;
    float scale_log2;
};

// A request's rows and keys, with what the caller's arrays say held to their bounds.
struct AttnReq {
    int len, n, first;  // keys, tokens, first token's row of q
    int rows;           // rows of a kv head that the call computes
};
__device__ inline AttnReq attn_request(const AttnArgs& a, int b) {
    AttnReq r;
    r.len = (int)min((int64_t)max(a.lens[b], 0), (int64_t)a.width * a.c.bs);
    r.first = min(max(a.q_offsets[b], 0), a.tokens);
    r.n = min(max(a.q_offsets[b + 1], r.first), a.tokens) - r.first;
    r.rows = min(r.n, a.max_q) * a.G;
    return r;
}

__device__ inline uint32_t pack_half2(float lo, float hi, bf16_t) {
    typedef __attribute__((ext_vector_type(2))) float f2;
    typedef __attribute__((ext_vector_type(2))) __bf16 h2;
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{lo, hi}, h2));
}

// Bit 7 of every byte that is a NaN code.
__device__ inline uint32_t nan_codes(uint32_t x) { return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// What a wave keeps for its 16 rows: lane l has row l % 16.
template <int D> struct AttnAcc {
    f32x4 o[D / 16];  // o[dt][i]: channel 16 dt + 4 (l / 16) + i
    float m, l;       // running maximum (base 2) and this lane's part of the sum
};

template <typename T, int D> struct AttnWave {
    static constexpr int KC = D / 64;  // 16-byte chunks of a key per lane
    u32x4 q[2 * KC];
    int limit;  // last key this lane's row sees, negative: none

    // Rows r0 .. r0 + 15 of kv head h.
    __device__ void load_q(const AttnArgs& a, const AttnReq& r, int h, int r0) {
        const int lane = threadIdx.x & 63, row = r0 + (lane & 15), g = lane >> 4;
        const bool live = row < r.rows;  // the others compute the first row's scores, which nobody reads
        const int i = live ? row / a.G : 0, hh = live ? row % a.G : 0;
        limit = live ? r.len - r.n + i : r.len - 1;
        const uint16_t* src = a.q + (int64_t)(r.first + i) * a.q_stride + (int64_t)(h * a.G + hh) * D + 16 * g;
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int u = 0; u < 2; ++u) q[2 * c + u] = *reinterpret_cast<const u32x4*>(src + 64 * c + 8 * u);
    }

    // Keys key0 .. key0 + 63 of request b.
    __device__ void tile(const AttnArgs& a, const AttnReq& r, int b, int h, int key0, AttnAcc<D>& acc) {
        const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4, bs = a.c.bs;
        // the block of chunk x of the tile, -1 where there is none
        auto page_of = [&](int x) {
            const int key = key0 + 16 * x;
            if (key >= r.len) return -1;
            const int id = a.table[b * a.table_stride + key / bs];
            return id >= 0 && id < a.c.blocks ? id : -1;
        };
        const int kp = page_of(l16 >> 2), vp = page_of(g);
        const int koff = (key0 + 16 * (l16 >> 2)) % bs + (l16 & 3), voff = (key0 + 16 * g) % bs;
        const uint8_t* ksrc = a.c.k + max(kp, 0) * a.c.k_stride + ((int64_t)h * bs + koff) * D + 16 * g;
        const uint8_t* vsrc = a.c.v + max(vp, 0) * a.c.v_stride + ((int64_t)h * D + l16) * bs + voff;
        const int valid = vp < 0 ? 0 : min(r.len - (key0 + 16 * g), 16);
        const float sk = a.c.k_scale[(int64_t)max(vp, 0) * a.c.heads + h] * a.scale_log2;
        const float sv = a.c.v_scale[(int64_t)max(vp, 0) * a.c.heads + h];

        f32x4 s[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            s[t] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(ksrc + 4 * t * D + 64 * c);
                s[t] = mfma16x16x32(fp8x8_to_half8(w[0], w[1], T{}), q[2 * c], s[t], T{});
                s[t] = mfma16x16x32(fp8x8_to_half8(w[2], w[3], T{}), q[2 * c + 1], s[t], T{});
            }
        }
        const int seen = min(valid, limit - (key0 + 16 * g) + 1);  // of this lane's 16 keys
        const bool masked = __any(seen < 16);
        float p[16], m = -INFINITY;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            p[j] = s[j >> 2][j & 3] * sk;
            if (masked && j >= seen) p[j] = -INFINITY;
            m = __builtin_elementwise_maximum(m, p[j]);
        }
        m = __builtin_elementwise_maximum(m, __shfl_xor(m, 16));
        m = __builtin_elementwise_maximum(m, __shfl_xor(m, 32));
        m = __builtin_elementwise_maximum(m, acc.m);
        const float ref = m == -INFINITY ? 0.f : m;  // a row that has seen no key yet
        const float keep = __builtin_amdgcn_exp2f(acc.m - ref);
        acc.m = m;
        acc.l *= keep;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) acc.o[dt] *= keep;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            p[j] = __builtin_amdgcn_exp2f(p[j] - ref);
            acc.l += p[j];
            p[j] *= sv;
            if (masked && j >= seen) p[j] = 0.f;  // sv may be anything
        }
        u32x4 hi[2], lo[2];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t x = pack_half2(p[2 * j], p[2 * j + 1], bf16_t{});
            hi[j >> 2][j & 3] = x;
            lo[j >> 2][j & 3] = pack_half2(p[2 * j] - __uint_as_float(x << 16),
                                           p[2 * j + 1] - __uint_as_float(x & 0xffff0000u), bf16_t{});
        }
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) {
            u32x4 w = *reinterpret_cast<const u32x4*>(vsrc + (int64_t)16 * dt * bs);
            uint32_t bad = 0;
            u32x4 ind{0, 0, 0, 0};
            if (masked) {
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int left = valid - 4 * x;  // codes of this word that are a token's
                    if (left < 4) w[x] &= left <= 0 ? 0u : (1u << (8 * left)) - 1u;
                    const uint32_t nan = nan_codes(w[x]) >> 7;
                    bad |= nan;
                    ind[x] = nan * 0x38u;  // 1.0
                    w[x] &= ~(nan * 0xffu);
                }
            }
            const u32x4 v0 = fp8x8_to_half8(w[0], w[1], bf16_t{}), v1 = fp8x8_to_half8(w[2], w[3], bf16_t{});
            acc.o[dt] = mfma16x16x32(v0, hi[0], acc.o[dt], bf16_t{});
            acc.o[dt] = mfma16x16x32(v1, hi[1], acc.o[dt], bf16_t{});
            if constexpr (sizeof(T) == 2 && __is_same(T, f16_t)) {
                acc.o[dt] = mfma16x16x32(v0, lo[0], acc.o[dt], bf16_t{});
                acc.o[dt] = mfma16x16x32(v1, lo[1], acc.o[dt], bf16_t{});
            }
            if (masked && __any(bad != 0)) {
                u32x4 one[2];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    one[j >> 2][j & 3] = (2 * j < seen ? 0x3f80u : 0u) | (2 * j + 1 < seen ? 0x3f800000u : 0u);
                f32x4 hit{0, 0, 0, 0};
                hit = mfma16x16x32(fp8x8_to_half8(ind[0], ind[1], bf16_t{}), one[0], hit, bf16_t{});
                hit = mfma16x16x32(fp8x8_to_half8(ind[2], ind[3], bf16_t{}), one[1], hit, bf16_t{});
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (hit[i] > 0.f) acc.o[dt][i] = __builtin_nanf("");
            }
        }
    }

    // The rows' output: o / sum, zero for a row without a key (or with -inf for every score).
    __device__ void store(const AttnArgs& a, const AttnReq& r, int h, int r0, AttnAcc<D>& acc) {
        const int lane = threadIdx.x & 63, row = r0 + (lane & 15), g = lane >> 4;
        float l = acc.l;
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (row >= r.rows) return;
        const float inv = acc.m == -INFINITY ? 0.f : 1.0f / l;
        uint16_t* dst = a.o + (int64_t)(r.first + row / a.G) * a.o_stride + (int64_t)(h * a.G + row % a.G) * D + 4 * g;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) {
            u32x2 w;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                w[i] = (uint32_t)elem<T>::from_f32(acc.o[dt][2 * i] * inv) |
                       ((uint32_t)elem<T>::from_f32(acc.o[dt][2 * i + 1] * inv) << 16);
            *reinterpret_cast<u32x2*>(dst + 16 * dt) = w;
        }
    }
};

template <typename T, int D>
__global__ void __launch_bounds__(kWave) kv_attn_kernel(AttnArgs a) {
    const int r0 = 16 * blockIdx.x, h = blockIdx.y;
    for (int b = blockIdx.z; b < a.B; b += gridDim.z) {
        const AttnReq r = attn_request(a, b);
        if (r0 >= r.rows) continue;
        AttnWave<T, D> w;
        w.load_q(a, r, h, r0);
        AttnAcc<D> acc;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) acc.o[dt] = f32x4{0, 0, 0, 0};
        acc.m = -INFINITY;
        acc.l = 0.f;
        // keys that the tile's last row sees
        const int last = min(r0 + 15, r.rows - 1) / a.G, end = max(0, r.len - r.n + last + 1);
        for (int key0 = 0; key0 < end; key0 += 64) w.tile(a, r, b, h, key0, acc);
        w.store(a, r, h, r0, acc);
    }
}

}  // namespace pyc

extern "C" size_t pyc_hip_kv_attention_workspace_bytes(int B, int hq, int hk, int d, int max_q) { return 16; }

extern "C" int pyc_hip_kv_attention_launch(int is_bf16, const pyc_hip_kv_cache* cache, int B, int tokens, int hq,
                                           int max_q, int max_len, const void* q, int64_t q_stride,
                                           const int32_t* table, int64_t table_stride, int width, const int32_t* lens,
                                           const int32_t* q_offsets, void* o, int64_t o_stride, float scale,
                                           void* workspace, void* stream) {
    using namespace pyc;
    AttnArgs a;
    a.c = kv_cache_of(cache);
    a.B = B;
    a.tokens = tokens;
    a.hq = hq;
    a.G = hq / a.c.heads;
    a.max_q = max_q;
    a.width = width;
    a.q = (const uint16_t*)q;
    a.q_stride = q_stride;
    a.table = table;
    a.table_stride = table_stride;
    a.lens = lens;
    a.q_offsets = q_offsets;
    a.o = (uint16_t*)o;
    a.o_stride = o_stride;
    a.scale_log2 = scale * 1.44269504088896340736f;
    const long rows = (long)(max_q < tokens ? max_q : tokens) * a.G;
    const dim3 grid((unsigned)((rows + 15) / 16), a.c.heads, B < 65535 ? B : 65535), block(kWave);
    hipStream_t s = (hipStream_t)stream;
    if (a.c.d == 128) {
        if (is_bf16) hipLaunchKernelGGL((kv_attn_kernel<bf16_t, 128>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((kv_attn_kernel<f16_t, 128>), grid, block, 0, s, a);
    } else {
        if (is_bf16) hipLaunchKernelGGL((kv_attn_kernel<bf16_t, 64>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((kv_attn_kernel<f16_t, 64>), grid, block, 0, s, a);
    }
    return hipGetLastError() == hipSuccess ? 0 : -2;
}

extern "C" int pyc_hip_kinfo_kv_attention(int is_bf16, pyc_hip_kinfo* out) {
    using namespace pyc;
    if (!out) return -1;
    out->fn = is_bf16 ? reinterpret_cast<const void*>(&kv_attn_kernel<bf16_t, 128>)
                      : reinterpret_cast<const void*>(&kv_attn_kernel<f16_t, 128>);
    out->name = "kv_attn_kernel<128>";
    out->lds_bytes = 0;
    out->threads = kWave;
    out->waves_per_simd = 2;
    return 0;
}
