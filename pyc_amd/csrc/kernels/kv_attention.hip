// kv_attention.hip — attention of a step's tokens over the paged 8-bit cache.
//
//   o[t,h] = sum_j softmax_j(scale * q[t,h].k_j * sk(block of j)) v_j * sv(block of j),
// token i of the n that a request of `len` tokens brings sees keys j <= len - n + i;
// head h reads kv head h / G, G = q heads / kv heads. Without a key: zero.
//
// Rows are (token, head of the group): row r of a request and kv head is token r / G, head
// r % G. Two kernels: the split kernel for requests of few rows, bound by reading the
// cache, and the chunk kernels for many, bound by matrix and softmax work; a batch that
// has both goes out in one launch. In the split kernel a wave works on 16 NT rows and 64
// keys at a time, on v_mfma_f32_16x16x32:
//   S^T = K Q^T: K's codes become 16-bit (exact) in registers, Q stays there.
//   Which key a row of the A operand is, is free: row 4g' + i of product t is
//   key 16 g' + 4 t + i, so that lane group g (lanes 16g .. 16g + 15) ends with
//   the scores of keys 16g .. 16g + 15, one chunk of one block: one pair of
//   scales per lane, and P is the B operand of the next product as it is.
//   O^T = V^T P^T: lane group g takes the 16 tokens of its chunk for one channel
//   from the transposed values with one 16-byte load.
// A block's value scale goes into P (p * sv), the sum of p stays without it.
// Statistics and sums are fp32. (8-bit matrix products of codes, q as two of them, would
// run at twice the rate for half the work, but add their 64 products with fewer
// bits: scores near 170 came out off by 0.01. So both operands are 16-bit.) P is
// rounded to 16 bits for the product: for bf16 output once (2^-8 of each p at most), which
// adds about as much as the output's own rounding: 2.3e-3 of the result's norm against
// 64 bits where 1.65e-3 is the output's alone. For f16 output P is split into two bf16
// parts (2^-16 left), as bf16 holds any block's scale and f16 does not; the second product
// takes 497 us where one takes 390 (4 chunks of 2048 tokens over 3800 keys) and 33.6 where
// one takes 32.6 (32 single tokens), too much for the half bit it would give bf16.
//
// Masked places never reach a sum: scores are selected away, tokens behind
// `len` (or of a block id outside the cache) have their value codes cleared, and
// where a row may not see a token that others see, a NaN code is taken out of the
// product and put back by a product of indicators.
#include <type_traits>

#include "kv_cache.hpp"
#include "lds_dma.hpp"

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

// Values that are the same in all lanes, into scalar registers.
__device__ inline int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ inline int64_t uniform(int64_t x) {
    return (int64_t)(((uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32) | (uint32_t)uniform((int)x));
}
__device__ inline AttnReq uniform(const AttnReq& r) {
    return AttnReq{uniform(r.len), uniform(r.n), uniform(r.first), uniform(r.rows)};
}

__device__ inline int64_t wave_prefix(int64_t x) {
    return wave_scan(x, (int64_t)0, [](int64_t a, int64_t b) { return a + b; });
}
__device__ inline float wave_sum(float x) {
    return read_lane(wave_scan(x, 0.f, [](float a, float b) { return a + b; }), 63);
}
__device__ inline float wave_max(float x) {
    return read_lane(wave_scan(x, -INFINITY, [](float a, float b) { return __builtin_elementwise_maximum(a, b); }), 63);
}
__device__ inline int wave_max(int x) {
    return __builtin_amdgcn_readlane(wave_scan(x, 0, [](int a, int b) { return max(a, b); }), 63);
}

__device__ inline uint32_t pack_half2(float lo, float hi, bf16_t) {
    typedef __attribute__((ext_vector_type(2))) float f2;
    typedef __attribute__((ext_vector_type(2))) __bf16 h2;
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{lo, hi}, h2));
}

// Bit 7 of every byte that is a NaN code.
__device__ inline uint32_t nan_codes(uint32_t x) { return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// The blocks and scales of 16 tiles of 64 keys: lane l has chunk l % 4 of tile l / 4.
struct AttnPages {
    int id;  // -1: none
    float sk, sv;
};
__device__ inline AttnPages attn_pages(const AttnArgs& a, const AttnReq& r, int b, int h, int tile0) {
    const int lane = threadIdx.x & 63;
    const int64_t key = 64 * ((int64_t)tile0 + (lane >> 2)) + 16 * (lane & 3);
    AttnPages p;
    p.id = -1;
    if (key < r.len) p.id = a.table[b * a.table_stride + key / a.c.bs];
    if (p.id < 0 || p.id >= a.c.blocks) p.id = -1;
    const int64_t at = (int64_t)max(p.id, 0) * a.c.heads + h;
    p.sk = a.c.k_scale[at] * a.scale_log2;
    p.sv = a.c.v_scale[at];
    return p;
}

// NT times 16 rows of one wave: lane l has rows l % 16, 16 + l % 16, ...
template <typename T, int D, int NT> struct AttnWave {
    static constexpr int KC = D / 64;   // 16-byte chunks of a key per lane
    static constexpr int DT = D / 16;   // 16-channel tiles of the output
    u32x4 q[NT][2 * KC];
    int limit[NT];  // last key the row sees, negative: none
    u32x4 k[4 * KC], v[DT];
    f32x4 o[NT][DT];        // o[n][dt][i]: channel 16 dt + 4 (l / 16) + i
    float m[NT], l[NT];     // running maximum (base 2) and this lane's part of the sum

    // Rows r0 .. r0 + 16 NT - 1 of kv head h.
    __device__ void begin(const AttnArgs& a, const AttnReq& r, int h, int r0) {
        const int lane = threadIdx.x & 63, g = lane >> 4;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int row = r0 + 16 * n + (lane & 15);
            const bool live = row < r.rows;  // the others compute the first row's scores, which nobody reads
            const int i = live ? row / a.G : 0, hh = live ? row % a.G : 0;
            limit[n] = live ? r.len - r.n + i : r.len - 1;
            const uint16_t* src = a.q + (int64_t)(r.first + i) * a.q_stride + (int64_t)(h * a.G + hh) * D + 16 * g;
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int u = 0; u < 2; ++u) q[n][2 * c + u] = *reinterpret_cast<const u32x4*>(src + 64 * c + 8 * u);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[n][dt] = f32x4{0, 0, 0, 0};
            m[n] = -INFINITY;
            l[n] = 0.f;
        }
    }

    // Tile j (of 16) of the pages: its keys, and its values.
    __device__ void load_k(const AttnArgs& a, const AttnPages& p, int h, int tile, int j) {
        const int lane = threadIdx.x & 63, l16 = lane & 15, bs = a.c.bs;
        const int id = max(__shfl(p.id, 4 * j + (l16 >> 2)), 0);
        const int off = ((64 * tile + 16 * (l16 >> 2)) & (bs - 1)) + (l16 & 3);
        const uint8_t* src = a.c.k + id * a.c.k_stride + ((int64_t)h * bs + off) * D + 16 * (lane >> 4);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int c = 0; c < KC; ++c) k[t * KC + c] = *reinterpret_cast<const u32x4*>(src + 4 * t * D + 64 * c);
    }
    __device__ void load_v(const AttnArgs& a, const AttnPages& p, int h, int tile, int j) {
        const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4, bs = a.c.bs;
        const int id = max(__shfl(p.id, 4 * j + g), 0);
        const uint8_t* src =
            a.c.v + id * a.c.v_stride + ((int64_t)h * D + l16) * bs + ((64 * tile + 16 * g) & (bs - 1));
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) v[dt] = *reinterpret_cast<const u32x4*>(src + (int64_t)16 * dt * bs);
    }

    __device__ void scores(f32x4 (&s)[NT][4]) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int t = 0; t < 4; ++t) s[n][t] = f32x4{0, 0, 0, 0};
        // two products at a time: a sum's next term waits for the one before it
#pragma unroll
        for (int t = 0; t < 4; t += 2)
#pragma unroll
            for (int c = 0; c < KC; ++c) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const u32x4 w0 = k[t * KC + c], w1 = k[(t + 1) * KC + c];
                    const u32x4 k0 = fp8x8_to_half8(w0[2 * u], w0[2 * u + 1], T{});
                    const u32x4 k1 = fp8x8_to_half8(w1[2 * u], w1[2 * u + 1], T{});
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        s[n][t] = mfma16x16x32(k0, q[n][2 * c + u], s[n][t], T{});
                        s[n][t + 1] = mfma16x16x32(k1, q[n][2 * c + u], s[n][t + 1], T{});
                    }
                }
                __builtin_amdgcn_sched_barrier(0);  // else every code is converted first, into registers there are not
            }
    }

    // Softmax and the product with the values, which are in v.
    __device__ void finish(const AttnReq& r, const AttnPages& pg, int tile, int j, f32x4 (&s)[NT][4]) {
        const int g = (threadIdx.x & 63) >> 4, key = 64 * tile + 16 * g;  // this lane's 16 keys
        const float sk = __shfl(pg.sk, 4 * j + g), sv = __shfl(pg.sv, 4 * j + g);
        const int valid = __shfl(pg.id, 4 * j + g) < 0 ? 0 : min(r.len - key, 16);
        int seen[NT];
        bool part = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            seen[n] = min(valid, limit[n] - key + 1);
            part |= seen[n] < 16;
        }
        const bool masked = __any(part);
        u32x4 hi[NT][2], lo[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float p[16], mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; ++i) p[i] = s[n][i >> 2][i & 3] * sk;
            if (masked) {
#pragma unroll
                for (int i = 0; i < 16; ++i) p[i] = i < seen[n] ? p[i] : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = __builtin_elementwise_maximum(mx, p[i]);
            mx = __builtin_elementwise_maximum(mx, __shfl_xor(mx, 16));
            mx = __builtin_elementwise_maximum(mx, __shfl_xor(mx, 32));
            mx = __builtin_elementwise_maximum(mx, m[n]);
            const float ref = mx == -INFINITY ? 0.f : mx;  // a row that has seen no key yet
            if (__any(mx != m[n])) {
                const float keep = __builtin_amdgcn_exp2f(m[n] - ref);
                l[n] *= keep;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) o[n][dt] *= keep;
            }
            m[n] = mx;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                p[i] = __builtin_amdgcn_exp2f(p[i] - ref);
                l[n] += p[i];
                p[i] *= sv;
            }
            if (masked) {  // sv may be anything
#pragma unroll
                for (int i = 0; i < 16; ++i) p[i] = i < seen[n] ? p[i] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t x = pack_half2(p[2 * i], p[2 * i + 1], bf16_t{});
                hi[n][i >> 2][i & 3] = x;
                if constexpr (__is_same(T, f16_t))
                    lo[n][i >> 2][i & 3] = pack_half2(p[2 * i] - __uint_as_float(x << 16),
                                                      p[2 * i + 1] - __uint_as_float(x & 0xffff0000u), bf16_t{});
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (masked) values_masked(valid, seen);
#pragma unroll
        for (int dt = 0; dt < DT; dt += 2) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const u32x4 v0 = fp8x8_to_half8(v[dt][2 * u], v[dt][2 * u + 1], bf16_t{});
                const u32x4 v1 = fp8x8_to_half8(v[dt + 1][2 * u], v[dt + 1][2 * u + 1], bf16_t{});
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    o[n][dt] = mfma16x16x32(v0, hi[n][u], o[n][dt], bf16_t{});
                    o[n][dt + 1] = mfma16x16x32(v1, hi[n][u], o[n][dt + 1], bf16_t{});
                    if constexpr (__is_same(T, f16_t)) {
                        o[n][dt] = mfma16x16x32(v0, lo[n][u], o[n][dt], bf16_t{});
                        o[n][dt + 1] = mfma16x16x32(v1, lo[n][u], o[n][dt + 1], bf16_t{});
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // Takes out of v what a row must not see: the codes behind `valid`, and NaN
    // codes, which become NaN sums of exactly the rows that see them.
    __device__ void values_masked(int valid, const int (&seen)[NT]) {
        uint32_t word[4], bad = 0;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int left = valid - 4 * x;  // codes of this word that are a token's
            word[x] = left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                v[dt][x] &= word[x];
                bad |= nan_codes(v[dt][x]);
            }
        if (!__any(bad != 0)) return;
        u32x4 one[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                one[n][i >> 2][i & 3] = (2 * i < seen[n] ? 0x3f80u : 0u) | (2 * i + 1 < seen[n] ? 0x3f800000u : 0u);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            u32x4 ind;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const uint32_t nan = nan_codes(v[dt][x]) >> 7;
                ind[x] = nan * 0x38u;  // 1.0
                v[dt][x] &= ~(nan * 0xffu);
            }
            const u32x4 i0 = fp8x8_to_half8(ind[0], ind[1], bf16_t{}), i1 = fp8x8_to_half8(ind[2], ind[3], bf16_t{});
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                f32x4 hit{0, 0, 0, 0};
                hit = mfma16x16x32(i0, one[n][0], hit, bf16_t{});
                hit = mfma16x16x32(i1, one[n][1], hit, bf16_t{});
#pragma unroll
                for (int i = 0; i < 4; ++i) o[n][dt][i] = hit[i] > 0.f ? __builtin_nanf("") : o[n][dt][i];
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // Tiles t0 .. t1 - 1 of request b: a tile's loads are in flight while the one
    // before it is computed, its keys from its scores on, its values to its end.
    __device__ void run(const AttnArgs& a, const AttnReq& r, int b, int h, int t0, int t1) {
        if (t0 >= t1) return;
        AttnPages pg = attn_pages(a, r, b, h, t0), nx = pg;
        load_k(a, pg, h, t0, 0);
        load_v(a, pg, h, t0, 0);
        for (int t = t0; t < t1; ++t) {
            const int j = (t - t0) & 15, jn = (j + 1) & 15;
            if (j == 0 && t + 16 < t1) nx = attn_pages(a, r, b, h, t + 16);
            const AttnPages ld = jn == 0 ? nx : pg;
            f32x4 s[NT][4];
            scores(s);
            if (t + 1 < t1) load_k(a, ld, h, t + 1, jn);
            finish(r, pg, t, j, s);
            if (t + 1 < t1) load_v(a, ld, h, t + 1, jn);
            pg = ld;
        }
    }

    // The rows' output: o / sum, zero for a row without a key (or with -inf for every score).
    __device__ void store(const AttnArgs& a, const AttnReq& r, int h, int r0) {
        const int lane = threadIdx.x & 63, g = lane >> 4;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int row = r0 + 16 * n + (lane & 15);
            float sum = l[n];
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (row >= r.rows) continue;
            const float inv = m[n] == -INFINITY ? 0.f : 1.0f / sum;
            uint16_t* dst = a.o + (int64_t)(r.first + row / a.G) * a.o_stride + (int64_t)(h * a.G + row % a.G) * D + 4 * g;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                u32x2 w;
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    w[i] = (uint32_t)elem<T>::from_f32(o[n][dt][2 * i] * inv) |
                           ((uint32_t)elem<T>::from_f32(o[n][dt][2 * i + 1] * inv) << 16);
                *reinterpret_cast<u32x2*>(dst + 16 * dt) = w;
            }
        }
    }

    // A part of the rows' keys: sums in rows of D + 4 (off the banks' stride), maximum and sum of p.
    __device__ void store_part(int live, float* sums, float* ml) {
        const int lane = threadIdx.x & 63, g = lane >> 4;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int row = 16 * n + (lane & 15);
            float sum = l[n];
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (row >= live) continue;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(sums + row * (D + 4) + 16 * dt + 4 * g) = o[n][dt];
            if (g == 0) {
                ml[2 * row] = m[n];
                ml[2 * row + 1] = sum;
            }
        }
    }
};

// ---------------------------------------------------------------------------
// Requests of few rows (decoding, draft tokens): reading the cache is the work, so
// it is cut evenly. A request of up to most_rows rows has, for every kv head and every
// 16 NT rows, a run of tiles of 64 keys; all runs, one after the other, are cut into
// one piece for each wave. What a wave finds of a run it leaves in LDS unless it has
// all of it; the workgroup joins what its waves have of one run, and where a run goes
// on in other workgroups, the last of these to be done joins all. Up to 256 short runs
// get a workgroup each instead: then no run crosses one.
// Even pieces against one workgroup for a request and head: no CU waits for the longest
// context, and two requests of 100000 keys use the card as 64 of 3000 do. Measured, 32
// heads of 128 in bf16: 2 contexts of 100000 to 131072 keys, 8 kv heads, 83.5 us (5.2
// TB/s, what a copy reaches); 64 of 300 to 6000, 32 kv heads, 216 us (5.4 TB/s); 32 of
// 200 to 4096, 8 kv heads, 27 us (3.8 TB/s: what it takes to start, to find the work and to
// join is 7 of them); one of 777, 10.3 us, which is latency: its 8 runs of 13 tiles are a
// workgroup's each, up to two tiles to a wave, one after the other, behind loads that wait for
// each other (lengths, ids, scales and codes), with a join in LDS and no counter. With 32
// rows to a wave (NT 2; four heads to a kv head): 16 requests over 3000 to 3750 keys, 5 tokens
// each, one run, 43 us; 16 tokens each, two runs, 70.
struct AttnSplit {
    int most_rows;
    float* part;     // two results of every workgroup: [16 NT][D] sums, [16 NT][2] maximum and sum
    uint32_t* done;  // for every run that workgroups share: how many are done; zero between calls
};
constexpr int kSplitGroups = 256;
// Two waves on a SIMD where their registers allow it.
__host__ __device__ constexpr int split_waves(int nt, int d) { return nt == 1 || d == 64 ? 8 : 4; }

struct SplitPart {  // a part of a run in LDS
    int b, h, rt, t0, t1, tiles, live, first;
    int64_t begin;  // the run's first unit
};
template <int D, int NT> struct SplitShare {
    static constexpr int WAVES = split_waves(NT, D), ROWS = 16 * NT;
    float sums[2 * WAVES][ROWS][D + 4];
    float ml[2 * WAVES][ROWS][2];
    SplitPart part[2 * WAVES];
    int last[2];
};

// Tiles of a request's runs (0: it is not the split kernel's), and its runs of a head.
__device__ inline int split_tiles(const AttnArgs& a, const AttnReq& r, int most_rows) {
    if (r.rows <= 0 || r.rows > most_rows) return 0;
    const int end = r.len - r.n + r.rows / a.G;  // keys that the last row sees
    return max(1, end / 64 + (end % 64 > 0 ? 1 : 0));
}
// 64-bit quotients are slow and rarely needed.
__device__ inline uint64_t div_u64(uint64_t n, uint64_t d) {
    return ((n | d) >> 32) == 0 ? (uint32_t)n / (uint32_t)d : n / d;
}
// Piece w of W begins at floor(total w / W); the last piece that begins at or before
// u. There are fewer than 2^12 pieces and 2^50 units: no product passes 64 bits.
__device__ inline int64_t piece_begin(int64_t total, int W, int w) { return (int64_t)div_u64((uint64_t)total * w, W); }
__device__ inline int piece_of(int64_t total, int W, int64_t u) {
    return (int)div_u64((uint64_t)(u + 1) * W - 1, (uint64_t)total);
}

template <typename T, int D> struct SplitRow {  // a row of results, D / 64 channels a lane
    static constexpr int E = D / 64;
    float x[E], m, l;
    __device__ void store(const AttnArgs& a, const SplitPart& p, int row) const {
        const int lane = threadIdx.x & 63, at = p.rt + row;  // row of the request and head
        const float inv = m == -INFINITY ? 0.f : 1.0f / l;
        uint16_t* dst = a.o + (int64_t)(p.first + at / a.G) * a.o_stride + (int64_t)(p.h * a.G + at % a.G) * D + E * lane;
        if constexpr (E == 2)
            *reinterpret_cast<uint32_t*>(dst) =
                (uint32_t)elem<T>::from_f32(x[0] * inv) | ((uint32_t)elem<T>::from_f32(x[1] * inv) << 16);
        else
            *dst = elem<T>::from_f32(x[0] * inv);
    }
};
__device__ inline uint64_t pack_floats(float a, float b) {
    return (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32);
}
// Accesses to what workgroups on other XCDs read or wrote (their L2 caches are not coherent).
__device__ inline void agent_store(uint64_t* p, uint64_t v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline uint64_t agent_load(const uint64_t* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Workgroup wg of `groups`.
template <typename T, int D, int NT>
__device__ inline void split_body(const AttnArgs& a, const AttnSplit& sp, SplitShare<D, NT>& sh, int wg, int groups) {
    constexpr int WAVES = split_waves(NT, D), ROWS = 16 * NT, E = D / 64;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    // Lane i's request is the i-th of a batch's first 64; larger batches are looked at again.
    const AttnReq near = lane < a.B ? attn_request(a, lane) : AttnReq{0, 0, 0, 0};
    auto request = [&](int b) {
        if (b >= kWave) return uniform(attn_request(a, b));
        return AttnReq{__builtin_amdgcn_readlane(near.len, b), __builtin_amdgcn_readlane(near.n, b),
                       __builtin_amdgcn_readlane(near.first, b), __builtin_amdgcn_readlane(near.rows, b)};
    };
    auto runs_of = [&](const AttnReq& r) { return (r.rows + ROWS - 1) / ROWS; };
    auto work_of = [&](int b0, int* runs) {  // tiles and runs of request b0 + lane
        const AttnReq r = b0 == 0 ? near : b0 + lane < a.B ? attn_request(a, b0 + lane) : AttnReq{0, 0, 0, 0};
        const int t = split_tiles(a, r, sp.most_rows);
        *runs = t ? runs_of(r) : 0;
        return t;
    };
    // All units (tiles of all runs), all runs, the longest run.
    int64_t total = 0, runs = 0, units0 = 0, runs0 = 0;  // and the first 64 requests' prefix sums
    int longest = 0;
    for (int b0 = 0; b0 < a.B; b0 += kWave) {
        int n;
        const int t = work_of(b0, &n);
        const int64_t ut = wave_prefix((int64_t)t * n), rn = wave_prefix((int64_t)n);
        if (b0 == 0) {
            units0 = ut;
            runs0 = rn;
        }
        total += read_lane(ut, kWave - 1);
        runs += read_lane(rn, kWave - 1);
        longest = max(longest, t);
    }
    total *= a.c.heads;
    runs *= a.c.heads;
    const bool aligned = runs <= groups && wave_max(longest) <= 2 * WAVES;
    const int W = (int)min((int64_t)groups * WAVES, total);

    // This wave's piece: `left` units from tile t0 of run (b, h, rt); unit u of all.
    int64_t u = 0, left = 0, before = 0;
    int b = 0, h = 0, rt = 0, t0 = 0;
    const int w = wg * WAVES + wave;
    if (aligned) {
        u = wg;  // a run here, counted below as a unit
        left = wg < runs ? 1 : 0;
    } else if (w < W) {
        u = piece_begin(total, W, w);
        left = piece_begin(total, W, w + 1) - u;
    }
    if (left > 0) {
        int64_t base = 0;
        for (int b0 = 0; b0 < a.B; b0 += kWave) {
            int64_t end = aligned ? runs0 : units0;
            if (b0) {
                int n;
                const int t = work_of(b0, &n);
                end = wave_prefix((int64_t)n * (aligned ? 1 : t));
            }
            end = base + end * a.c.heads;
            const uint64_t past = __ballot(end > u);
            if (past) {
                const int i = __builtin_ctzll(past);
                before = i ? read_lane(end, i - 1) : base;
                b = b0 + i;
                break;
            }
            base = read_lane(end, kWave - 1);
        }
    }
    b = uniform(b);
    before = uniform(before);
    AttnReq r = request(b);
    int tiles = split_tiles(a, r, sp.most_rows), n_rt = runs_of(r);
    if (left > 0) {
        const int64_t v = u - before;
        const int64_t run = aligned ? v : (int64_t)div_u64(v, tiles);
        h = (int)div_u64(run, n_rt);
        rt = (int)(run - (int64_t)h * n_rt);
        if (aligned) {  // the workgroup's run, a piece for each wave
            t0 = tiles * wave / WAVES;
            left = tiles * (wave + 1) / WAVES - t0;
            u = t0;  // not looked at again but for u - t0, the run's first unit
        } else {
            t0 = (int)(v - run * tiles);
        }
    }
    h = uniform(h);
    rt = uniform(rt);
    t0 = uniform(t0);
    u = uniform(u);
    left = uniform(left);
    if (lane < 2) sh.part[2 * wave + lane].t1 = 0;
    while (left > 0) {
        const int t1 = (int)min((int64_t)tiles, t0 + left);
        AttnWave<T, D, NT> wv;
        wv.begin(a, r, h, ROWS * rt);
        wv.run(a, r, b, h, t0, t1);
        if (t0 == 0 && t1 == tiles) {
            wv.store(a, r, h, ROWS * rt);
        } else {
            const int at = 2 * wave + (t0 == 0 ? 1 : 0), live = min(r.rows - ROWS * rt, ROWS);
            wv.store_part(live, &sh.sums[at][0][0], &sh.ml[at][0][0]);
            if (lane == 0) sh.part[at] = SplitPart{b, h, ROWS * rt, t0, t1, tiles, live, r.first, u - t0};
        }
        u += t1 - t0;
        left -= t1 - t0;
        if (left <= 0) break;
        t0 = 0;
        if (++rt == n_rt) {
            rt = 0;
            if (++h == a.c.heads) {
                h = 0;
                do {
                    r = request(++b);
                    tiles = split_tiles(a, r, sp.most_rows);
                } while (tiles == 0);  // ends: there are units left
                n_rt = runs_of(r);
            }
        }
    }
    __syncthreads();

    // Join the parts in LDS. Lane i has part i's head: a part at 2 w + 1 begins a run,
    // one at 2 w goes on with the part before it (of another workgroup, if it is the first).
    SplitPart mine = sh.part[min(lane, 2 * WAVES - 1)];
    if (lane >= 2 * WAVES) mine.t1 = 0;
    const uint64_t have = __ballot(mine.t1 > 0);
    uint64_t begins = __ballot(mine.t1 > 0 && (mine.t0 == 0 || (have & ((1ull << lane) - 1)) == 0));
    int shared = 0;             // runs that go beyond this workgroup: at most its first and its last
    int shared_at[2] = {0, 0};  // a part of each
    for (uint64_t left_runs = begins; left_runs; left_runs &= left_runs - 1) {
        const int i = __builtin_ctzll(left_runs);
        const uint64_t later = left_runs & (left_runs - 1);
        const uint64_t parts = have & (~0ull << i) & (later ? (1ull << __builtin_ctzll(later)) - 1 : ~0ull);
        const int last = 63 - __builtin_clzll(parts);
        const SplitPart& p = sh.part[i];
        const bool whole = p.t0 == 0 && sh.part[last].t1 == p.tiles;
        float* dst = sp.part + (2 * (int64_t)wg + (p.t0 == 0 ? 1 : 0)) * (ROWS * (D + 2));
        for (int row = wave; row < p.live; row += WAVES) {
            const bool in = (parts >> lane) & 1;
            const int li = min(lane, 2 * WAVES - 1);
            const float pm = in ? sh.ml[li][row][0] : -INFINITY, pl = in ? sh.ml[li][row][1] : 0.f;
            SplitRow<T, D> o;
            o.m = wave_max(pm);
            const float wgt = __builtin_amdgcn_exp2f(pm - (o.m == -INFINITY ? 0.f : o.m));
            o.l = wave_sum(in ? pl * wgt : 0.f);
#pragma unroll
            for (int e = 0; e < E; ++e) o.x[e] = 0.f;
            for (uint64_t k = parts; k;) {  // four at a time: an LDS read takes longer than the rest
                int j[4];
                float f[4], x[4][E];
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    j[y] = k ? __builtin_ctzll(k) : j[0];
                    f[y] = k ? read_lane(wgt, j[y]) : 0.f;
                    k &= k - 1;
                }
#pragma unroll
                for (int y = 0; y < 4; ++y)
#pragma unroll
                    for (int e = 0; e < E; ++e) x[y][e] = sh.sums[j[y]][row][E * lane + e];
#pragma unroll
                for (int y = 0; y < 4; ++y)
#pragma unroll
                    for (int e = 0; e < E; ++e) o.x[e] += f[y] * x[y][e];
            }
            if (whole) {
                o.store(a, p, row);
            } else {
                if constexpr (E == 2)
                    agent_store(reinterpret_cast<uint64_t*>(dst + row * D) + lane, pack_floats(o.x[0], o.x[1]));
                else
                    __hip_atomic_store(dst + row * D + lane, o.x[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                if (lane == 0) agent_store(reinterpret_cast<uint64_t*>(dst + ROWS * D) + row, pack_floats(o.m, o.l));
            }
        }
        if (!whole) shared_at[shared++ & 1] = i;
    }
    if (shared == 0) return;
    // Count the workgroup in; the last one of a run joins it.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's stores are where others see them
    __syncthreads();
    const int n_rt_most = (sp.most_rows + ROWS - 1) / ROWS;
    if (threadIdx.x < shared) {
        const SplitPart& p = sh.part[shared_at[threadIdx.x]];
        const int w0 = piece_of(total, W, p.begin) / WAVES, w1 = piece_of(total, W, p.begin + p.tiles - 1) / WAVES;
        uint32_t* done = sp.done + ((int64_t)p.b * a.c.heads + p.h) * n_rt_most + p.rt / ROWS;
        const uint32_t before_me = __hip_atomic_fetch_add(done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const bool last = before_me == (uint32_t)(w1 - w0);
        if (last) __hip_atomic_store(done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        sh.last[threadIdx.x] = last ? w1 - w0 + 1 : 0;
        sh.part[shared_at[threadIdx.x]].t1 = w0;  // t1 has been used
    }
    __syncthreads();
    for (int k = 0; k < shared; ++k) {
        const int n = sh.last[k];
        if (n == 0) continue;
        const SplitPart& p = sh.part[shared_at[k]];
        const int w0 = p.t1;
        // workgroup w0 + i's result: of the run that it ends with, for the others the one they begin with
        auto src = [&](int i) { return sp.part + (2 * (int64_t)(w0 + i) + (i == 0 ? 1 : 0)) * (ROWS * (D + 2)); };
        for (int row = wave; row < p.live; row += WAVES) {
            SplitRow<T, D> o;
            o.m = -INFINITY;
            o.l = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) o.x[e] = 0.f;
            for (int i0 = 0; i0 < n; i0 += kWave) {
                const int cnt = min(n - i0, kWave), mi = min(i0 + lane, n - 1);
                uint64_t x[8];
                auto load = [&](int i) {  // results i .. i + 7 of the 64
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float* from = src(i0 + min(i + j, cnt - 1)) + row * D;
                        if constexpr (E == 2) x[j] = agent_load(reinterpret_cast<const uint64_t*>(from) + lane);
                        else
                            x[j] = __float_as_uint(__hip_atomic_load(from + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
                    }
                };
                const uint64_t v = agent_load(reinterpret_cast<const uint64_t*>(src(mi) + ROWS * D) + row);
                load(0);  // while the weights are made
                const bool in = lane < cnt;
                const float pm = in ? __uint_as_float((uint32_t)v) : -INFINITY, pl = __uint_as_float((uint32_t)(v >> 32));
                const float mx = __builtin_elementwise_maximum(o.m, wave_max(pm)), ref = mx == -INFINITY ? 0.f : mx;
                const float keep = __builtin_amdgcn_exp2f(o.m - ref), wgt = __builtin_amdgcn_exp2f(pm - ref);
                o.m = mx;
                o.l = o.l * keep + wave_sum(in ? pl * wgt : 0.f);
#pragma unroll
                for (int e = 0; e < E; ++e) o.x[e] *= keep;
                for (int i = 0; i < cnt; i += 8) {
                    if (i) load(i);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float f = i + j < cnt ? read_lane(wgt, min(i + j, cnt - 1)) : 0.f;
                        o.x[0] += f * __uint_as_float((uint32_t)x[j]);
                        if constexpr (E == 2) o.x[1] += f * __uint_as_float((uint32_t)(x[j] >> 32));
                    }
                }
            }
            o.store(a, p, row);
        }
    }
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(split_waves(NT, D) * kWave, 1) kv_split_kernel(AttnArgs a, AttnSplit sp) {
    __shared__ SplitShare<D, NT> sh;
    split_body<T, D, NT>(a, sp, sh, blockIdx.x, gridDim.x);
}

// ---------------------------------------------------------------------------
// Requests of many rows (prompt chunks): matrix work. A workgroup's 8 waves have 32 rows
// each. On v_mfma_f32_32x32x16, as above: S^T = K Q^T with the keys of a tile of 64 ordered
// so that a lane ends with 16 keys of one chunk of each half tile, O^T += V^T P^T with P as
// it is. Tiles come by LDS-DMA, as codes, into a ring. A SIMD's two waves are one phase
// apart: while one runs matrix instructions (phase M: the products of this tile and
// the scores of the next), the other runs its softmax (phase V).
// GROUPS 2: 128 rows, 4 waves for them, twice; the two groups take tiles in turn and join at
// the end. GROUPS 1: 256 rows, all waves on the same tiles. A part costs 14 us that are
// not its tiles (start, first loads, join), so 256 rows are better where they save rounds of
// workgroups, and worse where the card is not full (figures at the launch). With one group LDS has room for the tiles converted to 16
// bits, once for the workgroup instead of once for each wave.
// Measured, 32 heads of 128, 8 kv heads, bf16: 4 chunks of 2048 tokens over 3500 to 4100 keys
// 370 to 390 us by the card, 0.92 to 0.98 PFLOP/s (1.10 over 16384 keys; a large
// library product reaches 1.44). Of a tile's 4000 cycles the matrix unit is busy for 2048: phase M takes 1850
// (its 34 16-byte reads a lane, for four waves, are 1100 cycles of LDS beside 1024 of
// products), phase V 1700 (32 exponentials, 32 scalings, 32 additions, 16 roundings:
// between the other wave's products a vector instruction issues about every 7 cycles).
constexpr int chunk_rows(int groups) { return 256 / groups; }
constexpr int kChunkRing = 4;
constexpr int kChunkThreads = 512;
__device__ inline f32x16 mfma32x32x16(const u32x4& a, const u32x4& b, const f32x16& c, bf16_t) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ inline f32x16 mfma32x32x16(const u32x4& a, const u32x4& b, const f32x16& c, f16_t) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Row tiles of a request in the chunk kernel.
__device__ inline int chunk_tiles(const AttnReq& r, int from_rows, int part_rows) {
    return r.rows > from_rows ? (r.rows + part_rows - 1) / part_rows : 0;
}

// The reference m of a row is its maximum over the first tile that shows it a key,
// raised only when a later tile's sum of p passes 2^14: p stays far from
// overflow in bf16 (whose exponents are fp32's), and the common path has no maximum.
constexpr float kChunkSumMax = 16384.0f;

template <int D, int GROUPS> struct ChunkShare {
    static constexpr int TILE = 64 * D;
    // One group: the codes go on as 16-bit numbers, converted once by the wave that loaded
    // them, into `keys` (rows of D, 16-byte chunks at c ^ row % 16) and `values` (channel rows
    // of 64 keys, chunks at c ^ row / 2 % 8: 16 lanes that read one chunk of 16 rows touch
    // all 64 banks once); two tiles of codes are enough then, a wave reads only its own. Two groups have no room for this: every wave converts what it multiplies.
    static constexpr int RING = GROUPS == 1 ? 2 : kChunkRing;
    __attribute__((aligned(1024))) uint8_t ring[GROUPS * RING * 2 * TILE];
    __attribute__((aligned(1024))) uint16_t keys[GROUPS == 1 ? 2 * TILE : 1];
    __attribute__((aligned(1024))) uint16_t values[GROUPS == 1 ? kChunkRing * TILE : 1];
    // Which codes of a value tile are NaN, a bit each, where a wave's part of it (with_nan)
    // has any; [group][tile % 4]. In the ring, or converted, these are 0: the product then says
    // nothing of them, and nan_values gives the NaN to the rows that see them.
    __attribute__((aligned(16))) uint16_t nans[4 * GROUPS][TILE / 16];
    __attribute__((aligned(16))) int with_nan[4 * GROUPS][8 / GROUPS];
    float joint[8][32][2];
};

template <typename T, int D, int GROUPS>
__device__ inline void chunk_body(const AttnArgs& a, int from_rows, ChunkShare<D, GROUPS>& sh, int part_index) {
    constexpr int ROWS = chunk_rows(GROUPS);
    constexpr int LOADERS = 8 / GROUPS;   // waves that load a tile together
    constexpr int KC = D / 16;            // 16-byte chunks of a key's row in LDS
    constexpr int KK = D / 32;            // pairs of k steps of S
    constexpr int DT = D / 32;            // 32-channel tiles of O^T
    constexpr int TILE = 64 * D;          // bytes of one operand of a tile
    constexpr int DMA = TILE / (LOADERS * 1024);  // wave loads of an operand for each of them
    static_assert(GROUPS == 2 || D == 128, "rows of 16 chunks");
    static_assert(DMA > 0, "each loads of both operands");
    constexpr bool SHARED = GROUPS == 1;  // converted codes in LDS
    constexpr int RING = ChunkShare<D, GROUPS>::RING;
    constexpr bool SPLIT = __is_same(T, f16_t);
    auto& ring = sh.ring;
    auto& nans = sh.nans;
    auto& with_nan = sh.with_nan;
    auto& joint = sh.joint;
    static_assert(GROUPS == 1 || 8 * 64 * (DT / 2) * 64 <= (int)sizeof(ring), "room to join in");

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int phase = wave >> 2;                                 // which of a SIMD's two waves
    const int grp = GROUPS == 2 ? phase : 0, wr = wave % LOADERS;  // whose tiles; place in the group
    const int l32 = lane & 31, hh = lane >> 5, bs = a.c.bs, bs_log2 = __builtin_ctz(bs);

    // The part: part_index counts (request, row tile from the last, head).
    int b = -1, h = 0, rt = 0;
    AttnReq r{0, 0, 0, 0};
    {
        int64_t base = 0;
        for (int b0 = 0; b0 < a.B && b < 0; b0 += kWave) {
            const int i = b0 + lane;
            const AttnReq near = i < a.B ? attn_request(a, i) : AttnReq{0, 0, 0, 0};
            const int tiles = chunk_tiles(near, from_rows, ROWS);
            const int64_t mine = (int64_t)tiles * a.c.heads;
            const int64_t end = base + wave_prefix(mine);
            const uint64_t past = __ballot(end > part_index);
            if (past) {
                const int i2 = __builtin_ctzll(past);
                const int v = (int)(part_index - read_lane(end - mine, i2));
                b = b0 + i2;
                h = v % a.c.heads;
                rt = __builtin_amdgcn_readlane(tiles, i2) - 1 - v / a.c.heads;
                r = AttnReq{__builtin_amdgcn_readlane(near.len, i2), __builtin_amdgcn_readlane(near.n, i2),
                            __builtin_amdgcn_readlane(near.first, i2), __builtin_amdgcn_readlane(near.rows, i2)};
            }
            base = read_lane(end, kWave - 1);
        }
    }
    b = __builtin_amdgcn_readfirstlane(b);
    h = __builtin_amdgcn_readfirstlane(h);
    rt = __builtin_amdgcn_readfirstlane(rt);
    if (b < 0) return;
    r = uniform(r);
    const int r0 = rt * ROWS, w0 = r0 + 32 * wr;  // the part's first row, the wave's
    const int keys = max(0, r.len - r.n + min(r0 + ROWS - 1, r.rows - 1) / a.G + 1);  // that its last row sees
    const int n = (keys + 64 * GROUPS - 1) / (64 * GROUPS);  // tiles of each group (the last of group 1 may have no key)

    // Q and what each row sees.
    const int row = w0 + l32;
    const bool live = row < r.rows;
    const int limit = live ? r.len - r.n + row / a.G : r.len - 1;
    // Blocks and scales of 16 of the group's tiles: lane l has chunk l % 4 of tile l / 4.
    auto page_ids = [&](int j0) {
        const int64_t key = 64 * (GROUPS * ((int64_t)j0 + (lane >> 2)) + grp) + 16 * (lane & 3);
        return key < r.len ? a.table[b * a.table_stride + (key >> bs_log2)] : -1;
    };
    struct Pages : AttnPages {
        float log_sv, inv_sv;
        uint64_t plain;  // bit l: lane l's chunk is there and its value scale an ordinary one
    };
    auto page_scales = [&](Pages& p) {
        if (p.id < 0 || p.id >= a.c.blocks) p.id = -1;
        const int64_t at = (int64_t)max(p.id, 0) * a.c.heads + h;
        p.sk = a.c.k_scale[at];
        p.sv = a.c.v_scale[at];
    };
    auto page_derive = [&](Pages& p) {
        p.log_sv = __builtin_amdgcn_logf(p.sv);
        p.inv_sv = __builtin_amdgcn_rcpf(p.sv);
        p.plain = __ballot(p.id >= 0 && p.sv >= 0x1p-64f && p.sv <= 0x1p64f);
    };
    // every row of the wave sees all keys below this
    const int open = w0 < r.rows ? min(r.len - r.n + w0 / a.G + 1, r.len) : r.len;
    const uint32_t lds0 = (uint32_t)(uintptr_t)&ring[0] + (uint32_t)(grp * RING * 2 * TILE);
    // LDS row m of a half tile holds key 16 (m / 4 % 2) + 4 (m / 8) + m % 4 of it; rows
    // are swizzled by 16-byte chunks so that 16 lanes reading one chunk of 16 rows
    // touch every bank once (rows of 128 bytes: c ^ m / 2 % 8, of 64: c ^ m / 4 % 4).
    auto swz = [](int row64, int m, int c) { return row64 ? c ^ ((m >> 2) & 3) : c ^ ((m >> 1) & 7); };
    // The loads of a tile are 2 DMA of this wave: x < DMA keys, else values. A lane's
    // load x is at one place of a block in every tile: `at` is that place in block 0, `from`
    // the lane (times 4) of AttnPages with its chunk of tile 0. (Two groups' tiles are
    // 128 keys apart, whole blocks; one group's odd tiles are the second half of a block of 128.)
    uint64_t at[2 * DMA];
    int from[2 * DMA];
#pragma unroll
    for (int x = 0; x < DMA; ++x) {
        const int i = wr + LOADERS * x;
        const int m = i * (1024 / D) + lane / KC, c = swz(D == 64, m, lane % KC), m32 = m & 31;
        const int key = (m & 32) + 16 * ((m32 >> 2) & 1) + 4 * (m32 >> 3) + (m32 & 3);
        at[x] = (uint64_t)(uintptr_t)a.c.k + ((int64_t)h * bs + ((64 * grp + key) & (bs - 1))) * D + 16 * c;
        from[x] = 4 * (key >> 4);
        const int d = 16 * i + lane / 4, vc = swz(1, d, lane & 3);
        at[DMA + x] = (uint64_t)(uintptr_t)a.c.v + ((int64_t)h * D + d) * bs + ((64 * grp + 16 * vc) & (bs - 1));
        from[DMA + x] = 4 * vc;
    }
    const uint32_t k_stride = (uint32_t)a.c.k_stride, v_stride = (uint32_t)a.c.v_stride;  // below 2^31
    auto load_id = [&](int x, int ids, int j) { return __builtin_amdgcn_ds_bpermute(from[x] + 16 * (j & 15), ids); };
    const uint32_t odd = GROUPS == 1 && bs > 64 ? 64 : 0;  // keys
    auto issue_one = [&](int x, int id, int j, int in) {  // of tile j, from block id into tile in's slot
        const uint32_t slot = lds0 + (uint32_t)((in % RING) * 2 * TILE + 1024 * (wr + LOADERS * (x % DMA)));
        const uint64_t src = at[x] + (uint64_t)(uint32_t)max(id, 0) * (x < DMA ? k_stride : v_stride) +
                             (j & 1 ? (x < DMA ? odd * D : odd) : 0u);
        lds_dma_b128((const void*)(uintptr_t)src, x < DMA ? slot : slot + TILE);
    };
    auto issue = [&](const Pages& p, int j, int in) {
#pragma unroll
        for (int x = 0; x < 2 * DMA; ++x) issue_one(x, load_id(x, p.id, j), j, in);
    };

    // What the first products wait for, in this order: the blocks' ids and Q together, then
    // the scales and the tiles.
    u32x4 q[2 * KK];
    Pages pg, nx;  // of the tile whose softmax is next; of the tiles 16 on
    pg.id = page_ids(0);
    {
        const int i = live ? row / a.G : 0, qh = live ? row % a.G : 0;
        const uint16_t* src = a.q + (int64_t)(r.first + i) * a.q_stride + (int64_t)(h * a.G + qh) * D;
#pragma unroll
        for (int k = 0; k < KK; ++k)
#pragma unroll
            for (int u = 0; u < 2; ++u) q[2 * k + u] = *reinterpret_cast<const u32x4*>(src + 32 * k + 16 * hh + 8 * u);
#pragma unroll
        for (int k = 0; k < 2 * KK; ++k) asm volatile("" : "+v"(q[k]));
    }
    page_scales(pg);
    nx = pg;
    if (n > 0)
        for (int j = 0; j < min(RING, 3); ++j) issue(pg, min(j, n - 1), j);
    f32x16 o[DT], s[2];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = 0.f;
    float m = -INFINITY, l = 0.f;
    u32x4 hi[4], lo[4];  // P^T: [2 e + u], half tile e, its keys 8 u .. of each lane half
    // What the next softmax needs of its tile's two chunks of this lane.
    float sk[2], log_sv[2], inv_sv[2];
    int any_nan = 0;  // lane x % LOADERS: NaN codes among the values that wave loaded
    auto of_chunk = [&](int x, int j, int e) { return __builtin_amdgcn_ds_bpermute(16 * (j & 15) + 8 * e + 4 * hh, x); };
    auto of_chunk_f = [&](float x, int j, int e) { return __int_as_float(of_chunk(__float_as_int(x), j, e)); };
    auto take_scales = [&](int j) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            sk[e] = of_chunk_f(pg.sk, j, e);
            log_sv[e] = of_chunk_f(pg.log_sv, j, e);
            inv_sv[e] = of_chunk_f(pg.inv_sv, j, e);
        }
        any_nan = with_nan[4 * grp + (j & 3)][lane % LOADERS];
    };
    // Value fragments, read AHEAD steps ahead; a tile's first ones before its M phase.
    constexpr int AHEAD = SHARED && !SPLIT ? 3 : 2;
    u32x4 vf[AHEAD + 1][SHARED ? 2 : 1];
    // A tile's values as this lane reads them: half tile e, made here so that the addresses
    // are not held over the loop for every slot of the ring.
    auto v_base = [&](int j, const uint8_t* (&vs)[2]) {
        uint32_t so = (uint32_t)(SHARED ? j % kChunkRing * 2 * TILE : (grp * RING + j % RING) * 2 * TILE + TILE);
        asm volatile("" : "+s"(so));
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if constexpr (SHARED) vs[e] = (const uint8_t*)sh.values + so + l32 * 128 + 16 * ((4 * e + 2 * hh) ^ ((l32 >> 1) & 7));
            else vs[e] = ring + so + l32 * 64 + 16 * swz(1, l32, 2 * e + hh);
    };
    // from a fragment's first chunk to its second
    const int other_v = (l32 & 2) ? -16 : 16, other_k = (l32 & 1) ? -16 : 16;
    auto load_v = [&](const uint8_t* const (&vs)[2], int st) {
        const uint8_t* p = vs[st / KK] + 32 * (st % KK) * (SHARED ? 128 : 64);
        vf[st % (AHEAD + 1)][0] = *reinterpret_cast<const u32x4*>(p);
        if constexpr (SHARED) vf[st % (AHEAD + 1)][1] = *reinterpret_cast<const u32x4*>(p + other_v);
    };
    auto put_values = [&](int j, int x, const u32x4& w) {  // this lane's chunk of codes into sh.values
        const int d = 16 * (wr + LOADERS * x) + lane / 4, c = 2 * swz(1, d, lane & 3);
        uint16_t* row = sh.values + j % kChunkRing * TILE + 64 * d;
#pragma unroll
        for (int u = 0; u < 2; ++u)
            *reinterpret_cast<u32x4*>(row + 8 * ((c + u) ^ ((d >> 1) & 7))) = fp8x8_to_half8(w[2 * u], w[2 * u + 1], bf16_t{});
    };

    auto put_keys = [&](int j, int x, const u32x4& w) {  // into sh.keys
        const int m = (wr + LOADERS * x) * (1024 / D) + lane / KC, c = 2 * swz(D == 64, m, lane % KC);
        uint16_t* row = sh.keys + j % 2 * TILE + D * m;
#pragma unroll
        for (int u = 0; u < 2; ++u)
            *reinterpret_cast<u32x4*>(row + 8 * ((c + u) ^ (m & 15))) = fp8x8_to_half8(w[2 * u], w[2 * u + 1], T{});
    };

    // This wave's part of tile j's values, which has landed: NaN codes out of it. (The
    // tile's softmax is behind the next barrier.)
    u32x4 part[DMA], key_part[SHARED ? DMA : 1];
    auto read_part = [&](int j) {
        const uint8_t* mine = ring + (grp * RING + j % RING) * 2 * TILE + TILE + 16 * lane;
#pragma unroll
        for (int x = 0; x < DMA; ++x) {
            part[x] = *reinterpret_cast<const u32x4*>(mine + 1024 * (wr + LOADERS * x));
            if constexpr (SHARED) key_part[x] = *reinterpret_cast<const u32x4*>(mine - TILE + 1024 * (wr + LOADERS * x));
        }
    };
    auto part_nans = [&](int j) {
        uint32_t bad = 0;
#pragma unroll
        for (int x = 0; x < DMA; ++x) {
            if constexpr (SHARED) {
                put_keys(j, x, key_part[x]);
                put_values(j, x, part[x]);  // and again should one be NaN
            }
#pragma unroll
            for (int y = 0; y < 4; ++y) bad |= (part[x][y] & 0x7f7f7f7fu) + 0x01010101u;
        }
        return bad & 0x80808080u;
    };
    auto check_part = [&](int j, uint32_t bad) {
        const bool any = __any(bad != 0);
        if (lane == 0) with_nan[4 * grp + (j & 3)][wr] = any;
        if (!any) return;
        uint8_t* mine = ring + (grp * RING + j % RING) * 2 * TILE + TILE + 16 * lane;
#pragma unroll
        for (int x = 0; x < DMA; ++x) {
            u32x4 w = part[x];
            uint32_t bits = 0;
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const uint32_t nan = nan_codes(w[y]) >> 7;
                bits |= (nan * 0x01020408u >> 24) << (4 * y);
                w[y] &= ~(nan * 0xffu);
            }
            nans[4 * grp + (j & 3)][64 * (wr + LOADERS * x) + lane] = (uint16_t)bits;
            if constexpr (SHARED) put_values(j, x, w);
            else *reinterpret_cast<u32x4*>(mine + 1024 * (wr + LOADERS * x)) = w;
        }
    };
    // NaN codes among tile j's values: NaN sums for the rows that see them, by a product of indicators.
    auto nan_values = [&](int j, const int (&seen)[2]) {
        const int which = 4 * grp + (j & 3);
#pragma unroll 1
        for (int e = 0; e < 2; ++e) {
            u32x4 one[2];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                one[i >> 2][i & 3] = (2 * i < seen[e] ? 0x3f80u : 0u) | (2 * i + 1 < seen[e] ? 0x3f800000u : 0u);
#pragma unroll
            for (int k = 0; k < DT; ++k) {
                uint32_t bits = nans[which][(32 * k + l32) * 4 + swz(1, l32, 2 * e + hh)];
                if (!with_nan[which][(2 * k + (l32 >> 4)) % LOADERS]) bits = 0;  // the part has none
                u32x4 w;
#pragma unroll
                for (int x = 0; x < 4; ++x) w[x] = (((bits >> (4 * x)) & 15u) * 0x00204081u & 0x01010101u) * 0x38u;  // 1.0
                f32x16 hit;
#pragma unroll
                for (int i = 0; i < 16; ++i) hit[i] = 0.f;
                hit = mfma32x32x16(fp8x8_to_half8(w[0], w[1], bf16_t{}), one[0], hit, bf16_t{});
                hit = mfma32x32x16(fp8x8_to_half8(w[2], w[3], bf16_t{}), one[1], hit, bf16_t{});
#pragma unroll
                for (int i = 0; i < 16; ++i) o[k][i] = hit[i] > 0.f ? __builtin_nanf("") : o[k][i];
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };

    // One M phase: S of tile jp + 1 and O += P V of tile jp (if DP: from the second on); on
    // its way the loads of tile ji are issued into the slot of tile jp + 3 (that of jp - 1, which
    // all are done with; with two slots that of jp + 1, whose codes this wave, their only
    // reader, converted a tile ago), the part of tile jp + 2 that this wave loaded is checked
    // and, with one group, converted, and the scales of jp + 1 are taken.
    auto m_phase = [&](auto dp_tag, int jp, int ids_of_ji, int ji) {
        const int js = jp + 1;
        constexpr bool DP = decltype(dp_tag)::value;
        constexpr int ST = 2 * KK;
        uint32_t so_k = (uint32_t)(SHARED ? js % 2 * 2 * TILE : (grp * RING + js % RING) * 2 * TILE);
        asm volatile("" : "+s"(so_k));
        // K fragments are read two steps before their products, which are two steps behind
        // V's: a read takes longer than a step.
        u32x4 kf[3][SHARED ? 2 : 1];
        auto load_k = [&](int st) {
            const int row = 32 * (st / KK) + l32, c = 2 * (st % KK) + hh;
            if constexpr (SHARED) {
                const uint8_t* p = (const uint8_t*)sh.keys + so_k + row * (2 * D) + 16 * ((2 * c) ^ (l32 & 15));
                kf[st % 3][0] = *reinterpret_cast<const u32x4*>(p);
                kf[st % 3][1] = *reinterpret_cast<const u32x4*>(p + other_k);
            } else {
                kf[st % 3][0] = *reinterpret_cast<const u32x4*>(ring + so_k + row * D + 16 * swz(D == 64, l32, c));
            }
        };
        int ids[2 * DMA];
        const uint8_t* vs[2];
        uint32_t bad = 0;
        if constexpr (DP) {
            v_base(jp, vs);
#pragma unroll
            for (int x = 0; x < 2 * DMA; ++x) ids[x] = load_id(x, ids_of_ji, ji);
        }
#pragma unroll
        for (int st = 0; st < ST + 2; ++st) {
            if (st < ST) load_k(st);
            if constexpr (DP) {
                if (st + AHEAD < ST) load_v(vs, st + AHEAD);
                if (st == ST / 2) read_part(jp + 2);
            }
            if (st == ST / 2 + 1) take_scales(js);
            // The two products of a step's O, and of its S, wait for each other: they take turns.
            auto pv = [&](int u) {
                if constexpr (DP) {
                    if (st < ST) {
                        const int e = st / KK, k = st % KK;
                        u32x4 v0;
                        if constexpr (SHARED) v0 = vf[st % (AHEAD + 1)][u];
                        else v0 = fp8x8_to_half8(vf[st % (AHEAD + 1)][0][2 * u], vf[st % (AHEAD + 1)][0][2 * u + 1], bf16_t{});
                        o[k] = mfma32x32x16(v0, hi[2 * e + u], o[k], bf16_t{});
                        if constexpr (SPLIT) o[k] = mfma32x32x16(v0, lo[2 * e + u], o[k], bf16_t{});
                    }
                }
            };
            auto qk = [&](int u) {
                if (st < 2) return;
                const int e = (st - 2) / KK, k = (st - 2) % KK;
                u32x4 k0;
                if constexpr (SHARED) k0 = kf[(st - 2) % 3][u];
                else k0 = fp8x8_to_half8(kf[(st - 2) % 3][0][2 * u], kf[(st - 2) % 3][0][2 * u + 1], T{});
                if (k == 0 && u == 0)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[e][i] = 0.f;
                s[e] = mfma32x32x16(k0, q[2 * k + u], s[e], T{});
            };
            pv(0);
            qk(0);
            pv(1);
            qk(1);
            if constexpr (DP) {
                if (st == ST) bad = part_nans(jp + 2);
            }
            if constexpr (DP) {
                if (st >= 1 && st <= 2 * DMA) issue_one(st - 1, ids[st - 1], ji, jp + 3);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        // used here: the compiler would move the products of S to the softmax, which
        // alone needs them, and so into the other phase
        asm volatile("" : "+v"(s[0]), "+v"(s[1]));
        if constexpr (DP) check_part(jp + 2, bad);
    };
    // The softmax of tile j, whose scores are in s: P into hi (and lo).
    auto v_phase = [&](int j) {
        const int key0 = 64 * (GROUPS * j + grp);
        // Nothing masked and ordinary scales: the value scale goes into the exponent,
        // p sv = 2^(x + log2 sv), and out of the chunk's sum once. Else p is
        // masked and multiplied.
        const bool plain = ((uint32_t)(pg.plain >> (4 * (j & 15))) & 15u) == 15u && key0 + 64 <= open;
        const float ref = m == -INFINITY ? 0.f : m, factor = a.scale_log2;
        float add[2], out[2], sv[2];
        int seen[2] = {16, 16};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            sk[e] *= factor;
            add[e] = log_sv[e] - ref;
            out[e] = inv_sv[e];
        }
        if (!plain) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int id = of_chunk(pg.id, j, e);
                sv[e] = of_chunk_f(pg.sv, j, e);
                seen[e] = id < 0 ? 0 : min(min(r.len, limit + 1) - (key0 + 32 * e + 16 * hh), 16);
                add[e] = -ref;
                out[e] = 1.0f;
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[e][i] = fmaf(s[e][i], sk[e], add[e]);
        if (!plain) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                int n_seen = seen[e];
                asm volatile("" : "+v"(n_seen));  // keeps the comparisons inside this branch
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float x = i < n_seen ? s[e][i] : -INFINITY;
                    asm volatile("" : "+v"(x));  // and the masking
                    s[e][i] = x;
                }
            }
        }
        auto pack = [&](int e, int i, float x0, float x1) {
            const uint32_t w = pack_half2(x0, x1, bf16_t{});
            hi[2 * e + (i >> 3)][(i & 7) >> 1] = w;
            if constexpr (SPLIT)
                lo[2 * e + (i >> 3)][(i & 7) >> 1] =
                    pack_half2(x0 - __uint_as_float(w << 16), x1 - __uint_as_float(w & 0xffff0000u), bf16_t{});
        };
        auto exponentiate = [&]() {  // s becomes what is rounded to P; the sum of p
            // Four at a time, summed and rounded while the next four are on their way: an
            // addition right behind its exponential waits for it.
            float p[8][4], sum[2][4];
#pragma unroll
            for (int g = 0; g <= 8; ++g) {
                if (g < 8) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) p[g][x] = __builtin_amdgcn_exp2f(s[g >> 2][4 * (g & 3) + x]);
                }
                if (g > 0) {
                    const int w = g - 1, e = w >> 2;
#pragma unroll
                    for (int x = 0; x < 4; ++x) sum[e][x] = w & 3 ? sum[e][x] + p[w][x] : p[w][x];
                    pack(e, 4 * (w & 3), p[w][0], p[w][1]);
                    pack(e, 4 * (w & 3) + 2, p[w][2], p[w][3]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            return ((sum[0][0] + sum[0][1]) + (sum[0][2] + sum[0][3])) * out[0] +
                   ((sum[1][0] + sum[1][1]) + (sum[1][2] + sum[1][3])) * out[1];
        };
        float sum = exponentiate();
        const bool fresh = m == -INFINITY && (seen[0] > 0 || seen[1] > 0);
        if (__any(fresh || !(sum <= kChunkSumMax))) {
            // both lane halves of a row move together
            float mx = -INFINITY;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float me = s[e][0];
#pragma unroll
                for (int i = 1; i < 16; ++i) me = __builtin_elementwise_maximum(me, s[e][i]);
                mx = __builtin_elementwise_maximum(mx, me - (add[e] + ref));
            }
            const float mo = __shfl_xor(mx, 32), so = __shfl_xor(sum, 32);
            mx = __builtin_elementwise_maximum(mx, mo);  // of the row, above ref
            const bool move = mx != -INFINITY && (m == -INFINITY || !(sum <= kChunkSumMax) || !(so <= kChunkSumMax));
            const float shift = move ? mx : 0.f, keep = __builtin_amdgcn_exp2f(-shift);
            if (m != -INFINITY) {
                l *= keep;
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[t][i] *= keep;
            }
            if (move) m = ref + shift;
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[e][i] -= shift;
            sum = exponentiate();
        }
        if (!plain) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                int n_seen = seen[e];
                asm volatile("" : "+v"(n_seen));
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const float p0 = __builtin_amdgcn_exp2f(s[e][i]), p1 = __builtin_amdgcn_exp2f(s[e][i + 1]);
                    pack(e, i, i < n_seen ? p0 * sv[e] : 0.f, i + 1 < n_seen ? p1 * sv[e] : 0.f);  // sv may be anything
                }
            }
        }
        l += sum;
        if (__any(any_nan)) nan_values(j, seen);
    };

    // One M phase and what comes with it; the last tiles' load the last tile once more, into
    // slots that nobody reads, and compute an S of whatever its slot holds.
    auto m_step = [&](int k) {
        wait_vmem_le<0>();  // tile k + 2, issued a tile's time ago
        if (((k + 1) & 15) == 0) pg = nx;
        const int ji = min(k + 3, n - 1);
        const int ids = ji > k + 1 && (ji >> 4) != ((k + 1) >> 4) ? nx.id : pg.id;
        // The wave in its M phase goes first: the softmax of the SIMD's other wave takes
        // the cycles that its matrix instructions leave.
        __builtin_amdgcn_s_setprio(2);
        m_phase(std::true_type{}, k, ids, ji);
        __builtin_amdgcn_s_setprio(0);
    };
    auto v_step = [&](int j) {
        // the next 16 tiles' blocks, then their scales: they have tiles' time to come
        if ((j & 15) == 1 && (j & ~15) + 16 < n) nx.id = page_ids((j & ~15) + 16);
        if ((j & 15) == 3) page_scales(nx);
        if ((j & 15) == 5) page_derive(nx);
        v_phase(j);
        const uint8_t* vs[2];
        v_base(j, vs);
#pragma unroll
        for (int st = 0; st < AHEAD; ++st) load_v(vs, st);
    };
    if (n > 0) {
        wait_vmem_le<2 * DMA>();  // tile 0, of three also tile 1
        page_derive(pg);
        read_part(0);
        check_part(0, part_nans(0));
        if constexpr (RING == 2) {  // tile 0's codes are read: its slot is tile 2's
            issue(pg, min(2, n - 1), 2);
            wait_vmem_le<2 * DMA>();
        }
        read_part(1);
        check_part(1, part_nans(1));
        __syncthreads();
        m_phase(std::false_type{}, -1, 0, 0);
        if constexpr (SHARED) __syncthreads();  // the next M phase overwrites tile 0's keys
        // A barrier a tile: a SIMD's first wave passes it before, its second behind a product, so they
        // stay half a tile apart and are free between. Behind it the tile that both
        // waited for and checked (and converted) is there, and the slot of the tile before
        // is free: keys are read a phase before their values, so two tiles of them are enough.
        for (int k = 0; k < n; ++k) {
            v_step(k);
            if (phase == 0 && k > 0) __syncthreads();
            m_step(k);
            if (phase == 1) __syncthreads();
        }
        if (phase == 0) __syncthreads();
    }
    wait_vmem_le<0>();  // no load into a ring is on its way

    l += __shfl_xor(l, 32);
    uint16_t* dst = a.o + (int64_t)(r.first + row / a.G) * a.o_stride + (int64_t)(h * a.G + row % a.G) * D + 8 * hh;
    // Channels 32 t + 8 i + 4 hh .. of i and i + 1: the lane halves exchange, so that each
    // stores 16 bytes, of i or of i + 1.
    auto store = [&](int t, int i, const float (&z)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int x = 0; x < 4; ++x)
            w[x] = (uint32_t)elem<T>::from_f32(z[2 * x]) | ((uint32_t)elem<T>::from_f32(z[2 * x + 1]) << 16);
        const auto lo = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
        const auto hi = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
        if (live) *reinterpret_cast<u32x4*>(dst + 32 * t + 8 * i) = u32x4{lo[0], hi[0], lo[1], hi[1]};
    };
    if constexpr (GROUPS == 1) {
        const float inv = m == -INFINITY ? 0.f : 1.0f / l;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                float z[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] = o[t][4 * i + e] * inv;
                store(t, i, z);
            }
        return;
    }
    __syncthreads();  // the rings are free
    // Join: group g ends with channels 32 t .. of t in its half.
    if (hh == 0) {
        joint[wave][l32][0] = m;
        joint[wave][l32][1] = l;
    }
    f32x4* give = reinterpret_cast<f32x4*>(ring) + (size_t)wave * (DT / 2) * 4 * kWave + lane;
#pragma unroll
    for (int t = 0; t < DT / 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x16& x = o[t];
            const f32x16& y = o[DT / 2 + t];
            give[(4 * t + i) * kWave] = grp == 0 ? f32x4{y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]}
                                                 : f32x4{x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]};
        }
    __syncthreads();
    const float m2 = joint[wave ^ 4][l32][0], l2 = joint[wave ^ 4][l32][1];
    const float mx = __builtin_elementwise_maximum(m, m2), ref = mx == -INFINITY ? 0.f : mx;
    const float f = __builtin_amdgcn_exp2f(m - ref), g = __builtin_amdgcn_exp2f(m2 - ref);
    const float inv = mx == -INFINITY ? 0.f : 1.0f / (l * f + l2 * g);
    const f32x4* take = reinterpret_cast<const f32x4*>(ring) + (size_t)(wave ^ 4) * (DT / 2) * 4 * kWave + lane;
#pragma unroll
    for (int t = 0; t < DT / 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const f32x4 y[2] = {take[(4 * t + i) * kWave], take[(4 * t + i + 1) * kWave]};
            float z[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float mine = grp == 0 ? o[t][4 * i + e] : o[DT / 2 + t][4 * i + e];
                z[e] = (mine * f + y[e >> 2][e & 3] * g) * inv;
            }
            store(grp * (DT / 2) + t, i, z);
        }
}

// A batch with requests of many rows: the first `parts` workgroups take parts of these,
// those behind them split what the requests of up to sp.most_rows rows read (and end at
// once where there are none). How many parts there are is known here only: the host counts
// as many as there may be, and those that find none end as well.
template <typename T, int D, int GROUPS>
__global__ void __launch_bounds__(kChunkThreads, 1) kv_chunk_kernel(AttnArgs a, AttnSplit sp, int parts) {
    static_assert(split_waves(1, 128) * kWave == kChunkThreads, "one workgroup size");
    union Share {
        SplitShare<D, 1> split;
        ChunkShare<D, GROUPS> chunk;
    };
    __shared__ Share sh;
    if ((int)blockIdx.x < parts) chunk_body<T, D, GROUPS>(a, sp.most_rows, sh.chunk, blockIdx.x);
    else split_body<T, D, 1>(a, sp, sh.split, blockIdx.x - parts, gridDim.x - parts);
}

// Rows of a request that the split kernel takes, 16 NT of them a wave: all up to 64 at
// NT = 2; of a batch with more, requests of up to 16 at NT = 1.
constexpr int kSplitRows = 64;
static int split_nt(long rows) { return rows <= 16 || rows > kSplitRows ? 1 : 2; }
static long split_most_rows(long rows) { return rows <= kSplitRows ? rows : 16; }
static long split_run_tiles(long rows) { return (split_most_rows(rows) + 16 * split_nt(rows) - 1) / (16 * split_nt(rows)); }
// A workspace is the workgroups' results, in room for the largest of any call, then the
// counters: these stay zero between calls whatever the calls' shapes. A call has as many as
// it has run tiles; calls of up to `rows` rows have the most at 33 to 64.
static long split_room_tiles(long rows) { return rows <= 32 ? 1 : split_run_tiles(kSplitRows); }
constexpr size_t kSplitPartBytes = (size_t)2 * kSplitGroups * 32 * (128 + 2) * sizeof(float);

template <typename T, int D> static void launch_attention(const AttnArgs& a, int max_q, void* workspace, int max_len,
                                                           hipStream_t s) {
    const long rows = (long)max_q * a.G, run_tiles = split_run_tiles(rows);
    const int nt = split_nt(rows), waves = split_waves(nt, D);
    AttnSplit sp;
    sp.most_rows = (int)split_most_rows(rows);
    sp.part = (float*)workspace;
    sp.done = (uint32_t*)((char*)workspace + kSplitPartBytes);
    // Workgroups of the split: for every wave a tile, for every run a workgroup, at most one on a CU.
    const long keys = max_len > 0 ? max_len : (long)a.width * a.c.bs;
    const double runs = (double)a.B * a.c.heads * run_tiles, units = runs * (double)((keys + 63) / 64);
    double groups = units / waves;
    if (groups < runs) groups = runs;
    const int split = groups < kSplitGroups ? (int)groups : kSplitGroups;
    if (rows <= kSplitRows) {
        if (nt == 1) hipLaunchKernelGGL((kv_split_kernel<T, D, 1>), dim3(split), dim3(waves * kWave), 0, s, a, sp);
        else hipLaunchKernelGGL((kv_split_kernel<T, D, 2>), dim3(split), dim3(waves * kWave), 0, s, a, sp);
        return;
    }
    // Parts: whole ones, and one more for each request that is large enough.
    const long all = (long)a.tokens * a.G, some = all / (sp.most_rows + 1);
    auto parts_of = [&](int groups) { return (all / chunk_rows(groups) + (some < a.B ? some : a.B)) * a.c.heads; };
    // Requests of few rows are split in any batch, also where the rows of q would let all have
    // max_q tokens: lengths are known on the device only, and a part walks all its keys alone.
    // With parts alone in such calls, a token over 100000 keys beside three chunks of 2048 over 3800
    // took 2855 us, now 342 (316 for the chunks and 40 for the token, each alone); 32 tokens over 3000
    // keys in a q with room for 512 each 111, now 41 (36 in one of their size). Split workgroups
    // without work cost a call of four such chunks nothing that can be seen (390).
    // Rounds of workgroups if every request has max_q tokens. A round of 256 rows takes 1.6 to
    // 1.85 times as long as one of 128. Measured (us, 128 rows against 256, 4 chunks over 4096 keys,
    // 32 heads of 128, 8 kv heads, bf16): 256 tokens 78 / 112 (1 round / 1), 320 137 / 115 (2 / 1),
    // 512 146 / 132 (2 / 1), 768 209 / 225 (3 / 2), 1024 267 / 246 (4 / 2); in f16 98 / 135,
    // 167 / 137, 186 / 171, 267 / 281, 340 / 320. Of 80 shapes, half of them in f16 (1 to 8 requests of 256 to
    // 2048 tokens, 5 to 32 kv heads) the rule took the slower side by more than 2 % in two (3 and 4 %:
    // one request of 2048).
    auto rounds = [&](int groups) {
        const long tiles = ((long)a.max_q * a.G + chunk_rows(groups) - 1) / chunk_rows(groups);
        return (tiles * a.B * a.c.heads + kSplitGroups - 1) / kSplitGroups;
    };
    const bool full = 4.0 * a.tokens >= 3.0 * (double)a.B * max_q;  // most requests may have about max_q
    if constexpr (D == 128)
        if (full && 7 * rounds(1) <= 4 * rounds(2)) {
            const long parts = parts_of(1);
            hipLaunchKernelGGL((kv_chunk_kernel<T, D, 1>), dim3((unsigned)(parts + split)), dim3(kChunkThreads), 0, s, a, sp,
                               (int)parts);
            return;
        }
    const long parts = parts_of(2);
    hipLaunchKernelGGL((kv_chunk_kernel<T, D, 2>), dim3((unsigned)(parts + split)), dim3(kChunkThreads), 0, s, a, sp,
                       (int)parts);
}

}  // namespace pyc

extern "C" size_t pyc_hip_kv_attention_workspace_bytes(int B, int hq, int hk, int d, int max_q) {
    using namespace pyc;
    const long rows = (long)max_q * (hq / hk);
    (void)d;
    return kSplitPartBytes + ((size_t)B * hk * split_room_tiles(rows) * sizeof(uint32_t) + 15) / 16 * 16;
}

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
    a.max_q = max_q < tokens ? max_q : tokens;
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
    hipStream_t s = (hipStream_t)stream;
    if (a.c.d == 128) {
        if (is_bf16) launch_attention<bf16_t, 128>(a, max_q, workspace, max_len, s);
        else launch_attention<f16_t, 128>(a, max_q, workspace, max_len, s);
    } else {
        if (is_bf16) launch_attention<bf16_t, 64>(a, max_q, workspace, max_len, s);
        else launch_attention<f16_t, 64>(a, max_q, workspace, max_len, s);
    }
    return hipGetLastError() == hipSuccess ? 0 : -2;
}

extern "C" int pyc_hip_kinfo_kv_attention(int is_bf16, pyc_hip_kinfo* out) {
    using namespace pyc;
    if (!out) return -1;
    out->fn = is_bf16 ? reinterpret_cast<const void*>(&kv_split_kernel<bf16_t, 128, 1>)
                      : reinterpret_cast<const void*>(&kv_split_kernel<f16_t, 128, 1>);
    out->name = "kv_split_kernel<128, 1>";
    out->lds_bytes = sizeof(SplitShare<128, 1>);
    out->threads = split_waves(1, 128) * kWave;
    out->waves_per_simd = 2;
    return 0;
}
