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

// Rows per request up to which the split kernel takes it; the others go to kv_attn_kernel.
struct AttnSplit {
    int most_rows;
    float* part;       // two partial results for each wave
    int64_t part_size; // floats of one: [most_rows][D] sums, then [most_rows][2] maximum and sum
};

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
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                const u32x4 w = k[t * KC + c];
                const u32x4 k0 = fp8x8_to_half8(w[0], w[1], T{}), k1 = fp8x8_to_half8(w[2], w[3], T{});
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    s[n][t] = mfma16x16x32(k0, q[n][2 * c], s[n][t], T{});
                    s[n][t] = mfma16x16x32(k1, q[n][2 * c + 1], s[n][t], T{});
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
        for (int dt = 0; dt < DT; ++dt) {
            const u32x4 v0 = fp8x8_to_half8(v[dt][0], v[dt][1], bf16_t{}), v1 = fp8x8_to_half8(v[dt][2], v[dt][3], bf16_t{});
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                o[n][dt] = mfma16x16x32(v0, hi[n][0], o[n][dt], bf16_t{});
                o[n][dt] = mfma16x16x32(v1, hi[n][1], o[n][dt], bf16_t{});
                if constexpr (__is_same(T, f16_t)) {
                    o[n][dt] = mfma16x16x32(v0, lo[n][0], o[n][dt], bf16_t{});
                    o[n][dt] = mfma16x16x32(v1, lo[n][1], o[n][dt], bf16_t{});
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

    // A part of the rows' keys: sums, maximum and sum of p.
    __device__ void store_part(const AttnReq& r, const AttnSplit& sp, int64_t slot) {
        const int lane = threadIdx.x & 63, g = lane >> 4;
        float* dst = sp.part + slot * sp.part_size;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int row = 16 * n + (lane & 15);
            float sum = l[n];
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (row >= r.rows) continue;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(dst + row * D + 16 * dt + 4 * g) = o[n][dt];
            if (g == 0) {
                float* ml = dst + (int64_t)sp.most_rows * D + 2 * row;
                ml[0] = m[n];
                ml[1] = sum;
            }
        }
    }
};

// The split kernel's work: for every request of at most most_rows rows and every kv
// head a run of tiles of 64 keys, all runs one after the other (request, head, tile),
// cut into equal pieces, one for each wave. A run that falls into several pieces is
// joined by kv_join_kernel.
__device__ inline int attn_tiles(const AttnArgs& a, const AttnReq& r, int most_rows) {
    if (r.rows <= 0 || r.rows > most_rows) return 0;
    const int end = r.len - r.n + r.rows / a.G;  // keys that the last row sees
    return max(1, end / 64 + (end % 64 > 0 ? 1 : 0));
}
__device__ inline int64_t attn_tiles64(const AttnArgs& a, int b, int most_rows) {
    return b < a.B ? attn_tiles(a, attn_request(a, b), most_rows) : 0;
}
__device__ inline int64_t wave_sum(int64_t x) {
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) x += __shfl_xor(x, d);
    return x;
}
__device__ inline int64_t attn_total(const AttnArgs& a, int most_rows) {
    int64_t sum = 0;
    for (int b0 = 0; b0 < a.B; b0 += kWave) sum += attn_tiles64(a, b0 + (threadIdx.x & 63), most_rows);
    return wave_sum(sum) * a.c.heads;
}
// The request that unit u (0 <= u < total) belongs to, and the units before it.
__device__ inline int attn_locate(const AttnArgs& a, int most_rows, int64_t u, int64_t* before) {
    const int lane = threadIdx.x & 63;
    int64_t base = 0;
    for (int b0 = 0; b0 < a.B; b0 += kWave) {
        const int64_t mine = attn_tiles64(a, b0 + lane, most_rows) * a.c.heads;
        int64_t end = mine;
#pragma unroll
        for (int d = 1; d < kWave; d *= 2) {
            const int64_t x = __shfl_up(end, d);
            if (lane >= d) end += x;
        }
        end += base;
        const uint64_t past = __ballot(end > u);
        if (past) {
            const int i = __builtin_ctzll(past);
            *before = __shfl(end - mine, i);
            return b0 + i;
        }
        base = __shfl(end, kWave - 1);
    }
    return -1;
}
// Piece w of W begins at floor(total w / W). There are fewer than 2^12 pieces and
// 2^50 units: no product passes 64 bits.
__device__ inline int64_t piece_begin(int64_t total, int W, int w) { return total * w / W; }
// The last piece that begins at or before u.
__device__ inline int piece_of(int64_t total, int W, int64_t u) { return (int)(((u + 1) * W - 1) / total); }

constexpr int kSplitWaves = 4;

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kSplitWaves* kWave, NT == 1 ? 2 : 1) kv_split_kernel(AttnArgs a, AttnSplit sp) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int w = blockIdx.x * kSplitWaves + wave;
    const int64_t total = attn_total(a, sp.most_rows);
    const int W = (int)min((int64_t)gridDim.x * kSplitWaves, total);
    if (w >= W) return;
    int64_t u = piece_begin(total, W, w);
    const int64_t end = piece_begin(total, W, w + 1);
    int64_t before;
    int b = __builtin_amdgcn_readfirstlane(attn_locate(a, sp.most_rows, u, &before));
    if (b < 0) return;
    AttnReq r = attn_request(a, b);
    int tiles = attn_tiles(a, r, sp.most_rows);
    int h = (int)((u - before) / tiles), t0 = (int)((u - before) % tiles);
    for (;;) {
        const int t1 = (int)min((int64_t)tiles, t0 + (end - u));
        AttnWave<T, D, NT> wv;
        wv.begin(a, r, h, 0);
        wv.run(a, r, b, h, t0, t1);
        if (t0 == 0 && t1 == tiles) wv.store(a, r, h, 0);
        else wv.store_part(r, sp, 2 * (int64_t)w + (t0 == 0 ? 1 : 0));
        u += t1 - t0;
        if (u >= end) return;
        t0 = 0;
        if (++h == a.c.heads) {
            h = 0;
            do {
                r = attn_request(a, ++b);
                tiles = attn_tiles(a, r, sp.most_rows);
            } while (tiles == 0);  // ends: there are units left
        }
    }
}

// Joins the parts of one row: thread 32 p + c takes channels D / 32 * c .. of parts p, p + 8, ...
constexpr int kJoinParts = 8;
template <typename T, int D>
__global__ void __launch_bounds__(32 * kJoinParts) kv_join_kernel(AttnArgs a, AttnSplit sp, int waves) {
    constexpr int C = D / 32;
    __shared__ float so[kJoinParts][D], sm[kJoinParts], sl[kJoinParts];
    const int row = blockIdx.x, h = blockIdx.y, c = threadIdx.x & 31, p = threadIdx.x / 32;
    const int64_t total = attn_total(a, sp.most_rows);
    const int W = (int)min((int64_t)waves, total);
    for (int b = blockIdx.z; b < a.B; b += gridDim.z) {
        const AttnReq r = attn_request(a, b);
        const int tiles = attn_tiles(a, r, sp.most_rows);
        if (tiles == 0 || row >= r.rows) continue;
        int64_t before = 0;
        for (int b0 = 0; b0 < b; b0 += kWave) {
            const int i = b0 + (threadIdx.x & 63);
            before += i < b ? attn_tiles64(a, i, sp.most_rows) : 0;
        }
        before = wave_sum(before) * a.c.heads + (int64_t)h * tiles;
        const int w0 = piece_of(total, W, before), w1 = piece_of(total, W, before + tiles - 1);
        if (w0 == w1) continue;
        float m = -INFINITY, l = 0.f, o[C];
#pragma unroll
        for (int i = 0; i < C; ++i) o[i] = 0.f;
        for (int w = w0 + p; w <= w1; w += kJoinParts) {
            const float* src = sp.part + (2 * (int64_t)w + (w == w0 ? 1 : 0)) * sp.part_size;
            const float* ml = src + (int64_t)sp.most_rows * D + 2 * row;
            const float pm = ml[0], pl = ml[1], mx = __builtin_elementwise_maximum(m, pm);
            const float ref = mx == -INFINITY ? 0.f : mx;
            const float f = __builtin_amdgcn_exp2f(m - ref), g = __builtin_amdgcn_exp2f(pm - ref);
            m = mx;
            l = l * f + pl * g;
#pragma unroll
            for (int i = 0; i < C; ++i) o[i] = o[i] * f + src[row * D + C * c + i] * g;
        }
#pragma unroll
        for (int i = 0; i < C; ++i) so[p][C * c + i] = o[i];
        if (c == 0) {
            sm[p] = m;
            sl[p] = l;
        }
        __syncthreads();
        if (threadIdx.x < D) {
            float mx = sm[0], sum = 0.f, x = 0.f;
            for (int i = 1; i < kJoinParts; ++i) mx = __builtin_elementwise_maximum(mx, sm[i]);
            const float ref = mx == -INFINITY ? 0.f : mx;
            for (int i = 0; i < kJoinParts; ++i) {
                const float g = __builtin_amdgcn_exp2f(sm[i] - ref);
                sum += sl[i] * g;
                x += so[i][threadIdx.x] * g;
            }
            a.o[(int64_t)(r.first + row / a.G) * a.o_stride + (int64_t)(h * a.G + row % a.G) * D + threadIdx.x] =
                elem<T>::from_f32(mx == -INFINITY ? 0.f : x / sum);
        }
        __syncthreads();
    }
}

// Requests of more rows than the split kernel takes: a wave for 16 of them.
template <typename T, int D>
__global__ void __launch_bounds__(kWave) kv_attn_kernel(AttnArgs a, int from_rows) {
    const int r0 = 16 * blockIdx.x, h = blockIdx.y;
    for (int b = blockIdx.z; b < a.B; b += gridDim.z) {
        const AttnReq r = attn_request(a, b);
        if (r0 >= r.rows || r.rows <= from_rows) continue;
        AttnWave<T, D, 1> w;
        w.begin(a, r, h, r0);
        // keys that the tile's last row sees
        const int last = min(r0 + 15, r.rows - 1) / a.G, end = max(0, r.len - r.n + last + 1);
        w.run(a, r, b, h, 0, (end + 63) / 64);
        w.store(a, r, h, r0);
    }
}

constexpr int kSplitMost = 2048;  // waves: 8 on each of 256 CUs

// Rows that the split kernel takes per request, as 16s: all of them up to 64, else 16.
static int split_tiles(long rows) { return rows <= 16 || rows > 64 ? 1 : rows <= 32 ? 2 : 4; }

template <typename T, int D> static void launch_attention(const AttnArgs& a, float* part, int max_len, hipStream_t s) {
    const long rows = (long)a.max_q * a.G;
    const int nt = split_tiles(rows);
    AttnSplit sp;
    sp.most_rows = (int)(rows < 16 * nt ? rows : 16 * nt);
    sp.part = part;
    sp.part_size = (int64_t)sp.most_rows * (D + 2);
    const long keys = max_len > 0 ? max_len : (long)a.width * a.c.bs;
    const double units = (double)a.B * a.c.heads * (double)((keys + 63) / 64);
    const int most = nt == 1 ? kSplitMost : kSplitMost / 2;
    const int waves = units < most ? (int)units : most;
    const int groups = (waves + kSplitWaves - 1) / kSplitWaves;
    const unsigned zb = a.B < 65535 ? a.B : 65535;
    const dim3 block(kSplitWaves * kWave);
    if (nt == 1) hipLaunchKernelGGL((kv_split_kernel<T, D, 1>), dim3(groups), block, 0, s, a, sp);
    else if (nt == 2) hipLaunchKernelGGL((kv_split_kernel<T, D, 2>), dim3(groups), block, 0, s, a, sp);
    else hipLaunchKernelGGL((kv_split_kernel<T, D, 4>), dim3(groups), block, 0, s, a, sp);
    hipLaunchKernelGGL((kv_join_kernel<T, D>), dim3(sp.most_rows, a.c.heads, zb), dim3(32 * kJoinParts), 0, s, a, sp,
                       groups * kSplitWaves);
    if (rows > sp.most_rows)
        hipLaunchKernelGGL((kv_attn_kernel<T, D>), dim3((unsigned)((rows + 15) / 16), a.c.heads, zb), dim3(kWave), 0, s,
                           a, sp.most_rows);
}

}  // namespace pyc

extern "C" size_t pyc_hip_kv_attention_workspace_bytes(int B, int hq, int hk, int d, int max_q) {
    using namespace pyc;
    const long rows = (long)max_q * (hq / hk);
    const int nt = split_tiles(rows);
    const long most = rows < 16 * nt ? rows : 16 * nt;
    return (size_t)2 * kSplitMost * most * (d + 2) * sizeof(float);
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
    float* part = (float*)workspace;
    if (a.c.d == 128) {
        if (is_bf16) launch_attention<bf16_t, 128>(a, part, max_len, s);
        else launch_attention<f16_t, 128>(a, part, max_len, s);
    } else {
        if (is_bf16) launch_attention<bf16_t, 64>(a, part, max_len, s);
        else launch_attention<f16_t, 64>(a, part, max_len, s);
    }
    return hipGetLastError() == hipSuccess ? 0 : -2;
}

extern "C" int pyc_hip_kinfo_kv_attention(int is_bf16, pyc_hip_kinfo* out) {
    using namespace pyc;
    if (!out) return -1;
    out->fn = is_bf16 ? reinterpret_cast<const void*>(&kv_split_kernel<bf16_t, 128, 1>)
                      : reinterpret_cast<const void*>(&kv_split_kernel<f16_t, 128, 1>);
    out->name = "kv_split_kernel<128, 1>";
    out->lds_bytes = 0;
    out->threads = kSplitWaves * kWave;
    out->waves_per_simd = 2;
    return 0;
}
