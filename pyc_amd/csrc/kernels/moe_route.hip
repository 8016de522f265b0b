// moe_route.hip — the k experts of each token, their weights, and the order that puts
// the tokens of one expert together.
//
//   chosen_t   the k largest logits of row t, ties to the lower expert; -infinity and NaN
//              are never chosen (a token may have fewer than k, or none: id -1, weight 0)
//   weight     e^(l_i - m) / s, m the row's largest, s the sum over all experts or
//              (normalize) over the chosen ones. m = +infinity: its limit, 1 at each
//              +infinity and 0 elsewhere, before the division.
//   offsets    where each expert's rows begin; rows[offsets[e] ..] its flat indexes
//              t * k + j in ascending order, -1 behind the last expert's;
//              places[t * k + j] the position of a flat index in rows, -1 without expert.
//
// A wave for two tokens, their logits in registers (E <= 1024: up to 16 a lane). One of the k
// steps: the largest value by lanes, the lowest expert that has it by ballots, which
// costs no more with ties. A token takes an expert once, so 32 tokens' choices are one
// word of bits for each expert: setting bits needs no order, and the rank of a token
// among its expert's is a count of lower bits. So no sum depends on the order of
// atomics, and equal inputs give equal outputs.
// Up to 64 tokens one workgroup does it all; above, the first launch leaves each
// 32 tokens' words in the workspace and the second adds up the words before its own.
//
// Bound by vector instructions: the logits are read once (2 MB of 8200 tokens by 128 experts, under
// 1 us), but each of a token's choices takes a maximum over all 64 lanes, 37 instructions in all (a wave makes the
// choices of two tokens side by side). 32 tokens by 64 experts, 8 chosen: 7.8 us a call, 7.6 on the
// device, where one CU issues them in 14,200 of its 18,400 cycles (8.8 one token after the other, ids read back
// from memory). 8200 tokens by 128 experts 17 us, 10 and 7 on the device: 88 % of the first launch's cycles
// issue them, 54 % of the second's, which waits for the first (27 with the wave's maximum through LDS and eight
// blocks to every workgroup of the second launch).
#include "common.hpp"

namespace pyc {

constexpr int kRouteThreads = 1024;
constexpr int kRouteWaves = kRouteThreads / kWave;
constexpr int kRouteBlock = 32;     // tokens to a word
constexpr int kRouteExperts = 1024;
constexpr int kOneBlocks = 2;       // blocks one workgroup does alone
constexpr int kScatterMost = 8;     // blocks to a workgroup of the second launch, at most

struct Route {
    const void* logits;
    int64_t stride;
    int T, E, k, normalize;
    int32_t* ids;
    float* weights;
    int32_t* offsets;
    int32_t* rows;
    int32_t* places;
    uint32_t* words;  // [blocks][E]
};

template <int DT> __device__ inline float route_logit(const void* p, int64_t i) {
    if constexpr (DT == 0) return static_cast<const float*>(p)[i];
    else if constexpr (DT == 1) return elem<bf16_t>::to_f32(static_cast<const uint16_t*>(p)[i]);
    else return elem<f16_t>::to_f32(static_cast<const uint16_t*>(p)[i]);
}

// Over the wave's lanes, by DPP: four steps in each row of 16, then the rows' last lanes; lane 63 has it.
template <int CTRL, int ROWS> __device__ inline float dpp_f(float old, float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(v), CTRL, ROWS, 0xf, false));
}
__device__ inline float last_lane(float v) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63)); }
__device__ inline float wave_max(float v) {
    v = fmaxf(v, dpp_f<0x111, 0xf>(v, v));
    v = fmaxf(v, dpp_f<0x112, 0xf>(v, v));
    v = fmaxf(v, dpp_f<0x114, 0xf>(v, v));
    v = fmaxf(v, dpp_f<0x118, 0xf>(v, v));
    v = fmaxf(v, dpp_f<0x142, 0xa>(v, v));
    v = fmaxf(v, dpp_f<0x143, 0xc>(v, v));
    return last_lane(v);
}
__device__ inline float wave_sum(float v) {
    v += dpp_f<0x111, 0xf>(0.f, v);
    v += dpp_f<0x112, 0xf>(0.f, v);
    v += dpp_f<0x114, 0xf>(0.f, v);
    v += dpp_f<0x118, 0xf>(0.f, v);
    v += dpp_f<0x142, 0xa>(0.f, v);
    v += dpp_f<0x143, 0xc>(0.f, v);
    return last_lane(v);
}

// One wave: the choices of tokens t and t + kRouteWaves (below t1), side by side, for each depends on the one before;
// their bits in the words of blocks (LDS), and the ids there too where `kept` is given.
template <int DT, int NV>
__device__ inline void route_tokens(const Route& r, int t, int t1, uint32_t* words, int16_t* kept, int lane) {
    constexpr float kNone = -INFINITY;
    constexpr int NT = 2;
    float v[NT][NV], m[NT], s[NT], p[NT], top[NT];
    int mine[NT];  // lane j: choice j
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = i * kWave + lane, tn = min(t + n * kRouteWaves, t1 - 1);
            v[n][i] = route_logit<DT>(r.logits, (int64_t)tn * r.stride + min(e, r.E - 1));
        }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const float l = v[n][i];
            v[n][i] = i * kWave + lane < r.E && l == l ? l : kNone;
        }
        m[n] = v[n][0];
#pragma unroll
        for (int i = 1; i < NV; ++i) m[n] = fmaxf(m[n], v[n][i]);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) top[n] = m[n] = wave_max(m[n]);
    auto power = [&](int n, float l) { return l == m[n] ? 1.0f : expf(l - m[n]); };  // m infinite: 1 or 0
    if (!r.normalize) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            s[n] = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i) s[n] += v[n][i] > kNone ? power(n, v[n][i]) : 0.f;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n] = wave_sum(s[n]);
    }
    float chosen[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        mine[n] = -1;
        chosen[n] = kNone;
    }
    for (int j = 0; j < r.k; ++j) {
        float left[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            int best = -1;
#pragma unroll
            for (int i = NV - 1; i >= 0; --i) {
                const uint64_t is = __ballot(v[n][i] == top[n] && top[n] > kNone);
                best = is ? i * kWave + __builtin_ctzll(is) : best;
            }
            mine[n] = lane == j ? best : mine[n];
            chosen[n] = lane == j ? top[n] : chosen[n];
            left[n] = kNone;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                v[n][i] = i * kWave + lane == best ? kNone : v[n][i];
                left[n] = fmaxf(left[n], v[n][i]);
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) top[n] = wave_max(left[n]);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) p[n] = mine[n] >= 0 ? power(n, chosen[n]) : 0.f;
    if (r.normalize) {
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n] = wave_sum(p[n]);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int tn = t + n * kRouteWaves;
        if (tn < t1 && lane < r.k) {
            r.ids[(int64_t)tn * r.k + lane] = mine[n];
            r.weights[(int64_t)tn * r.k + lane] = mine[n] >= 0 ? p[n] / s[n] : 0.f;
            if (mine[n] >= 0) atomicOr(&words[mine[n]], 1u << (tn % kRouteBlock));
            if (kept) kept[tn * r.k + lane] = (int16_t)mine[n];
        }
    }
}

// Exclusive sums over the experts of n[e] (LDS, E of them) into first[], the total returned.
__device__ inline int route_scan(const int* n, int* first, int E, int* part, int tid) {
    const int v = tid < E ? n[tid] : 0;  // E <= the workgroup's threads
    const int lane = tid & 63, wave = tid >> 6;
    int sum = v;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const int o = __shfl_up(sum, d);
        sum = lane >= d ? sum + o : sum;
    }
    if (lane == 63) part[wave] = sum;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kRouteWaves; ++w) {
        before += w < wave ? part[w] : 0;
        all += part[w];
    }
    if (tid < E) first[tid] = before + sum - v;
    __syncthreads();
    return all;
}

// Place and row of flat index f, which chose e, of token t of its block of 32, whose words and first positions are given.
__device__ inline void route_place(const Route& r, int64_t f, int e, const uint32_t* words, const int* first, int t) {
    int at = -1;
    if (e >= 0) {
        at = first[e] + __popc(words[e] & ((1u << t) - 1u));
        // inside rows, whatever a second call on the same workspace left in the words
        if ((unsigned)at < (unsigned)(r.T * r.k)) r.rows[at] = (int32_t)f;
    }
    r.places[f] = at;
}

template <int DT, int NV, bool ONE>
__global__ void __launch_bounds__(kRouteThreads) moe_route_kernel(Route r) {
    constexpr int BLOCKS = ONE ? kOneBlocks : 1;
    __shared__ uint32_t words[BLOCKS][NV * kWave];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int b0 = ONE ? 0 : blockIdx.x;
    for (int i = tid; i < BLOCKS * NV * kWave; i += kRouteThreads) (&words[0][0])[i] = 0;
    __syncthreads();
    const int t0 = b0 * kRouteBlock, t1 = min(r.T, t0 + BLOCKS * kRouteBlock);
    __shared__ int16_t kept[ONE ? kOneBlocks * kRouteBlock * kWave : 1];  // k <= 64
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
        const int t = t0 + b * kRouteBlock + wave;
        if (t < t1) route_tokens<DT, NV>(r, t, t1, words[b], ONE ? kept : nullptr, lane);
    }
    __syncthreads();
    if constexpr (ONE) {
        __shared__ int count[NV * kWave], first[BLOCKS][NV * kWave], part[kRouteWaves];
        if (tid < r.E) {
            int n = 0;
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) n += __popc(words[b][tid]);
            count[tid] = n;
        }
        __syncthreads();
        const int all = route_scan(count, first[0], r.E, part, tid);
        if (tid < r.E) {
            r.offsets[tid] = first[0][tid];
#pragma unroll
            for (int b = 1; b < BLOCKS; ++b) first[b][tid] = first[b - 1][tid] + __popc(words[b - 1][tid]);
        }
        if (tid == 0) r.offsets[r.E] = all;
        __syncthreads();
        const int each = kRouteBlock * r.k;
        for (int i = tid; i < r.T * r.k; i += kRouteThreads) {
            const int b = i / each;
            route_place(r, i, kept[i], words[b], first[b], (i - b * each) / r.k);
        }
        for (int i = all + tid; i < r.T * r.k; i += kRouteThreads) r.rows[i] = -1;
    } else {
        for (int e = tid; e < r.E; e += kRouteThreads) r.words[(int64_t)b0 * r.E + e] = words[0][e];
    }
}

// nb blocks to a workgroup. Every workgroup adds up all blocks' words by itself, which up to 65536 tokens costs less than
// a third launch: the words (1 MB by 128 experts) stay in L2. That work grows with the square of the tokens and takes over
// from 2^18 on (by 128 experts, 8 chosen: 2^16 tokens 75 us, 2^17 172, 2^18 479, 2^20 5.4 ms).
__global__ void __launch_bounds__(kRouteThreads) moe_scatter_kernel(Route r, int blocks, int nb) {
    __shared__ uint32_t own[kScatterMost][kRouteExperts];
    __shared__ int first[kScatterMost + 1][kRouteExperts];
    __shared__ int count[kRouteExperts], before[kRouteExperts], part[kRouteWaves];
    const int tid = threadIdx.x;
    const int b0 = blockIdx.x * nb, mine = min(nb, blocks - b0);
    for (int e = tid; e < r.E; e += kRouteThreads) count[e] = before[e] = 0;
    const int each = kRouteBlock * r.k;
    const int n = min(mine * each, (r.T - b0 * kRouteBlock) * r.k);
    int e0 = tid < n ? r.ids[(int64_t)b0 * each + tid] : -1;  // on its way from the start
    for (int i = tid; i < mine * r.E; i += kRouteThreads) own[i / r.E][i % r.E] = r.words[(int64_t)b0 * r.E + i];
    __syncthreads();
    const int per = kRouteThreads / r.E;  // threads to an expert, each a share of the blocks
    if (tid < per * r.E) {
        const int e = tid % r.E;
        int n = 0, low = 0;
        for (int b = tid / r.E; b < blocks; b += 8 * per) {
            uint32_t w[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) w[u] = r.words[(int64_t)min(b + u * per, blocks - 1) * r.E + e];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int c = b + u * per < blocks ? __popc(w[u]) : 0;
                n += c;
                low += b + u * per < b0 ? c : 0;
            }
        }
        atomicAdd(&count[e], n);
        atomicAdd(&before[e], low);
    }
    __syncthreads();
    const int all = route_scan(count, first[0], r.E, part, tid);
    if (blockIdx.x == 0) {
        if (tid < r.E) r.offsets[tid] = first[0][tid];
        if (tid == 0) r.offsets[r.E] = all;
    }
    __syncthreads();
    if (tid < r.E) {
        int at = first[0][tid] + before[tid];
        for (int b = 0; b < mine; ++b) {
            first[b][tid] = at;
            at += __popc(own[b][tid]);
        }
    }
    __syncthreads();
    for (int i = tid; i < n; i += kRouteThreads) {
        const int b = i / each, t = (i - b * each) / r.k;
        route_place(r, (int64_t)b0 * each + i, min(e0, r.E - 1), own[b], first[b], t);
        if (i + kRouteThreads < n) e0 = r.ids[(int64_t)b0 * each + i + kRouteThreads];
    }
    for (int i = all + blockIdx.x * kRouteThreads + tid; i < r.T * r.k; i += gridDim.x * kRouteThreads) r.rows[i] = -1;
}

template <int DT, int NV> static int route_launch(const Route& r, hipStream_t s) {
    const int blocks = (r.T + kRouteBlock - 1) / kRouteBlock;
    if (blocks <= kOneBlocks) {
        hipLaunchKernelGGL((moe_route_kernel<DT, NV, true>), dim3(1), dim3(kRouteThreads), 0, s, r);
        return hipGetLastError() == hipSuccess ? 0 : -2;
    }
    hipLaunchKernelGGL((moe_route_kernel<DT, NV, false>), dim3(blocks), dim3(kRouteThreads), 0, s, r);
    // two blocks to a workgroup; eight where the words that each of them reads are many
    const int nb = (int64_t)blocks * r.E <= 65536 ? 2 : kScatterMost;
    hipLaunchKernelGGL(moe_scatter_kernel, dim3((blocks + nb - 1) / nb), dim3(kRouteThreads), 0, s, r, blocks, nb);
    return hipGetLastError() == hipSuccess ? 0 : -2;
}

}  // namespace pyc

// Workspace of a call: a word for each expert and 32 tokens where it takes two launches.
extern "C" size_t pyc_hip_moe_route_workspace_bytes(int T, int E) {
    const size_t blocks = ((size_t)T + pyc::kRouteBlock - 1) / pyc::kRouteBlock;
    return blocks <= (size_t)pyc::kOneBlocks ? 0 : blocks * (size_t)E * 4;
}

extern "C" int pyc_hip_moe_route_launch(int dtype, int T, int E, int k, int normalize, const void* logits, int64_t stride,
                                        int32_t* ids, float* weights, int32_t* offsets, int32_t* rows, int32_t* places,
                                        void* workspace, void* stream) {
    using namespace pyc;
    const Route r{logits, stride, T, E, k, normalize, ids, weights, offsets, rows, places, (uint32_t*)workspace};
    const hipStream_t s = (hipStream_t)stream;
#define PYC_ROUTE(DT)                                       \
    (E <= 64 ? route_launch<DT, 1>(r, s) : E <= 128 ? route_launch<DT, 2>(r, s) \
     : E <= 256 ? route_launch<DT, 4>(r, s) : route_launch<DT, 16>(r, s))
    return dtype == 0 ? PYC_ROUTE(0) : dtype == 1 ? PYC_ROUTE(1) : PYC_ROUTE(2);
#undef PYC_ROUTE
}

extern "C" int pyc_hip_kinfo_moe_route(int dtype, pyc_hip_kinfo* out) {
    using namespace pyc;
    if (!out) return -1;
    out->fn = dtype == 0   ? reinterpret_cast<const void*>(&moe_route_kernel<0, 2, false>)
              : dtype == 1 ? reinterpret_cast<const void*>(&moe_route_kernel<1, 2, false>)
                           : reinterpret_cast<const void*>(&moe_route_kernel<2, 2, false>);
    out->name = "moe_route_kernel";
    out->lds_bytes = 2 * kWave * 4;
    out->threads = kRouteThreads;
    out->waves_per_simd = 8;
    return 0;
}
