// kv_plan.hip — block tables, slot map, positions and query offsets of one
// serving step, from what each request holds in the paged cache and what it brings.
//
// With have = ceil(cached / bs) blocks per request and the free blocks a stack:
//   released (fresh < 0): table[b][0 .. have) is pushed, in request order;
//   asked, if cached + fresh fits the table: need = ceil((cached + fresh) / bs) - have;
//   granted: need == 0 or sum_{c <= b} need <= blocks on the stack, and
//            sum_{c <= b} fresh <= tokens (both sums over what was asked);
//   the new blocks are popped in request order; lens, q_offsets (exclusive sum
//   of the granted tokens), and per token its position and slot
//   table[b][pos / bs] * bs + pos % bs.
// Whole numbers only: prefix sums over the requests, in one workgroup, and one lookup
// per token. Latency bounds it: a handful of dependent loads and stores of a few
// hundred nanoseconds each. So everything that can be known is loaded at once, blocks
// move a wave at a time, a step whose requests bring a token each writes it from the
// request's own thread, and many tokens get a launch over all CUs (from 4096 on: below,
// the one workgroup has them sooner than a second launch starts). 32 requests of a token
// each: 2.1 us on the device, 7.5 with the call; 1024 requests that bring 55206 tokens:
// 9.0 and 4.1 on the device, 13.1 with the call.
#include "kv_cache.hpp"

namespace pyc {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / kWave;
constexpr uint32_t kPlanMost = 0x7fffffffu;  // sums stop here: more than there is of anything

struct PlanSum {
    uint32_t blocks, tokens;
};
__device__ inline PlanSum plan_add(PlanSum a, PlanSum b) {
    return PlanSum{min(a.blocks + b.blocks, kPlanMost), min(a.tokens + b.tokens, kPlanMost)};
}

// Inclusive sum over the workgroup's threads; `all` is the sum of all of them.
__device__ inline PlanSum plan_scan(PlanSum v, PlanSum* all, PlanSum* waves) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, n = blockDim.x / kWave;
    auto add = [](int a, int b) { return (int)min((uint32_t)a + (uint32_t)b, kPlanMost); };
    v = PlanSum{(uint32_t)wave_scan((int)v.blocks, 0, add), (uint32_t)wave_scan((int)v.tokens, 0, add)};
    if (n == 1) {
        *all = PlanSum{(uint32_t)__builtin_amdgcn_readlane((int)v.blocks, kWave - 1),
                       (uint32_t)__builtin_amdgcn_readlane((int)v.tokens, kWave - 1)};
        return v;
    }
    __syncthreads();  // the last use of `waves`
    if (lane == kWave - 1) waves[wave] = v;
    __syncthreads();
    // every wave scans the waves' sums
    PlanSum w = lane < n ? waves[lane] : PlanSum{0, 0};
    w = PlanSum{(uint32_t)wave_scan((int)w.blocks, 0, add), (uint32_t)wave_scan((int)w.tokens, 0, add)};
    auto at = [&](int i) {
        return PlanSum{(uint32_t)__builtin_amdgcn_readlane((int)w.blocks, i),
                       (uint32_t)__builtin_amdgcn_readlane((int)w.tokens, i)};
    };
    *all = at(kWave - 1);
    const int uw = __builtin_amdgcn_readfirstlane(wave);
    return uw ? plan_add(v, at(uw - 1)) : v;
}

// The workgroup's threads' bits, or-ed.
__device__ inline uint32_t plan_vote(uint32_t bits, uint32_t* votes) {
    const int n = blockDim.x / kWave;
    const uint32_t mine = (__any(bits & 1) ? 1u : 0u) | (__any(bits & 2) ? 2u : 0u);
    if (n == 1) return mine;
    __syncthreads();  // the last use of `votes`
    if ((threadIdx.x & (kWave - 1)) == 0) votes[threadIdx.x / kWave] = mine;
    __syncthreads();
    const uint32_t theirs = votes[min((int)(threadIdx.x & (kWave - 1)), n - 1)];
    return (__any(theirs & 1) ? 1u : 0u) | (__any(theirs & 2) ? 2u : 0u);
}

struct PlanArgs {
    int B, width, bs, shift, tokens, free_cap;  // bs == 1 << shift
    const int32_t* cached;
    const int32_t* fresh;
    int32_t* table;
    int64_t table_stride;
    int32_t* free_list;
    const int32_t* free_count;
    int32_t* lens;
    int32_t* q_offsets;
    int32_t* slots;
    int32_t* positions;
    int32_t* free_after;
};

// Slot and position of token t < q_offsets[B]: the request is the last one whose
// offset is <= t (offsets in LDS or global memory).
__device__ inline void plan_token(const PlanArgs& a, const int32_t* offsets, const int32_t* lens, int t) {
    int lo = 0, hi = a.B;  // offsets[lo] <= t < offsets[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (offsets[mid] <= t) lo = mid;
        else hi = mid;
    }
    // the request was granted: its length now, less its tokens behind this one
    const int pos = lens[lo] - (offsets[lo + 1] - t);
    a.slots[t] = a.table[lo * a.table_stride + (pos >> a.shift)] * a.bs + (pos & (a.bs - 1));
    a.positions[t] = pos;
}

// Moves one block id for every j < count of every thread of the workgroup: from(i, j,
// k) to to(i, j, k), with i the thread and k counting all; `end` is the inclusive sum
// of count over the threads. Counts of up to two everywhere (`few`): each thread
// does its own, else all are dealt out, four to a thread at a time.
constexpr uint32_t kPlanFew = 2;
template <typename From, typename To>
__device__ inline void plan_move(bool few, uint32_t count, uint32_t end, uint32_t all, uint32_t* s_end, From from, To to) {
    if (few) {
        for (uint32_t j = 0; j < count; ++j) {
            int32_t* dst = to((int)threadIdx.x, j, end - count + j);
            if (dst) *dst = *from((int)threadIdx.x, j, end - count + j);
        }
        return;
    }
    const int T = (int)blockDim.x;
    __syncthreads();  // the last use of s_end
    s_end[threadIdx.x] = end;
    __syncthreads();
    for (uint32_t k0 = threadIdx.x; k0 < all; k0 += 4 * T) {
        int32_t id[4], *dst[4];
        int i[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) i[x] = 0;
        for (int step = T / 2; step > 0; step /= 2)  // the first thread whose end is past k
#pragma unroll
            for (int x = 0; x < 4; ++x)
                if (s_end[i[x] + step - 1] <= k0 + x * T) i[x] += step;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const uint32_t k = k0 + x * T;
            dst[x] = nullptr;
            if (k >= all) continue;
            const uint32_t j = k - (i[x] ? s_end[i[x] - 1] : 0u);
            dst[x] = to(i[x], j, k);
            if (dst[x]) id[x] = *from(i[x], j, k);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x)
            if (dst[x]) *dst[x] = id[x];
    }
}

__global__ void __launch_bounds__(kPlanThreads) kv_plan_kernel(PlanArgs a, int with_tokens) {
    __shared__ PlanSum waves[kPlanWaves];
    __shared__ uint32_t votes[kPlanWaves];
    __shared__ int32_t s_offsets[kPlanThreads + 4], s_lens[kPlanThreads], s_have[kPlanThreads];
    __shared__ uint32_t s_end[kPlanThreads];
    const int tid = threadIdx.x, T = blockDim.x;
    const int cap_tokens = a.width * a.bs;
    const uint32_t F = (uint32_t)min(max(a.free_count[0], 0), a.free_cap);

    PlanSum asked{0, 0}, given{0, 0};
    uint32_t top = F;
    bool long_asks = false;
    auto load = [&](int b, int* held, int* fresh, int* block) {
        *held = *fresh = *block = 0;
        if (b < a.B) {
            *held = min(max(a.cached[b], 0), cap_tokens);
            *fresh = a.fresh[b];
            *block = a.table[b * a.table_stride + min(*held >> a.shift, a.width - 1)];
        }
    };
    int held, fresh, block;  // block: the entry that the next token falls into
    load(tid, &held, &fresh, &block);
    // Ended requests give their blocks back. (A first request is looked at before
    // any sum: most steps have none that ends.)
    for (int b0 = 0; b0 < a.B; b0 += T) {
        const int b = b0 + tid, f = b0 == 0 ? fresh : b < a.B ? a.fresh[b] : 0;
        if (!plan_vote(f < 0, votes)) continue;
        uint32_t back = 0;
        if (f < 0) back = (uint32_t)((b0 == 0 ? held : min(max(a.cached[b], 0), cap_tokens)) + a.bs - 1) >> a.shift;
        PlanSum all;
        const PlanSum end = plan_scan(PlanSum{back, 0}, &all, waves);
        plan_move(
            false, back, end.blocks, all.blocks, s_end,
            [&](int i, uint32_t j, uint32_t) { return a.table + (b0 + i) * a.table_stride + j; },
            [&](int, uint32_t, uint32_t k) { return top + k < (uint32_t)a.free_cap ? a.free_list + top + k : nullptr; });
        top = min(top + all.blocks, (uint32_t)a.free_cap);
    }
    if (top != F) __syncthreads();  // the pushed entries are read below

    for (int b0 = 0; b0 < a.B; b0 += T) {
        const int b = b0 + tid;
        if (b0 != 0) load(b, &held, &fresh, &block);
        const int have = (int)((uint32_t)(held + a.bs - 1) >> a.shift);
        uint32_t ask = 0, need = 0;
        if (fresh > 0 && fresh <= cap_tokens - held) {
            ask = (uint32_t)fresh;
            need = (((uint32_t)held + ask + a.bs - 1) >> a.shift) - have;
        }
        PlanSum all;
        PlanSum end = plan_add(asked, plan_scan(PlanSum{need, ask}, &all, waves));
        const bool refused = ask > 0 && ((need > 0 && end.blocks > top) || end.tokens > (uint32_t)a.tokens);
        asked = plan_add(asked, all);
        if (plan_vote(refused, votes)) {
            if (refused) ask = need = 0;
            end = plan_add(given, plan_scan(PlanSum{need, ask}, &all, waves));
        } else {
            end = plan_add(given, PlanSum{end.blocks - (asked.blocks - all.blocks), end.tokens - (asked.tokens - all.tokens)});
        }
        const uint32_t first = end.tokens - ask, pop = top - 1 - (end.blocks - need);  // its first token and new block
        if (need > 0 && have == held >> a.shift) block = a.free_list[pop];
        const uint32_t vote = plan_vote((ask > 1 ? 1 : 0) | (need > kPlanFew ? 2 : 0), votes);
        long_asks |= (vote & 1) != 0;
        s_have[tid] = have;  // read behind plan_move's barriers, or by this thread
        plan_move(
            !(vote & 2), need, end.blocks - given.blocks, all.blocks, s_end,
            [&](int, uint32_t, uint32_t k) { return a.free_list + (top - 1 - (given.blocks + k)); },
            [&](int i, uint32_t j, uint32_t) { return a.table + (b0 + i) * a.table_stride + s_have[i] + j; });
        given = plan_add(given, all);
        if (b < a.B) {
            const int len = fresh < 0 ? 0 : held + (int)ask;
            a.lens[b] = len;
            a.q_offsets[b] = (int)first;
            if (a.B <= T) {
                s_lens[tid] = len;
                s_offsets[tid] = (int)first;
            }
            if (with_tokens && !long_asks && ask == 1) {
                a.slots[first] = block * a.bs + (held & (a.bs - 1));
                a.positions[first] = held;
            }
        }
    }
    const int total = (int)given.tokens;
    if (tid == 0) {
        a.q_offsets[a.B] = total;
        s_offsets[a.B <= T ? a.B : 0] = total;
        a.free_after[0] = (int)(top - given.blocks);
    }
    if (!with_tokens) return;
    if (long_asks) {
        __syncthreads();  // lens, offsets and the table are read below
        const bool near = a.B <= T;
        for (int t = tid; t < total; t += T) plan_token(a, near ? s_offsets : a.q_offsets, near ? s_lens : a.lens, t);
    }
    for (int t = total + tid; t < a.tokens; t += T) a.slots[t] = a.positions[t] = -1;
}

// Many tokens: the search runs in LDS where the offsets fit.
constexpr int kSlotsNear = 1024;
__global__ void __launch_bounds__(256) kv_slots_kernel(PlanArgs a) {
    __shared__ int32_t s_offsets[kSlotsNear + 1];
    const int t = blockIdx.x * 256 + threadIdx.x;
    const bool near = a.B <= kSlotsNear;
    if (near) {
        for (int i = threadIdx.x; i <= a.B; i += 256) s_offsets[i] = a.q_offsets[i];
        __syncthreads();
    }
    if (t >= a.tokens) return;
    if (t < (near ? s_offsets[a.B] : a.q_offsets[a.B])) plan_token(a, near ? s_offsets : a.q_offsets, a.lens, t);
    else a.slots[t] = a.positions[t] = -1;
}

}  // namespace pyc

extern "C" int pyc_hip_kv_plan_launch(int B, int width, int64_t table_stride, int bs, int tokens,
                                      const int32_t* cached, const int32_t* fresh, int32_t* table, int32_t* free_list,
                                      int free_cap, const int32_t* free_count, int32_t* lens, int32_t* q_offsets,
                                      int32_t* slots, int32_t* positions, int32_t* free_after, void* stream) {
    using namespace pyc;
    const PlanArgs a{B,      width,        bs,        __builtin_ctz(bs), tokens, free_cap,  cached, fresh,
                     table,  table_stride, free_list, free_count,        lens,   q_offsets, slots,  positions,
                     free_after};
    hipStream_t s = (hipStream_t)stream;
    // One workgroup looks up 4096 tokens in about the time of another launch.
    const int one = tokens <= 4 * kPlanThreads;
    int threads = kWave;
    while (threads < kPlanThreads && (threads < B || (one && 4 * threads < tokens))) threads *= 2;
    hipLaunchKernelGGL(kv_plan_kernel, dim3(1), dim3(threads), 0, s, a, one);
    if (!one) hipLaunchKernelGGL(kv_slots_kernel, dim3((tokens + 255) / 256), dim3(256), 0, s, a);
    return hipGetLastError() == hipSuccess ? 0 : -2;
}

extern "C" int pyc_hip_kinfo_kv_plan(pyc_hip_kinfo* out) {
    using namespace pyc;
    if (!out) return -1;
    out->fn = reinterpret_cast<const void*>(&kv_plan_kernel);
    out->name = "kv_plan_kernel";
    out->lds_bytes = (sizeof(PlanSum) + sizeof(uint32_t)) * kPlanWaves + sizeof(int32_t) * (4 * kPlanThreads + 4);
    out->threads = kPlanThreads;
    out->waves_per_simd = 8;
    return 0;
}
