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
// Whole numbers only: three prefix sums over the requests and one lookup per token.
#include "common.hpp"

namespace pyc {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / kWave;

struct PlanSum {
    int64_t blocks, tokens;
};

// Inclusive sum over the workgroup's threads; `all` is the sum of all of them.
__device__ inline PlanSum plan_scan(PlanSum v, PlanSum* all, PlanSum* waves) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const int64_t b = __shfl_up(v.blocks, d), t = __shfl_up(v.tokens, d);
        if (lane >= d) {
            v.blocks += b;
            v.tokens += t;
        }
    }
    __syncthreads();  // the last use of `waves`
    if (lane == kWave - 1) waves[wave] = v;
    __syncthreads();
    PlanSum before{0, 0};
    *all = PlanSum{0, 0};
    for (int w = 0; w < kPlanWaves; ++w) {
        if (w < wave) {
            before.blocks += waves[w].blocks;
            before.tokens += waves[w].tokens;
        }
        all->blocks += waves[w].blocks;
        all->tokens += waves[w].tokens;
    }
    v.blocks += before.blocks;
    v.tokens += before.tokens;
    return v;
}

struct PlanArgs {
    int B, width, bs, tokens, free_cap;
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

// Slot and position of token t: the request is the last one whose offset is <= t.
__device__ inline void plan_token(const PlanArgs& a, int t, int total) {
    int slot = -1, pos = -1;
    if (t < total) {
        int lo = 0, hi = a.B;  // q_offsets[lo] <= t < q_offsets[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.q_offsets[mid] <= t) lo = mid;
            else hi = mid;
        }
        // the request was granted: its length now, less its tokens behind this one
        pos = a.lens[lo] - (a.q_offsets[lo + 1] - t);
        slot = a.table[lo * a.table_stride + pos / a.bs] * a.bs + pos % a.bs;
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
}

__global__ void __launch_bounds__(kPlanThreads) kv_plan_kernel(PlanArgs a, int with_tokens) {
    __shared__ PlanSum waves[kPlanWaves];
    const int tid = threadIdx.x;
    const int64_t cap_tokens = (int64_t)a.width * a.bs;
    const int64_t F = min(max(a.free_count[0], 0), a.free_cap);
    auto held = [&](int b) { return min((int64_t)max(a.cached[b], 0), cap_tokens); };

    // Ended requests give their blocks back.
    int64_t pushed = 0;
    for (int b0 = 0; b0 < a.B; b0 += kPlanThreads) {
        const int b = b0 + tid;
        int64_t back = 0;
        if (b < a.B && a.fresh[b] < 0) back = (held(b) + a.bs - 1) / a.bs;
        PlanSum all;
        const PlanSum end = plan_scan(PlanSum{back, 0}, &all, waves);
        for (int64_t j = 0; j < back; ++j) {
            const int64_t at = F + pushed + end.blocks - back + j;
            if (at < a.free_cap) a.free_list[at] = a.table[b * a.table_stride + j];
        }
        pushed += all.blocks;
    }
    const int64_t top = min(F + pushed, (int64_t)a.free_cap);
    __syncthreads();  // the pushed entries are read below

    PlanSum asked{0, 0}, given{0, 0};
    for (int b0 = 0; b0 < a.B; b0 += kPlanThreads) {
        const int b = b0 + tid;
        int64_t have_tokens = 0, ask = 0, need = 0, have = 0;
        int f = 0;
        if (b < a.B) {
            f = a.fresh[b];
            have_tokens = held(b);
            have = (have_tokens + a.bs - 1) / a.bs;
            if (f > 0 && have_tokens + f <= cap_tokens) {
                ask = f;
                need = (have_tokens + f + a.bs - 1) / a.bs - have;
            }
        }
        PlanSum all;
        const PlanSum end = plan_scan(PlanSum{need, ask}, &all, waves);
        const bool granted = ask > 0 && (need == 0 || asked.blocks + end.blocks <= top) &&
                             asked.tokens + end.tokens <= a.tokens;
        asked.blocks += all.blocks;
        asked.tokens += all.tokens;
        if (!granted) ask = need = 0;
        const PlanSum mine = plan_scan(PlanSum{need, ask}, &all, waves);
        for (int64_t j = 0; j < need; ++j)
            a.table[b * a.table_stride + have + j] = a.free_list[top - 1 - (given.blocks + mine.blocks - need + j)];
        if (b < a.B) {
            a.lens[b] = f < 0 ? 0 : (int)(have_tokens + ask);
            a.q_offsets[b] = (int)(given.tokens + mine.tokens - ask);
        }
        given.blocks += all.blocks;
        given.tokens += all.tokens;
    }
    if (tid == 0) {
        a.q_offsets[a.B] = (int)given.tokens;
        a.free_after[0] = (int)(top - given.blocks);
    }
    if (!with_tokens) return;
    __syncthreads();  // lens, q_offsets and the table are read below
    for (int t = tid; t < a.tokens; t += kPlanThreads) plan_token(a, t, (int)given.tokens);
}

__global__ void __launch_bounds__(256) kv_slots_kernel(PlanArgs a) {
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t < a.tokens) plan_token(a, t, a.q_offsets[a.B]);
}

}  // namespace pyc

extern "C" int pyc_hip_kv_plan_launch(int B, int width, int64_t table_stride, int bs, int tokens,
                                      const int32_t* cached, const int32_t* fresh, int32_t* table, int32_t* free_list,
                                      int free_cap, const int32_t* free_count, int32_t* lens, int32_t* q_offsets,
                                      int32_t* slots, int32_t* positions, int32_t* free_after, void* stream) {
    using namespace pyc;
    const PlanArgs a{B,          width,     bs,        tokens,     free_cap, cached,    fresh,     table,
                     table_stride, free_list, free_count, lens,     q_offsets, slots, positions, free_after};
    hipStream_t s = (hipStream_t)stream;
    const int one = tokens <= 4 * kPlanThreads;
    hipLaunchKernelGGL(kv_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a, one);
    if (!one) hipLaunchKernelGGL(kv_slots_kernel, dim3((tokens + 255) / 256), dim3(256), 0, s, a);
    return hipGetLastError() == hipSuccess ? 0 : -2;
}

extern "C" int pyc_hip_kinfo_kv_plan(pyc_hip_kinfo* out) {
    using namespace pyc;
    if (!out) return -1;
    out->fn = reinterpret_cast<const void*>(&kv_plan_kernel);
    out->name = "kv_plan_kernel";
    out->lds_bytes = sizeof(PlanSum) * kPlanWaves;
    out->threads = kPlanThreads;
    out->waves_per_simd = 4;
    return 0;
}
