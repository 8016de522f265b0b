// grouped_tile.hip — products by expert of many rows, 16-bit weights: bound by the matrix
// units from about 270 rows of an expert on, by the stream of the weights below.
//
// 256 rows of one expert x 256 rows of its W per tile, four waves of 128 x 128, K in stages of 64
// that LDS-DMA brings in (two of them, XOR-swizzled), the matrix instructions of a stage laid
// out in order with the fragment reads and the loads between them; one workgroup per CU walks
// tiles, and the next tile's first stages load while this one is written out. What is
// particular to experts:
//  * The ragged tiles are counted on the device: at its start a workgroup sums up the
//    experts' tiles into LDS, and finds a tile's expert there with one ballot per 64
//    experts. So nothing is read back and a captured graph follows its routing.
//  * Tiles of one expert are neighbours, its rows (up to 8 tiles of them) first: the CUs of an
//    XCD, which has a contiguous part of the list, share W's and x's lines in their L2.
//  * Rows come through the index: the next tile's are fetched while this one is multiplied.
//    Indexes outside x, rows past the expert's end and k past K get offsets past the
//    buffer's end, which read zeros; rows past the end are stored nowhere the same way.
//  * Gated: 16 rows of gates and 16 of values alternate in the tile, so a lane holds
//    both of a column and 128 columns go out.
// 4096 tokens by 2 of 8 experts of 4096 x 22016, gated: 1270 to 1320 us over cards, 1.12 to 1.16 PFLOP/s, the matrix
// units busy 63 % of the cycles (on one card 1285; 1336 with tiles of 256 rows only, 1315 with the two lists, then a quotient's reciprocal).
// Its registers are full: 16 to 37 values of a tile's start and end lie in scratch, none of the loop over K.
#include <type_traits>

#include "grouped.hpp"
#include "lds_dma.hpp"

namespace pyc {

constexpr int kTile = 256, kTileK = 64;
constexpr int kTileStageRows = 16;  // rows of y a wave stages at once
constexpr uint32_t kTilePastEnd = 0xFFFFFFF0u;
constexpr size_t kTileRing = 2 * 2 * kTile * kTileK * 2;
constexpr size_t kTileOut = 4 * kTileStageRows * 128 * 2;
constexpr size_t kTileLds = kTileRing + kTileOut + 4 * (3 * (kMaxExperts + 1) + kTile);

// TAIL: K is no multiple of 64 (but of 8).
template <typename T, bool GATE, bool TAIL>
__global__ void __launch_bounds__(256, 1) grouped_tile_kernel(Grouped g, int tiles_n) {
    constexpr int BK = kTileK, CH = 8, NT = 256;
    constexpr int LOADS = kTile * CH / NT;              // 8 for each operand, stage and wave
    constexpr uint32_t STAGE_BYTES = kTile * BK * 2;
    constexpr int COLS = GATE ? 64 : 128;               // columns of y to a wave
    constexpr int SR = kTileStageRows;
    constexpr int ROWS_PER_STORE = kWave / (COLS / 8);  // 16-byte stores
    constexpr int STORES = SR / ROWS_PER_STORE;         // per 16 rows of a wave
    __shared__ __attribute__((aligned(1024))) uint8_t smem[kTileLds];
    uint16_t* const As = reinterpret_cast<uint16_t*>(smem);
    uint16_t* const Bs = As + 2 * kTile * BK;
    uint16_t* const Cs = reinterpret_cast<uint16_t*>(smem + kTileRing);
    int* const first = reinterpret_cast<int*>(smem + kTileRing + kTileOut);  // [E + 1] first rows
    int* const high = first + kMaxExperts + 1;                               // [E + 1] row tiles of more than 128 rows before
    int* const low = high + kMaxExperts + 1;                                 // the expert's, and of fewer (at most one each)
    uint32_t* const src = reinterpret_cast<uint32_t*>(low + kMaxExperts + 1);  // offsets of the tile's rows of x

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    const int lrow = lane & 15, lgrp = lane >> 4;
    const int ktiles = (g.K + BK - 1) / BK;
    const int F = GATE ? g.N / 2 : g.N;

    // the experts' first rows and tiles; one wave
    if (wave == 0) {
        int held = 0, nh = 0, nl = 0;
        for (int e0 = 0; e0 < g.E; e0 += kWave) {
            const int e = e0 + lane;
            const bool in = e < g.E;
            const int lo = g.offsets ? min(g.offsets[min(e, g.E)], g.P) : in ? 0 : g.P;
            const int hi = g.offsets ? min(g.offsets[min(e + 1, g.E)], g.P) : g.P;
            const int b = scan_max(max(held, lo));
            const int end = max(b, hi);
            const int h = (end - b + kTile / 2 - 1) / kTile, l = end - b > h * kTile ? 1 : 0;
            const int sh = scan_add(h), sl = scan_add(l);
            if (in) {
                first[e] = b;
                high[e] = nh + sh - h;
                low[e] = nl + sl - l;
                if (e == g.E - 1) {
                    first[g.E] = end;
                    high[g.E] = nh + sh;
                    low[g.E] = nl + sl;
                }
            }
            nh += __builtin_amdgcn_readlane(sh, kWave - 1);
            nl += __builtin_amdgcn_readlane(sl, kWave - 1);
            held = __builtin_amdgcn_readlane(end, kWave - 1);
        }
    }
    __syncthreads();
    // Two lists, of the high tiles and of the low ones, which take half as long or less: XCD x (workgroups b
    // with b % 8 == x) has the x-th eighth of each, and its workgroups take turns through the one, then the other
    const int nhigh = __builtin_amdgcn_readfirstlane(high[g.E]) * tiles_n;  // uniform: what the loop carries stays scalar
    const int nlow = __builtin_amdgcn_readfirstlane(low[g.E]) * tiles_n;
    const int xcd = blockIdx.x & 7, per = gridDim.x >> 3;
    const int h0 = (int)((int64_t)nhigh * xcd / 8), hn = (int)((int64_t)nhigh * (xcd + 1) / 8) - h0;
    const int l0 = (int)((int64_t)nlow * xcd / 8), t_end = hn + (int)((int64_t)nlow * (xcd + 1) / 8) - l0;
    int t = blockIdx.x >> 3;
    if (t >= t_end) return;

    struct Tile {
        int e, row, end, col;  // expert, first row of y, the expert's end, first column of y
    };
    auto tile_of = [&](int t) __attribute__((always_inline)) {
        const bool is_low = t >= hn;
        const int q = is_low ? l0 + t - hn : h0 + t;
        const int* const table = is_low ? low : high;
        const int tm = q / tiles_n;
        int e = 0;
        for (int e0 = 0; e0 < g.E; e0 += kWave) {
            const uint64_t in = __ballot(e0 + lane < g.E && table[min(e0 + lane, g.E - 1) + 1] > tm);
            if (in) {
                e = e0 + __builtin_ctzll(in);
                break;
            }
        }
        e = __builtin_amdgcn_readfirstlane(e);
        const int b0 = __builtin_amdgcn_readfirstlane(table[e]);
        const int mt = __builtin_amdgcn_readfirstlane(table[e + 1]) - b0;
        const int tl = q - b0 * tiles_n;
        const int span = 8 * tiles_n, grp = tl / span, m0 = grp * 8, gsz = min(mt - m0, 8), in = tl - grp * span;
        const int hi = __builtin_amdgcn_readfirstlane(high[e + 1]) - __builtin_amdgcn_readfirstlane(high[e]);
        Tile r;
        r.e = e;
        r.row = __builtin_amdgcn_readfirstlane(first[e]) + (is_low ? hi : m0 + in % gsz) * kTile;
        r.end = __builtin_amdgcn_readfirstlane(first[e + 1]);
        r.col = in / gsz * (GATE ? 128 : 256);
        return r;
    };

    const uint32_t as_base = (uint32_t)(uintptr_t)As, bs_base = (uint32_t)(uintptr_t)Bs;
    const i32x4 a_rsrc = make_buf_rsrc(g.x, (uint32_t)(((int64_t)(g.x_rows - 1) * g.x_stride + g.K) * 2));
    i32x4 b_rsrc;
    auto swz = [](int row, int chunk) { return chunk ^ (row & 7); };
    // Load j of a wave fills LDS rows (4 j + wave) * 8 + lane / 8 of its operand, chunk lane % 8
    // holding logical chunk (lane % 8) ^ (row % 8): the same for every j.
    const int lch = swz(lane / CH, lane % CH);
    uint32_t voff[2 * LOADS], ldso[2 * LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const uint32_t off = (uint32_t)((j * 4 + wave) * 8 * BK * 2);
        ldso[j] = __builtin_amdgcn_readfirstlane(as_base + off);
        ldso[LOADS + j] = __builtin_amdgcn_readfirstlane(bs_base + off);
    }
    // offset of x's row behind row r of y, for thread r of the workgroup's 256
    auto source = [&](const Tile& c) __attribute__((always_inline)) {
        const int p = c.row + tid;
        const int r = source_row(g, p, c.end);
        return r < 0 ? kTilePastEnd : (uint32_t)((int64_t)r * g.x_stride * 2);
    };
    auto set_tile = [&](const Tile& c) __attribute__((always_inline)) {
        b_rsrc = make_buf_rsrc(static_cast<const uint16_t*>(g.w) + (int64_t)c.e * g.w_stride, (uint32_t)g.N * (uint32_t)g.K * 2u);
        int ln = lane;
        asm volatile("" : "+v"(ln));  // keeps what follows here instead of in registers all along
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int row = (j * 4 + wave) * 8 + ln / CH;
            const uint32_t s = src[row];
            voff[j] = s == kTilePastEnd ? s : s + (uint32_t)lch * 16;
            int n;
            if constexpr (GATE) {
                const int col = c.col + (row >> 7) * 64 + ((row & 127) >> 5) * 16 + (row & 15);
                n = col < F ? col + ((row >> 4) & 1) * F : -1;
            } else {
                n = c.col + row < F ? c.col + row : -1;
            }
            voff[LOADS + j] = n < 0 ? kTilePastEnd : ((uint32_t)n * (uint32_t)g.K + (uint32_t)lch * 8) * 2u;
        }
        // complete before the first load goes out: the compiler's own waits would count the loads
#pragma unroll
        for (int j = 0; j < 2 * LOADS; ++j) asm volatile("" : "+v"(voff[j]));
    };
    const bool lane_in = lch * 8 < g.K - (ktiles - 1) * BK;  // this lane's chunk of the last stage
    auto dma = [&](int j, int kt, int buf) __attribute__((always_inline)) {
        uint32_t off = voff[j];
        if constexpr (TAIL) off = lane_in || kt < ktiles - 1 ? off : kTilePastEnd;
        lds_dma_buf_b128(j < LOADS ? a_rsrc : b_rsrc, off, (uint32_t)(kt * BK * 2), ldso[j] + (uint32_t)buf * STAGE_BYTES);
    };
    auto issue_prologue = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 2 * LOADS; ++j) dma(j, 0, 0);
#pragma unroll
        for (int j = 0; j < 2 * LOADS; ++j) dma(j, min(1, ktiles - 1), 1);
    };

    const uint16_t* a_rd[2];  // of the wave's first 16 rows, but for wm
    const uint16_t* b_rd[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int pc = (h * 4 + lgrp) ^ (lrow & 7);
        a_rd[h] = As + lrow * BK + pc * 8;
        b_rd[h] = Bs + (wn * 128 + lrow) * BK + pc * 8;
    }
    f32x4 acc[8][8];
    u32x4 fa[2][8], fb[2][8];
    uint16_t* const stage = Cs + wave * (SR * 128);
    const __amdgpu_buffer_rsrc_t y_rsrc = __builtin_amdgcn_make_buffer_rsrc(
        g.y, 0, (uint32_t)(((int64_t)(g.P - 1) * g.y_stride + F) * 2), 0x00020000);
    const bool has_bias = g.epi & kEpiBias, relu = g.epi & kEpiRelu;

    Tile cur = tile_of(t);
    src[tid] = source(cur);
    __syncthreads();
    set_tile(cur);
    issue_prologue();
    int pending = 0;  // the stores of the tile before, behind this one's first loads
    bool more = true;

    // One tile, 2 FM fragments of rows high (two waves of FM): as many as it has rows for.
    auto run_tile = [&](auto fm) __attribute__((always_inline)) {
        constexpr int FM = decltype(fm)::value;
        constexpr int GROUPS = 8 * FM;               // of two products to a step
        constexpr int READS = FM + 8;                // fragment reads of half a stage
        constexpr int GA = FM == 8 ? 24 : FM == 4 ? 12 : 5;
        constexpr int DPG = FM == 8 ? 1 : FM == 4 ? 2 : 4;  // loads to a group
        constexpr int RPG = FM == 2 ? 2 : 1;                // reads to a group
        constexpr int GB = GA + 16 / DPG;
        static_assert(READS <= RPG * GA && READS <= RPG * (GROUPS - GB) && GB >= GROUPS / 2, "order of a step");
        if (pending == 8 * STORES) wait_vmem_le<2 * LOADS + 8 * STORES>();
        else if (pending == 4 * STORES) wait_vmem_le<2 * LOADS + 4 * STORES>();
        else if (pending == 2 * STORES) wait_vmem_le<2 * LOADS + 2 * STORES>();
        else wait_vmem_le<2 * LOADS>();
        __syncthreads();
        // the next tile and its rows, on the way while this one is multiplied
        const int tn = t + per;
        more = tn < t_end;
        const Tile next = tile_of(more ? tn : t);
        const int np = min(next.row + tid, next.end - 1);
        const bool nin = next.row + tid < next.end;
        const int nidx = g.rows ? g.rows[np] : 0;
        auto read_a = [&](int h, int f, uint32_t buf) {
            return *reinterpret_cast<const u32x4*>(a_rd[h] + buf + (wm * FM + f) * 16 * BK);
        };
        auto read_b = [&](int h, int f, uint32_t buf) { return *reinterpret_cast<const u32x4*>(b_rd[h] + buf + f * 16 * BK); };
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i < FM) fa[0][i] = read_a(0, i, 0);
            fb[0][i] = read_b(0, i, 0);
        }
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

        // A step: half of its groups on each half of the stage. First the second half is read;
        // by group GA all waves have, and the loads of the stage after next follow; by group GB
        // the next stage has landed, and its first half is read.
        for (int kt = 0; kt < ktiles; ++kt) {
            const uint32_t now = (uint32_t)(kt & 1) * (kTile * BK), nxt = (uint32_t)((kt + 1) & 1) * (kTile * BK);
            const int dkt = min(kt + 2, ktiles - 1);
            auto read = [&](int h, int q, uint32_t buf) {  // read q of a half: A and B in turn
                if (q < 2 * FM) {
                    if ((q & 1) == 0) fa[h][q >> 1] = read_a(h, q >> 1, buf);
                    else fb[h][q >> 1] = read_b(h, q >> 1, buf);
                } else {
                    fb[h][q - FM] = read_b(h, q - FM, buf);
                }
            };
#pragma unroll
            for (int s = 0; s < GROUPS; ++s) {
                if (s == GA) {
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    __syncthreads();
                }
                if (s == GB) {
                    wait_vmem_le<2 * LOADS>();
                    __syncthreads();
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int m = (s % (GROUPS / 2)) * 2 + u, i = m >> 3, j = m & 7;
                    if (s < GROUPS / 2) acc[i][j] = mfma16x16x32(fb[0][j], fa[0][i], acc[i][j], T{});
                    else acc[i][j] = mfma16x16x32(fb[1][j], fa[1][i], acc[i][j], T{});
                }
#pragma unroll
                for (int u = 0; u < RPG; ++u) {
                    const int q = s * RPG + u;
                    if (q < READS) read(1, q, now);
                }
#pragma unroll
                for (int u = 0; u < DPG; ++u) {
                    const int q = (s - GA) * DPG + u;
                    if (q >= 0 && q < 16) dma(q, dkt, kt & 1);
                }
#pragma unroll
                for (int u = 0; u < RPG; ++u) {
                    const int q = (s - GB) * RPG + u;
                    if (q >= 0 && q < READS) read(0, q, nxt);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        wait_vmem_le<0>();
        {
            const int r = g.rows ? (int)((unsigned)max(nidx, 0) / (unsigned)g.fan) : np;
            src[tid] = (nin & (nidx >= 0) & (r < g.x_rows)) ? (uint32_t)((int64_t)r * g.x_stride * 2) : kTilePastEnd;
        }
        __syncthreads();  // the stages are free, the next tile's rows are there

        float4 bv[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            bv[j] = float4{0.f, 0.f, 0.f, 0.f};
            if (has_bias) {
                const float* b = g.bias + (int64_t)cur.e * g.N;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int c = GATE ? cur.col + wn * 64 + (j >> 1) * 16 + 4 * lgrp + q : cur.col + wn * 128 + j * 16 + 4 * lgrp + q;
                    (&bv[j].x)[q] = b[c < F ? (GATE && (j & 1) ? c + F : c) : 0];
                }
            }
        }
        if (more) {
            set_tile(next);
            issue_prologue();
        }
        // 16 rows of a wave at a time through its part of LDS, whole row segments to y
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            if (FM == 8 && i == 4 && more) wait_vmem_le<4 * LOADS>();  // the counter holds 63
#pragma unroll
            for (int j = 0; j < 8; j += GATE ? 2 : 1) {
                float v[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    v[q] = acc[i][j][q] + (&bv[j].x)[q];
                    if constexpr (GATE) v[q] = silu_gate(v[q], acc[i][j + 1][q] + (&bv[j + 1].x)[q]);
                    else if (relu) v[q] = relu_of(v[q]);
                }
                uint2 packed;
                packed.x = (uint32_t)elem<T>::from_f32(v[0]) | ((uint32_t)elem<T>::from_f32(v[1]) << 16);
                packed.y = (uint32_t)elem<T>::from_f32(v[2]) | ((uint32_t)elem<T>::from_f32(v[3]) << 16);
                const int c = (GATE ? j / 2 : j) * 16 + 4 * lgrp;
                *reinterpret_cast<uint2*>(stage + lrow * COLS + (((c >> 3) ^ (lrow & (COLS / 8 - 1))) << 3) + (c & 4)) = packed;
            }
#pragma unroll
            for (int p = 0; p < STORES; ++p) {
                const int r = p * ROWS_PER_STORE + lane / (COLS / 8), ch = lane % (COLS / 8);
                const u32x4 val = *reinterpret_cast<const u32x4*>(stage + r * COLS + ((ch ^ (r & (COLS / 8 - 1))) << 3));
                const int gm = cur.row + (wm * FM + i) * 16 + r, gn = cur.col + wn * COLS + ch * 8;
                const uint32_t off = gm < cur.end && gn < F ? (uint32_t)(((int64_t)gm * g.y_stride + gn) * 2) : kTilePastEnd;
                __builtin_amdgcn_raw_buffer_store_b128(val, y_rsrc, off, 0, 0);
            }
        }
        t = tn;
        cur = next;
        pending = FM * STORES;
    };
    while (more) {
        const int rows = cur.end - cur.row;
        if (rows > 128) run_tile(std::integral_constant<int, 8>{});
        else if (rows > 64) run_tile(std::integral_constant<int, 4>{});
        else run_tile(std::integral_constant<int, 2>{});
    }
    wait_vmem_le<0>();
}

}  // namespace pyc

// What the kernel needs: 16-byte pieces of x, W and y, and byte counts that a descriptor holds.
extern "C" int pyc_hip_grouped_tile_takes(const pyc_grouped* g) {
    const int64_t most = 0xFFFFFFF0ll;
    const int cols = g->epi & pyc::kEpiGate ? g->N / 2 : g->N;
    if (g->x_rows == 0 || (((uintptr_t)g->x | (uintptr_t)g->w | (uintptr_t)g->y) & 15) || g->K % 8 || cols % 8 ||
        (g->x_rows > 1 && g->x_stride % 8) || (g->P > 1 && g->y_stride % 8) || (g->E > 1 && g->w_stride % 8))
        return 0;
    return ((int64_t)(g->x_rows - 1) * g->x_stride + g->K) * 2 <= most && (int64_t)g->N * g->K * 2 <= most &&
           ((int64_t)(g->P - 1) * g->y_stride + cols) * 2 <= most;
}

extern "C" int pyc_hip_grouped_tile_launch(int is_bf16, const pyc_grouped* gp, void* stream) {
    using namespace pyc;
    const Grouped& g = *gp;
    const bool gate = g.epi & kEpiGate, tail = g.K % kTileK != 0;
    const int cols = gate ? g.N / 2 : g.N, per = gate ? 128 : 256;
    const int tiles_n = (cols + per - 1) / per;
    if (expert_tiles_most(g.offsets ? g.E : 1, g.P, kTile) * tiles_n > 0x7FFF0000) return -1;
    const dim3 grid(256), block(256);
    const hipStream_t s = (hipStream_t)stream;
#define PYC_TILE(G, TL)                                                                                       \
    if (gate == G && tail == TL) {                                                                            \
        if (is_bf16) hipLaunchKernelGGL((grouped_tile_kernel<bf16_t, G, TL>), grid, block, 0, s, g, tiles_n); \
        else hipLaunchKernelGGL((grouped_tile_kernel<f16_t, G, TL>), grid, block, 0, s, g, tiles_n);          \
    }
    PYC_TILE(false, false)
    PYC_TILE(false, true)
    PYC_TILE(true, false)
    PYC_TILE(true, true)
#undef PYC_TILE
    return hipGetLastError() == hipSuccess ? 0 : -2;
}
