/* pyc/hip_backend.h — MI355X (gfx950) extensions of the GPU backend ABI.
 *
 * These entry points are additions next to the reference ABI in
 * pyc/cuda_backend.h (reference cuda_backend.h:105-138 defines the
 * single-head/no-bias family they generalise). All pointers are DEVICE
 * pointers, stream is a hipStream_t (NULL = the null stream), nothing is
 * allocated except where a workspace is said to be. Every function returns
 *   0  success (kernels enqueued),
 *  -1  unknown symbol or invalid argument (nothing enqueued),
 *  -2  HIP launch error (hipGetLastError after the launch). */
#ifndef PYC_HIP_BACKEND_H
#define PYC_HIP_BACKEND_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* GEMM epilogue flags: applied to the fp32 accumulator before the store. */
#define PYC_HIP_EPI_NONE 0
#define PYC_HIP_EPI_BIAS 1 /* out[m,n] += bias[n] (fp32 bias) */
#define PYC_HIP_EPI_RELU 2 /* out = max(out, 0) after bias. NaN: 0, but from the products by expert
                            * and with 4-bit weights NaN */
/* Products by expert and with 4-bit weights only, not with RELU: rows 0 .. N/2 - 1 of
 * the weights are gates, the others values, and column c of out (N/2 of them) is
 * silu(gate c) * value c, each with its bias. silu(g) = g / (1 + e^-g), 0 where e^-g leaves
 * fp32 (g below -88.7). */
#define PYC_HIP_EPI_SILU_GATE 4

/* Generalises reference gemm/kernel.cu:151-203 (pyc_cutlass_gemm_dispatch):
 * C[M,N] = epilogue(alpha * A[M,K] * op(B) + beta * C), fp32 accumulate.
 * The symbol fixes the element type and B's layout:
 *   hip_gemm_bf16_nt  bf16  B stored [N,K] (column-major B)
 *   hip_gemm_bf16_nn  bf16  B stored [K,N]
 *   hip_gemm_f16_nt / hip_gemm_f16_nn   fp16, same layouts
 *   hip_gemm_f32_nn / hip_gemm_f32_nt   fp32 (true fp32 MFMA, no TF32)
 * A and C are row-major. Any M,N,K >= 1. */
int pyc_hip_gemm_dispatch(
    const char* symbol,
    int M, int N, int K,
    const void* A, const void* B, void* C,
    float alpha, float beta,
    const float* bias, int epilogue,
    void* stream);

/* Measured autotune of the [M,K]x[K,N] GEMM at a live shape (the reference's
 * compiler_api.c:3000-3044 records one estimated candidate per run instead):
 * every registered variant of `dtype` (PYC_DTYPE_F32/BF16/F16) whose right
 * operand is [K,N] is timed by HIP events on scratch operands of uniform
 * [-1,1) values, after 50 ms of settling load, in three interleaved rounds of
 * `iters` launches; the fastest median becomes the symbol the backend plans
 * for GEMMs of that dtype and shape. Writes up to `cap` symbols (each in a
 * slot of `sym_stride` bytes of `syms`) and their median per-launch ms.
 * Returns the number timed, 0 without a GPU, -1 on bad arguments. */
int pyc_hip_autotune_gemm(
    pyc_dtype dtype, int M, int N, int K, int iters,
    char* syms, size_t sym_stride, double* ms, int cap);

/* Generalises reference attention/kernel.cu:95-122 to batch and heads:
 * O[b,h] = softmax(Q[b,h] K[b,h]^T * scale (+ causal mask)) V[b,h],
 * Q,K,V,O [B,H,S,D] contiguous (BHSD), fp32 softmax and accumulation.
 * Symbol "hip_attention_bf16" (bf16) or "hip_attention_f16". D in {64,128}. */
int pyc_hip_attention_dispatch(
    const char* symbol,
    int B, int H, int S, int D, int causal,
    const void* Q, const void* K, const void* V, void* O,
    float scale, void* stream);

/* Generalises reference conv2d/kernel.cu:80-112 with a fused epilogue:
 * y[n,p,q,k] = relu?(bias[k] + sum_{r,s,c} x[n,p*sh-ph+r,q*sw-pw+s,c] w[k,r,s,c]),
 * x NHWC, w KRSC, y NPQK; out-of-image taps read zero. bias may be NULL.
 * C_in % 8 == 0. The symbol fixes the element type and the kernel path:
 *   hip_conv2d_bf16 / _f16          by shape: whole 256 x 256 tiles on the
 *                                   persistent kernel, a second partial round
 *                                   on 144-pixel tail tiles, or LDS-DMA tiles of
 *                                   32 to 128 pixels, whichever is estimated
 *                                   fastest, else the tiles below
 *   hip_conv2d_bf16_persist / _f16_persist   every tile on the persistent kernel
 *                                   (no tail kernel), else the tiles below
 *   hip_conv2d_bf16_tiled / _f16_tiled       the register-staged implicit-GEMM
 *                                   tiles (256 x 256 when they fill the chip, else 128)
 * All three give the same results up to fp32 summation order. */
int pyc_hip_conv2d_dispatch(
    const char* symbol,
    int N, int H, int W, int C_in,
    int K, int R, int S,
    int pad_h, int pad_w, int stride_h, int stride_w,
    const void* x, const void* w, const float* bias, int relu,
    void* y, void* stream);

/* Weight-only fp8 GEMM for decode (no reference counterpart: the reference
 * has no fp8 type, reference include/pyc/ir.h:16-23):
 * Y[M,N] = relu?( (X[M,K] * dequant(Wq)^T)[m,n] * scale[n] )
 * X bf16 row-major [M,K]; Wq OCP e4m3fn stored [N,K] (each output channel's
 * K weights contiguous); scale fp32 [N]; Y bf16 [M,N]. 1 <= M <= 32, K % 16 == 0.
 * Symbol "hip_gemm_w8a16_e4m3". */
int pyc_hip_w8a16_gemm_dispatch(
    const char* symbol,
    int M, int N, int K,
    const void* X, const void* Wq, const float* scale, int relu,
    void* Y, void* stream);

/* The decode MLP chain in one call (no reference counterpart; see
 * pyc_hip_w8a16_gemm_dispatch): for s = 0..nsteps-1,
 *   X_{s+1} = relu_s?( (X_s * dequant(Wq[s])^T) * scale[s] ),  Y = X_nsteps,
 * X_0 = X bf16 [M, K[0]], Wq[s] e4m3fn [N[s], K[s]], scale[s] fp32 [N[s]],
 * Y bf16 [M, N[nsteps-1]]. 1 <= M <= 32, 1 <= nsteps <= 32, K[s] % 128 == 0,
 * N[s] % 64 == 0, K[s+1] == N[s]. It runs in one persistent launch, or as one launch
 * per layer where that is estimated to be faster (few tokens, small layers).
 * Intermediate activations live in a library-owned device workspace. Returns -1 on
 * bad arguments, and also when the stream is being captured and
 * pyc_hip_w8a16_chain_reserve was not called for this shape first; -2 on a HIP
 * error.
 * Symbol "hip_w8a16_chain_e4m3". */
int pyc_hip_w8a16_chain_dispatch(
    const char* symbol,
    int M, int nsteps,
    const void* X, const void* const* Wq, const float* const* scale,
    const int* N, const int* K, const int* relu,
    void* Y, void* stream);

/* pyc_hip_w8a16_chain_dispatch without any allocation. No counterpart in the
 * reference: for callers that cannot allocate device memory (code under HIP
 * graph capture, tight serving loops, harnesses that forbid hipMalloc). Same
 * arguments, kernels and results; the workspace (counters, intermediate
 * activations, split-K slots) lives in a static device array of
 * PYC_HIP_CHAIN_NOALLOC_SCRATCH_BYTES that each GPU the library runs on holds
 * until the process ends, so no reserve call is needed before capturing it.
 * A call that takes the one-launch chain kernel clears its counters with a small
 * kernel on `stream` first (no memset node); layer launches have none. Calls on one GPU share the array: calls
 * whose executions overlap race. The timeout flag is read by
 * pyc_hip_w8a16_chain_error. Returns 0, -1 on bad arguments, -2 on a HIP
 * error, -3 when the chain's workspace exceeds the scratch size (config 5,
 * 8 x [32x4096 -> 11008 -> 4096], needs 63.6 MiB). */
#define PYC_HIP_CHAIN_NOALLOC_SCRATCH_BYTES (64u << 20)
int pyc_hip_w8a16_chain_dispatch_noalloc(
    const char* symbol,
    int M, int nsteps,
    const void* X, const void* const* Wq, const float* const* scale,
    const int* N, const int* K, const int* relu,
    void* Y, void* stream);

/* Allocates the chain workspace for this shape on the current device; call it
 * outside stream capture before capturing a chain launch. 0, -1 (bad shape),
 * -2 (HIP error). */
int pyc_hip_w8a16_chain_reserve(int M, int nsteps, const int* N, const int* K);

/* 1 if a chain launch on the current device gave up waiting for another
 * workgroup (its output is then invalid), 0 if not, -2 on a HIP error.
 * Synchronizes the device; clear != 0 resets the flag. pyc_run_model reads
 * the flag after every run that launched a chain and turns a set flag into a
 * native failure (reason "hip_chain_wait_timeout"). */
int pyc_hip_w8a16_chain_error(int clear);

/* 1 when pyc_hip_w8a16_chain_dispatch takes a chain of this shape (the
 * preconditions above plus the kernel's unit and split-K slot limits), 0
 * otherwise. Host only; the backend fuses fp8 steps into a chain launch only
 * while this holds. */
int pyc_hip_w8a16_chain_supported(int M, int nsteps, const int* N, const int* K);

/* Sets the current device's chain timeout flag as a wait that ran out would,
 * for tests of the failure handling (no kernel has to time out). 0, or -2 on
 * a HIP error. */
int pyc_hip_w8a16_chain_error_raise(void);

/* GELU, exact erf form: y = 0.5 x (1 + erf(x / sqrt(2))), elementwise over n
 * elements (no reference kernel: the reference reports PYC_IR_OP_GELU as a
 * graph break and executes it nowhere, reference
 * src/compiler/passes/pass_manager.c:313-373). fp32 statistics, one rounding.
 * Symbols "hip_gelu_f32", "hip_gelu_bf16", "hip_gelu_f16". 0, -1 (bad
 * arguments), -2 (HIP error). */
int pyc_hip_gelu_dispatch(const char* symbol, size_t n, const void* x, void* y, void* stream);

/* LayerNorm over the last dimension of a [rows, D] row-major tensor:
 * y = (x - mean) / sqrt(var + eps) * gamma + beta, var the population
 * variance, gamma and beta [D] of x's type or NULL (1 and 0). Same reference
 * status as GELU (PYC_IR_OP_LAYERNORM). Symbols "hip_layernorm_f32",
 * "hip_layernorm_bf16", "hip_layernorm_f16". 0, -1, -2 as above. */
int pyc_hip_layernorm_dispatch(const char* symbol, int rows, int D, float eps, const void* x, const void* gamma,
                               const void* beta, void* y, void* stream);

/* The paged 8-bit key/value cache (no reference counterpart: the reference
 * holds no state between runs). A block holds block_size tokens of every kv head:
 *   k [num_blocks][kv_heads][block_size][head_dim]  e4m3fn codes,
 *   v [num_blocks][kv_heads][head_dim][block_size]  e4m3fn codes (a channel's
 *     tokens run on: the operand of the product over tokens, as it is),
 *   k_scale, v_scale [num_blocks][kv_heads] fp32: an element is code * scale.
 * A block's codes are dense; k_block_stride and v_block_stride are the bytes
 * from a block to the next (at least kv_heads * block_size * head_dim, multiples
 * of 16, below 2^31; k and v on 16-byte boundaries). block_size 16, 32, 64 or 128, head_dim 64
 * or 128, num_blocks * block_size < 2^31. Slot s is token s % block_size of block
 * s / block_size. */
typedef struct {
    void* k;
    void* v;
    float* k_scale;
    float* v_scale;
    int64_t k_block_stride;
    int64_t v_block_stride;
    int num_blocks;
    int kv_heads;
    int block_size;
    int head_dim;
} pyc_hip_kv_cache;

/* The plan of one serving step, made on the device from what B requests hold in
 * the cache (cached[b] tokens, their blocks in table[b][0 ..]) and what they bring
 * (fresh[b] tokens; negative: the request is over). table is [B][width], rows
 * table_stride apart; free_list[0 .. free_count[0]) is a stack of free blocks of
 * room for free_capacity. In order of b:
 *  - a request that is over pushes its ceil(cached / block_size) blocks;
 *  - then fresh[b] > 0 is granted if cached + fresh fits the table row and
 *    needs no new block or the stack holds the new blocks of all that was asked up
 *    to and with b, and if all tokens asked up to and with b are at most `tokens`
 *    (what does not fit its row counts as not asked);
 *  - granted requests pop their new blocks into their table rows.
 * Outputs: lens[b] = cached + granted (0 when over); q_offsets[B + 1], where each
 * request's granted tokens begin; for each token its slot and its position in the
 * request, -1 behind the last one up to `tokens`; free_after[0], the blocks left.
 * A refused request keeps its length and its blocks, and has no tokens in the step.
 * Entries of table and free_list that are not pushed or popped stay as they are.
 * lens may be cached, free_after may be free_count; with neither, the call can be
 * made again. B >= 1, width >= 1, 0 <= tokens < 2^24, block_size as above,
 * width * block_size < 2^31 - 255. Symbol "hip_kv_plan". 0, -1 (bad argument, nothing
 * launched), -2 (HIP error). */
int pyc_hip_kv_plan_dispatch(
    const char* symbol, int B, int width, int64_t table_stride, int block_size, int tokens,
    const int32_t* cached, const int32_t* fresh, int32_t* table,
    int32_t* free_list, int free_capacity, const int32_t* free_count,
    int32_t* lens, int32_t* q_offsets, int32_t* slots, int32_t* positions, int32_t* free_after,
    void* stream);

/* Keys and values of a step into the cache: row t of k and v (kv_heads x
 * head_dim dense, rows k_stride and v_stride elements apart) goes to slot slots[t];
 * a slot outside the cache (-1) is skipped. For a block and head with new rows, a
 * their largest finite magnitude and s_new the smallest power of two with a <= 448
 * s_new, at least 2^-100, its scale becomes
 *   s_new               where the block's first slot is written: the block
 *                       starts anew, what it held counts as gone,
 *   max(old, s_new)     else; codes already there are re-rounded to it (with an
 *                       old scale that is not finite and positive: s_new, and the
 *                       codes stay).
 * code = e4m3(x * (1 / scale)), to nearest even; infinities and NaN become NaN.
 * The rows of one block have to stand together in slots, as the plan lays them
 * out, and no slot may come twice; otherwise which of the rows a block keeps is
 * undefined. k and v on 16-byte boundaries, strides multiples of 8 and at least
 * kv_heads * head_dim. 0 <= tokens < 2^24. Symbols "hip_kv_append_bf16",
 * "hip_kv_append_f16". 0, -1, -2 as above. */
int pyc_hip_kv_append_dispatch(
    const char* symbol, const pyc_hip_kv_cache* cache, int tokens,
    const void* k, int64_t k_stride, const void* v, int64_t v_stride, const int32_t* slots,
    void* stream);

/* Attention of a step's tokens over the cache. Request b has rows q_offsets[b] ..
 * q_offsets[b + 1] - 1 of q and o (q_heads x head_dim dense, rows q_stride and
 * o_stride elements apart) and lens[b] tokens in the blocks table[b][..], the
 * step's own last among them; with n rows, row i sees keys j <= lens[b] - n + i:
 *   o = sum_j softmax_j(scale q.k_j) v_j,  head h reading kv head h / (q_heads / kv_heads).
 * One token each is decoding; more are draft tokens or a prompt chunk; a batch may
 * mix them. fp32 softmax and sums. A row without a key
 * (or with -infinity for every score) is zero; keys of a block id outside the cache
 * count as absent; rows outside every request stay as they are.
 * max_q: no request has more rows (what is past it is left); max_len: the longest
 * of lens if known, else 0 (how the work is split goes by it, results do not but for
 * the order of sums). workspace: pyc_hip_kv_attention_workspace bytes on a 16-byte
 * boundary, zero before its first call and left zeroed where that matters: for one
 * call at a time (calls that may overlap need one each). q_heads a multiple of
 * kv_heads; q, o on 16-byte boundaries, strides multiples of 8, o overlapping
 * nothing. 0 <= tokens < 2^24, tokens * q_heads / kv_heads < 2^31 - 255. Symbols "hip_kv_attention_bf16",
 * "hip_kv_attention_f16". 0, -1, -2 as above. */
int pyc_hip_kv_attention_dispatch(
    const char* symbol, const pyc_hip_kv_cache* cache, int B, int tokens, int q_heads, int max_q, int max_len,
    const void* q, int64_t q_stride, const int32_t* table, int64_t table_stride, int width,
    const int32_t* lens, const int32_t* q_offsets, void* o, int64_t o_stride, float scale,
    void* workspace, size_t workspace_bytes, void* stream);

/* Bytes of workspace that a call of up to B requests and max_q rows each needs
 * (0: bad arguments): never less for more of either. Host only. */
size_t pyc_hip_kv_attention_workspace(int B, int q_heads, int kv_heads, int head_dim, int max_q);

/* Layers of experts (no reference counterpart: the reference's graph ops name no
 * routing and its one matmul has one weight). Rows of tokens that go to the same expert
 * stand together: expert e has rows offsets[e] .. offsets[e + 1] - 1.
 *
 * Routing. For each row of logits [tokens][experts] (rows logits_stride apart): the k
 * largest, in descending order, ties to the lower expert: ids [tokens][k], and weights
 * [tokens][k] fp32 = softmax over all experts, with normalize over the chosen ones. -infinity and
 * NaN are never chosen and weigh nothing; a choice that there is none for has id -1 and
 * weight 0 (padding: a row of -infinity). +infinity: all weight, in equal parts, on those that have it.
 * With flat index f = t * k + j of choice j of token t:
 *   offsets [experts + 1]  where each expert's rows begin, and how many there are,
 *   rows [tokens * k]      the flat indexes by expert, ascending in each; -1 behind the last,
 *   places [tokens * k]    where f stands in rows, -1 without an expert.
 * 1 <= experts <= 1024, 1 <= k <= min(experts, 64), 0 <= tokens <= 2^22; above about 2^17 tokens the time
 * grows with their square (2^20 by 128 experts: 5.4 ms). workspace:
 * pyc_hip_moe_route_workspace bytes on a 4-byte boundary, of any content, for one call at a time
 * (calls that may overlap need one each); up to 64 tokens it may be NULL.
 * Symbols "hip_moe_route_f32", "hip_moe_route_bf16", "hip_moe_route_f16". 0, -1 (bad
 * argument, nothing launched), -2 (HIP error). */
int pyc_hip_moe_route_dispatch(
    const char* symbol, int tokens, int experts, int k, int normalize, const void* logits, int64_t logits_stride,
    int32_t* ids, float* weights, int32_t* offsets, int32_t* rows, int32_t* places,
    void* workspace, size_t workspace_bytes, void* stream);

/* Bytes of workspace of a routing (0: bad arguments): never less for more tokens. Host only. */
size_t pyc_hip_moe_route_workspace(int tokens, int experts, int k);

/* out[t] = base[t] + sum_j weights[t][j] y[places[t][j]]: a token's experts' rows back onto it.
 * y [rows][width], out and base [tokens][width] of the symbol's type (rows their strides
 * apart, base NULL: 0), weights fp32 and places [tokens][k]. fp32 sums, base first, then j
 * in order, one rounding. A place outside y (-1) counts as absent. out may be base; else it
 * overlaps nothing. Any width and alignment; 16-byte rows are fastest. 1 <= k <= 64, tokens * width below 2^32.
 * Symbols "hip_moe_combine_bf16", "hip_moe_combine_f16". 0, -1, -2 as above. */
int pyc_hip_moe_combine_dispatch(
    const char* symbol, int rows, int tokens, int k, int width, const void* y, int64_t y_stride,
    const float* weights, const int32_t* places, const void* base, int64_t base_stride,
    void* out, int64_t out_stride, void* stream);

/* Products grouped by expert, of ragged sizes that the device knows:
 *   y[p] = epi(x[src[p] / fan] w[e]^T + bias[e])   for offsets[e] <= p < offsets[e + 1],
 * fp32 sums, one rounding. x [x_rows][K] (rows x_stride apart), w [experts][N][K] (experts w_stride
 * elements apart, each dense), bias fp32 [experts][N] with PYC_HIP_EPI_BIAS; y [rows][N], with
 * PYC_HIP_EPI_SILU_GATE [rows][N / 2] (rows y_stride apart). src NULL: row p of x; with the
 * routing's rows and fan = k, a token's row goes to each of its experts. An index outside x reads a row of zeros.
 * offsets are held to 0 .. rows and to never decrease; rows of y before the first and
 * behind the last expert's stay as they are. Experts without rows are not read. y overlaps nothing.
 * Any N, K, strides and 2-byte alignment; K, strides and bases in whole 16 bytes are fastest.
 * 1 <= experts <= 1024, rows and x_rows up to 2^28, N and K up to 2^24.
 * Symbols "hip_grouped_gemm_bf16", "hip_grouped_gemm_f16". 0, -1, -2 as above. */
int pyc_hip_grouped_gemm_dispatch(
    const char* symbol, int experts, int rows, int N, int K, const void* x, int64_t x_stride, int x_rows,
    const int32_t* src, int fan, const int32_t* offsets, const void* w, int64_t w_stride,
    const float* bias, int epilogue, void* y, int64_t y_stride, void* stream);

/* Products with 4-bit weights: w[n][k] = (code - zero) * scale, with a scale of x's type and
 * a zero point for each `group` (32, 64 or 128) k of a row:
 *   codes [N][K / 2]  the even k in the low half of a byte, 0 .. 15,
 *   scale [N][K / group], zeros [N][K / group] bytes, or NULL: 8.
 *   y[M][N] = epi(x[M][K] w^T + bias), epilogues as above (bias fp32 [N]).
 * Whole numbers times x are summed as they are, the scale comes in fp32: weights are
 * never rounded. x finite, the sums of |x| and |scale x| along K below 2^122 (those of x (16 + code) and of
 * x (16 + zero) are taken apart). Any M and N, K a multiple of group; x and codes on 16-byte boundaries, x_stride a multiple of 8. Symbols "hip_gemm_w4a16_bf16", "hip_gemm_w4a16_f16". 0, -1, -2 as above. */
int pyc_hip_w4a16_gemm_dispatch(
    const char* symbol, int M, int N, int K, int group, const void* x, int64_t x_stride,
    const void* codes, const void* scale, const uint8_t* zeros, const float* bias, int epilogue,
    void* y, int64_t y_stride, void* stream);

/* The same by expert: codes [experts][N][K / 2] (experts codes_stride bytes apart, a multiple of 16),
 * scale and zeros [experts][N][K / group] dense, bias [experts][N]; the rest as in
 * pyc_hip_grouped_gemm_dispatch. Symbols "hip_grouped_gemm_w4a16_bf16", "hip_grouped_gemm_w4a16_f16". */
int pyc_hip_w4a16_grouped_gemm_dispatch(
    const char* symbol, int experts, int rows, int N, int K, int group, const void* x, int64_t x_stride, int x_rows,
    const int32_t* src, int fan, const int32_t* offsets, const void* codes, int64_t codes_stride,
    const void* scale, const uint8_t* zeros, const float* bias, int epilogue,
    void* y, int64_t y_stride, void* stream);

/* Device properties the bench and the registry report. */
typedef struct {
    char gcn_arch[64];       /* e.g. "gfx950:sramecc+:xnack-" */
    int compute_units;
    int clock_khz;           /* peak shader clock */
    int memory_clock_khz;
    int memory_bus_width;
    size_t total_global_mem;
    size_t lds_per_block;
    int xcds;                /* best-effort; 8 on MI355X */
} pyc_hip_device_info;

/* Returns 0 and fills info for the current device, -1 when no HIP device. */
int pyc_hip_device_query(pyc_hip_device_info* info);

/* Measured choice between the conv2d paths above at a live shape: every
 * registered conv2d variant of `dtype` (PYC_DTYPE_BF16/F16) is timed as in
 * pyc_hip_autotune_gemm (scratch operands of uniform [0,1) activations and
 * [-1,1) weights, bias and ReLU on, settle, three interleaved rounds of
 * `iters` launches); the fastest median becomes the symbol the backend plans
 * for conv2d steps of that dtype and geometry. Outputs and return value as
 * pyc_hip_autotune_gemm. */
int pyc_hip_autotune_conv2d(
    pyc_dtype dtype, int N, int H, int W, int C_in, int K, int R, int S,
    int pad_h, int pad_w, int stride_h, int stride_w, int iters,
    char* syms, size_t sym_stride, double* ms, int cap);

/* Resources of the kernel a registered symbol launches (at the large shapes
 * its registry entry describes; shape-chosen symbols may launch another kernel
 * for small shapes). The products by expert and with 4-bit weights are described by their
 * forms of 64 rows and columns; calls of many rows launch tiles of 256 x 256 or 128 x 256, which
 * take nearly all LDS of a CU and one or two waves a SIMD. The registry's shared_mem_bytes and
 * estimated_occupancy (waves_per_simd / 8) are the compiled-in figures;
 * with a HIP device present the attr_* fields are read from the loaded code
 * object (hipFuncGetAttributes, hipOccupancyMaxActiveBlocksPerMultiprocessor)
 * and device is 1. Returns 0, or -1 for an unknown symbol. */
typedef struct {
    char kernel[64];           /* kernel (template instance) name */
    size_t lds_bytes;          /* LDS per workgroup, as registered */
    int threads;               /* workgroup size */
    int waves_per_simd;        /* resident waves per SIMD, as registered */
    int device;                /* 1 when the attr_ fields are filled */
    size_t attr_lds_bytes;     /* sharedSizeBytes (all LDS here is static) */
    int attr_regs;             /* numRegs */
    size_t attr_scratch_bytes; /* localSizeBytes: spill per lane */
    int attr_max_threads;      /* maxThreadsPerBlock (launch bounds) */
    int attr_blocks_per_cu;    /* resident workgroups per CU at `threads` */
} pyc_hip_kernel_resources;
int pyc_hip_kernel_resources_query(const char* symbol, pyc_hip_kernel_resources* out);

/* Number of kernel symbols compiled into this library for op_key
 * ("matmul", "attention", "conv2d", "matmul_w8a16", "matmul_w8a16_chain",
 * "gelu", "layernorm", "kv_plan", "kv_append", "kv_attention", "moe_route",
 * "moe_combine", "grouped_gemm", "matmul_w4a16", "grouped_w4a16"), independent of the
 * registry's state. */
int pyc_hip_kernel_symbol_count(const char* op_key);

#ifdef __cplusplus
}
#endif

#endif
