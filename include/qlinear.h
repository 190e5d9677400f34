/*
 * qlinear.h — C ABI of libqlinear.so: GPTQ int4 quantized linears on MI355X (gfx950).
 *
 * Drop-in for the quantized-linear hot path of intplusplus/webllm. Plain pointers, sizes and
 * byte offsets only; every function returns an int status (QL_OK = 0, negative = error class)
 * and ql_last_error() holds the message of the calling thread's last failure. No exceptions
 * cross the ABI. Weights stay GPTQ-packed in device memory; dequantization is fused into the
 * kernels.
 *
 * Reference interfaces each entry point replaces (paths relative to the reference checkout):
 *   ql_create / ql_destroy        src/gpu/device.ts:40-98 initGpu (one device, one queue)
 *   ql_arena_*                    src/gpu/buffer.ts:20-34 createStorageBuffer, :103-120 writeF16 /
 *                                 device.queue.writeBuffer, :123-170 readback; src/gpu/arena.ts:17-59
 *   ql_gptq_desc / ql_gptq_check  src/weights/quant.ts:16-30 GptqInt4Params, :44-79 validation
 *   ql_unpack_f16                 src/weights/qwen-loader.ts:55-67 dequantGptqLinear +
 *                                 src/model/qwen.ts:262-266 uploadF16 (CPU dequant + f16 encode)
 *   ql_unpack_f32, ql_unpack_f32_ex  src/weights/quant.ts:42-118 dequantizeGptqInt4
 *   ql_plan_linear                src/model/qwen.ts:61-74 planGemvSplit + the branch in :568-618
 *   ql_linear                     src/model/qwen.ts:568-618 QwenGpt.gemm (GEMV / split-K / GEMM)
 *   ql_linear_batch               src/model/qwen.ts:411-413, :464-465 (q/k/v and gate/up issued
 *                                 back to back on one input inside one CommandBatch pass)
 *   ql_sync, ql_timer_*           src/gpu/buffer.ts:123-145 mapAsync readback,
 *                                 src/gpu/pipeline.ts:119-161 timestamp-query profiling
 *   ql_graph_*                    src/gpu/pipeline.ts:55-117 CommandBatch (one submit per forward)
 *   ql_plan_seq, ql_seq_*         src/gpu/pipeline.ts:71-116 CommandBatch.dispatch/endPass/submit
 *                                 with src/model/qwen.ts:556-559 passBreak, as runForward uses
 *                                 them (qwen.ts:382-387, :411-473): a forward's linears recorded
 *                                 once, then submitted as one unit per step
 *   ql_seq_fuse, ql_plan_seq_fused, ql_seq_create_fused
 *                                 the same, with the layer's elementwise dispatches around the
 *                                 linears folded in: rmsnorm before q/k/v and gate/up
 *                                 (qwen.ts:403-405, :458-460, src/gpu/kernels/norm/rmsnorm.wgsl),
 *                                 the residual vec_add after o and down (qwen.ts:453-455,
 *                                 :476-478, src/gpu/kernels/misc/vec_add.wgsl) and silu_mul
 *                                 before down (qwen.ts:468-470,
 *                                 src/gpu/kernels/activation/silu_mul.wgsl)
 */
#ifndef QLINEAR_H
#define QLINEAR_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes. -1..-7 are the failure classes of quant.ts:46-79, in its check order. */
#define QL_OK 0
#define QL_E_BITS (-1)          /* bits != 4                                    quant.ts:46 */
#define QL_E_GROUP (-2)         /* group <= 0                                   quant.ts:47 */
#define QL_E_DIMS (-3)          /* K <= 0 or N <= 0                             quant.ts:48 */
#define QL_E_QWEIGHT_SHORT (-4) /* qweight [ceil(K/8), N] int32 outside arena   quant.ts:58 */
#define QL_E_SCALES_SHORT (-5)  /* scales [ceil(K/group), N] outside arena      quant.ts:62 */
#define QL_E_QZEROS_SHORT (-6)  /* qzeros [ceil(K/group), ceil(N/8)] outside    quant.ts:69 */
#define QL_E_GROUP_PACK (-7)    /* group % 8 != 0                               quant.ts:76 */
#define QL_E_INVALID (-10)      /* null handle/pointer, bad M, bad dtype                     */
#define QL_E_RANGE (-11)        /* activation/output/scratch range outside its arena         */
#define QL_E_ALIGN (-12)        /* misaligned offset (int32/f32: 4 B, f16: 2 B)              */
#define QL_E_HIP (-13)          /* HIP runtime failure (message in ql_last_error)            */
#define QL_E_STATE (-14)        /* call not valid in the current state (graph capture)       */

/* Sentinel for optional offsets (no qzeros -> symmetric zero 8, quant.ts:73-74; no bias). */
#define QL_NONE UINT64_MAX

#define QL_DTYPE_F32 0
#define QL_DTYPE_F16 1
#define QL_DTYPE_F8 2 /* e4m3 values (largest 448) under powers of two: paged caches only */

/* kernel families returned by ql_plan_linear */
#define QL_KIND_GEMV_MFMA 1   /* M <= 16: packed-int4 GEMV on MFMA, hi/lo split activations */
#define QL_KIND_GEMV_SIMPLE 2 /* any shape: one lane per output column, fp32                */
#define QL_KIND_GEMM_MFMA 3   /* M > 16: LDS-dequant f16 tiles, MFMA f16, fp32 accumulate   */
#define QL_KIND_GEMM_SIMPLE 4 /* any shape: f16 operands, fp32 accumulate, no MFMA          */

typedef struct ql_ctx ql_ctx;
typedef struct ql_arena ql_arena;
typedef struct ql_graph ql_graph;

/* GPTQ int4 linear inside a weight arena (byte offsets). Mirrors GptqInt4Params
 * (quant.ts:16-30) except that scales stay raw fp16 as stored in the checkpoint.
 *   qweight int32 [ceil(K/8), N]   8 nibbles per word, low nibble = smallest input index
 *   qzeros  int32 [ceil(K/group), ceil(N/8)] stored zero - 1, or QL_NONE (zero = 8)
 *   scales  fp16  [ceil(K/group), N]
 *   bias    fp32  [N] or QL_NONE
 * W[n,k] = (q[k,n] - (qz[g,n] + 1)) * s[g,n], g = k / group. */
typedef struct ql_gptq_desc {
    uint64_t qweight_off;
    uint64_t qzeros_off;
    uint64_t scales_off;
    uint64_t bias_off;
    int32_t K;     /* in_features  */
    int32_t N;     /* out_features */
    int32_t group; /* group size (128 for Qwen2.5 GPTQ) */
    int32_t bits;  /* must be 4 */
} ql_gptq_desc;

typedef struct ql_plan {
    int32_t kind;          /* QL_KIND_* */
    int32_t split;         /* K segments; partial sums reduced in fixed ascending order */
    int32_t waves;         /* waves per workgroup splitting each segment */
    int32_t grid_x;        /* workgroups along N */
    int32_t grid_y;        /* workgroups along K (split) or M (GEMM) */
    int32_t block;         /* threads per workgroup */
    uint64_t scratch_bytes;/* bytes the caller must provide at scratch_off (0 if none) */
    int32_t ref_split;     /* planGemvSplit(ceil(N/256), K) of the reference, for comparison */
    int32_t reserved;
} ql_plan;

/* ---- context: one device, one HIP stream (default priority). */
int ql_create(int device, ql_ctx** out);
int ql_destroy(ql_ctx* ctx);
const char* ql_last_error(void);
int ql_device_info(ql_ctx* ctx, char* name, int name_len, int* cu_count, uint64_t* hbm_bytes);

/* ---- arenas: one device allocation addressed by byte offset (256-B aligned base). */
int ql_arena_reserve(ql_ctx* ctx, uint64_t bytes, ql_arena** out);
int ql_arena_release(ql_arena* arena);
uint64_t ql_arena_size(const ql_arena* arena);
/* device address of arena byte 0, for interop (e.g. wrapping as a framework tensor) */
uint64_t ql_arena_device_ptr(const ql_arena* arena);
/* synchronous host<->device copies; the host pointer is borrowed for the call only */
int ql_arena_write(ql_arena* arena, uint64_t off, const void* src, uint64_t bytes);
int ql_arena_read(ql_arena* arena, uint64_t off, void* dst, uint64_t bytes);
/* device-side copy between arenas, enqueued on the context stream */
int ql_arena_copy(ql_ctx* ctx, ql_arena* dst, uint64_t dst_off, const ql_arena* src,
                  uint64_t src_off, uint64_t bytes);

/* ---- GPTQ descriptors (host only, no GPU work). */
/* sizes in bytes of the three packed tensors of a K x N linear */
int ql_gptq_sizes(int32_t K, int32_t N, int32_t group, uint64_t* qweight_bytes,
                  uint64_t* qzeros_bytes, uint64_t* scales_bytes);
/* validates like quant.ts:44-79 (same classes, same order) against a weight arena of
 * arena_bytes bytes, then the bias range (QL_E_RANGE) and alignment (QL_E_ALIGN). Host only. */
int ql_gptq_validate(const ql_gptq_desc* desc, uint64_t arena_bytes);
/* ql_gptq_validate against the arena's size */
int ql_gptq_check(const ql_gptq_desc* desc, const ql_arena* weights);

/* ---- load time: fp16 [N,K] row-major, bit-identical to
 * f32ToF16Bits(dequantizeGptqInt4(...)) (quant.ts:42-118, buffer.ts:57-100). */
int ql_unpack_f16(ql_ctx* ctx, const ql_gptq_desc* desc, const ql_arena* weights,
                  ql_arena* out, uint64_t out_off);
/* many tensors at once (the loader's whole weight set, qwen-loader.ts:146-162 calling
 * dequantGptqLinear + uploadF16 per linear): tensor i into out_offs[i], same bits as
 * ql_unpack_f16. Tensors are batched into few launches (up to 84 tensors each); every descriptor
 * and output range is validated before anything is enqueued. */
int ql_unpack_f16_batch(ql_ctx* ctx, int32_t count, const ql_gptq_desc* descs,
                        const ql_arena* weights, ql_arena* out, const uint64_t* out_offs);
/* fp32 [N,K] row-major, bit-identical to dequantizeGptqInt4(...) itself (quant.ts:42-118) with
 * the scales decoded from fp16 as the loader does (safetensors.ts:180-182, qwen-loader.ts:65).
 * out_off must be 16-byte aligned. */
int ql_unpack_f32(ql_ctx* ctx, const ql_gptq_desc* desc, const ql_arena* weights,
                  ql_arena* out, uint64_t out_off);
/* ql_unpack_f32 with the scales' dtype stated: QL_DTYPE_F16 (as stored in the checkpoint; the same
 * as ql_unpack_f32) or QL_DTYPE_F32, where desc->scales_off holds f32 scales [ceil(K/group), N]
 * (4-byte aligned) — GptqInt4Params.scales as the reference takes it, any Float32Array
 * (quant.ts:22-23, :62 sizes it in values). Each weight is (q - zero) * scale rounded once to f32,
 * bit-identical to dequantizeGptqInt4 for every f32 scale (quant.ts:111-112). */
int ql_unpack_f32_ex(ql_ctx* ctx, const ql_gptq_desc* desc, const ql_arena* weights, int32_t scales_dtype,
                     ql_arena* out, uint64_t out_off);

/* ---- dispatch plan (host only, deterministic, pure): the kernel family, and the shape and scratch of its split-K
 * form. scratch_bytes is what the caller has to provide (and what ql_linear_noalloc checks), an upper bound of what
 * runs: where offsets are aligned, a call may take a kernel of the same family that splits nothing and leaves the
 * scratch alone, which the plan does not tell because it depends on the offsets and the batch too:
 *   M = 3..16, groups of 128, K up to a length that grows with M: products over an image of x (two launches; at 3 and
 *     4 rows for K from 2304 and 2048 on and few columns);
 *   M > 16, groups a multiple of 128, up to about a thousand tiles of 64 columns x 32 rows (fewer where K is long):
 *     the same over an fp16 image;
 *   M > 16, enough tiles of 128 x 256: the prefill launch.
 * ql_plan_batch likewise. */
int ql_plan_linear(int32_t M, int32_t N, int32_t K, int32_t group, ql_plan* out);

/* ---- y[M,N] (fp32) = x[M,K] * W^T (+ bias), enqueued on the context stream.
 * x_dtype: QL_DTYPE_F32 (decode path) or QL_DTYPE_F16. Offsets are into `act`.
 * M <= 16: weights (q - zero) exact, fp16 scales, fp32 sums; x to 2^-30 of its group's largest value, or as two fp16
 * parts of about 22 bits each (products over an image); fp16 weights and x rounded to fp16 above, as the reference.
 * scratch_off: plan.scratch_bytes bytes in `act` for split-K partial sums (ignored when 0).
 * Images of x (M = 3..16 and prompts of some tens of rows, see ql_plan_linear) go through the context's 64 MiB
 * workspace: calls on one context run in its stream's order.
 * The caller orders work by issuing it on this one stream (stream order replaces the
 * reference's passBreak, qwen.ts:556-559). */
int ql_linear(ql_ctx* ctx, const ql_gptq_desc* desc, const ql_arena* weights, ql_arena* act,
              uint64_t x_off, int32_t x_dtype, int32_t M, uint64_t y_off, uint64_t scratch_off);

/* ql_linear with no scratch argument and no allocation. No counterpart in the reference: it is
 * for callers that cannot allocate or carve out a workspace (code under HIP graph capture, tight
 * serving loops, harnesses that forbid hipMalloc). Same kernels, plan and results as ql_linear.
 * Split-K partial sums go to a static device array of QL_NOALLOC_SCRATCH_BYTES per GPU, resolved
 * at ql_create; a plan needing more scratch (ql_plan_linear's scratch_bytes: at most 6.94 MiB for
 * the Qwen2.5-0.5B and -7B decode shapes at M <= 16) fails with QL_E_RANGE before anything is
 * enqueued. Nothing in the array must
 * start at zero (every partial is written before it is read; the arrival counters are the
 * context's and every launch leaves them at zero). Every call on a GPU shares its array and it
 * keeps the last call's contents: calls that overlap on one GPU (several streams, contexts or
 * threads) race. */
#define QL_NOALLOC_SCRATCH_BYTES (8u << 20)
int ql_linear_noalloc(ql_ctx* ctx, const ql_gptq_desc* desc, const ql_arena* weights, ql_arena* act,
                      uint64_t x_off, int32_t x_dtype, int32_t M, uint64_t y_off);

/* y[M,N] (fp32) = x[M,K] (fp32) . W^T (+ bias) for an fp16 weight W [N,K] row-major at w_off in
 * `weights` (bias f32 [N] at bias_off or QL_NONE): the tied lm_head / embedding product,
 * QwenGpt.gemm(lnf, 'embed', logits, null, M, V, C) (qwen.ts:488-489) on gemm_gemv_f16.wgsl's
 * arithmetic (fp32 x, fp16 weights, fp32 accumulation). M = 1..65535: up to 16 rows one pass over
 * the weights; more rows run as a tiled product that reads them once for up to about 1000 rows (K = 896), with
 * an image of x in the context's 4 MiB workspace (calls on one context run in its stream's order). x is fp32 at
 * M = 1, two scaled fp16 parts of about 22 bits above.
 * x, y, w offsets 16-byte aligned, K % 8 == 0. */
int ql_gemv_f16w(ql_ctx* ctx, const ql_arena* weights, uint64_t w_off, uint64_t bias_off,
                 ql_arena* act, uint64_t x_off, int32_t M, int32_t N, int32_t K, uint64_t y_off);

/* ---- decode attention over the KV cache (qwen.ts:424-442).
 * Cache: per layer one fp32 K and one fp32 V region of [max_t, n_kv_head * D], row t holding the
 * vectors of position t (the reference's kCache[i] / vCache[i], qwen.ts:200-205).
 *
 * ql_kv_store: cache[(pos0 + r) * row_len + c] = src[r * row_len + c] for r < rows
 *   (misc/kv_store.wgsl); pos0 + rows > max_t fails with QL_E_RANGE (qwen.ts:352-355 throws).
 *   row_len % 4 == 0, offsets 16-byte aligned. */
int ql_kv_store(ql_ctx* ctx, const ql_arena* act, uint64_t src_off, ql_arena* cache, uint64_t cache_off,
                int32_t max_t, int32_t rows, int32_t row_len, int32_t pos0);

/* ql_attention_decode: out[m, h, :] = softmax_s(q[m, h] . K[s, h / (H / KV)] / sqrt(D)) V[s, ...]
 *   over s = 0 .. past_len + m (causal; attention/attention_gqa_cache.wgsl, CPU form
 *   reference/qwen-ref.ts:65-111 attentionGqaRef). q and out are [M, n_head, D] fp32 in `act`;
 *   D = 4..256 (multiple of 4); past_len + M <= max_t and <= 8192. fp32 inputs, sums and results.
 *   Few rows x heads (decode) split the keys over workgroups, with partials in a 4 MiB workspace the context owns:
 *   calls on one context run in its stream's order, so they never share it at the same time. Many rows
 *   (prefill: M >= 96, D 64 or 128, past_len + M / 2 at least 896 times the nsplit of ql_plan_attention) run as tiles
 *   of 128 (row, head) pairs on the matrix cores, with a 64 MiB workspace of the context's: q, K, V and the
 *   probabilities enter as two fp16 parts each (about 22 bits, no less exact than the other form's sums), in fp32
 *   where their values lie too far apart for that. */
int ql_attention_decode(ql_ctx* ctx, ql_arena* act, uint64_t q_off, const ql_arena* cache, uint64_t k_off,
                        uint64_t v_off, int32_t max_t, int32_t M, int32_t n_head, int32_t n_kv_head, int32_t D,
                        int32_t past_len, uint64_t out_off);
/* ql_plan_attention (diagnostic, host only): the launch shape ql_attention_decode's row-per-workgroup
 *   kernel has for these dimensions, with the same checks (no counterpart in the reference, whose attention is one
 *   dispatch per layer, qwen.ts:430-442). heads_per_run query heads share each K/V row read;
 *   nsplit key splits (1 = no merge launch); workgroups of the attention launch. */
typedef struct ql_attn_info {
    int32_t heads_per_run;
    int32_t nsplit;
    int32_t workgroups;
    int32_t keys_per_split;
} ql_attn_info;
int ql_plan_attention(int32_t max_t, int32_t M, int32_t n_head, int32_t n_kv_head, int32_t D, int32_t past_len,
                      ql_attn_info* info);

/* ql_embed_f16: out[r, :] = f32(embed[tokens[r], :]) for r < rows: the embedding lookup that
 *   starts a forward (embedding_f16.wgsl, dispatched at qwen.ts:392), over the fp16 [vocab, D]
 *   table at embed_off in `weights` (the tied table ql_gemv_f16w reads as lm_head), with uint32
 *   token ids [rows] at tokens_off and the fp32 [rows, D] output at out_off in `act`. Exact
 *   (binary16 -> binary32, as f16BitsToF32, safetensors.ts:144-152). A token id >= vocab writes a
 *   row of zeros (the WGSL reads past the table there; WebGPU's robust access makes that read
 *   implementation-defined). rows 1..65535; embed 2-byte, tokens and out 4-byte aligned (D % 8 == 0
 *   with 16-byte embed/out offsets takes the 16-byte path). */
int ql_embed_f16(ql_ctx* ctx, const ql_arena* weights, uint64_t embed_off, int32_t vocab, int32_t D,
                 ql_arena* act, uint64_t tokens_off, int32_t rows, uint64_t out_off);

/* ---- the elementwise work around the linears (qwen.ts:401-405, :447-478).
 * ql_add_rmsnorm: s = x + d (misc/vec_add.wgsl: the residual add after o_proj / down_proj), stored
 *   at sum_off unless QL_NONE, then y = s * rstd * w, rstd = 1 / sqrt(mean(s^2) + eps)
 *   (norm/rmsnorm.wgsl; CPU form reference/qwen-ref.ts:12-28). d_off = QL_NONE: plain RMSNorm of x.
 *   One launch where the reference runs two; fp32; x, d, sum, y [M, C] in `act`, w [C] in
 *   `weights`; offsets 4-byte aligned (16-byte and C % 4 == 0 take the vector path). The sum may
 *   be stored in place over x or d (sum_off == x_off or d_off); any other overlap of the sum with
 *   x or d, or of y with anything, fails with QL_E_INVALID. */
int ql_add_rmsnorm(ql_ctx* ctx, ql_arena* act, uint64_t x_off, uint64_t d_off, const ql_arena* weights,
                   uint64_t w_off, float eps, int32_t M, int32_t C, uint64_t sum_off, uint64_t y_off);
/* ql_silu_mul: y[i] = (g / (1 + exp(-g))) * up[i], g = gate[i] (activation/silu_mul.wgsl;
 *   siluMulRef, qwen-ref.ts:114-121); offsets 16-byte aligned. */
int ql_silu_mul(ql_ctx* ctx, ql_arena* act, uint64_t gate_off, uint64_t up_off, int64_t n, uint64_t y_off);

/* ---- speculative decoding: a pass over M drafted tokens (a tree) after past_len cached positions.
 * Row m of a pass lies in the cache at slot past_len + m, whatever its depth in the tree; its position, which turns it, is
 * past_len + depth. The order of a step: linears, ql_qk_norm_rope, ql_attention_tree, linears, lm_head, ql_token_logprobs;
 * then the host accepts a path and ql_kv_move brings its rows together. Caches are as ql_kv_store's, fp32 or fp16. */

/* Heads, rotation and cache type of ql_qk_norm_rope (the model's, made once). */
typedef struct ql_rope_desc {
    uint64_t q_norm_off;   /* fp32 [D] RMSNorm weight of every query head in `weights`, or QL_NONE */
    uint64_t k_norm_off;   /* of every key head, or QL_NONE */
    uint64_t table_off;    /* fp32 [max_pos, rot_dim] in `weights`: a position's rot_dim/2 cosines, then its sines */
    int32_t max_pos;
    int32_t n_head, n_kv_head, D;   /* D: 8..256, a multiple of 8 */
    int32_t rot_dim;       /* values of a head that turn, from its first: 8..D, a multiple of 8 */
    int32_t interleaved;   /* 0: pairs (i, i + rot_dim/2), as ropeHalfRef; 1: pairs (2i, 2i + 1) */
    int32_t q_stride, k_stride, v_stride;   /* values from a row to the next, a multiple of 4; 0: heads * D */
    int32_t cache_dtype;   /* QL_DTYPE_F32 or QL_DTYPE_F16 */
    float norm_eps;
    int32_t reserved;      /* 0 */
} ql_rope_desc;
/* fills a table: cos and sin of p * theta^(-2i / rot_dim), the angle in fp64, rounded once (ropeHalfRef,
 * reference/qwen-ref.ts). A program with other frequencies writes its own with ql_arena_write. table_off 16-byte aligned. */
int ql_rope_table(ql_ctx* ctx, ql_arena* weights, uint64_t table_off, int32_t max_pos, int32_t rot_dim, double theta);
/* q and k RMSNormed per head (where the descriptor has weights) and turned by pos[m], q to q_out [M, n_head, D], k and v
 * to rows slot0 + m of the caches [max_t, n_kv_head * D] (fp16: rounded once). pos is int32 [M] in `act`. A row whose position
 * is not in 0..max_pos-1 is padding: its q_out row and its cache rows stay as they were. q_out may be q itself (same
 * offset, dense rows); any other overlap of what is written with what is read fails with QL_E_INVALID. M = 1..65535,
 * M * (n_head + 2 n_kv_head) <= 2^26; slot0 + M > max_t fails with QL_E_RANGE. Offsets 16-byte aligned (pos: 4). */
int ql_qk_norm_rope(ql_ctx* ctx, const ql_rope_desc* desc, const ql_arena* weights, ql_arena* act, uint64_t q_off, uint64_t k_off,
                    uint64_t v_off, uint64_t pos_off, int32_t M, uint64_t q_out_off, ql_arena* cache, uint64_t k_cache_off,
                    uint64_t v_cache_off, int32_t max_t, int32_t slot0);
/* Host only: masks [M, ceil(M/64)] (bit j % 64 of word j / 64 of row m: token j is m or one that m continues) and depths [M]
 * (0: continues the context) of a tree. parents[m] is -1 or an earlier row (< m); anything else fails with QL_E_INVALID.
 * masks or depths may be null. M = 1..256. */
int ql_tree_masks(int32_t M, const int32_t* parents, uint64_t* masks, int32_t* depths);
/* out[m, h, :] = softmax_s(q[m, h] . K[s, h / (n_head / n_kv_head)] / sqrt(D)) V[s, ...] over s < past_len and the drafted rows
 * s = past_len + j whose bit j is set in row m of mask (uint64 [M, ceil(M/64)] at mask_off in `act`; bits from M on are ignored;
 * QL_NONE: j <= m, causal rows). A row that sees nothing, or no score above -inf, is zero. What a row does not see adds nothing to it,
 * infinities and NaN included. M = 1..256, D = 8..256 (a multiple of 8), past_len <= 2^30, past_len + M <= max_t (the cache may be
 * longer than ql_attention_decode's 8192); fp32 q and out, sums and softmax in fp32; caches fp32 or fp16. Offsets 16-byte
 * aligned (mask: 8). Uses the context's 64 MiB workspace, as ql_attention_decode. */
int ql_attention_tree(ql_ctx* ctx, ql_arena* act, uint64_t q_off, const ql_arena* cache, uint64_t k_off, uint64_t v_off,
                      int32_t cache_dtype, int32_t max_t, int32_t M, int32_t n_head, int32_t n_kv_head, int32_t D, int32_t past_len,
                      uint64_t mask_off, uint64_t out_off);
/* The launch shape ql_attention_tree picks for these dimensions (host only, with the same checks): `pairs` (row, head) pairs of a
 * kv head share a workgroup of `waves` waves and its reads of K and V; nsplit key ranges (1: no merge launch). */
typedef struct ql_tree_info {
    int32_t pairs;
    int32_t waves;
    int32_t nsplit;
    int32_t keys_per_split;
    int32_t workgroups;    /* of the attention launch */
} ql_tree_info;
int ql_plan_attention_tree(int32_t cache_dtype, int32_t max_t, int32_t M, int32_t n_head, int32_t n_kv_head, int32_t D, int32_t past_len,
                           ql_tree_info* info);
/* Log probabilities over M rows of V fp32 logits (stride values apart, stride >= V; ql_gemv_f16w's y has stride V), natural
 * logarithms, no temperature:
 *   logprob [M, n_tok] fp32    of tokens [M, n_tok] int32; 0 for an id outside 0..V-1 (a padding entry)
 *   entropy [M] fp32           -sum p log p of the row (entropy_off QL_NONE: not wanted)
 *   top_id, top_logprob [M, top_k] int32, fp32: the largest logits in order, equal ones by the lower id; beyond V
 *                              entries -1 and -inf
 * all in `act`. -inf logits are tokens of no probability; a row of nothing else has log probabilities of -inf and entropy 0. A
 * NaN or +inf in a row makes its log probabilities and its entropy NaN; NaN comes first among the alternatives. M = 1..65535, V =
 * 1..2^24, n_tok 0..256, top_k 0..32 (the offsets of what is not wanted are ignored). Offsets 4-byte aligned; nothing
 * written may overlap anything else. Uses the context's 64 MiB workspace. */
int ql_token_logprobs(ql_ctx* ctx, ql_arena* act, uint64_t logits_off, int32_t stride, int32_t M, int32_t V, uint64_t tokens_off,
                      int32_t n_tok, int32_t top_k, uint64_t logprob_off, uint64_t entropy_off, uint64_t top_id_off, uint64_t top_logprob_off);
/* Rows of `count` cache regions: row dst_row + i of region r of `dst` (at dst_offs[r], dst_max_t rows of row_bytes) becomes row
 * src_row + rows[i] of region r of `src` (at src_offs[r], src_max_t rows), for i < n. rows is int32 [n] at rows_off in
 * `act`; QL_NONE: rows src_row + i (act may be null). An entry that is negative or leads outside the source leaves its destination
 * row as it was. A region may be moved onto itself (same arena and offset; n <= 256): every row is read before any is
 * written, so the list may have any order and name a row twice. Any other overlap of a written row with a source region, with
 * rows, or with another written row fails with QL_E_INVALID. count 1..256, n 0..2^24 (0: nothing is done), row_bytes a multiple of 16,
 * offsets 16-byte aligned (rows: 4). Ordered on ctx's stream only: where another context works on dst or src, the caller syncs. */
int ql_kv_move(ql_ctx* ctx, ql_arena* dst, const uint64_t* dst_offs, int32_t dst_max_t, const ql_arena* src, const uint64_t* src_offs,
               int32_t src_max_t, int32_t count, int32_t row_bytes, int32_t dst_row, int32_t src_row, int32_t n, const ql_arena* act,
               uint64_t rows_off);

/* ---- a pass over many requests at once: paged caches, a batch's rows of several sequences, low-rank adapters.
 * The order of a layer: linears over all M rows, ql_lora_add where requests have adapters, ql_paged_append,
 * ql_paged_attention, linears.
 *
 * A batch has n_seq sequences, whose rows lie one behind the other: sequence s has rows row_start[s] .. row_start[s + 1] - 1, one
 * of a request that decodes, many of a prompt or a piece of one. kv_len[s] counts its tokens with those of this pass: the last of its n
 * rows is token kv_len[s] - 1, the first kv_len[s] - n, and a row's position is its token. Token t lies in page pages[s][t / page_size].
 * The tables are int32 in `act` and read on the device, so a captured graph serves every pass of its sizes. What they may not say is
 * skipped, not followed: a sequence with row_start descending or outside 0..M, with more than max_rows rows, or with kv_len outside n..max_len has no
 * rows at all; a token whose page is outside 0..n_page - 1 is not stored, and no row sees it. Rows that two sequences claim have either's result, or none. Rows behind
 * the last sequence are padding.
 * Rows of q_out and out that belong to no sequence stay as they were. No two sequences may append to one page; they may share pages that they
 * only read. */
typedef struct ql_batch_desc {
    uint64_t row_start_off; /* int32 [n_seq + 1], ascending */
    uint64_t kv_len_off;    /* int32 [n_seq] */
    uint64_t pages_off;     /* int32 [n_seq, max_pages] */
    int32_t n_seq;          /* 1..4096 */
    int32_t max_pages;      /* pages of a sequence's list */
    int32_t max_rows;       /* no sequence has more rows in this pass, */
    int32_t max_len;        /* none more tokens: at most max_pages * page_size, and 2^26. Both choose the launches; bounds near what the tables hold serve best */
} ql_batch_desc;
/* A layer's paged cache, regions of n_page pages in a cache arena, offsets 16-byte aligned. A page holds page_size tokens of all kv heads, each
 * head's behind the other. D is a multiple of 16, u = 16 bytes of values: 8 (fp16) or 16 (e4m3).
 *   K  [n_page, n_kv_head, page_size / 16, D / u, 16, u]: value d of token t at (t / 16, d / u, t % 16, d % u)
 *   V  [n_page, n_kv_head, page_size / 4u, D / 16, 4, 16, u]: at (t / 4u, d / 16, t / 4 % 4, d % 16, t / 16 % (u / 4) * 4 + t % 4)
 *   QL_DTYPE_F8: fp32 scales [n_page, n_kv_head, page_size / 16] of K and of V, powers of two 2^-120 .. 2^120; a value is its e4m3
 *   number times the scale of its 16 tokens.
 * Pages are copied with ql_kv_move: a page is a row of n_kv_head * page_size * D values. */
typedef struct ql_paged_desc {
    uint64_t k_off, v_off;
    uint64_t k_scale_off, v_scale_off;   /* QL_DTYPE_F8 (otherwise ignored) */
    int32_t n_page;
    int32_t page_size;      /* 64, 128 or 256 */
    int32_t n_kv_head;
    int32_t D;              /* 16..256, a multiple of 16 */
    int32_t cache_dtype;    /* QL_DTYPE_F16 or QL_DTYPE_F8 */
    int32_t reserved;       /* 0 */
} ql_paged_desc;
/* ql_qk_norm_rope over a batch's rows: q and k RMSNormed per head (where the descriptor has weights) and turned by their positions, q to
 * q_out [M, n_head, D] in q_dtype (fp32, or fp16 rounded once), k and v to their tokens' places in the cache. `rope` is ql_qk_norm_rope's
 * descriptor, with the cache's n_kv_head, D and cache_dtype, and max_pos at least max_len.
 * fp16: rounded once; beyond 65504 infinite. e4m3: a group of 16 tokens of a head has one scale. Where the pass brings the group's first token, it is the smallest
 * 2^e (e >= -120) under which its largest new value is at most 448; otherwise that or the one the group has, whichever is larger, and
 * where it grows, the group's earlier tokens are rounded anew under it (exact but for values below 2^-6 of the new scale). Each value is rounded
 * once to e4m3; an infinity or NaN is stored as NaN and does not enter the scale.
 * q_out may be q itself (fp32, same offset, dense rows); any other overlap of what is written with what is read, tables included, fails with
 * QL_E_INVALID. M = 1..65535 rows of the buffers, M * (n_head + 2 n_kv_head) <= 2^23. Offsets 16-byte aligned (tables: 4). */
int ql_paged_append(ql_ctx* ctx, const ql_rope_desc* rope, const ql_arena* weights, ql_arena* act, uint64_t q_off, uint64_t k_off,
                    uint64_t v_off, const ql_batch_desc* batch, int32_t M, uint64_t q_out_off, int32_t q_dtype, ql_arena* cache,
                    const ql_paged_desc* paged);
/* out[m, h, :] = softmax_t(q[m, h] . K[t, h / (n_head / n_kv_head)] / sqrt(D)) V[t, ...] over the tokens t <= the row's own of its
 * sequence, which the cache holds (ql_paged_append has run). q and out are [M, n_head, D] in `act`, both of q_dtype: fp32 (q as two fp16
 * parts of about 22 bits under its row's exponent, probabilities likewise, down to 2^-33 of the row's largest), or fp16 (probabilities rounded once to fp16, with
 * the same end, as the result is). Sums and softmax in fp32. e4m3 values of V count by their own scales, whatever others have; where these lie more than 2^15 apart in 64 tokens
 * of a head (zeros aside) the tokens may be gone through a second, slower time. A row that sees nothing, or no score above -inf, is zero. What a row does not see adds nothing to it, infinities and NaN included;
 * a value of q that is not finite gives its head's row what the formula gives: NaN, or zero where every score is -inf. M * n_head <= 2^23,
 * n_seq * n_kv_head <= 2^22. Offsets 16-byte aligned. Uses the context's 64 MiB workspace. */
int ql_paged_attention(ql_ctx* ctx, ql_arena* act, uint64_t q_off, int32_t q_dtype, const ql_arena* cache, const ql_paged_desc* paged,
                       const ql_batch_desc* batch, int32_t M, int32_t n_head, uint64_t out_off);
/* Low-rank adapters of one projection, all n_adapter of them, in `weights`. */
typedef struct ql_lora_desc {
    uint64_t a_off;         /* fp16 [n_adapter, rank, K] */
    uint64_t b_off;         /* fp16 [n_adapter, N, rank] */
    uint64_t scale_off;     /* fp32 [n_adapter], or QL_NONE: 1 */
    int32_t K, N;           /* the projection's; K a multiple of 8, N of 4 */
    int32_t rank;           /* 8..128, a multiple of 8; an adapter of a lower rank has zeros behind its own */
    int32_t n_adapter;      /* 1..65536 */
} ql_lora_desc;
/* For each of `count` (1..8) projections: y[m, :] = base[m, :] + scale[a] * (x[m, :] . A_a^T) . B_a^T, a = ids[m]; y = base where ids[m] is outside
 * 0..n_adapter - 1 (-1: a row without an adapter). ids is int32 [M] in `act`; x [M, K] in x_dtype (fp32 or fp16), base and y fp32 [M, N] at
 * x_offs[i], base_offs[i], y_offs[i] in `act`. y_offs[i] may be base_offs[i] (a row without an adapter is not touched);
 * any other overlap of what is written with what is read fails with QL_E_INVALID. Sums in fp32, fp16 products exact; many rows take fp32 x, and x . A^T, as
 * two fp16 parts of about 22 bits each under the exponent of 64 columns, or of the row's ranks. A value of x that is not finite makes its own row's y infinite or
 * NaN, no other's.
 * M = 1..65535. Offsets 16-byte aligned (ids, scales: 4). Uses the context's 64 MiB workspace. */
int ql_lora_add(ql_ctx* ctx, int32_t count, const ql_lora_desc* descs, const ql_arena* weights, ql_arena* act, uint64_t ids_off,
                const uint64_t* x_offs, int32_t x_dtype, int32_t M, const uint64_t* base_offs, const uint64_t* y_offs);

/* several independent linears in one launch (e.g. q/k/v on one input, gate/up on another);
 * linear i reads x_offs[i] and writes y_offs[i]; scratch for all of them starts at scratch_off
 * (ql_plan_batch gives the size). M and x_dtype are shared; at most 8 linears. */
int ql_plan_batch(int32_t count, const ql_gptq_desc* descs, int32_t M, uint64_t* scratch_bytes);
int ql_linear_batch(ql_ctx* ctx, int32_t count, const ql_gptq_desc* descs,
                    const ql_arena* weights, ql_arena* act, const uint64_t* x_offs,
                    int32_t x_dtype, int32_t M, const uint64_t* y_offs, uint64_t scratch_off);

/* ---- linear sequences: many decode linears (M = 1..16) in ONE persistent launch.
 * Linear i reads x_offs[i] and writes y_offs[i] (fp32 [M, N_i]) in `act`. When x_offs[i] equals
 * y_offs[j] of an earlier linear j (with N_j == K_i), linear i consumes linear j's output and the
 * kernel orders the two on the device (the reference's passBreak); every other input is external
 * (x_dtype) and must not overlap any output; outputs must not overlap each other. All linears
 * share one group size (64, 128 or 256), need N % 4 == 0, and 16-byte aligned qweight, bias, x
 * and y offsets (scales 8-byte).
 * ql_seq_create validates, plans and allocates the sequence's device tables and exchange
 * buffers (the arenas are bound by address and must outlive it). ql_seq_run enqueues its launch
 * (one, except pass-by-pass sequences, below) on the context stream; it allocates nothing and
 * may be captured into a graph and replayed.
 * Runs of one sequence must not overlap (one stream). ql_seq_status waits for the stream and
 * reports whether a run was aborted (a bounded device-side wait ran out: QL_E_STATE).
 * Prefill (M = 17..65536): a sequence of independent linears (no linear reads another's output)
 * with fp16 x, N % 4 == 0 and groups a multiple of 128 runs as ONE persistent prefill GEMM
 * launch (kernel QL_SEQ_PREFILL): tasks of 128 rows x 256 columns over all of K, planned longest
 * first onto one workgroup per CU; y = f16(x) . f16(W)^T in fp32, as ql_linear's MFMA GEMM. */
#define QL_SEQ_TILES 0
#define QL_SEQ_STRIPS 1
#define QL_SEQ_PREFILL 2
#define QL_SEQ_STRIP_PASSES 3
#define QL_SEQ_PREFILL_PASSES 4
typedef struct ql_seq ql_seq;
typedef struct ql_seq_info {
    int32_t linears;
    int32_t passes;       /* dependency depth: linears that must run one after another */
    int32_t tiles;        /* GEMV tiles (64 columns x a K segment) */
    int32_t reduces;      /* split-K reductions (one per column tile of a split linear) */
    int32_t grid;         /* resident workgroups */
    int32_t max_split;    /* most parts (K pieces) of one 64-column block */
    uint64_t lds_bytes;   /* dynamic LDS per workgroup */
    uint64_t device_bytes;/* tables + exchange buffers ql_seq_create allocates */
    uint64_t total_units; /* block-groups (64 columns x one quantization group) of all linears */
    uint64_t busiest_units; /* block-groups of the most loaded workgroup: balance = busiest*grid/total */
    int32_t kernel;       /* QL_SEQ_TILES: dependency-ordered tiles; QL_SEQ_STRIPS: column strips;
                             QL_SEQ_PREFILL: prefill GEMM tiles (units: 128-k chunks);
                             QL_SEQ_STRIP_PASSES: one strip launch per pass (figures summed over
                             the passes) */
    int32_t split;        /* strips: waves per 64-column block (1: strips of 8 blocks, 2: of 4) */
    int32_t stream;       /* strips: 1 when the packed weights are read with streaming loads (the
                             weights exceed what the 256 MB MALL keeps between steps) */
    int32_t variant;      /* strips: 1 when the launch is the no-padding kernel on streamed
                             weights (every linear: group 128, K a multiple of 512, N a multiple
                             of 512; M = 5..16, or 2..16 pass by pass); QL_SEQ_PREFILL_PASSES: the
                             passes that run the chunked split-K GEMM. ql_seq_get_info, QL_SEQ_TILES: 2
                             when the created sequence runs its passes as products over activation
                             images (below; the other figures are then the tiles' plan, launches and
                             device_bytes its own). 0 otherwise */
    int32_t launches;     /* kernel launches one ql_seq_run enqueues */
} ql_seq_info;
/* plan only (host, pure) for a given grid size: validation and the figures above */
int ql_plan_seq(int32_t n, const ql_gptq_desc* descs, int32_t M, const uint64_t* x_offs,
                int32_t x_dtype, const uint64_t* y_offs, int32_t grid, ql_seq_info* info);
int ql_seq_create(ql_ctx* ctx, int32_t n, const ql_gptq_desc* descs, const ql_arena* weights,
                  ql_arena* act, const uint64_t* x_offs, int32_t x_dtype, int32_t M,
                  const uint64_t* y_offs, ql_seq** out);
int ql_seq_get_info(const ql_seq* seq, ql_seq_info* info);
int ql_seq_run(ql_ctx* ctx, ql_seq* seq);
int ql_seq_status(ql_ctx* ctx, ql_seq* seq);
/* Fused sequences (M = 1..16, fp32 x): per linear, elementwise work folded into the launch.
 *   norm_w_off  QL_NONE, or the weights-arena offset of an fp32 [K] RMSNorm weight: the linear
 *               reads rmsnorm(x) = x * rsqrt(mean(x^2) + norm_eps) * w per row (rmsNormRef)
 *               instead of x;
 *   x2_off      QL_NONE, or the activation-arena offset of an fp32 [M, K] second operand: the
 *               linear reads silu(x) * x2 (siluMulRef) instead of x; like x_offs it is another
 *               linear's output when it equals that linear's y offset, else external;
 *   res_off     QL_NONE, or the activation-arena offset of an fp32 [M, N] residual added to the
 *               linear's output (y = W.x + bias + res); another linear's output when it equals
 *               that linear's y offset, else external.
 * norm and x2 exclude each other. A linear runs after every producer it reads (x, x2 or res).
 * A fused sequence runs as dependency-ordered tiles (QL_SEQ_TILES) in one launch, except as
 * below. ql_plan_seq_fused and ql_seq_create_fused with fuse == NULL behave as ql_plan_seq and
 * ql_seq_create.
 * Chained sequences (fused or not) at M = 2..16 with fp32 x whose weights exceed what the MALL
 * keeps (192 MiB) and whose linears all have groups of 128, K % 512 == 0, K >= 1024 and
 * N % 512 == 0 run pass by pass instead (QL_SEQ_STRIP_PASSES): ql_seq_run enqueues, per pass,
 * the pass's column-strip launch (every strip cut into K parts of whole 512-k chunks, each part's
 * sums stored apart; each linear's activations formed as they are staged: as is, times an
 * RMSNorm weight, or SiLU-mul of two producers) and one launch that adds each linear's parts in a
 * fixed order, times the row's 1/rms for an RMSNorm'd input, with bias and residual (and the row
 * sums of squares of outputs a later linear RMSNorms); an external input that is RMSNorm'd adds
 * one launch before its pass. Stream order replaces the device-side waits (nothing can abort).
 * Other chained sequences (fused or not) with fp32 x, groups of 128, K % 128 == 0 and 16-byte aligned
 * norm weights run pass by pass over activation images at M = 5..16, and at M = 2..4 where a pass reads
 * 16 MiB of weights or more on average (and, at 2 and 3 rows, a pass with K above 8192 has at most 4096
 * columns): per pass, a launch for its distinct inputs of each kind (RMSNorms, SiLU-muls, rows as they are, as
 * scaled fp16 parts) and one for its linears, up to eight inputs or linears a launch. ql_plan_seq(_fused)
 * reports the tiles' plan for them, ql_seq_get_info variant 2 and the launches enqueued.
 * QL_SEQ_PASSES=0 in the environment keeps the tiles. */
typedef struct ql_seq_fuse {
    uint64_t norm_w_off;
    uint64_t x2_off;
    uint64_t res_off;
    float norm_eps;
    int32_t reserved;
} ql_seq_fuse;
int ql_plan_seq_fused(int32_t n, const ql_gptq_desc* descs, int32_t M, const uint64_t* x_offs,
                      int32_t x_dtype, const uint64_t* y_offs, const ql_seq_fuse* fuse, int32_t grid,
                      ql_seq_info* info);
int ql_seq_create_fused(ql_ctx* ctx, int32_t n, const ql_gptq_desc* descs, const ql_arena* weights,
                        ql_arena* act, const uint64_t* x_offs, int32_t x_dtype, int32_t M,
                        const uint64_t* y_offs, const ql_seq_fuse* fuse, ql_seq** out);
/* diagnostic: polls a device-side wait makes before aborting the run (default 4M, min 64) */
int ql_seq_set_spin_limit(ql_seq* seq, uint32_t polls);
int ql_seq_destroy(ql_seq* seq);

/* ---- ordering and timing on the context stream */
int ql_sync(ql_ctx* ctx);
int ql_timer_start(ql_ctx* ctx);
int ql_timer_stop(ql_ctx* ctx, float* elapsed_ms); /* waits for the stop event */

/* ---- stream capture into a HIP graph (one replayable submit per forward).
 * A graph may be launched on any context of the device. Where its calls pass data through a workspace of the context
 * (attention, ql_gemv_f16w, ql_linear and ql_linear_batch, as said there), it has one of its own, allocated while it
 * is captured and freed with it, so it does not meet the context's other work. It does hold the capturing context's
 * split-K arrival counters (ql_linear and ql_linear_batch with a plan that splits K): such a graph must not run
 * beside that context's linears on another stream, nor outlive the context. ql_linear_noalloc allocates nothing:
 * its captured launches use the static array, or the context's workspace where that is too small. */
int ql_graph_begin(ql_ctx* ctx);
int ql_graph_end(ql_ctx* ctx, ql_graph** out);
int ql_graph_launch(ql_ctx* ctx, ql_graph* graph);
int ql_graph_destroy(ql_graph* graph);

#ifdef __cplusplus
}
#endif
#endif /* QLINEAR_H */
