/*
 * mlxq.h — C ABI of libmlxq_hip.so, the MI355X (gfx950) implementation of mlx-gen's group-wise
 * affine Q4/Q8 quantized-linear path.
 *
 * The reference reaches this arithmetic through three MLX ops and one MLX layer, all external to
 * the reference (pmetal-mlx-rs 0.25.8 -> MLX 0.31.2, reference Cargo.toml:38,43):
 *   mlx_rs::ops::quantize            called at src/quant.rs:140, src/nn.rs:91-93, and via
 *                                    nn::QuantizedLinear::try_from_linear at src/adapters.rs:533-537
 *   mlx_rs::ops::dequantize          called at src/nn.rs:55, mlx-gen-flux/src/text_encoder.rs:78
 *   mlx_rs::ops::quantized_matmul    called at src/adapters.rs:309-317 (LinearBase::forward)
 * Each entry point below replaces one of them; a Rust -sys crate binds these symbols one-to-one.
 *
 * Conventions
 *   - All tensor pointers are DEVICE pointers owned by the caller; the library allocates nothing
 *     on these paths except where a workspace size query says so.
 *   - Work is enqueued asynchronously on `stream` (a hipStream_t; NULL = the default stream).
 *   - Row-major, contiguous.  Packing: 32/bits codes per uint32, element i of a word at bit offset
 *     i*bits (low bits first); wq [N, K*bits/32]; scales/biases [N, K/group_size].
 *   - group_size in {32, 64, 128}, bits in {4, 8}, K % group_size == 0.
 *   - Alignment: activations, packed weights, outputs and workspaces 16 bytes; scales and biases
 *     4 bytes.  Misaligned pointers are rejected with MLXQ_EINVAL.
 *   - Every call returns an mlxq_status; on failure mlxq_last_error() (thread-local) describes
 *     it.  Arguments that contradict each other here (dtype codes, group_size/bits, K % gs,
 *     alignment, null pointers) are rejected with MLXQ_EINVAL.  This layer sees pointers, not
 *     tensor shapes: the C++ and Python hosts check every operand's shape and dtype against x
 *     before they call in (the reference's packed_bits panics on malformed triples,
 *     src/quant.rs:38-41).
 *   - Dtypes follow MLX's promotion: an op on a bf16 and an f32 operand computes and returns f32
 *     (quantized_matmul returns promote(x, scales); a bias add and a LoRA residual promote the
 *     output the same way).  mlxq_linear_out_dtype gives the dtype y must have.
 *   - Re-entrant per stream.  Process-wide state, all of it per device and written once: the two
 *     GELU tables (device memory in the code object, filled by the first GELU GEMM on a device),
 *     the cached CU count, the decode GEMV's raised dynamic-LDS limit (atomic flags), the device
 *     address of mlxq_linear_noalloc's static scratch (guarded by a mutex), plus the thread-local
 *     error string.
 */
#ifndef MLXQ_H
#define MLXQ_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum {
  MLXQ_FLOAT32 = 0,
  MLXQ_BFLOAT16 = 1,
  /* fp16 is taken as the activation x of quantized_matmul, qmv, qmv_valu, linear, linear_noalloc,
   * lora_residual and qmm_experts: the dtype SDXL's U-Net, CLIP encoders and ControlNets run in
   * (mlx-gen-sdxl/src/model.rs:216) over bf16-packed weights (src/adapters.rs:508-537).  MLX
   * promotes fp16 against bf16 or f32 to f32, so those products and their results are f32.
   * Elsewhere (weights, scales, biases, LoRA factors, outputs) fp16 returns MLXQ_EUNSUPPORTED. */
  MLXQ_FLOAT16 = 2,
} mlxq_dtype;

typedef enum {
  MLXQ_OK = 0,
  MLXQ_EINVAL = 1,       /* bad shape / dtype / group_size / bits / null pointer */
  MLXQ_EUNSUPPORTED = 2, /* valid for MLX but not implemented here (e.g. transpose=false) */
  MLXQ_EDEVICE = 3,      /* HIP launch or runtime error */
} mlxq_status;

typedef enum {
  MLXQ_ACT_NONE = 0,
  /* mlx_rs::nn::gelu, the exact-erf GELU of FLUX's FeedForward (mlx-gen-flux/src/transformer.rs:975;
   * also mlx-gen-qwen-image/src/text_encoder/vision/merger.rs:49, mlx-gen-ltx/src/connector.rs:252):
   * its constants are f32 arrays, so a bf16 input promotes and the result is f32 (src/nn.rs:335-338) */
  MLXQ_ACT_GELU = 1,
  /* tanh-approximate GELU as separate ops in the input dtype, src/nn.rs:321-329 (FLUX
   * single-stream FFN and GeluApprox, mlx-gen-flux/src/transformer.rs:506,708,979) */
  MLXQ_ACT_GELU_TANH = 2,
  /* dtype-preserving exact GELU, src/nn.rs:344-355 gelu_exact (x * (1 + erf(x / sqrt2))) / 2; the
   * GELU of most crates' FFNs (bernini, boogu, pid, svd, ...).  In bf16 each op of the sequence is
   * rounded to bf16 (the uncompiled op sequence).  The reference runs it under compile(f, true),
   * whose fused kernel its own comments say rounds 16-bit types differently from the separate ops
   * (src/nn.rs:339-343): bf16 parity with the reference is unpinned.  f32 is unaffected. */
  MLXQ_ACT_GELU_EXACT = 3,
} mlxq_activation;

/* Thread-local description of the last failure on this thread ("" if none). */
const char* mlxq_last_error(void);
/* Library version string. */
const char* mlxq_version(void);

/*
 * quantize — replaces mlx_rs::ops::quantize(w, group_size, bits) (src/quant.rs:140;
 * src/adapters.rs:533-537 through QuantizedLinear::try_from_linear).
 * w [N,K] in w_dtype; writes wq [N, K*bits/32] and scales/biases [N, K/group_size] in w_dtype.
 */
int mlxq_quantize(const void* w, int w_dtype, int64_t N, int64_t K, int group_size, int bits,
                  uint32_t* wq, void* scales, void* biases, void* stream);

/*
 * quantize over `count` weights of one shape [N,K] and dtype: the same outputs as `count`
 * mlxq_quantize calls (w[i] -> wq[i], scales[i], biases[i]), in launches of up to 16 weights,
 * which pay a launch's ramp and its partly filled last round once for all of them.  No single
 * counterpart in the reference, which quantizes weight by weight (quantize_map, src/quant.rs:125-149,
 * calling a-1 per target); for converters that pack many same-shaped weights.  The pointer arrays
 * are host memory; count == 0 does nothing.
 */
int mlxq_quantize_batched(const void* const* w, int count, int w_dtype, int64_t N, int64_t K, int group_size,
                          int bits, uint32_t* const* wq, void* const* scales, void* const* biases, void* stream);

/*
 * dequantize — replaces mlx_rs::ops::dequantize(wq, scales, biases, group_size, bits)
 * (src/nn.rs:55).  out [N,K] in sb_dtype (the scales dtype, as MLX returns).
 */
int mlxq_dequantize(const uint32_t* wq, const void* scales, const void* biases, int sb_dtype,
                    int64_t N, int64_t K, int group_size, int bits, void* out, void* stream);

/*
 * quantized_matmul — replaces mlx_rs::ops::quantized_matmul(x, wq, scales, biases, transpose,
 * group_size, bits) (src/adapters.rs:309-317).  x [M,K] in x_dtype (batch dims flattened into
 * M); y [M,N] in promote(x_dtype, sb_dtype) (bf16 only when both are bf16, as MLX casts x, scales
 * and biases to their result type); fp32 accumulation.  Only transpose=1 (y = x . W^T, the only
 * form the reference uses) is implemented; transpose=0 returns MLXQ_EUNSUPPORTED.
 * Dispatch: bf16 x and scales with M > 8 run the MFMA GEMM (weights dequantized to bf16 tiles);
 * bf16 with M <= 8 runs the bandwidth-bound GEMV (weights dequantized in f32, factored per
 * group); an f32 operand, or fp16 x (which MLX promotes to f32 against bf16 or f32 scales), runs
 * the f32 kernels (exact f32 dequant, f32 result).
 */
int mlxq_quantized_matmul(const void* x, int x_dtype, int64_t M, int64_t K, const uint32_t* wq,
                          const void* scales, const void* biases, int sb_dtype, int64_t N,
                          int transpose, int group_size, int bits, void* y, void* stream);

/*
 * Quantized token-embedding lookup — replaces TokenEmbedding::forward's quantized arm
 * (src/nn.rs:42-58: take_axis of wq/scales/biases by ids, dequantize, cast to f32) in one pass.
 * ids [T] int32 device array; table wq [vocab, hidden*bits/32] with scales/biases
 * [vocab, hidden/group_size] in sb_dtype; out [T, hidden] in out_dtype (MLXQ_FLOAT32 reproduces
 * the reference's cast).  Each value is dequantize()'s, i.e. rounded to sb_dtype first.  Ids
 * outside [0, vocab) produce a row of NaN.
 */
int mlxq_embedding(const int32_t* ids, int64_t T, const uint32_t* wq, const void* scales,
                   const void* biases, int sb_dtype, int64_t vocab, int64_t hidden, int group_size,
                   int bits, void* out, int out_dtype, void* stream);

/* Forced-kernel variants of quantized_matmul (same arguments, transpose implied = 1). */
/* MFMA bf16-tile GEMM; x must be bf16; any M >= 1; y is bf16 whatever sb_dtype is (the kernel's
 * native output: with f32 scales this is not quantized_matmul's promoted f32 result). */
int mlxq_qmm(const void* x, int x_dtype, int64_t M, int64_t K, const uint32_t* wq,
             const void* scales, const void* biases, int sb_dtype, int64_t N, int group_size,
             int bits, void* y, void* stream);
/* GEMV; bf16, f32 or fp16 x; 1 <= M <= 8; y in promote(x_dtype, sb_dtype). */
int mlxq_qmv(const void* x, int x_dtype, int64_t M, int64_t K, const uint32_t* wq,
             const void* scales, const void* biases, int sb_dtype, int64_t N, int group_size,
             int bits, void* y, void* stream);

/* A GEMV on the VALU only (no matrix cores); any x / scales dtype; 1 <= M <= 8; y in
 * promote(x_dtype, sb_dtype).  The VALU GEMV with exact f32 dequant (the kernel quantized_matmul
 * uses for f32 operands), except at M = 1 with bf16 x and scales, Q4, group
 * 64/128 and K <= 8192, where it is the M = 1 matrix-core kernel's loads and fold with VALU dot
 * products.  Forced here so it can be measured against the matrix-core GEMV on bf16 decode
 * shapes. */
int mlxq_qmv_valu(const void* x, int x_dtype, int64_t M, int64_t K, const uint32_t* wq,
                  const void* scales, const void* biases, int sb_dtype, int64_t N, int group_size,
                  int bits, void* y, void* stream);

/*
 * Fused AdaptableLinear forward over a quantized base — replaces the op sequence of
 * LinearBase::forward's quantized arm plus AdaptableLinear::forward (src/adapters.rs:300-322,
 * 543-549) for one LoRA adapter (Adapter::residual, src/adapters.rs:260-270), optionally followed
 * by the caller's activation (FeedForward::forward, mlx-gen-flux/src/transformer.rs:970-977):
 *   y0 = qmm(x)                 in D0 = promote(x_dtype, sb_dtype)          (:309-317)
 *   y1 = y0 + bias              in D1 = promote(D0, bias_dtype)             (:318-320)
 *   r  = ((x.A).B) * scale      in DR = promote(x_dtype, lora_dtype), each op rounded to DR and
 *                               scale cast to DR first (the factors keep their file dtype, :243-252)
 *   y2 = y1 + r                 in D2 = promote(D1, DR), not cast back     (:546)
 *   y  = act(y2)                GELU_TANH / GELU_EXACT per op in D2; GELU in f32
 * Each round() happens exactly where the reference's separate MLX ops round, and y has dtype
 * mlxq_linear_out_dtype().  bias [N] (bias_dtype), lora_a [K,rank] and lora_b [rank,N]
 * (lora_dtype) are nullable (rank 0 = no LoRA); rank <= 256.  workspace must hold
 * mlxq_linear_workspace_size() bytes (NULL when that is 0).
 */
typedef struct {
  const void* bias;
  const void* lora_a;
  const void* lora_b;
  int64_t lora_rank;
  float lora_scale;
  int activation; /* mlxq_activation */
  int bias_dtype; /* mlxq_dtype of bias (ignored when bias is NULL) */
  int lora_dtype; /* mlxq_dtype of lora_a and lora_b (ignored when lora_rank is 0) */
} mlxq_epilogue;

/* The dtype y of mlxq_linear has for these operands (an mlxq_dtype), or -1 (with
 * mlxq_last_error set) when a dtype code or the activation is invalid.  epilogue may be NULL. */
int mlxq_linear_out_dtype(int x_dtype, int sb_dtype, const mlxq_epilogue* epilogue);

/* Bytes of device workspace mlxq_linear needs (0: pass NULL): the LoRA staging (x.A and B^T
 * padded to rank 16, 4 bytes per element) and, when a bf16 product promotes to an f32 result,
 * the bf16 product itself [M, N].  0 as well for invalid arguments (mlxq_linear reports them). */
size_t mlxq_linear_workspace_size(int x_dtype, int sb_dtype, int64_t M, int64_t N,
                                  const mlxq_epilogue* epilogue);

int mlxq_linear(const void* x, int x_dtype, int64_t M, int64_t K, const uint32_t* wq,
                const void* scales, const void* biases, int sb_dtype, int64_t N, int group_size,
                int bits, const mlxq_epilogue* epilogue, void* y, void* workspace,
                size_t workspace_bytes, void* stream);

/*
 * mlxq_linear without a workspace argument: the workspace mlxq_linear_workspace_size reports
 * (LoRA staging, and the bf16 product of a promoted result) lives in a static device array of
 * MLXQ_NOALLOC_SCRATCH_BYTES that each GPU holds from the first call on it until the process ends.
 * No counterpart in the reference: this entry point exists for callers that cannot allocate
 * device memory (code under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc).  It calls no allocator.  A problem that needs more scratch than the array holds is
 * rejected with MLXQ_EINVAL before any device work.  The first call on each device resolves the
 * array's device address (hipGetSymbolAddress), so make it outside graph capture.  Every call on
 * one GPU shares that GPU's array: calls that overlap on one GPU (several streams or threads)
 * race and must be serialised by the caller.  Same arguments, results and errors as mlxq_linear
 * otherwise.
 */
#define MLXQ_NOALLOC_SCRATCH_BYTES (8u << 20)

int mlxq_linear_noalloc(const void* x, int x_dtype, int64_t M, int64_t K, const uint32_t* wq,
                        const void* scales, const void* biases, int sb_dtype, int64_t N,
                        int group_size, int bits, const mlxq_epilogue* epilogue, void* y,
                        void* stream);

/*
 * Stacked-expert projection — Proj::forward of the quantized MoE experts
 * (mlx-gen-lens/src/text_encoder/gpt_oss.rs:412-425, quantized_matmul(x, wq, s, b, true) + bias)
 * run for every expert of a stacked pack split along axis 0 (mlx-gen-lens/src/quant.rs:93-137):
 *   for e in [0, E):  y[e] = round(round(x[e] . dequant(wq[e])^T) + bias[e])
 * rounded to D0 = promote(x_dtype, sb_dtype) and then promote(D0, bias_dtype), as mlxq_linear.
 * wq [E, N, K*bits/32], scales/biases [E, N, K/group_size] (sb_dtype), bias [E, N] in bias_dtype
 * or NULL, y [E, M, N].  The reference's stacked packs carry a bf16 bias (gpt_oss.rs:478-487); an
 * f32 bias over a bf16 product would need a promoted second pass and returns MLXQ_EUNSUPPORTED.
 * x is [M, K] shared by every expert when x_per_expert == 0 (the gate_up projection of
 * gpt_oss.rs:702), else [E, M, K] (the down projection of :714).  Each expert's result is the
 * single-matrix mlxq_linear's with that bias: the same products, rounded at the same points.  How the f32
 * sums over K are split follows the whole launch, so with 9 rows or more (and one row of Q8 with a ragged
 * K) an expert's last bf16 bit may depend on how many share the stack.  bf16 x and scales run every expert in one launch with
 * M <= 8 (the GEMV's shapes), with M <= 64, K a multiple of 64 and K >= 512, and with K a multiple of
 * 64 and at least 128 GEMM tiles over all experts; otherwise the experts run one after another
 * through mlxq_linear.  All but the last of these need each expert's slices aligned: M*N elements of
 * y a multiple of 16 bytes and N*K/group_size scales (biases) a multiple of 4 bytes; shapes that none
 * then takes return MLXQ_EUNSUPPORTED (the Python and C++ hosts run those experts on aligned copies).
 */
int mlxq_qmm_experts(const void* x, int x_dtype, int x_per_expert, int64_t E, int64_t M, int64_t K,
                     const uint32_t* wq, const void* scales, const void* biases, int sb_dtype,
                     const void* bias, int bias_dtype, int64_t N, int group_size, int bits, void* y,
                     void* stream);

/*
 * Fused SwiGLU gate/up for decode — the first two ops of Mlp::forward
 * (mlx-gen-sensenova/src/qwen3.rs:178-181): h = multiply(silu(gate.forward(x)), up.forward(x))
 * with gate/up quantized linears [F,K] sharing x [M,K]; one launch streams both weight matrices
 * (launches of four or two activation rows when the M rows do not fit one workgroup):
 *   h = round(round(silu(round(x.Wg^T))) * round(x.Wu^T))      (round() to bf16)
 * Decode form only: bf16 x and scales, 1 <= M <= 8, group_size 32, 64 or 128, K a multiple of
 * 512/bits within the fused kernels' reach (Q4: K <= 16384 at M = 1, 12288 at M = 2..8, 8192
 * with group 32; Q8: 8192 at M = 1, 6144 at M = 2..8, 4096 with group 32); anything else
 * returns MLXQ_EUNSUPPORTED (callers then run the two linears).
 * This entry point has no single counterpart in the reference; it replaces a three-op sequence.
 */
int mlxq_swiglu(const void* x, int x_dtype, int64_t M, int64_t K, const uint32_t* wq_gate,
                const void* scales_gate, const void* biases_gate, const uint32_t* wq_up,
                const void* scales_up, const void* biases_up, int sb_dtype, int64_t F,
                int group_size, int bits, void* h, void* stream);

/*
 * One more LoRA adapter on an already computed output — the `out + adapter.residual(x)` step of
 * AdaptableLinear::forward (src/adapters.rs:543-549, Adapter::residual :260-270) for adapter
 * stacks beyond the one mlxq_linear fuses:
 *   y_out = y_in + r,  r = ((x.A).B) * scale in DR = promote(x_dtype, lora_dtype) (each op rounded
 *   to DR, scale cast to DR), the sum in promote(y_dtype, DR) — the dtype y_out must have.
 * A [K,rank], B [rank,N] in lora_dtype, 1 <= rank <= 256.  y_out may be y_in when the sum keeps
 * y_dtype; otherwise the two must not overlap.  workspace: mlxq_lora_residual_workspace_size().
 */
size_t mlxq_lora_residual_workspace_size(int x_dtype, int lora_dtype, int64_t M, int64_t N,
                                         int64_t rank);
int mlxq_lora_residual(const void* x, int x_dtype, int64_t M, int64_t K, const void* lora_a,
                       const void* lora_b, int lora_dtype, int64_t N, int64_t rank,
                       float lora_scale, const void* y_in, int y_dtype, void* y_out,
                       void* workspace, size_t workspace_bytes, void* stream);

/*
 * One LoKr adapter on an already computed output — the Adapter::Lokr arm of Adapter::residual
 * (src/adapters.rs:263-266) in AdaptableLinear::forward's residual sum (:543-549):
 *   d = delta cast to x_dtype;  r = x . d^T in x_dtype (f32 accumulation, rounded once);
 *   r = r * scale (scale cast to x_dtype first);  y_out = y_in + r in promote(y_dtype, x_dtype).
 * delta [N, K] in delta_dtype is the reconstructed kron delta (reconstruct_lokr_delta,
 * src/adapters.rs:26-128; the reference stores it bf16).  K must be a multiple of 32.  y_out may be
 * y_in when the sum keeps y_dtype; otherwise the two must not overlap.  workspace:
 * mlxq_lokr_residual_workspace_size() bytes (the f32 product, M*N*4).
 */
size_t mlxq_lokr_residual_workspace_size(int x_dtype, int64_t M, int64_t N);
int mlxq_lokr_residual(const void* x, int x_dtype, int64_t M, int64_t K, const void* delta,
                       int delta_dtype, int64_t N, float scale, const void* y_in, int y_dtype,
                       void* y_out, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Element-wise dtype conversion f32 <-> bf16 (round to nearest even) — the `as_dtype(Bfloat16)`
 * casts that precede packing in AdaptableLinear::quantize (src/adapters.rs:508-521) and
 * quant::quantize_map (src/quant.rs:140).  src/dst 4-byte aligned.
 */
int mlxq_cast(const void* src, int src_dtype, void* dst, int dst_dtype, int64_t n, void* stream);

/*
 * ---- Serving a decoder from a paged key/value cache ------------------------------------------
 *
 * The step between a decoder block's qkv projection and its output projection: rotate the new
 * queries and keys by their positions, write keys and values into the pages of a cache, attend
 * over the pages, and copy pages when sequences fork or the pool is compacted.  No counterpart in
 * the reference, whose attention runs in MLX (mlx-gen-sensenova/src/qwen3.rs:463, forward_cached).
 *
 * Queries, keys, values, cache and result have one dtype (f32, bf16 or fp16).  Scores, softmax
 * statistics and sums are f32, and the result is rounded once.  f32 rounds nothing between.  16-bit
 * types round the softmax weights to the type before the product with the values: weights are taken
 * against a running maximum, so that fp16's below 2^-25 of it are 0.  Chunks (more than 32 rows, pairs
 * of a token and a query head, a key head; 16 for heads past 128) sum the rounded weights, shorter calls
 * the f32 ones: the same row may differ between the two by what that rounding is.
 *
 * Cache: a pool of pages of page_size tokens, one pool for a layer's keys and one for its values.
 * With C = 16 / sizeof(element) (8 for 16-bit types, 4 for f32), page p of the keys starts
 * p * k_page_stride elements into k and holds [heads, page_size/16, head_dim/C, 16, C]: blocks of
 * 16 tokens, each a run of 16-byte pieces with the token the faster index.  A page of the values
 * holds [heads, page_size/C, head_dim, C]: C tokens of a feature side by side.  These are the
 * operands of the matrix instructions as they lie, so the attention kernels read both without
 * moving an element between lanes.  The pages of a pool need no order; head_dim is a multiple of 16
 * up to 256, page_size a power of two from 16 to 1024.
 *
 * A page id that a call needs and that is outside [0, pages) is never followed: the token is not
 * written (cache_append, copy_pages), the rows that see it become NaN (paged_attention).
 */
typedef struct {
  void* data;             /* element (t, h, d) at data[t * token_stride + h * head_stride + d] */
  int64_t heads;
  int64_t token_stride;   /* elements; both strides a multiple of 16 bytes */
  int64_t head_stride;
} mlxq_heads;

typedef struct {
  void* k;
  void* v;
  int64_t k_page_stride;  /* elements from one page to the next, a multiple of 16 bytes */
  int64_t v_page_stride;
  int64_t pages, page_size, heads, head_dim;
  int dtype;              /* mlxq_dtype of cache, queries, keys, values and result */
} mlxq_paged_cache;

/* The sequences of a step.  Sequence b owns the new tokens q_starts[b] .. q_starts[b+1] - 1 of the
 * step's T (n of them, 0 allowed) and has kv_lens[b] tokens in the cache counting those: the i-th new
 * one is its token kv_lens[b] - n + i.  Token j lies in page block_tables[b * table_stride +
 * j / page_size].  All arrays are device int32.  A token past table_width pages (or past 2^30 - 16) has no
 * page: it is not written, and rows that see it become NaN.
 * max_q and max_kv are what the launch is planned for (the longest n and kv length expected): any values
 * give right results, which differ in their last bits where the plan sums in another order.  Steps' tokens
 * outside every sequence are left alone. */
typedef struct {
  const int32_t* block_tables;
  const int32_t* q_starts;  /* [sequences + 1], not decreasing */
  const int32_t* kv_lens;   /* [sequences] */
  int64_t sequences, table_width, table_stride;
  int64_t max_q, max_kv;
} mlxq_paged_batch;

/* Long-context scalings of the rotation frequencies f_i = base^(-2i/rotary_dim). */
typedef enum {
  MLXQ_ROPE_NONE = 0,
  MLXQ_ROPE_LINEAR = 1,  /* f_i / factor */
  MLXQ_ROPE_NTK = 2,     /* base * factor^(r / (r - 2)), r = rotary_dim */
  /* Blend by wavelength: with n_i = original_context * f_i / 2 pi turns over the trained context,
   * f_i is kept where n_i >= high, divided by factor where n_i <= low, and between them mixed:
   * YARN linearly in the pair index i between the (fractional) indexes of the two bounds, rounded
   * outwards, LLAMA3 linearly in n_i.  YARN also scales cos and sin by 0.1 ln(factor) + 1. */
  MLXQ_ROPE_YARN = 3,
  MLXQ_ROPE_LLAMA3 = 4,
} mlxq_rope_kind;

typedef struct {
  int kind;                 /* mlxq_rope_kind */
  double factor;            /* >= 1; not read for NONE */
  double original_context;  /* trained context, tokens (YARN, LLAMA3) */
  double low, high;         /* turns, 0 < low < high (YARN: 1 and 32 are common, LLAMA3: 1 and 4) */
} mlxq_rope_scaling;

/* Host function: inv_freq[i], i < rotary_dim / 2, in radians a position, and the factor of cos and
 * sin.  scaling NULL = none. */
int mlxq_rotary_frequencies(int64_t rotary_dim, double base, const mlxq_rope_scaling* scaling,
                            double* inv_freq, double* magnitude);

/* table[p, i] = magnitude * (cos, sin)(p * inv_freq[i]) for positions p < positions, f32, each angle
 * in 64 bits.  inv_freq is a host array of rotary_dim / 2 <= 128; table is
 * [positions, rotary_dim/2, 2], 16-byte aligned. */
int mlxq_rotary_table(const double* inv_freq, int64_t rotary_dim, double magnitude, int64_t positions,
                      float* table, void* stream);

/*
 * Rotary positions: y[t, h] = x[t, h] with each pair (a, b) of its first rotary_dim features turned
 * by the table's row positions[t]: (a c - b s, b c + a s).  Pair i is features (i, i + rotary_dim/2),
 * or (2i, 2i + 1) when interleaved.  Features past rotary_dim are copied.  inverse != 0 turns by -s:
 * the transpose, which takes the gradient of y to the gradient of x.  positions [T] int32; one outside
 * [0, table_rows) gives NaN in the rotated features.  head_dim is a multiple of 16 bytes.  y may be x
 * (same strides); otherwise they must not overlap.
 */
int mlxq_rotary(const mlxq_heads* x, int dtype, int64_t T, int64_t head_dim, const int32_t* positions,
                const float* table, int64_t table_rows, int64_t rotary_dim, int interleaved,
                int inverse, const mlxq_heads* y, void* stream);

/*
 * Writes a step's keys and values into the cache, in one launch with the rotation of its queries and
 * keys.  k and v hold the T new tokens; the keys are rotated as mlxq_rotary does by the token's place
 * in its sequence, or by positions[t] when positions is not NULL; table NULL (rotary_dim 0) writes
 * them as they are.  q (NULL = none) is rotated alike into q_out, which may be q.  Tokens whose place
 * is negative (more new tokens than kv_lens) are not written to the cache.
 */
int mlxq_cache_append(const mlxq_heads* k, const mlxq_heads* v, int64_t T, const mlxq_paged_cache* cache,
                      const mlxq_paged_batch* batch, const int32_t* positions, const float* table,
                      int64_t table_rows, int64_t rotary_dim, int interleaved, const mlxq_heads* q,
                      const mlxq_heads* q_out, void* stream);

/* Options of the attention.  Row h of the new token at place p of a sequence of L tokens sees the
 * tokens j with  lo <= j < hi,  hi = causal ? min(L, max(p + 1, prefix)) : L,  lo = window ?
 * max(0, p + 1 - window) : 0. */
typedef struct {
  float scale;                 /* > 0: z_j = scale * q.k_j */
  int causal;
  int64_t window;              /* 0 = none; counts the token itself */
  float softcap;               /* 0 = none; z_j = softcap * tanh(z_j / softcap), any finite one; 16-bit types
                                * are off by up to 5 2^-24 softcap of a score for caps up to 256 */
  const int32_t* prefix_lens;  /* [sequences] or NULL: tokens that every row of the sequence sees */
  const float* alibi_slopes;   /* [q heads] or NULL: z_j -= slope * |p - j|, after the cap */
  const float* sinks;          /* [q heads] or NULL: a score without a value, in the denominator only */
} mlxq_attention;

/*
 * Attention of the step's new tokens over their sequences' cached tokens (a chunk of a prompt, drafted
 * tokens or one token each, mixed at will):
 *   out[t, h] = sum_j exp(z_j) v_j / (sum_j exp(z_j) + exp(sink_h))   over the visible j,
 * zero for a row that sees nothing.  Query head h reads key head h / (q heads / cache heads).  What the
 * masked and unwritten places of the cache hold (NaN and infinities included) does not reach the
 * result.  out must not overlap q.  workspace: mlxq_paged_attention_workspace_size() bytes, whatever
 * they hold (NULL when that is 0), at most some 300 MB.  T * (q heads / cache heads) must be below 2^31 - 128.
 * Launch shapes follow T, the batch's sizes and hints and the strides
 * only, so a captured graph may be replayed with other lengths and tables.
 */
size_t mlxq_paged_attention_workspace_size(int64_t T, int64_t q_heads, const mlxq_paged_cache* cache,
                                           const mlxq_paged_batch* batch, const mlxq_attention* options);
int mlxq_paged_attention(const mlxq_heads* q, int64_t T, const mlxq_paged_cache* cache,
                         const mlxq_paged_batch* batch, const mlxq_attention* options,
                         const mlxq_heads* out, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Copies pages src[i] to dst[i], i < count, in each of `planes` pools (the layers' keys and values):
 * page p of plane l is the page_bytes bytes at cache + l * plane_stride_bytes + p * page_stride_bytes
 * (strides and page_bytes multiples of 16).  tables (NULL = none): entries [rows, width], rows
 * table_stride apart, that equal some src[i] become dst[i].  src and dst are device int32; no dst may
 * be a src or appear twice, and a src that tables are to follow appears once.
 */
int mlxq_cache_copy_pages(void* cache, int64_t planes, int64_t plane_stride_bytes, int64_t pages,
                          int64_t page_bytes, int64_t page_stride_bytes, const int32_t* src,
                          const int32_t* dst, int64_t count, int32_t* tables, int64_t rows,
                          int64_t width, int64_t table_stride, void* stream);

/*
 * ---- A decoder block in microscaled types: quantisation, products, norms, routing to experts ------
 *
 * No counterpart in the reference, whose norms, routers and microscaled products run in MLX
 * (mlx-gen-sensenova/src/qwen3.rs:178-181; mlx-gen-lens/src/text_encoder/gpt_oss.rs:396-440 turns its
 * microscaled experts into affine packs).
 *
 * A microscaled matrix [rows, K], K a multiple of 32: blocks of 32 values of a row share a scale, a byte
 * b that stands for 2^(b - 127) (255: NaN, and so the whole block).  Codes are e2m1 (0, 0.5, 1, 1.5, 2,
 * 3, 4, 6 and their negatives, two to a byte, the first in the low half) or e4m3 (a byte each, largest
 * 448, 0x7f and 0xff NaN), the Open Compute Project's types.  Codes are contiguous, rows * K / 2 or
 * rows * K bytes, 16-byte aligned; the scales of a row, K / 32 bytes, start scale_stride bytes after the
 * row before's, a multiple of 4 and at least K / 32, and 4-byte aligned.  Bytes between them are not
 * read for a result and may hold anything; up to the next multiple of 4 quantisation writes them as 0.
 */
typedef enum { MLXQ_MX_E2M1 = 0, MLXQ_MX_E4M3 = 1 } mlxq_mx_format;

typedef struct {
  void* codes;
  void* scales;
  int64_t scale_stride; /* bytes */
  int format;           /* mlxq_mx_format */
} mlxq_mx;

/*
 * x [rows, K] (f32, bf16, fp16; row_stride elements from one row to the next, rows 16-byte aligned) to
 * microscaled codes.  A block's scale is the smallest power of two from 2^-127 on by which its largest
 * magnitude divided is at most 6 (e2m1) or 448 (e4m3), so that nothing saturates; values are rounded to
 * nearest, ties to even.  A block with an infinity or a NaN has scale 255 and codes 0.  Every step
 * but the rounding is exact.  The types are the Open Compute Project's; the choice of a scale is not its
 * conversion's, which takes the power of two of the largest magnitude and saturates: codes differ from such a
 * quantiser's wherever that magnitude's significand is above 1.5 (e2m1) or 1.75 (e4m3).
 */
int mlxq_mx_quantize(const void* x, int dtype, int64_t rows, int64_t K, int64_t row_stride,
                     const mlxq_mx* out, void* stream);

/* out [rows, K] in out_dtype: code times scale, rounded once.  f32 holds all of them and bf16 those from 2^-126 on,
 * but for the largest codes under the largest scales, which are infinite from 2^128 on (a block of the largest f32
 * has one: it is quantised to 2^128); fp16 overflows past 65504. */
int mlxq_mx_dequantize(const mlxq_mx* x, int64_t rows, int64_t K, void* out, int out_dtype, void* stream);

/*
 * y [M, N] = x . w^T + bias: x [M, K] in either format, w [N, K] e2m1, bias [N] in bias_dtype or NULL; y
 * in y_dtype (f32, bf16, fp16).  Products of codes and scales are exact, sums f32 in an order that follows
 * M, N, K, the format and y_dtype only, one rounding at the end.  But for e4m3 with a bf16 y: the matrix cores
 * then add eight neighbouring products at a time and cut each below 2^-13 of the largest, so that up to 7 2^-13 of
 * the largest of every eight is lost, less than 2^-10 of sum |x w| and than half a rounding to bf16 of a result
 * that does not cancel; y_dtype f32 asks for f32 sums.  f32 and fp16 y of e4m3: values of x or w from 2^128 on are
 * infinite, and those below 2^-126 have the bits of bf16's subnormals.  Sizes that take more tiles than a launch
 * has (2^30 features, or results of some 100 GB) are MLXQ_EUNSUPPORTED.
 */
int mlxq_mx_matmul(const mlxq_mx* x, int64_t M, int64_t K, const mlxq_mx* w, int64_t N, const void* bias,
                   int bias_dtype, void* y, int y_dtype, void* stream);

/*
 * Root-mean-square norm over the last dimension of [T, heads, D]:
 *   h = x + residual (rounded to dtype and written to sum; without residual h = x and sum is NULL)
 *   y = h * (mean(h^2) + eps)^(-1/2) * weight            (weight [D] in weight_dtype, NULL: ones)
 * x, residual, sum and y have one dtype and any strides that are whole elements. Sums are f32, and y is
 * rounded once: a row whose squares add up past f32's range counts as infinite, and with eps 0 squares
 * below 2^-126 lose bits (rows from 1e-18 to 1e16 are in range at any D). Exactly one of y and y_mx is
 * given: y_mx (e4m3, rows T * heads of D, D a multiple of 32) is what mlxq_mx_quantize would make of the
 * exact norm, which is taken in 64 bits wherever it matters, so that no code depends on the order of a
 * sum. sum may be x or residual (same strides), y may be x; otherwise nothing may overlap. D up to 32768.
 */
int mlxq_rms_norm(const mlxq_heads* x, int dtype, int64_t T, int64_t D, const mlxq_heads* residual,
                  const mlxq_heads* sum, const void* weight, int weight_dtype, float eps,
                  const mlxq_heads* y, const mlxq_mx* y_mx, void* stream);

/*
 * Its gradient.  With r = (mean(x^2) + eps)^(-1/2), n = x r and g = dy * weight:
 *   dx = r (g - n mean(g n)) + dsum,     dweight = sum over tokens and heads of dy n
 * x is what was normed (the sum, if there was a residual: dx is then the gradient of both), dsum (NULL =
 * none) the gradient that arrives at the sum from elsewhere. dweight [D] in weight_dtype, NULL when weight
 * is. f32 sums in a fixed order, each result rounded once, over the norm's range (and the sum of g x
 * within f32's). dx may be dy or dsum (same strides).
 * workspace: mlxq_rms_norm_backward_workspace_size() bytes, 16-byte aligned, whatever they hold.
 */
size_t mlxq_rms_norm_backward_workspace_size(int64_t T, int64_t heads, int64_t D, int dtype);
int mlxq_rms_norm_backward(const mlxq_heads* dy, const mlxq_heads* x, int dtype, int64_t T, int64_t D,
                           const void* weight, int weight_dtype, const mlxq_heads* dsum, float eps,
                           const mlxq_heads* dx, void* dweight, void* workspace, size_t workspace_bytes,
                           void* stream);

/* How a router chooses. */
typedef enum { MLXQ_ROUTE_SOFTMAX = 0, MLXQ_ROUTE_SIGMOID = 1 } mlxq_route_scoring;

typedef struct {
  int scoring;          /* mlxq_route_scoring: s = softmax(z) over all experts, or sigmoid(z) */
  int64_t top_k;        /* experts a token goes to, 1 to 64 */
  const float* bias;    /* [experts] or NULL: added to s for the choice only */
  int64_t groups;       /* equal runs of experts, 1 to 64; only those of the kept_groups best groups are chosen */
  int64_t kept_groups;  /* from */
  int64_t group_best;   /* a group counts as the sum of its 1 or 2 best experts */
  int normalize;        /* weights are divided by their sum */
  float scale;          /* and multiplied by this */
} mlxq_router;

/* Where tokens go: ids [tokens, top_k] and weights [tokens, top_k], and the plan of the experts' products:
 * rows lists the choices t * top_k + j in the order of their experts (those of one expert ascending), expert
 * e's from starts[e] up to starts[e + 1]; choices without an expert (an id outside [0, experts)) come last.
 * All device arrays, int32 but for the f32 weights. */
typedef struct {
  int32_t* ids;
  float* weights;
  int32_t* starts; /* [experts + 1] */
  int32_t* rows;   /* [tokens * top_k] */
  int64_t tokens, top_k, experts;
} mlxq_routing;

/*
 * Routes tokens by their logits [T, experts] (dtype, row_stride elements from row to row).  The top_k
 * experts with the largest s + bias (without a bias: the largest logits) among the kept groups, best first,
 * the lowest expert first among equal ones; weights are s of the chosen, normalized and scaled.  The choice
 * is made in 64 bits.  active (NULL = all): tokens whose byte is 0 get ids -1 and weights 0.
 * NaN logits come after all others of the kept groups.  Under softmax a row with a NaN or +infinity has no
 * scores: its logits alone choose (no bias, a group by its best) and its weights are NaN.  Where the chosen
 * scores sum to 0 in 64 bits (all -infinity, or some 709 below 0 or 745 below the row's largest) the weights are 0.
 * top_k is at most kept_groups * (experts / groups).  experts up to 1024, tokens * top_k below 2^31 - 2^20.
 * workspace: mlxq_route_workspace_size() bytes, 16-byte aligned, whatever they hold.
 */
size_t mlxq_route_workspace_size(int64_t choices, int64_t experts);
int mlxq_route_experts(const void* logits, int dtype, int64_t row_stride, const mlxq_router* router,
                       const uint8_t* active, const mlxq_routing* out, void* workspace,
                       size_t workspace_bytes, void* stream);

/* starts and rows for given ids (of out; its weights are not read). */
int mlxq_route_plan(const mlxq_routing* out, void* workspace, size_t workspace_bytes, void* stream);

/*
 * The gradient of the logits from that of the weights, dweights [tokens, top_k] f32, for the choice that
 * ids holds (ids outside [0, experts) pass nothing on; no expert twice in a row): dlogits [tokens, experts]
 * contiguous, in dtype.  f32 arithmetic; normalized weights by their shares, so that scores may be of any size, and
 * where the weights are 0 the gradient is.  A token without an expert has a gradient of 0 whatever its logits
 * hold; under softmax another row with a NaN or +infinity has NaN.  Of router, scoring, normalize and scale are read.
 */
int mlxq_route_experts_backward(const float* dweights, const void* logits, int dtype, int64_t row_stride,
                                const mlxq_router* router, const mlxq_routing* routing, void* dlogits,
                                void* stream);

/*
 * The products of the experts that tokens were routed to: y[t, j] = x[t] . w[ids[t, j]]^T + bias[ids[t,
 * j]] with w [experts, N, K] e2m1 (one stack of experts * N rows), bias [experts, N] in bias_dtype or
 * NULL, x [tokens, K], or with x_per_choice [tokens, top_k, K]. y is [tokens, top_k, N] in y_dtype, zero
 * for choices without an expert; with combine it is [tokens, N], sum_j weights[t, j] y[t, j]: each product
 * is rounded to y_dtype first, as separate products would be (fp16: past 65504 infinite), and the sum is
 * f32 and rounded again; y_dtype f32 keeps the products in f32. Sums and sizes otherwise as
 * mlxq_mx_matmul's. starts and rows must be ids' plan; entries outside their ranges are skipped.
 * workspace: mlxq_mx_experts_workspace_size() bytes, 16-byte aligned, whatever they hold (NULL when that
 * is 0: without combine).
 */
size_t mlxq_mx_experts_workspace_size(int64_t tokens, int64_t top_k, int64_t N, int combine, int y_dtype);
int mlxq_mx_experts(const mlxq_mx* x, int x_per_choice, int64_t K, const mlxq_mx* w, int64_t N,
                    const void* bias, int bias_dtype, const mlxq_routing* routing, int combine, void* y,
                    int y_dtype, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Host-side shape helper — replaces quant::packed_bits (src/quant.rs:38-41): from the packed
 * shapes infer bits = wq_cols*32 / (scales_cols*group_size).  Returns 4 or 8, or -1 (with
 * mlxq_last_error set) for a malformed triple instead of panicking.
 */
int mlxq_packed_bits(int64_t wq_cols, int64_t scales_cols, int group_size);

#ifdef __cplusplus
}
#endif

#endif /* MLXQ_H */
