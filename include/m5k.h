/*
 * m5k.h -- C ABI of libm5k.so, the MI355X (gfx950) quantized-projection hot path.
 *
 * Every entry point takes device pointers to row-major, contiguous buffers,
 * 64-bit sizes and an opaque HIP stream (hipStream_t passed as void*; NULL is
 * the default stream). Launches are asynchronous on that stream. Inputs are
 * never written, but for the caches that m5k_paged_append fills; the attention
 * entries take rows by strides. The library never allocates device memory: the caller owns
 * every buffer, outputs included.
 *
 * Return value: 0 on success; a nonzero M5K_E* code otherwise, with a
 * human-readable message available from m5k_last_error() on the calling
 * thread. Argument checks here cover only what the kernels rely on for memory
 * safety and launch validity; the Python layer reproduces the reference's
 * ValueError / NotImplementedError contract before calling in.
 *
 * Reference interfaces replaced (paths relative to the reference repository):
 *   quantize                 src/m5kernels/metal.py:27-44 (int8, fp8, mxint8)
 *   gemm                     src/m5kernels/metal.py:158-269
 *   rotate                   src/m5kernels/hadamard.py:33-77
 *   fused_norm_hadamard_quantize
 *                            src/m5kernels/norm_hadamard.py:122-176
 *   fused_gated_residual_norm_hadamard_quantize
 *                            src/m5kernels/norm_hadamard.py:198-265
 *   gated_residual_add       src/m5kernels/norm_hadamard.py:280-300
 *   unfused_norm             src/m5kernels/norm_hadamard.py:321-348
 *   projection_qk_rope       src/m5kernels/qk_rope.py:120-182
 *   qk_norm_rope             src/m5kernels/qk_rope.py:185-203
 *   rms_quantize             src/m5kernels/rms_quant.py:41-117
 *   grouped QKV projection   integrations/h3/qkv_candidate.metal:1-20
 *   shift-split conditioning src/m5kernels/norm_hadamard_gemm.py:233-247,459-460
 */
#ifndef M5K_H
#define M5K_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element type codes. */
#define M5K_F32 0
#define M5K_F16 1
#define M5K_BF16 2
#define M5K_I8 3
#define M5K_U8 4
#define M5K_I32 5

/* Quantization modes. */
#define M5K_QUANT_INT8 0 /* symmetric [-127,127], scale = peak/127 */
#define M5K_QUANT_FP8 1  /* OCP E4M3 codes in uint8, scale = peak/448 */

/* Normalization kinds for the fused prep. */
/* Prep parameter-table dtypes (param_dtype of m5k_norm_hadamard_quantize and m5k_norm_modulate):
 * one float dtype code for every table, or one code per table packed by M5K_PARAM_TABLES (the
 * gate field is ignored by calls without a gate). */
#define M5K_PARAM_PER_TABLE 0x100
#define M5K_PARAM_TABLES(gamma, scale, shift, gate) \
  (M5K_PARAM_PER_TABLE | (gamma) | ((scale) << 2) | ((shift) << 4) | ((gate) << 6))

#define M5K_NORM_RMS 0
#define M5K_NORM_LAYER 1

/* Status codes. */
#define M5K_OK 0
#define M5K_EINVAL 1  /* argument outside what the kernels support */
#define M5K_ELAUNCH 2 /* HIP launch or runtime error */

/* Message for the last failure on this thread ("" if none). */
const char* m5k_last_error(void);

/* ABI version (major*100 + minor).  Entries are added under the same number; what an argument was documented to mean
 * stays.  m5k_attention_plan once took any `paged` other than 0 for a paged call: it takes 1 for it now, as it was
 * documented, gives 2 and 4 (plus 8, 16) their own meaning, and refuses the rest. */
#define M5K_ABI_VERSION 100
int m5k_abi_version(void);

/*
 * Per-row symmetric quantizer.  Replaces metal.quantize(x, mode) for modes
 * "int8" and "fp8" (src/m5kernels/metal.py:27-44, shaders/quantize.metal:1-38).
 * x: [rows,k] of x_dtype (F32/F16/BF16).  q: [rows,k] int8 (INT8) or uint8
 * E4M3 codes (FP8).  scales: [rows] float32.
 * peak = max|x|; scale = peak==0 ? 1 : peak/127 (or /448), IEEE fp32 division;
 * INT8 code = clamp(rint_even(x/scale), -127, 127); FP8 code = nearest E4M3
 * (ties to even, saturating at 448, sign from the sign bit).
 */
int m5k_quantize_rows(const void* x, int x_dtype, int64_t rows, int64_t k, int mode,
                      void* q, float* scales, void* stream);

/*
 * MXINT8 block quantizer.  Replaces metal.quantize(x, "mxint8") (src/m5kernels/metal.py:27-44,
 * block mode of shaders/quantize.metal:13-37; spec numerics.py:33-41).  x: [rows,k] F32/F16/BF16
 * with k % 32 == 0.  Per 32-element block: e = 0 for an all-zero block, else
 * clamp(floor(log2(peak)) - 6, -127, 127) with log2 rounded to FP32 before the floor;
 * q = clamp(rint(x / 2^e), -127, 127) int8 [rows,k]; exponents[rows, k/32] = e + 127 (uint8,
 * the E8M0 scale byte of the OCP S1.6 convention with the /64 folded in).
 */
int m5k_quantize_mxint8(const void* x, int x_dtype, int64_t rows, int64_t k, int8_t* q,
                        uint8_t* exponents, void* stream);

/*
 * MXINT8 codes to BF16 values q * 2^(exponent - 127), exact.  Operand expansion for the MXINT8
 * linear (metal.gemm(..., "mxint8", ...), src/m5kernels/metal.py:81-86, plane scales of
 * 32 x 1 blocks): y[rows,k] BF16, 16-byte aligned; q 8-byte aligned; k % 32 == 0.
 */
int m5k_mxint8_to_bf16(const int8_t* q, const uint8_t* exponents, int64_t rows, int64_t k, void* y,
                       void* stream);

/* The same for both operands of a product, codes a [m,k] and b [n,k], in one launch. */
int m5k_mxint8_pair_to_bf16(const int8_t* qa, const uint8_t* ea, int64_t m, const int8_t* qb, const uint8_t* eb,
                            int64_t n, int64_t k, void* ya, void* yb, void* stream);

/*
 * W8A8 linear.  Replaces metal.gemm(a, b, "int8", ...) (src/m5kernels/metal.py:158-269,
 * epilogues :88-128).  a: [m,k] int8, b: [n,k] int8 (weights, K-contiguous).
 * c[m,n] = O(float(sum_k a*b) * a_scales[m] * b_scales[n] [+ bias]) with int32
 * accumulation and the FP32 products evaluated left to right; O = c_dtype
 * (F32/F16/BF16, round to nearest even).
 * bias (optional, may be NULL): float32 [n], or [P,n] selected by
 *   bias_row_map[m] (int32) when bias_row_map is non-NULL.
 * residual/gate (optional, both or neither; excludes bias; c_dtype must be BF16):
 *   residual bf16 [m,n], gate bf16 [n] or [P,n] with gate_row_map[m];
 *   c = bf16(float(residual) + float(bf16(branch)) * float(gate)).
 */
int m5k_gemm_i8(const int8_t* a, const int8_t* b, int64_t m, int64_t n, int64_t k,
                const float* a_scales, const float* b_scales, void* c, int c_dtype,
                const float* bias, const int32_t* bias_row_map,
                const void* residual, const void* gate, const int32_t* gate_row_map,
                void* stream);

/*
 * The same W8A8 linear as m5k_gemm_i8 for short M: each output tile may be split over up to
 * `splits` contiguous ranges of K (1..64).  The library takes the tile and the number of ranges
 * that it expects to be fastest (m5k_gemm_split_plan reports them; m5k_gemm_set_exact_splits makes
 * it run `splits`); with one range it is m5k_gemm_i8's launch and the workspace stays untouched.
 * Otherwise the raw INT32 partial tiles go to workspace[splits][m][n] (int32, caller-owned, at
 * least splits*m*n elements), and a second kernel sums them in split order and applies the
 * identical epilogue.  INT32 sums are exact, so c is bit-identical to m5k_gemm_i8's.  Needs
 * k % 16 == 0 and 16-byte aligned a/b (any operand size).  Same contract as
 * metal.gemm(a, b, "int8", ...) (src/m5kernels/metal.py:158-269); the split is this library's
 * schedule for outputs whose tiles leave CUs idle (few rows, or few columns).
 */
int m5k_gemm_i8_splitk(const int8_t* a, const int8_t* b, int64_t m, int64_t n, int64_t k,
                       const float* a_scales, const float* b_scales, void* c, int c_dtype,
                       const float* bias, const int32_t* bias_row_map, const void* residual,
                       const void* gate, const int32_t* gate_row_map, int splits, int32_t* workspace,
                       int64_t workspace_elems, void* stream);

/*
 * m5k_gemm_i8_splitk without the caller's workspace: the INT32 partials go to a scratch array
 * of the library (M5K_SCRATCH_ELEMS int32 = 64 MiB per GPU, a static device array held until
 * the process ends), so the call allocates nothing -- no hipMalloc, no hipFree, no allocating
 * library routine.  No counterpart in the reference: it is for callers that cannot allocate
 * (HIP graph capture, tight serving loops, harnesses that forbid allocation).
 * splits * m * n must not exceed M5K_SCRATCH_ELEMS (M5K_EINVAL otherwise).  The array used is
 * the one on the device of `stream` (the current device for the null stream); its address is
 * looked up once per device, the first call on that device.  Every call on one GPU shares that
 * GPU's array: calls that overlap on one GPU (other streams, other host threads) race.  Results
 * are bit-identical to m5k_gemm_i8_splitk and m5k_gemm_i8.
 */
#define M5K_SCRATCH_ELEMS (16 * 1024 * 1024)
int m5k_gemm_i8_splitk_noalloc(const int8_t* a, const int8_t* b, int64_t m, int64_t n, int64_t k,
                               const float* a_scales, const float* b_scales, void* c, int c_dtype,
                               const float* bias, const int32_t* bias_row_map, const void* residual,
                               const void* gate, const int32_t* gate_row_map, int splits, void* stream);

/*
 * Launch plan of the MFMA GEMMs (host only, launches nothing).  No counterpart in the
 * reference; it lets a host scheduler compose with the library's own choice.  For an
 * [m,n] output with operands of ab_dtype (M5K_I8, M5K_U8 for FP8 codes, M5K_BF16, M5K_F16,
 * M5K_F32) on a device of `cus` compute units, *schedule receives
 *   0  plain: 256 x 256 tiles;
 *   1  mixed: the leading *full_tiles 256 x 256 tiles (whole rounds), every other tile as
 *      two 256 x 128 halves in the same launch;
 *   2  narrow: 256 x 224 tiles (I8 / BF16 / F16 only);
 *   3  quad: 256 x 256 tiles on four waves of 128 x 128 (I8 only; only when forced, below);
 * and *full_tiles is -1 unless the schedule is 1.  Every m5k_gemm_* entry point makes this
 * choice with the device's CU count for operands on the direct-to-LDS path (row bytes a
 * multiple of 16, 16-byte aligned bases) whose tile is 0 in m5k_gemm_tile_plan.  Results are
 * bit-identical under every schedule.  M5K_GEMM_MIXED_TILES=0 / M5K_GEMM_NARROW_TILES=0 in
 * the environment switch schedule 1 / 2 off.
 */
int m5k_gemm_launch_plan(int ab_dtype, int64_t m, int64_t n, int cus, int* schedule, int64_t* full_tiles);

/*
 * Force the schedule of the MFMA GEMM launches made by the calling host thread: -1 restores the
 * library's own plan (m5k_gemm_launch_plan), 0 plain, 1 mixed, 2 narrow (plain for FP8/FP32),
 * 3 quad (plain for all but I8; never the library's own choice, as it measured slower).
 * *previous (may be NULL) receives the thread's earlier setting.  No counterpart in the
 * reference, whose tuner searches Metal threadgroup tiles through gemm's `tile` argument
 * (src/m5kernels/cli.py:66-151); this is the gfx950 knob the harness tuner searches instead.
 * The setting is thread-local, so other host threads keep their own plan; for tools outside the
 * process, M5K_GEMM_SCHEDULE=plain|mixed|narrow|quad in the environment does the same when no thread
 * setting is made.  Results are bit-identical under every schedule.  Under a forced schedule aligned
 * operands run that schedule's 256-row tiles whatever m5k_gemm_tile_plan would choose.
 */
int m5k_gemm_set_schedule(int schedule, int* previous);

/*
 * What decides the calling thread's schedules besides the shape, as one value (a key for host-side
 * plan caches; no counterpart in the reference): bits 0-2 the thread's forced schedule + 1, bit 3 a
 * schedule in M5K_GEMM_SCHEDULE, bits 4 and 5 M5K_GEMM_MIXED_TILES=0 and M5K_GEMM_NARROW_TILES=0,
 * bit 6 the thread's exact K ranges (m5k_gemm_set_exact_splits).
 */
int m5k_gemm_schedule_state(void);

/*
 * Tile of the MFMA GEMMs for an [m,n,k] product (host only, launches nothing; no counterpart in the
 * reference).  `aligned`: row bytes a multiple of 16 and at most 2^23, 16-byte aligned bases.  *tile
 * receives
 *   0  the 256-row schedules of m5k_gemm_launch_plan;
 *   1  128 x 128 tiles, K over two groups of waves;
 *   2  64 x 64 tiles, two workgroups per CU, K over two groups of waves;
 *   3  64 x 64 tiles with longer stages, the same sums;
 *   4  16 columns per workgroup, K over eight waves (m <= 32).
 * INT8 results are bit-identical under every tile.  Float results (FP32 sums) are the same bits for
 * tiles 1 to 3, and for tile 0 under every schedule; between these groups and tile 4 the order of the
 * sum differs.  Aligned float rows of under 1 KiB always take tile 0.  Unaligned I8 rows of at most
 * 128 bytes run on 256 x 256 tiles where the tile reported here would take several rounds longer.
 * max_splits (1..64, more than 1 for I8 and U8 only) offers K ranges of tiles 1 to 3 too; *splits
 * receives how many the choice takes (1: no partial sums; tiles 0 and 4 always).  K ranges of
 * 256-row tiles are not weighed here: m5k_gemm_split_plan has the split entry points' whole choice.
 */
int m5k_gemm_tile_plan(int ab_dtype, int64_t m, int64_t n, int64_t k, int cus, int aligned, int max_splits, int* tile,
                       int* splits);

/*
 * What a split entry point (m5k_gemm_i8_splitk[_noalloc]: I8; m5k_gemm_f8_splitk: U8) launches on a
 * device of `cus` compute units for `splits` (1..64), under the calling thread's settings (host only,
 * launches nothing; no counterpart in the reference).  *ranges receives the K ranges that run; 1: the
 * unsplit launch, which leaves the workspace alone.  *tile receives the tile as in m5k_gemm_tile_plan,
 * with 5 for 256 x 128 tiles; tile 0 with ranges above 1 is 256 x 256.
 */
int m5k_gemm_split_plan(int ab_dtype, int64_t m, int64_t n, int64_t k, int cus, int splits, int* tile, int* ranges);

/*
 * Whether the split entry points of the calling host thread run exactly the K ranges that a call names
 * (on != 0; fewer only where a range would be empty), or up to as many as the library expects to pay
 * (0, the default).  A forced schedule (m5k_gemm_set_schedule) does the same, on its 256-row tiles.
 * *previous (may be NULL) receives the earlier setting.  No counterpart in the reference: the harness
 * tuner times split counts through it, and tests run each split kernel.
 */
int m5k_gemm_set_exact_splits(int on, int* previous);

/*
 * Raw INT32 accumulators of the W8A8 GEMM (test hook for bit-exact parity):
 * acc[m,n] = sum_k a[m,k]*b[n,k].  Same kernel main loop as m5k_gemm_i8.
 */
int m5k_gemm_i8_acc(const int8_t* a, const int8_t* b, int64_t m, int64_t n, int64_t k,
                    int32_t* acc, void* stream);

/*
 * FP8 E4M3 linear with FP32 accumulation.  Replaces metal.gemm(a, b, "fp8", ...)
 * (src/m5kernels/metal.py:75-80,191-194).  a: [m,k], b: [n,k] uint8 E4M3 codes;
 * k % 128 == 0.  c = O(acc * a_scales[m] * b_scales[n]).
 */
int m5k_gemm_f8(const uint8_t* a, const uint8_t* b, int64_t m, int64_t n, int64_t k,
                const float* a_scales, const float* b_scales, void* c, int c_dtype,
                void* stream);

/*
 * Split-K FP8 linear for short M: the same contract as m5k_gemm_f8 (metal.gemm(a, b, "fp8", ...),
 * src/m5kernels/metal.py:75-80,191-194), computed as `splits` K ranges per output tile into
 * FP32 partials workspace[splits][m][n] (workspace_elems >= splits*m*n floats, caller-owned),
 * summed in split order before the scale epilogue.  Deterministic; its FP32 sums may differ
 * from m5k_gemm_f8's in the last bits (FP8 accumulation order is not pinned).  splits in
 * [1, 64]; operands 16-byte aligned.
 */
int m5k_gemm_f8_splitk(const uint8_t* a, const uint8_t* b, int64_t m, int64_t n, int64_t k,
                       const float* a_scales, const float* b_scales, void* c, int c_dtype, int splits,
                       float* workspace, int64_t workspace_elems, void* stream);

/*
 * Floating GEMM with FP32 accumulation.  Replaces metal.gemm(a, b, "bf16"|"fp16", ...)
 * (src/m5kernels/metal.py:59-74,101-107).  a: [m,k], b: [n,k] of ab_dtype (BF16/F16).
 * c = O(acc).  Optional gated residual epilogue as for m5k_gemm_i8 (BF16 only).
 */
int m5k_gemm_float(const void* a, const void* b, int ab_dtype, int64_t m, int64_t n, int64_t k,
                   void* c, int c_dtype, const void* residual, const void* gate,
                   const int32_t* gate_row_map, void* stream);

/*
 * Signed block-Hadamard rotation  Y = (X * signs) H_B, FP32 output.
 * Replaces hadamard.rotate (src/m5kernels/hadamard.py:33-77, shaders/hadamard.metal:1-26).
 * x: [rows,k] of x_dtype, signs: int8 [k] (+-1), block in {32,...,1024}, k % block == 0.
 * Natural-order Sylvester butterflies in FP32, then one multiply by the FP32
 * constant 1/sqrt(block).
 */
int m5k_hadamard_rotate(const void* x, int x_dtype, int64_t rows, int64_t k, int block,
                        const int8_t* signs, float* y, void* stream);

/*
 * Fused rotation + per-row INT8 quantization: the codes and scales of
 * quantize(rotate(x, block, signs), "int8") without materializing the FP32
 * rotation (the online composition of src/m5kernels/hadamard_gemm.py:27-69).
 */
int m5k_hadamard_quantize_rows(const void* x, int x_dtype, int64_t rows, int64_t k, int block,
                               const int8_t* signs, int8_t* q, float* scales, void* stream);

/*
 * Fused row preparation (one dispatch): [gated residual update] -> RMS or LayerNorm ->
 * modulation -> O cast -> signs -> block Hadamard -> per-row INT8.
 * Replaces norm_hadamard.fused_norm_hadamard_quantize (branch == NULL) and
 * fused_gated_residual_norm_hadamard_quantize (src/m5kernels/norm_hadamard.py:122-265,
 * shaders/norm_hadamard.metal:1-121).
 *   x: [rows,k] of x_dtype (the residual when gated); k % block == 0.
 *   gated: branch [rows,k] of branch_dtype (BF16, F16 or F32, independent of x_dtype, read as
 *          is), gate [k] or [P,k] with gate_row_map[rows]; residual_out[rows,k] (x_dtype)
 *          receives R(x + branch*gate), written once.  branch_dtype is ignored when branch is
 *          NULL.
 *   gamma [k]; scale/shift [k], or [P,k] tables selected by row_map[rows]; param_dtype gives
 *   the tables' dtypes: one float code for all, or M5K_PARAM_TABLES(gamma, scale, shift,
 *   gate).  signs int8 [k].
 *   norm: M5K_NORM_RMS / M5K_NORM_LAYER; round_to_input: 1 rounds the modulated value to
 *   x_dtype before the signs (round_output="input"), 0 keeps FP32.
 *   Outputs: q int8 [rows,k], scales float32 [rows].
 */
int m5k_norm_hadamard_quantize(const void* x, int x_dtype, int64_t rows, int64_t k, const void* branch,
                               int branch_dtype, const void* gate, const int32_t* gate_row_map,
                               const void* gamma,
                               const void* scale, const void* shift, int param_dtype,
                               const int32_t* row_map, const int8_t* signs, int block, int norm,
                               float epsilon, int round_to_input, int8_t* q, float* scales,
                               void* residual_out, void* stream);

/*
 * Staged norm + modulation with the fused kernel's arithmetic and reduction tree.
 * Replaces norm_hadamard.unfused_norm (src/m5kernels/norm_hadamard.py:321-348,
 * shaders/norm_modulate.metal:1-37).  y: [rows,k] of x_dtype (round_to_input=1) or F32.
 */
int m5k_norm_modulate(const void* x, int x_dtype, int64_t rows, int64_t k, const void* gamma,
                      const void* scale, const void* shift, int param_dtype, const int32_t* row_map,
                      int norm, float epsilon, int round_to_input, void* y, void* stream);

/*
 * Staged gated residual update out = R(float(residual) + float(branch) * float(gate)).
 * Replaces norm_hadamard.gated_residual_add (src/m5kernels/norm_hadamard.py:280-300,
 * shaders/gated_residual.metal:1-9).  gate [k] or [P,k] of gate_dtype with gate_row_map[rows];
 * branch of branch_dtype; both BF16, F16 or F32, independent of the residual dtype.
 */
int m5k_gated_residual_add(const void* residual, int dtype, int64_t rows, int64_t k, const void* branch,
                           int branch_dtype, const void* gate, int gate_dtype, const int32_t* gate_row_map,
                           void* out, void* stream);

/*
 * Q or K projection + per-head RMSNorm + split-half RoPE, head-major BF16 output.
 * Replaces qk_rope.projection_qk_rope (src/m5kernels/qk_rope.py:120-182,
 * shaders/qk_rope_projection.metal:1-39, shaders/qk_rope_body.metal:1-20).
 *   a [m,k], b [n,k] of ab_dtype: M5K_I8 (with float32 a_scales[m], b_scales[n]; k <= 131071)
 *   or M5K_BF16 (scales NULL); n % 128 == 0.  gamma bf16 [128]; cos, sin bf16 [m, rope_half],
 *   0 <= rope_half <= 64.  y bf16 [n/128, m, 128].
 *   z = bf16(projection); inv = 1/sqrt(sum(z^2)/128 + eps); u = z*inv*gamma;
 *   y[d] = u[d]*c - u[d+R]*s (d < R), u[d]*c + u[d-R]*s (R <= d < 2R), u[d] otherwise.
 */
int m5k_projection_qk_rope(const void* a, const void* b, int ab_dtype, int64_t m, int64_t n, int64_t k,
                           const float* a_scales, const float* b_scales, const void* gamma, const void* cos,
                           const void* sin, int rope_half, float epsilon, void* y, void* stream);

/*
 * Staged postprocess of a BF16 [m,n] projection with the fused kernel's per-(row, head) code.
 * Replaces qk_rope.qk_norm_rope (src/m5kernels/qk_rope.py:185-203, shaders/qk_rope_norm.metal).
 */
int m5k_qk_norm_rope(const void* projected, int64_t m, int64_t n, const void* gamma, const void* cos,
                     const void* sin, int rope_half, float epsilon, void* y, void* stream);

/*
 * The same for a BF16 projection in the grouped layout of m5k_projection_qkv_rope, [m, heads*3*128]:
 * Q and K blocks are normalized and rotated, V blocks copied, to [heads, m, 128] each (16-byte aligned).
 */
int m5k_qkv_norm_rope(const void* projected, int64_t m, int64_t heads, const void* q_gamma, const void* k_gamma,
                      const void* cos, const void* sin, int rope_half, float epsilon, void* q_out, void* k_out,
                      void* v_out, void* stream);

/*
 * Grouped Q/K/V projection in the H3 runtime's native layout
 * (integrations/h3/qkv_candidate.metal:5-81, reference math qkv_reference.h:15-35).
 * b: [heads*3*128, k] weight rows ordered [head][stream Q,K,V][channel]; a: [m,k] (INT8
 * with a_scales/b_scales, or BF16).  Every 128-column block is rounded to BF16 as in
 * m5k_projection_qk_rope; Q blocks then take q_gamma and K blocks k_gamma through the same
 * per-head RMSNorm + split-half RoPE (cos/sin [m, rope_half]); V blocks are the rounded
 * projection.  q_out, k_out, v_out: BF16 [heads, m, 128], 16-byte aligned.
 */
int m5k_projection_qkv_rope(const void* a, const void* b, int ab_dtype, int64_t m, int64_t heads,
                            int64_t k, const float* a_scales, const float* b_scales,
                            const void* q_gamma, const void* k_gamma, const void* cos,
                            const void* sin, int rope_half, float epsilon, void* q_out,
                            void* k_out, void* v_out, void* stream);

/*
 * RMS dynamic INT8 quantization with the inverse RMS folded into the row scales.  Replaces
 * rms_quant.rms_quantize (src/m5kernels/rms_quant.py:41-117, shaders/rms_quant.metal:1-97).
 * x: [rows,k] F32/F16/BF16; gamma: FP32 [k]; signs: int8 +-1 [k]; block 1 (no transform, any
 * k) or a power of two in [32,1024] dividing k.  ss = sum x^2, inv = 1/sqrt(ss/k + eps);
 * v = fold ? (x*gamma)*s : ((x*inv)*gamma)*s; z = blockdiag(H_B) v; peak = max|z|;
 * scales[row] = peak == 0 ? 1 : (peak * (fold ? inv : 1)) / 127;
 * q = peak == 0 ? 0 : clamp(rint((z/peak)*127), -127, 127) int8 [rows,k].
 */
int m5k_rms_quantize(const void* x, int x_dtype, int64_t rows, int64_t k, const float* gamma,
                     const int8_t* signs, int block, int fold_scale, float epsilon, int8_t* q,
                     float* scales, void* stream);

/*
 * Conditioning tables of the shift-split projection.  Replaces condition_prepare and
 * bias_prepare of the norm-shift-split backend (src/m5kernels/norm_hadamard_gemm.py:233-247,
 * 459-460).  gamma: [k]; scale, shift: [p_rows,k] (param_dtype and operand_dtype
 * respectively; F32/F16/BF16); w: [n,k] original projection weights (operand_dtype).
 * combined[p,j] = float(gamma[j]) * (1 + float(scale[p,j]))  FP32 [p_rows,k];
 * bias[p,n] = sum_j float(shift[p,j]) * float(w[n,j])       FP32 [p_rows,n] (FP32
 * accumulation; p_rows <= 8 one pass over w, more rows on the MFMA GEMM of m5k_gemm_float).
 * The online projection is m5k_rms_quantize(x, combined[p], fold) followed by m5k_gemm_i8 with
 * bias[p].
 */
int m5k_shift_split_condition(const void* gamma, const void* scale, int param_dtype,
                              const void* shift, const void* w, int operand_dtype, int64_t p_rows,
                              int64_t k, int64_t n, float* combined, float* bias, void* stream);

/*
 * Attention behind the Q/K/V projections.  out[token, head * head_dim] = softmax over the visible keys of
 * scale * q . k (FP32 statistics, probabilities rounded to `dtype` for the second product) times v; query
 * head h reads key head h / (heads / kv_heads).  dtype M5K_BF16 or M5K_F16, head_dim 64 or 128.  q
 * [heads, tokens, head_dim] and k, v [kv_heads, keys, head_dim] by strides in elements (multiples of 8, rows
 * contiguous, bases 16-byte aligned); out [tokens, heads * head_dim] contiguous.
 *   Row i stands at key position p = i + keys - tokens.  Scores: softcap > 0 replaces s by
 *   softcap * tanh(s / softcap); slopes (float32 [heads]) then adds -slopes[h] * |p - j|.
 *   Mask: causal keeps j <= p (and j below the document's first key + prefix_lengths[document]); window > 0
 *   keeps p - j < window, and j - p < window without causal; document_starts (int32 [documents + 1],
 *   nondecreasing from 0; needs keys == tokens) keeps the row's own document.  A row that sees no key is 0;
 *   so is a row behind the last document.  What a masked key or value holds does not matter, NaN included.
 *   Scores are FP32 numbers of any size; a row that sees only keys of score -infinity is NaN.
 *   Infinities and NaN in values that a row sees are in its output, however small their weight.  Sums of weights, up to
 *   2^8, times values are FP32 numbers: values up to 2^119 over the number of keys.
 *   scale and a softcap other than 0 are normal FP32 numbers, scale / softcap at most 1e37.
 *   prefix_lengths: int32 [documents], or [1] without document_starts; only with causal, not with window.
 *   splits: key ranges joined by a second launch (m5k_attention_plan gives the number that pays); above 1
 *   workspace holds splits * tokens * heads * (head_dim + 2) floats that the call may overwrite.
 */
int m5k_attention(const void* q, int dtype, int64_t tokens, int64_t heads, int head_dim, int64_t q_head,
                  int64_t q_token, const void* k, int64_t k_head, int64_t k_key, const void* v, int64_t v_head,
                  int64_t v_key, int64_t keys, int64_t kv_heads, float scale, int causal, int64_t window,
                  float softcap, const float* slopes, const int32_t* document_starts, int64_t documents,
                  const int32_t* prefix_lengths, void* out, int splits, float* workspace, int64_t workspace_elems,
                  void* stream);

/*
 * m5k_attention with a window (above 0) of which the first `sinks` keys of the row's document stay visible: of the keys
 * that the other masks leave, those with p - j < window (and j - p < window without causal), and those below the
 * document's first key + sinks.  sinks 0: m5k_attention.  The plan's keys: at most window (twice it without causal)
 * + sinks + 64.
 */
int m5k_attention_sinks(const void* q, int dtype, int64_t tokens, int64_t heads, int head_dim, int64_t q_head,
                        int64_t q_token, const void* k, int64_t k_head, int64_t k_key, const void* v, int64_t v_head,
                        int64_t v_key, int64_t keys, int64_t kv_heads, float scale, int causal, int64_t window,
                        int64_t sinks, float softcap, const float* slopes, const int32_t* document_starts,
                        int64_t documents, const int32_t* prefix_lengths, void* out, int splits, float* workspace,
                        int64_t workspace_elems, void* stream);

/* The plan of m5k_attention (paged 0, sequences = documents), m5k_paged_attention (paged 1,
 * keys = table_width * page_size) or m5k_paged_attention_codes (paged 2 for FP8 codes or 4 for INT8, plus 8 with
 * head_dim 128, plus 16 with a softcap or slopes) on `cus` compute units (host only; cus <= 0: those of the current
 * device): the key splits that pay, and whether the waves of a workgroup share 32 rows (few 1) or take 32 each (few 0;
 * few may be NULL). */
int m5k_attention_plan(int paged, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t sequences, int64_t keys,
                       int cus, int* splits, int* few);

/*
 * Attention of new tokens over a paged cache: k_cache, v_cache [pages, kv_heads, page_size, head_dim] by
 * strides; page_table int32 [sequences, table_width].  Sequence b's new tokens are rows
 * [query_starts[b], query_starts[b + 1]) of q and out (query_starts int32 [sequences + 1], nondecreasing from 0)
 * and the last of the context_lengths[b] keys of its cache (int32 [sequences], new tokens included, at most
 * table_width * page_size): the mask is causal on those positions, the other arguments are m5k_attention's, with
 * prefix_lengths int32 [sequences].  Rows behind the last sequence, and of a sequence whose context is empty,
 * are 0.  A table entry outside [0, pages) names no page; its keys are left out.  page_size is any number.
 */
int m5k_paged_attention(const void* q, int dtype, int64_t tokens, int64_t heads, int head_dim, int64_t q_head,
                        int64_t q_token, const void* k_cache, int64_t k_page, int64_t k_head, int64_t k_slot,
                        const void* v_cache, int64_t v_page, int64_t v_head, int64_t v_slot, int64_t pages,
                        int64_t page_size, int64_t kv_heads, const int32_t* page_table, int64_t table_width,
                        int64_t sequences, const int32_t* query_starts, const int32_t* context_lengths, float scale,
                        int64_t window, float softcap, const float* slopes, const int32_t* prefix_lengths, void* out,
                        int splits, float* workspace, int64_t workspace_elems, void* stream);

/* m5k_paged_attention with a window of which the first `sinks` keys of each sequence stay visible (as in
 * m5k_attention_sinks). */
int m5k_paged_attention_sinks(const void* q, int dtype, int64_t tokens, int64_t heads, int head_dim, int64_t q_head,
                              int64_t q_token, const void* k_cache, int64_t k_page, int64_t k_head, int64_t k_slot,
                              const void* v_cache, int64_t v_page, int64_t v_head, int64_t v_slot, int64_t pages,
                              int64_t page_size, int64_t kv_heads, const int32_t* page_table, int64_t table_width,
                              int64_t sequences, const int32_t* query_starts, const int32_t* context_lengths,
                              float scale, int64_t window, int64_t sinks, float softcap, const float* slopes,
                              const int32_t* prefix_lengths, void* out, int splits, float* workspace,
                              int64_t workspace_elems, void* stream);

/*
 * A cache in 8 bits.  Codes [pages, kv_heads, page_size, head_dim], E4M3 (mode M5K_QUANT_FP8) or INT8 in [-127, 127]
 * (M5K_QUANT_INT8), by strides in bytes; exponents [pages, kv_heads, page_size / block] bytes, the last axis
 * contiguous, ke_page and ke_head apart.  A code of a block of `block` tokens (a multiple of 16 that divides
 * page_size) and head stands for code * 2^(exponent - 127); under exponent 255 every code is NaN.
 *
 * m5k_paged_attention_codes: m5k_paged_attention_sinks over such a cache, whose values are taken in q's dtype (exact in
 * BF16 down to its subnormals; in FP16 rounded; infinities above either's range).  Rows of codes are 16-byte aligned,
 * head_dim to 2^23 bytes apart.
 */
int m5k_paged_attention_codes(
    const void* q, int dtype, int64_t tokens, int64_t heads, int head_dim, int64_t q_head, int64_t q_token, int mode,
    const void* k_codes, int64_t k_page, int64_t k_head, int64_t k_slot, const uint8_t* k_exponents, int64_t ke_page,
    int64_t ke_head, const void* v_codes, int64_t v_page, int64_t v_head, int64_t v_slot, const uint8_t* v_exponents,
    int64_t ve_page, int64_t ve_head, int64_t block, int64_t pages, int64_t page_size, int64_t kv_heads,
    const int32_t* page_table, int64_t table_width, int64_t sequences, const int32_t* query_starts,
    const int32_t* context_lengths, float scale, int64_t window, int64_t sinks, float softcap, const float* slopes,
    const int32_t* prefix_lengths, void* out, int splits, float* workspace, int64_t workspace_elems, void* stream);

/*
 * Rotary positions: y = x with channel pairs of the first 2 * pairs channels turned by
 * a = positions[token] * frequencies[j] (float64 radians a position; the angle is reduced in 64 bits) and
 * scaled by `magnitude`: (x1 c - x2 s, x2 c + x1 s), pair j being channels (j, j + pairs), or
 * (2j, 2j + 1) with interleaved != 0; the other channels are copied.  x [heads, tokens, head_dim] of F32, F16 or
 * BF16 by strides in elements (channels contiguous), y [heads, tokens, head_dim] contiguous; positions int32.
 */
int m5k_rope(const void* x, int dtype, int64_t tokens, int64_t heads, int64_t head_dim, int64_t x_head,
             int64_t x_token, const int32_t* positions, const double* frequencies, int64_t pairs, int interleaved,
             float magnitude, void* y, void* stream);

/*
 * Append keys and values of new tokens to a paged cache (layout, page_table, query_starts and context_lengths as in
 * m5k_paged_attention): token i of sequence b goes to position context_lengths[b] - n + i, keys turned as in
 * m5k_rope when pairs > 0.  k, v [kv_heads, tokens, head_dim] and the caches by strides, dtype F16, BF16 or F32.
 * q (or NULL) [heads, tokens, head_dim] is turned too, into q_out [heads, tokens, head_dim] contiguous, whose rows
 * behind the last sequence become 0.  A token whose position is negative or lies behind the table, or whose table
 * entry is outside [0, pages), is not stored; nothing else in the cache is written.
 * Two tokens that name the same place leave a mixture there, each channel of each head one token's or the other's.
 */
int m5k_paged_append(const void* k, int64_t k_head, int64_t k_token, const void* v, int64_t v_head, int64_t v_token,
                     int dtype, int64_t tokens, int64_t kv_heads, int64_t head_dim, void* k_cache, int64_t kc_page,
                     int64_t kc_head, int64_t kc_slot, void* v_cache, int64_t vc_page, int64_t vc_head,
                     int64_t vc_slot, int64_t pages, int64_t page_size, const int32_t* page_table,
                     int64_t table_width, int64_t sequences, const int32_t* query_starts,
                     const int32_t* context_lengths, const void* q, int64_t heads, int64_t q_head, int64_t q_token,
                     void* q_out, const double* frequencies, int64_t pairs, int interleaved, float magnitude,
                     void* stream);

/*
 * m5k_paged_append into a cache in 8 bits (layout: see m5k_paged_attention_codes; block at most 128; the caches are
 * written, with their exponents).  A block's exponent is the least e with max |x| <= 448 * 2^e (FP8) or 127 * 2^e
 * (INT8) over the new tokens in it and, where the block holds older ones (at positions below context - n), at least
 * the exponent that it has; a code is x / 2^e to the nearest, ties to even, and where the exponent grows the older
 * codes are rounded again under it.  Slots behind the context stay as they are.  A block that gets an infinity or NaN
 * takes exponent 255.
 * Keys are turned in 64 bits, and infinities beyond FP32's range; q, in 32, as m5k_rope's.  head_dim 64 or 128; rows of
 * k, v and q 16-byte aligned.
 * Two tokens that name the same place, or two sequences that name the same block, leave unspecified codes there.
 */
int m5k_paged_append_codes(
    const void* k, int64_t k_head, int64_t k_token, const void* v, int64_t v_head, int64_t v_token, int dtype,
    int64_t tokens, int64_t kv_heads, int64_t head_dim, int mode, void* k_codes, int64_t kc_page, int64_t kc_head,
    int64_t kc_slot, uint8_t* k_exponents, int64_t ke_page, int64_t ke_head, void* v_codes, int64_t vc_page,
    int64_t vc_head, int64_t vc_slot, uint8_t* v_exponents, int64_t ve_page, int64_t ve_head, int64_t block,
    int64_t pages, int64_t page_size, const int32_t* page_table, int64_t table_width, int64_t sequences,
    const int32_t* query_starts, const int32_t* context_lengths, const void* q, int64_t heads, int64_t q_head,
    int64_t q_token, void* q_out, const double* frequencies, int64_t pairs, int interleaved, float magnitude,
    void* stream);

/* The same with a magnitude that FP32 need not have: keys are turned with it as it is, q with the FP32 number next to
 * it. */
int m5k_paged_append_codes64(
    const void* k, int64_t k_head, int64_t k_token, const void* v, int64_t v_head, int64_t v_token, int dtype,
    int64_t tokens, int64_t kv_heads, int64_t head_dim, int mode, void* k_codes, int64_t kc_page, int64_t kc_head,
    int64_t kc_slot, uint8_t* k_exponents, int64_t ke_page, int64_t ke_head, void* v_codes, int64_t vc_page,
    int64_t vc_head, int64_t vc_slot, uint8_t* v_exponents, int64_t ve_page, int64_t ve_head, int64_t block,
    int64_t pages, int64_t page_size, const int32_t* page_table, int64_t table_width, int64_t sequences,
    const int32_t* query_starts, const int32_t* context_lengths, const void* q, int64_t heads, int64_t q_head,
    int64_t q_token, void* q_out, const double* frequencies, int64_t pairs, int interleaved, double magnitude,
    void* stream);

/*
 * Read a cache in 8 bits back: k, v [kv_heads, tokens, head_dim] (F32, F16 or BF16, contiguous, 16-byte aligned) are
 * the values of the last n of each sequence's context_lengths[b] keys, n = query_starts[b + 1] - query_starts[b]: what
 * m5k_paged_append_codes with the same arguments wrote.  Rows behind the last sequence, at negative positions, behind
 * the table or on no page are 0.
 */
int m5k_paged_read(int mode, const void* k_codes, int64_t kc_page, int64_t kc_head, int64_t kc_slot,
                   const uint8_t* k_exponents, int64_t ke_page, int64_t ke_head, const void* v_codes, int64_t vc_page,
                   int64_t vc_head, int64_t vc_slot, const uint8_t* v_exponents, int64_t ve_page, int64_t ve_head,
                   int64_t block, int64_t pages, int64_t page_size, int64_t kv_heads, int64_t head_dim,
                   const int32_t* page_table, int64_t table_width, int64_t sequences, const int32_t* query_starts,
                   const int32_t* context_lengths, int64_t tokens, void* k, void* v, int dtype, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* M5K_H */
