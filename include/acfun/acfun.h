/*
 * acfun.h — public C API of the B200 (sm_100a) implementation of the Acfun inference path.
 *
 * Drop-in for the reference's include/acfun/acfun.h: every declaration below keeps the
 * reference signature, argument meaning, layouts and error behaviour (void functions
 * return silently on invalid shapes; acfun_model_load returns NULL on failure;
 * acfun_model_infer returns 0 for a NULL model).  The comment on each names the
 * reference declaration it replaces (path:line in the hit-droid/Acfun tree).
 *
 * Memory: every tensor argument may be a host pointer (pageable or pinned) or a CUDA
 * device pointer, detected per call.  Host-pointer calls are synchronous, like the
 * reference.  Calls whose tensors are all device-resident are stream-ordered on the
 * stream set with acfun_set_stream() (default: the legacy default stream) and return
 * without synchronising; call acfun_synchronize() before reading results on the host.
 *
 * Layouts (row-major, NHWC activations):
 *   GEMM         A[M,K], B[K,N], C[M,N]
 *   conv weight  [KH*KW*Cin, Cout]      index ((kh*KW+kw)*Cin+ic)*Cout+oc
 *   depthwise    [C, KH, KW]
 *   grouped      [groups][KH*KW*Cin_per][Cout_per]
 *   FC weight    [Cin, Cout]
 */
#ifndef ACFUN_ACFUN_H
#define ACFUN_ACFUN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- runtime / dispatch (reference acfun.h:19-30) ---- */
void acfun_set_threads(int n);                 /* acfun.h:20 — kept for ABI; CPU thread count has no meaning here */
int acfun_backend(void);                       /* acfun.h:23 — returns 4 (ACFUN_BACKEND_CUDA_SM100A) */
const char* acfun_backend_name(void);          /* acfun.h:24 — "CUDA-sm100a" */
/* acfun.h:29 — measures, on the current GPU, the fastest tcgen05 tile variant of the plain
 * fp32 (3xBF16), bf16 and int8 GEMMs per shape class (M, N, K rounded up to powers of two) and
 * writes the table to $ACFUN_TUNE_CACHE or ~/.cache/acfun/tile_table_<gpu>.txt; later runs load
 * it on first use.  Without a table the built-in size heuristics choose.  Results do not
 * depend on the table (it only picks among tested kernels). */
void acfun_autotune(void);
/* acfun.h:30 — "tuned: <n> shape classes ..." or "static heuristics: ..." */
const char* acfun_tune_status(void);

#define ACFUN_BACKEND_CUDA_SM100A 4

/* ---- GEMM (reference acfun.h:33-51) ---- */
/* acfun.h:33 — fp32 C = A*B; computed as 3xBF16 on tcgen05 tensor cores (3xTF32 with
 * acfun_set_fp32_math(1)), fp32-class error */
void acfun_gemm(int M, int N, int K, const float* A, const float* B, float* C);
/* acfun.h:43 — C = A*B + bias[j] (bias may be NULL), then ReLU if act==1 */
void acfun_gemm_epi(int M, int N, int K, const float* A, const float* B, float* C,
                    const float* bias, int act);
/* acfun.h:51 — fp32 in/out, operands rounded to bf16 (RNE), fp32 accumulation */
void acfun_gemm_bf16(int M, int N, int K, const float* A, const float* B, float* C);

/* ---- convolution (reference acfun.h:61-97) ---- */
/* acfun.h:61 */
void acfun_conv2d(const float* input, int N, int H, int W, int Cin,
                  const float* weight, const float* bias,
                  int KH, int KW, int Cout, int stride, int pad, float* output);
/* acfun.h:67 */
void acfun_conv2d_relu(const float* input, int N, int H, int W, int Cin,
                       const float* weight, const float* bias,
                       int KH, int KW, int Cout, int stride, int pad, float* output);
/* acfun.h:77 — depthwise, weight [C,KH,KW] */
void acfun_conv2d_dw(const float* input, int N, int H, int W, int C,
                     const float* weight, const float* bias,
                     int KH, int KW, int stride, int pad, float* output, int act);
/* acfun.h:86 — grouped; groups==Cin==Cout routes to depthwise */
void acfun_conv2d_g(const float* input, int N, int H, int W, int Cin,
                    const float* weight, const float* bias,
                    int KH, int KW, int Cout, int stride, int pad, int groups,
                    float* output, int act);
/* acfun.h:92 — out[N,Cout] = in[N,Cin] * W[Cin,Cout] + bias */
void acfun_fc(const float* input, int N, int Cin, const float* weight, const float* bias,
              int Cout, float* output);
/* acfun.h:97 — FC + bias + ReLU */
void acfun_fc_relu(const float* input, int N, int Cin, const float* weight, const float* bias,
                   int Cout, float* output);

/* ---- elementwise / pooling / normalisation (reference acfun.h:101-117) ---- */
void acfun_relu(float* data, size_t len);      /* acfun.h:101 */
void acfun_relu6(float* data, size_t len);     /* acfun.h:102 */
/* acfun.h:105 — NHWC max pool, square window */
void acfun_maxpool(const float* input, int N, int H, int W, int C,
                   int pool, int stride, int pad, float* output);
/* acfun.h:111 — max pool with ReLU applied to the pooled value */
void acfun_maxpool_relu(const float* input, int N, int H, int W, int C,
                        int pool, int stride, int pad, float* output);
/* acfun.h:114 — row softmax over the last dimension */
void acfun_softmax(const float* input, int rows, int cols, float* output);
/* acfun.h:117 — in place y = (x-mean)/sqrt(var+eps)*gamma + beta over NHWC channels */
void acfun_batchnorm(float* data, int size, int channels, const float* mean, const float* var,
                     const float* gamma, const float* beta, float eps);

/* ---- int8 (reference acfun.h:126-131) ---- */
/* acfun.h:126 — per-column symmetric weight quantisation (host-side, exact lroundf) */
void acfun_quantize_weights(const float* w, int K, int N, float* scales, int8_t* wq);
/* acfun.h:128 — int8 conv with per-tensor dynamic activation scale (s_in is ignored,
 * as in the reference), per-channel weight scales, fp32 output */
void acfun_conv2d_int8(const float* input, int N, int H, int W, int Cin,
                       const int8_t* wq, const float* wscale, const float* bias,
                       int KH, int KW, int Cout, int stride, int pad,
                       float s_in, float* output, int act);

/* ---- model (reference acfun.h:136-144) ---- */
typedef struct AcfunModel AcfunModel;
AcfunModel* acfun_model_load(const char* path);                          /* acfun.h:138 */
void acfun_model_destroy(AcfunModel* m);                                 /* acfun.h:139 */
int acfun_model_infer(AcfunModel* m, const float* input, float* output); /* acfun.h:141 */
int acfun_model_output_size(AcfunModel* m);                              /* acfun.h:142 */
void acfun_model_input_dims(AcfunModel* m, int* Cin, int* Hin, int* Win); /* acfun.h:144 */

/* ======================= extensions (no reference counterpart) ======================= */

/* Batched inference: n images of [Hin,Win,Cin] -> n * output_size floats.  Each image is
 * processed with batch-1 semantics (Softmax per image).  Returns the per-image output
 * element count, 0 on error. */
int acfun_model_infer_batch(AcfunModel* m, int n, const float* input, float* output);

/* int8 mode for a loaded model (no counterpart in the reference, whose int8 path has no
 * model format): enable != 0 runs every dense convolution through the int8 router
 * (acfun_quantize_weights of the folded weights + acfun_conv2d_int8) with one activation
 * scale per image -- the result of the reference harness that calls acfun_conv2d_int8 per
 * image -- while FC, pooling, BN and softmax stay fp32; 0 switches back to fp32.  Returns
 * 0 or an error code. */
int acfun_model_set_int8(AcfunModel* m, int enable);

/* s8 x s8 GEMM with int32 accumulation and a fused requantising epilogue:
 *   C[i,j] = sat_s8(rne(relu?((float)(acc[i,j] + bias[j]) * scale[j])))
 * bias may be NULL.  This is the int8 GEMM the BASELINE int8 config names; the reference
 * expresses it as acfun_gemm_int8 on A+128 followed by a -128*colsum(B) correction. */
void acfun_gemm_s8_requant(int M, int N, int K, const int8_t* A, const int8_t* B,
                           const int32_t* bias, const float* scale, int8_t* C, int act);

/* acfun_gemm_epi for callers that cannot allocate device memory (no counterpart in the
 * reference).  Such callers exist: processes that reserve all device memory up front in
 * their own pool, code running in an out-of-memory handler or allocator callback, and
 * latency-critical loops where cudaMalloc/cudaFree would synchronise the device.  Same
 * result as acfun_gemm_epi in 3xTF32 mode (acfun_set_fp32_math(1)), but nothing is
 * allocated: the 3xTF32 operand copies live in one
 * fixed 16 MiB device array compiled into the library (held by every GPU that loads it),
 * so 2*(M*K + K*N) must stay <= 4 Mi floats (K, N rounded up to 4).  All tensors must be
 * device pointers on the acfun device.  The first call on a device resolves the array's
 * address.  Calls share the array: calls that overlap on the GPU race.  Runs on the acfun
 * stream and synchronises with it before returning (so it cannot be called while that
 * stream is being captured): returns 0, or an error code. */
int acfun_gemm_epi_noalloc(int M, int N, int K, const float* A, const float* B, float* C,
                           const float* bias, int act);

/* fp32 math on tensor cores.  Every fp32 product is split into hi + lo parts and three
 * tensor-core products are accumulated in fp32 (the dropped lo*lo term and the split residuals
 * bound the error):
 *   1  3xTF32 everywhere   (tf32 parts, ~2^-21 relative per product)
 *   2  3xBF16 everywhere   (bf16 parts, ~2^-17 per product; twice the tensor rate and half the
 *                           operand bytes of 3xTF32)
 *   0  default: 3xBF16 everywhere (measured max-rel vs float64 on the parity shapes is at
 *      or below 3xTF32's there: the fp32 accumulation dominates both).
 * The initial mode comes from $ACFUN_FP32_MATH ("tf32x3" / "bf16x3").  Returns 0 or 1 (bad
 * mode).  Process-wide. */
int acfun_set_fp32_math(int mode);

/* ---- attention over an int8 key / value cache (no reference counterpart) ----
 *
 * The pieces of a decoder block between its projections: rotary positions, a paged cache that
 * holds keys and values as int8 codes, and attention that reads the codes.  Activations are
 * fp32, fp16 or bf16 (`dtype`); a tensor [tokens, heads, dim] is given by its address and its
 * token and head strides in elements (dim is contiguous), so a slice of a packed q/k/v row can
 * be passed in place.  All functions return 0 or an error code (also in acfun_last_error()) and
 * check their arguments on the host; entries of device arrays (table, start, length) are checked
 * in the kernels: a bad one skips its sequence (a bad offset those on both sides of it; where offsets
 * decrease, rows of other sequences may be left as they are too) and is reported, as code 1, by the
 * next acfun_synchronize().  Activations and index arrays may be host memory; the cache itself must be
 * device memory.
 *
 * Calls on device memory may be recorded into a CUDA graph, once the library has been used on the
 * device: while the stream set with acfun_set_stream() is being captured, what a call needs besides its
 * arguments is allocated and freed by the graph, so replays share nothing with other calls. */
#define ACFUN_F32 0
#define ACFUN_F16 1
#define ACFUN_BF16 2

/* Codes [pages][heads][page][dim] and one positive scale per (page, head): value = code * scale.
 * page is 16, 32, 64 or 128 tokens; dim is 64, 128 or 256. */
typedef struct AcfunKvCache8 {
  int8_t* k;
  int8_t* v;
  float* k_scale; /* [pages][heads] */
  float* v_scale;
  int pages, heads, page, dim;
} AcfunKvCache8;

/* A batch of sequences.  Sequence i has length[i] tokens in the cache, token j of it in page
 * table[i * table_cols + j / page] at slot j % page.  Its new tokens are its last ones,
 * start[i+1] - start[i] of them, rows start[i].. of the packed activations.  max_new and max_len
 * bound the new tokens and the length of any sequence; tokens is start[seqs]. */
typedef struct AcfunKvBatch {
  const int32_t* table;
  const int32_t* start;  /* [seqs + 1] */
  const int32_t* length; /* [seqs] */
  int seqs, table_cols, tokens, max_new, max_len;
} AcfunKvBatch;

/* Rotary positions: pair i of the first `rot` elements of a head turns by pos * freq[i] and is
 * scaled by amplitude; the elements after them are copied.  Pairs are (i, i + rot/2), or
 * (2i, 2i + 1) when interleaved. */
typedef struct AcfunRope {
  const float* freq; /* [rot / 2] */
  int rot, interleaved;
  float amplitude;
} AcfunRope;

/* Frequencies base^(-2i/rot) for i < rot/2, adapted to contexts `factor` times as long as the
 * `trained` one, written to host memory, and the amplitude that goes with them (may be NULL):
 *   0  none
 *   1  positions divided by factor
 *   2  base enlarged by factor^(rot/(rot-2)), so the lowest frequency is divided by factor
 *   3  by wavelength: pairs that turn more than `fast` times in the trained length keep their
 *      frequency, those below `slow` turns are divided by factor, linear in the pair's index
 *      between; amplitude 0.1 ln(factor) + 1
 *   4  as 3, linear in the number of turns between, amplitude 1
 *   5  as 3 with the ends of the linear part rounded outward to whole pairs (and kept within [0,
 *      rot - 1]): the form that checkpoints of this scaling are made with unless they say otherwise */
int acfun_rope_frequencies(int rot, double base, int scaling, double factor, double trained,
                           double fast, double slow, float* freq, float* amplitude);
/* y = x with positions pos[token] in [0, 2^31) applied; rot even and at most dim; y may be x. */
int acfun_rope(const void* x, void* y, int dtype, int tokens, int heads, int dim,
               long long x_token, long long x_head, long long y_token, long long y_head,
               const int32_t* pos, const AcfunRope* rope);
/* Quantise the batch's new keys and values into the cache; keys are rotated by their position in
 * the sequence first when rope is given (rot a multiple of 16).  The scale of a (page, head) is
 * max(max|x|, 127 * 2^-60) / 127 over the new tokens in the page, code = rint(x * (1 / scale))
 * clamped to +-127.  A page that holds older tokens keeps the larger of its scale and the new
 * one, and when that grows, older codes become rint(code * (old / new)).  Within a page the angles are
 * turned on from token to token in 32 bits, where acfun_rope reduces each in 64: a rotated key is within
 * 2^-13 of the page's largest element, so a code may differ by a rounding from that of a key which
 * acfun_rope turned before.  Infinities saturate
 * to +-127 and NaN becomes 0; neither enters a scale.  Pages written must not be shared between
 * sequences. */
int acfun_kv8_append(const AcfunKvCache8* cache, const AcfunKvBatch* batch, const void* k, const void* v,
                     int dtype, long long k_token, long long k_head, long long v_token, long long v_head,
                     const AcfunRope* rope);
/* The batch's last start[i+1] - start[i] tokens as values, k and v [tokens, heads, dim] contiguous
 * (either may be NULL). */
int acfun_kv8_read(const AcfunKvCache8* cache, const AcfunKvBatch* batch, void* k, void* v, int dtype);
/* out = softmax(scale * q k^T) v over each sequence's cached tokens.  q and out are [tokens,
 * q_heads, dim] in fp16 or bf16, q head h reads cache head h / (q_heads / heads).  causal: a new
 * token sees the tokens up to itself, and with window > 0 only the last `window` of them.  A row
 * that sees nothing is 0.  lse (fp32 [tokens, q_heads], may be NULL) is the natural logarithm of
 * the softmax denominator, -inf for a row that sees nothing. */
int acfun_kv8_attention(const AcfunKvCache8* cache, const AcfunKvBatch* batch, const void* q, void* out,
                        int dtype, int q_heads, long long q_token, long long q_head, long long o_token,
                        long long o_head, float scale, int causal, int window, float* lse);

/* Stream for device-pointer calls (a cudaStream_t passed as void*; NULL = legacy default). */
void acfun_set_stream(void* stream);
void* acfun_get_stream(void);
/* Select the CUDA device used by subsequent calls of this thread (default: device 0 or
 * $ACFUN_DEVICE). */
int acfun_set_device(int device);
/* Wait for all work issued on the current stream; returns 0 on success, else the error
 * code also reported by acfun_last_error(). */
int acfun_synchronize(void);
/* Last error of this thread (0 / "" when none); acfun_clear_error() resets it.
 * Codes: 1 invalid argument, 2 CUDA runtime error, 3 device-side wait timeout,
 *        4 out of memory, 5 model format error. */
int acfun_last_error_code(void);
const char* acfun_last_error(void);
void acfun_clear_error(void);

#ifdef __cplusplus
}
#endif

#endif /* ACFUN_ACFUN_H */
