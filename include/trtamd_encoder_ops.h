/*
 * C-ABI of the encoder operations that sit BETWEEN the BERT plugins in a TensorRT engine: the INT8
 * linear layers (QKV projection, attention output projection, the two feed-forward layers) and the
 * layout / quantisation reformats either side of the interleaved plugins.  In the reference these
 * are not plugin code: TensorRT's closed core executes them (the only open counterpart is the
 * deprecated cuBLASLt plugin plugin/fcPlugin, FP32/FP16 only, plugin/fcPlugin/README.md:41-45), so
 * the semantics below are this library's own statement of an INT8 fully-connected layer with
 * folded quantisation scales.  Same calling rules as trtamd_bert_kernels.h: plain device pointers,
 * asynchronous on the given stream, int status, nothing allocates or synchronises.
 */
#ifndef TRTAMD_ENCODER_OPS_H
#define TRTAMD_ENCODER_OPS_H

#include "trtamd_bert_kernels.h"

#ifdef __cplusplus
extern "C"
{
#endif

/* What happens to the INT32 accumulator acc[t][n] = sum_k a[t][k] * w[n][k] (exact, modulo 2^32: rows of 131072 values or
 * more can pass its range, and whether theirs do is the caller's to know). */
enum
{
    /* y = fmaf(float(acc), alpha[n], beta[n]);  out8 = sat8(rne(y)).  alpha = s_a * s_w[n] / s_out and
     * beta = bias[n] / s_out: the caller folds the output scale, as a TensorRT build does. */
    TRTAMD_LINEAR_AFFINE = 0,
    /* y as above with alpha = s_a * s_w[n], beta = bias[n];  g = 0.5 * y * (1 + erf(y / sqrt(2)));
     * out8 = sat8(rne(g * out_scale)), out_scale = 1 / s_out. */
    TRTAMD_LINEAR_GELU = 1,
    /* out32[t][n] = acc, linear layout: the accumulators themselves, for bit-exact checks. */
    TRTAMD_LINEAR_RAW_INT32 = 2,
    /* out16[t][n] = binary16(y), linear layout: the de-quantised result (e.g. the last layer). */
    TRTAMD_LINEAR_AFFINE_FP16 = 3
};

typedef struct trtamd_int8_linear_params
{
    int8_t const* a;    /* activations: linear [T][K], or 32-interleaved [K/32][T][32] */
    int8_t const* w;    /* weights: linear [N][K] (one row of K per output channel), or 32-interleaved
                           [K/32][N][32] (the faster one: a build step reformats constant weights once).  For the QKV
                           projection the rows are ordered [head][q|k|v][64], the packing
                           plugin/bertQKVToContextPlugin/README.md:27-30 asks for. */
    float const* alpha; /* [N] */
    float const* beta;  /* [N] */
    void* out;          /* int8 [T][N] or [N/32][T][32]; int32 / binary16 [T][N] */
    int32_t T, K, N;    /* K % 64 == 0, N % 32 == 0 */
    int32_t a_interleaved;
    int32_t w_interleaved;
    int32_t out_interleaved;
    int32_t epilogue;
    float out_scale;    /* TRTAMD_LINEAR_GELU only */
} trtamd_int8_linear_params;

/* Stands where TensorRT's own INT8 fully-connected / 1x1-convolution layer runs between the plugins
 * (closed source; engine-side placement described in plugin/bertQKVToContextPlugin/README.md:25-30). */
TRTAMD_API int trtamd_int8_linear(trtamd_stream_t stream, trtamd_int8_linear_params const* params);

/* FP16 linear layer for the FP16 encoder: out[t][n] = binary16(f(fmaf(acc, alpha[n], beta[n]))), acc = sum_k
 * a[t][k] * w[n][k] accumulated in binary32 on the FP16 matrix cores, f = identity (TRTAMD_LINEAR_AFFINE) or erf-GELU
 * (TRTAMD_LINEAR_GELU).  alpha = 1 and beta = bias give the usual fully-connected layer.  All tensors linear:
 * a [T][K], w [N][K], out [T][N]; K % 32 == 0, N % 32 == 0.  The order in which the K products are added (one after the
 * other, or in eight sums that meet at the end) depends on T, K and N, so a row can come out a binary16 step apart in calls
 * of different T; calls of the same sizes give the same bits.  The open counterpart in the reference is the deprecated
 * cuBLASLt GEMM plugin CustomFCPluginDynamic (plugin/fcPlugin/README.md:20-45, FP16 without bias or activation);
 * bias and GELU are what TensorRT's core fuses onto it. */
typedef struct trtamd_fp16_linear_params
{
    trtamd_half_t const* a;
    trtamd_half_t const* w;
    float const* alpha; /* [N] */
    float const* beta;  /* [N] */
    trtamd_half_t* out;
    int32_t T, K, N;
    int32_t epilogue;   /* TRTAMD_LINEAR_AFFINE or TRTAMD_LINEAR_GELU */
} trtamd_fp16_linear_params;

TRTAMD_API int trtamd_fp16_linear(trtamd_stream_t stream, trtamd_fp16_linear_params const* params);

/* ------------------------------------------------------------------------------------------
 * INT8 arithmetic without calibration: every token is quantised with a scale of its own when it is there, every output
 * channel's weights have theirs.  Activations between the layers are FP16, all tensors are linear.  No counterpart in the
 * reference's plugins.
 * ------------------------------------------------------------------------------------------ */

/* amax[t] = max_c |in[t][c]|;  scales[t] = amax[t] / 127;  out[t][c] = round_half_even(in[t][c] * 127 / amax[t]), exact
 * (the quotient is rounded once, ties as such).  A token of zeros has scale 0 and zeros.  A token that holds an infinity
 * or a NaN has scale NaN and zeros, so that whatever is computed from it is NaN, and nothing else is.
 * in [T][C] with in_stride elements between rows (a multiple of 8, no less than C); out [T][C]; C % 32 == 0; T < 2^24 and C < 2^30.
 * As everywhere below, what a call writes overlaps nothing that it reads. */
TRTAMD_API int trtamd_quantize_fp16_per_token(trtamd_stream_t stream, int32_t T, int32_t C, trtamd_half_t const* in,
    int64_t in_stride, int8_t* out, float* scales);

/* out[t][n] = binary16(f(acc * token_scale[t] * channel_scale[n] + bias[n])), acc = sum_k a[t][k] * w[n][k] (exact), f =
 * identity (TRTAMD_LINEAR_AFFINE) or erf-GELU (TRTAMD_LINEAR_GELU), which before the rounding to binary16 is within 8.5e-5 of its
 * value where that is a normal binary16, 2^-14 or more, and within 5.2e-9 where it is less; of infinities, which products past the
 * end of binary32 give, it is infinity and 0.  Scales, sums and f are binary32, with one rounding at the end; a token's results do
 * not depend on what other tokens are in the call. */
typedef struct trtamd_int8_token_linear_params
{
    int8_t const* a;            /* [T][K] */
    int8_t const* w;            /* [N][K] */
    float const* token_scale;   /* [T] */
    float const* channel_scale; /* [N] */
    float const* bias;          /* [N], or NULL for none */
    trtamd_half_t* out;         /* [T][N] */
    int32_t T, K, N;            /* K % 64 == 0, N % 32 == 0; K < 131072, so that no sum passes INT32 */
    int32_t epilogue;           /* TRTAMD_LINEAR_AFFINE or TRTAMD_LINEAR_GELU */
} trtamd_int8_token_linear_params;

TRTAMD_API int trtamd_int8_token_linear(trtamd_stream_t stream, trtamd_int8_token_linear_params const* params);

/* The two in one call, for a layer whose input no other layer takes: the same bits as trtamd_quantize_fp16_per_token and
 * trtamd_int8_token_linear behind it (few tokens: in one launch, which leaves the workspace alone).  The quantised tokens go to the
 * workspace (16-byte aligned; calls that may overlap need one each). */
typedef struct trtamd_int8_dynamic_linear_params
{
    trtamd_half_t const* a;     /* [T][K] */
    int64_t a_stride;           /* elements between rows: a multiple of 8, no less than K */
    int8_t const* w;            /* [N][K] */
    float const* channel_scale; /* [N] */
    float const* bias;          /* [N], or NULL for none */
    trtamd_half_t* out;         /* [T][N] */
    void* workspace;
    size_t workspace_bytes;     /* trtamd_int8_dynamic_linear_workspace_size(T, K, N) or more */
    int32_t T, K, N;            /* K % 64 == 0, N % 32 == 0; K < 131072, so that no sum passes INT32 */
    int32_t epilogue;           /* TRTAMD_LINEAR_AFFINE or TRTAMD_LINEAR_GELU */
} trtamd_int8_dynamic_linear_params;

TRTAMD_API size_t trtamd_int8_dynamic_linear_workspace_size(int32_t T, int32_t K, int32_t N);
TRTAMD_API int trtamd_int8_dynamic_linear(trtamd_stream_t stream, trtamd_int8_dynamic_linear_params const* params);

/* ------------------------------------------------------------------------------------------
 * Norms of queries and keys for each head and their rotation by position, between the QKV projection and the attention, in
 * one pass over them.  No counterpart in the reference's plugins, which add position embeddings to the tokens instead.
 * ------------------------------------------------------------------------------------------ */
enum
{
    TRTAMD_QK_NORM_NONE = 0,
    TRTAMD_QK_NORM_RMS = 1,  /* y = x / sqrt(mean(x^2) + eps) * weight */
    TRTAMD_QK_NORM_LAYER = 2 /* y = (x - mean) / sqrt(variance + eps) * weight + bias */
};
enum
{
    TRTAMD_ROTARY_MAX_AXES = 4,
    TRTAMD_ROTARY_MAX_HEAD = 256
};

/* A head's values 0 .. rotary_dim-1 are rotary_dim / 2 pairs, pair i being the values i and i + rotary_dim / 2, or 2 i and
 * 2 i + 1 (adjacent_pairs); the values behind them are normed and not rotated.  Pair i (a, b) of token t becomes
 *   (a cos(p f) - b sin(p f), b cos(p f) + a sin(p f)),   p = positions[axis(i)][t],  f = frequencies[i]
 * with the angle formed and reduced in binary64 (no table: any position, negative ones too), all else in binary32 and one rounding
 * at the end.  Several axes (time, height, width) share the pairs: the first sections[0] pairs go to axis 0, the next
 * sections[1] to axis 1 and so on; with axes_cycled pair i goes to axis i % axes while that axis has pairs left
 * (i / axes < sections[i % axes]), otherwise to axis 0.  Either way the sections add up to rotary_dim / 2.
 *
 * q and k are read at q + t * q_token_stride + head * q_head_stride (elements), each head's d values in a row, and written
 * to q_out and k_out in the same way: the packed layouts of the attention plugins ([token][head][q|k|v][d] has token strides
 * of 3 N d and head strides of 3 d) as well as tensors of their own, with fewer heads of k than of q or none.  q_out = q with the
 * same strides works in place, if no two heads overlap (heads that are only read may: a stride of 0 is one head for all); other
 * overlaps of what is written with anything else in the call are not allowed.  T * (q_heads + k_heads) < 2^26. */
typedef struct trtamd_qk_norm_rotary_params
{
    void const* q;
    void const* k;
    void* q_out;
    void* k_out;
    int64_t q_token_stride, q_head_stride, k_token_stride, k_head_stride;
    int64_t q_out_token_stride, q_out_head_stride, k_out_token_stride, k_out_head_stride;
    int32_t T, q_heads, k_heads, d; /* d <= 256; q_heads or k_heads may be 0 (its pointers are not used then) */
    int32_t norm;                   /* TRTAMD_QK_NORM_* */
    float eps;
    float const* q_weight;          /* [d], with a norm */
    float const* k_weight;
    float const* q_bias;            /* [d], TRTAMD_QK_NORM_LAYER */
    float const* k_bias;
    int32_t rotary_dim;             /* even, <= d; 0: no rotation */
    int32_t adjacent_pairs;
    float const* frequencies;       /* [rotary_dim / 2] */
    int32_t const* positions;       /* [axes][T] */
    int32_t axes;                   /* 1 .. 4 */
    int32_t axes_cycled;
    int32_t sections[4];            /* [axes]; one axis: not used */
} trtamd_qk_norm_rotary_params;

/* data_type of q, k and the outputs: 0 = FP32, 1 = FP16 (nvinfer1::DataType values). */
TRTAMD_API int trtamd_qk_norm_rotary(
    trtamd_stream_t stream, int32_t data_type, trtamd_qk_norm_rotary_params const* params);

/* ------------------------------------------------------------------------------------------
 * A cache of keys and values in 8 bits, in pages, for sequences that grow: written as the projection leaves them (with
 * trtamd_qk_norm_rotary before it where the layer has that), attended to, and read back.  No counterpart in the reference's plugins,
 * whose attention has all of a sequence in one call.
 *
 * Token t of sequence b is token t % page_tokens of page page_table[b * max_pages + t / page_tokens]; the keys of head h of page p
 * are k[p][h][token][d], its values v[p][h][d][token] (a value's tokens side by side, as the second product wants them), one byte
 * each, INT8 or E4M3 (a sign, 4 bits of exponent, 3 of mantissa, no infinities), and what they stand for is the byte's value times
 * k_scale[p][h] or v_scale[p][h].
 *
 * A call has cu_seqlens[b + 1] - cu_seqlens[b] tokens of sequence b, rows cu_seqlens[b] on of its tensors, which are the LAST ones
 * of the lengths[b] that the sequence has.  Lengths, rows and pages are read on the GPU, so a captured call follows them: B, T,
 * max_tokens and max_pages are what may not be passed.  What does not fit is left out and harms nothing: rows at or behind T,
 * a sequence's rows from the max_tokens-th on (neither read nor written), tokens before a sequence's first one or behind its
 * max_pages pages, and pages whose number is not in 0 .. pages - 1 (not written; read as zeros; not attended to, so that
 * pages that a window has left behind can go back to the pool with -1 in their place).
 *
 * No page may be written for two sequences, or two rows, of a call; reading them may be shared, also with a sequence that writes: one
 * without rows in the call writes nothing.
 *
 * max_tokens and T may be bounds, of a captured call for one, and every row is served; but attention's kernels are chosen by them. Where T
 * is about B * max_tokens, every sequence is taken to have as many rows, and a lone one then waits for its keys 64 at a time (a row over
 * 131070 keys, 8 key heads of 128: 54 us with max_tokens = T = 1, 1.0 ms with 512, 3.9 ms with 8192).  Capture steps of single tokens apart
 * from those of prompts.
 * ------------------------------------------------------------------------------------------ */
typedef struct trtamd_kv_cache
{
    void* k;                   /* [pages][kv_heads][page_tokens][d] */
    void* v;                   /* [pages][kv_heads][d][page_tokens] */
    float* k_scale;            /* [pages][kv_heads] */
    float* v_scale;            /* [pages][kv_heads] */
    int32_t const* page_table; /* [B][max_pages] */
    int32_t const* lengths;    /* [B]: tokens of each sequence, those of the call included */
    int32_t const* cu_seqlens; /* [B + 1]: rows of each sequence in the call's tensors */
    int32_t data_type;         /* of k and v: 2 = INT8, 6 = FP8 E4M3 (nvinfer1::DataType values) */
    int32_t pages;             /* in the pool */
    int32_t page_tokens;       /* 16, 32, 64 or 128 */
    int32_t kv_heads;          /* at most 16383; pages * kv_heads < 2^31 */
    int32_t d;                 /* a multiple of 16, at most 256 */
    int32_t B;                 /* sequences, at most 65535 */
    int32_t max_pages;         /* entries of a sequence in page_table; max_pages * page_tokens at most 2^30 */
    int32_t max_tokens;        /* rows of a sequence in the call, or more */
    int32_t T;                 /* rows of the call's tensors */
} trtamd_kv_cache;

/* Quantises the call's rows into the cache.  top = 127 (INT8) or 448 (E4M3); for each page and head that gets new tokens, for keys and
 * values by themselves, a = the largest absolute value among the new ones:
 *   where the new tokens begin the page, or what it held had the scale 0: scale = a / top;
 *   otherwise the scale s stays while a <= s * top, and else becomes s * 2^n with the smallest n that makes it so, and what the page
 *   held becomes round_half_even(byte * 2^-n).
 *   byte = round_half_even(x * (1 / scale)), within -top .. top; 0 where the scale is 0.
 * All of it in binary32, each operation rounded correctly.  Doubling keeps what a page goes through as it fills bounded: whatever
 * the order, an INT8 token is within one step of its last scale (half a step where the scale never grew), and in E4M3 only what
 * falls below its normal numbers is rounded again.  New values that hold an infinity or a NaN leave the scale NaN and zeros in their
 * place, so that whatever is computed from this page and head is NaN, and nothing else is; a scale of NaN stays until the page is
 * begun again.  Other pages, heads and tokens are left as they were.  k and v: row t, head h at k + t * k_token_stride + h * k_head_stride, multiples of 8
 * elements, d values in a row. */
typedef struct trtamd_kv_cache_write_params
{
    trtamd_kv_cache cache;
    trtamd_half_t const* k;
    trtamd_half_t const* v;
    int64_t k_token_stride, k_head_stride, v_token_stride, v_head_stride;
} trtamd_kv_cache_write_params;

TRTAMD_API int trtamd_kv_cache_write(trtamd_stream_t stream, trtamd_kv_cache_write_params const* params);

/* The call's rows from the cache, binary16(byte * scale): the last cu_seqlens[b + 1] - cu_seqlens[b] tokens of each sequence.  (A value
 * within half a step of the largest binary16 can come back as an infinity; attention does not round it.) */
typedef struct trtamd_kv_cache_read_params
{
    trtamd_kv_cache cache;
    trtamd_half_t* k;
    trtamd_half_t* v;
    int64_t k_token_stride, k_head_stride, v_token_stride, v_head_stride;
} trtamd_kv_cache_read_params;

TRTAMD_API int trtamd_kv_cache_read(trtamd_stream_t stream, trtamd_kv_cache_read_params const* params);

/* Attention of the call's rows over their sequences in the cache, causal: row i of a sequence, its token p = begin + i, sees the
 * tokens j <= p, with a window only those with j > p - window, and the first `sinks` tokens whatever the window is.
 *   out = binary16(sum_j w_j v_j / sum_j w_j),  w_j = exp(scale * q k_j),  k_j and v_j what the cache's bytes stand for.
 * Products of the bytes' values are exact, sums, maxima and exponentials binary32; the weights of the second product are rounded
 * to binary16 once, half to even, each times its page's v_scale and the largest at 2^7 or more: by 2^-11 of themselves, or 2^-32 of the
 * largest where that is more.
 * A score of minus infinity weighs nothing.  A row that sees nothing is zeros.  Query head h reads head h / (q_heads / kv_heads) of the cache.
 * A result can differ in its last bits between calls of other sizes or estimates, not between calls of the same.
 * q: row t, head h at q + t * q_token_stride + h * q_head_stride, multiples of 8 elements, d values in a row; out alike.  What is
 * written overlaps nothing that is read, but out may be q with the same strides. */
typedef struct trtamd_kv_cache_attention_params
{
    trtamd_kv_cache cache;
    trtamd_half_t const* q;
    trtamd_half_t* out;
    int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;
    int32_t q_heads;        /* a multiple of kv_heads; T * q_heads < 2^30 */
    float scale;            /* of the scores; finite and not negative */
    int32_t window;         /* tokens that a row sees, itself the last of them; 0: all */
    int32_t sinks;          /* 0 or more */
    int32_t max_length;     /* about the longest of the lengths, by which work is shared out (longer ones are served as well); 0:
                               as long as max_pages allows */
    void* workspace;        /* 16-byte aligned; calls that may overlap need one each */
    size_t workspace_bytes; /* trtamd_kv_cache_attention_workspace_size(params) or more */
} trtamd_kv_cache_attention_params;

/* Of the parameters' sizes alone: no pointer is looked at.  0: none is needed, or the call refuses the sizes (trtamd_last_error() then
 * says why). */
TRTAMD_API size_t trtamd_kv_cache_attention_workspace_size(trtamd_kv_cache_attention_params const* params);
TRTAMD_API int trtamd_kv_cache_attention(trtamd_stream_t stream, trtamd_kv_cache_attention_params const* params);

/* ------------------------------------------------------------------------------------------
 * Attention in windows, over packed sequences in FP16: row i of a sequence sees the rows i - left .. i + right and the first `sinks`
 * rows, of them none behind i + right; left or right -1: all on that side (right = 0: causal).
 *   out = binary16(sum_j w_j v_j / sum_j w_j),  w_j = exp(scale * q k_j)
 * Sums, maxima and exponentials are binary32, the weights of the second product rounded to binary16 once, as above.  Rows that
 * are not seen do not take part whatever they hold, infinities and NaNs included (a NaN or an infinity anywhere near makes the
 * rows around it slow, some hundred times where all are).  A score of minus infinity weighs nothing.
 * A query head h reads head h / (q_heads / kv_heads) of k and v.  Rows at or behind T, and a sequence's rows from the
 * max_tokens-th on, are left out: neither read nor written.  Row t, head h of q at q + t * q_token_stride + h * q_head_stride, d
 * values in a row, multiples of 8 elements; k, v and out alike: the attention plugins' packing ([token][head][q|k|v][d]) as well
 * as tensors of their own.  What is written overlaps nothing that is read.  No counterpart in the reference's plugins.
 * ------------------------------------------------------------------------------------------ */
typedef struct trtamd_window_attention_params
{
    trtamd_half_t const* q;
    trtamd_half_t const* k;
    trtamd_half_t const* v;
    trtamd_half_t* out;
    int64_t q_token_stride, q_head_stride, k_token_stride, k_head_stride;
    int64_t v_token_stride, v_head_stride, out_token_stride, out_head_stride;
    int32_t const* cu_seqlens; /* [B + 1] */
    int32_t B;                 /* sequences, at most 65535 */
    int32_t T;                 /* rows of the tensors; T * q_heads < 2^30 */
    int32_t max_tokens;        /* of a sequence, or more */
    int32_t q_heads;           /* a multiple of kv_heads */
    int32_t kv_heads;          /* at most 65535 */
    int32_t d;                 /* a multiple of 8, at most 256 */
    float scale;               /* finite and not negative */
    int32_t left, right;       /* -1 or more */
    int32_t sinks;             /* 0 or more */
} trtamd_window_attention_params;

TRTAMD_API int trtamd_window_attention(trtamd_stream_t stream, trtamd_window_attention_params const* params);

/* ------------------------------------------------------------------------------------------
 * Reformats either side of the interleaved plugins.  TensorRT inserts these itself when a plugin asks
 * for TensorFormat::kCHW32 (include/NvInferRuntime.h:1471; the INT8 interleaved plugins do:
 * plugin/bertQKVToContextPlugin/qkvToContextInt8InterleavedPlugin.cpp:124-127,
 * plugin/skipLayerNormPlugin/skipLayerNormInt8InterleavedPlugin.cpp supportsFormatCombination); here
 * they are explicit calls.  "linear" is [T][C] (token-major); "interleaved" is [C/32][T][32], the
 * memory image of a [1,C,T,1] kCHW32 tensor.  C % 32 == 0.
 * ------------------------------------------------------------------------------------------ */

/* Pure layout change of INT8 data (also used once per weight matrix: [N][K] -> [K/32][N][32]). */
TRTAMD_API int trtamd_int8_linear_to_interleaved(trtamd_stream_t stream, int32_t T, int32_t C, int8_t const* in,
    int8_t* out);
TRTAMD_API int trtamd_int8_interleaved_to_linear(trtamd_stream_t stream, int32_t T, int32_t C, int8_t const* in,
    int8_t* out);

/* IQuantizeLayer with a per-tensor scale (include/NvInfer.h:5333-5345): out = clamp(round_half_even(in / scale),
 * -128, 127), fused with the reformat to the interleaved layout. */
TRTAMD_API int trtamd_quantize_fp16_to_interleaved(trtamd_stream_t stream, int32_t T, int32_t C,
    trtamd_half_t const* in, float scale, int8_t* out);

/* IDequantizeLayer with a per-tensor scale (include/NvInfer.h:5493-5500): out = binary16(in * scale), fused with
 * the reformat back to the linear layout. */
TRTAMD_API int trtamd_dequantize_interleaved_to_fp16(trtamd_stream_t stream, int32_t T, int32_t C, int8_t const* in,
    float scale, trtamd_half_t* out);

#ifdef __cplusplus
}
#endif

#endif /* TRTAMD_ENCODER_OPS_H */
