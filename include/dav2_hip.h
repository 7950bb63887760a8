/*
 * Thin C-ABI HIP launcher layer: one extern "C" entry per gfx950 kernel.
 *
 * Every entry takes raw device pointers, plain sizes and a hipStream_t passed
 * as void* (NULL = the null stream), enqueues asynchronously and returns the
 * hipError_t value as int (0 = hipSuccess; hipErrorInvalidValue = 1 for
 * rejected arguments). No entry allocates memory. The C++ operator surface
 * (dav2::HipOperators, mirroring the reference's src/operators.h) calls only
 * these; tests and FFI callers may call them directly.
 *
 * int8 matrices are row-major [rows][ld] bytes, ld a multiple of 64 and bytes
 * [K, ld) zero: the first K bytes of a row are the byte view of the
 * reference's packed 4x int8 words (quantize_rows_int8_fused.glsl:51).
 */
#ifndef DAV2_HIP_H
#define DAV2_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifndef DAV2_API
#define DAV2_API __attribute__((visibility("default")))
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* Replaces quantize_rows_int8_fused.glsl:20-55 as dispatched by
 * VulkanOperators::linear_int8 (src/operators.cpp:810-818) and
 * project_tokens_int8 (:1514-1522). Row r reads input[input_offset + r*columns + c].
 * columns % 4 == 0, input_offset % 4 == 0. */
DAV2_API int dav2_hip_quantize_rows_i8(const float* input, uint64_t input_offset,
                                       uint32_t rows, uint32_t columns, int8_t* q,
                                       uint32_t ldq, float* scales, void* stream);

/* gelu.glsl:16-49 followed by quantize_rows_int8_fused.glsl:20-55 in one pass:
 * the row quantized is gelu(input row), bit for bit what the reference's
 * GELU pass after fc1 (linear_int8 with gelu, src/operators.cpp:837-843,
 * called from src/encoder.cpp:525-528) and fc2's input quantization
 * (src/operators.cpp:810-818) produce. Arguments as dav2_hip_quantize_rows_i8;
 * columns <= 4096. */
DAV2_API int dav2_hip_gelu_quantize_rows_i8(const float* input, uint64_t input_offset,
                                            uint32_t rows, uint32_t columns, int8_t* q,
                                            uint32_t ldq, float* scales, void* stream);

/* int8 weight rows of `columns` bytes -- the reference GpuModel layout,
 * [rows][columns/4] little-endian words (src/gpu_model.cpp:241-284) -- to the
 * GEMM layout [rows][ld] (ld % 16 == 0, ld >= columns), bytes [columns, ld)
 * zero. rows <= 65535. No reference counterpart (a layout conversion). */
DAV2_API int dav2_hip_pad_rows_i8(const int8_t* src, uint32_t rows, uint32_t columns, int8_t* dst, uint32_t ld,
                                  void* stream);
/* The reference's transposed int8 weight layout (src/gpu_model.cpp:241-258,
 * int8_transposed_buffer: [K][N] bytes, byte k*N + n = weight of output n,
 * input k), consumed by linear_int8(..., weight_transposed=true)
 * (src/operators.cpp:819-832), to the GEMM layout: N rows of ld bytes
 * (ld % 64 == 0, ld >= K), zero beyond K. */
DAV2_API int dav2_hip_transpose_rows_i8(const int8_t* src, uint32_t k_rows, uint32_t n_columns, int8_t* dst,
                                        uint32_t ld, void* stream);

/* Replaces im2col_quantize_int8.glsl:26-83 (src/operators.cpp:1284-1298,
 * :1787-1801, :1946-1960). CHW input; rows = output_width*output_height.
 * scratch (optional, dav2_hip_im2col_scratch_floats() floats) enables the
 * tiled 3x3-stride-1 and 1x1 kernels and, for other geometries, row scales
 * from per-pixel channel-group maxima; without it the generic gather runs.
 * All produce the same bytes. */
DAV2_API uint64_t dav2_hip_im2col_scratch_floats(uint32_t input_width, uint32_t input_height,
                                                 uint32_t input_channels);
DAV2_API int dav2_hip_im2col_quantize_i8(const float* input, uint32_t input_width,
                                         uint32_t input_height, uint32_t input_channels,
                                         uint32_t output_width, uint32_t output_height,
                                         uint32_t kernel, uint32_t stride, int32_t padding,
                                         int8_t* q, uint32_t ldq, float* scales,
                                         float* scratch, uint64_t scratch_floats, void* stream);
/* The same for max(input, 0) (relu.glsl ahead of the convolution, as the DPT
 * residual units apply it), without materialising the ReLU: any geometry on
 * maps of up to 8192 output pixels (rows of up to 9216 columns), else kernel
 * 3 / stride 1 / padding 1 (channels % 16 == 0) or kernel 1 / stride 1 /
 * padding 0 with scratch only; other calls return hipErrorInvalidValue. No
 * reference counterpart (a fusion of two reference passes). */
DAV2_API int dav2_hip_im2col_quantize_relu_i8(const float* input, uint32_t input_width,
                                              uint32_t input_height, uint32_t input_channels,
                                              uint32_t output_width, uint32_t output_height,
                                              uint32_t kernel, uint32_t stride, int32_t padding,
                                              int8_t* q, uint32_t ldq, float* scales,
                                              float* scratch, uint64_t scratch_floats, void* stream);

/* Replaces layer_norm.glsl:27-68 (src/operators.cpp:1016-1042). */
DAV2_API int dav2_hip_layer_norm(float* out, const float* input, const float* weight,
                                 const float* bias, uint32_t rows, uint32_t columns,
                                 float epsilon, void* stream);

/* layer_norm.glsl followed by quantize_rows_int8_fused.glsl in one pass (the
 * reference runs them back to back at src/encoder.cpp:443-452, :500-528);
 * out may be NULL when the fp32 row is not needed. columns <= 4096. */
DAV2_API int dav2_hip_layer_norm_quantize_i8(int8_t* q, uint32_t ldq, float* scales,
                                             float* out, const float* input,
                                             const float* weight, const float* bias,
                                             uint32_t rows, uint32_t columns,
                                             float epsilon, void* stream);

/* GEMM epilogues. Reference: linear_int8_tiled.glsl:99-116,
 * gelu.glsl:16-49, add_scaled.glsl:23-32, conv_transpose_int8.glsl:31-58. */
enum {
    DAV2_GEMM_EPI_RAW_I32 = 0,        /* out_i32[m*n + n'] = int32 accumulator        */
    DAV2_GEMM_EPI_ROW = 1,            /* out[(m+off)*n + n'] = acc*sa*sb + bias        */
    DAV2_GEMM_EPI_ROW_GELU = 2,       /* ... then exact-erf GELU                        */
    DAV2_GEMM_EPI_ROW_LAYERSCALE = 3, /* out = residual + (acc*sa*sb + bias)*gamma[n'] */
    DAV2_GEMM_EPI_TRANSPOSED = 4,     /* out[n'*stride + m + off] (channel-major), plus
                                         residual at the same index when given, then
                                         max(., 0) when relu_output                     */
    DAV2_GEMM_EPI_CONVT = 5,          /* stride==kernel ConvTranspose scatter           */
    DAV2_GEMM_EPI_ROW_COLMAX = 6      /* ROW, and per tile of rows the max |out| of each
                                         column n' >= col_absmax_begin                  */
};

typedef struct dav2_gemm_i8_args {
    const int8_t* a;        /* activations [m][lda], 16-byte aligned          */
    uint64_t lda;
    const int8_t* b;        /* weights [n][ldb], 16-byte aligned              */
    uint64_t ldb;
    uint32_t m, n, k;       /* k: multiple of 64, padding bytes zero          */
    uint32_t epilogue;      /* DAV2_GEMM_EPI_*                                */
    const float* a_scales;  /* [m] per-row activation scales                  */
    const float* b_scales;  /* [n] per-row weight scales                      */
    const float* bias;      /* [n] (CONVT: [convt_channels]) or NULL = 0      */
    int32_t* out_i32;
    float* out;
    uint64_t out_row_offset;
    uint64_t out_row_stride;
    const float* residual;  /* LAYERSCALE (may alias out) or TRANSPOSED        */
    const float* gamma;
    uint32_t convt_kernel, convt_width, convt_height, convt_channels;
    /* ROW_COLMAX: col_absmax[t][n' - col_absmax_begin] = max |out[m][n']| over
     * the rows m of row tile t (dav2_hip_gemm_i8_row_tiles() tiles); the
     * begin is a multiple of 64, n % 4 == 0 and out 16-byte aligned. */
    float* col_absmax;
    uint32_t col_absmax_begin;
    uint32_t relu_output;   /* TRANSPOSED only: max(out, 0) after the residual */
    /* TRANSPOSED only: split_k > 1 runs K in that many slices on more
     * workgroups (for GEMMs with few output tiles), their int32 sums in
     * split_scratch (dav2_hip_gemm_i8_split_scratch_bytes), then one pass
     * adds them (exact) and applies the epilogue. Same output bits. */
    uint32_t split_k;
    int32_t* split_scratch;
} dav2_gemm_i8_args;

/* Replaces linear_int8_tiled.glsl:40-117 (src/operators.cpp:847-880) and
 * conv_transpose_int8.glsl:31-58 (:1969-1975). */
DAV2_API int dav2_hip_gemm_i8(const dav2_gemm_i8_args* args, void* stream);
/* Timing hook, no reference counterpart: hipEvent_t start / stop for the
 * calling thread's next dav2_hip_gemm_i8, recorded by its kernel dispatches
 * (the GEMM's start, the last kernel's end); NULL, NULL clears. */
DAV2_API void dav2_hip_gemm_i8_events(void* start, void* stop);
/* Timing hook, no reference counterpart: hipEvent_t start / stop for the
 * calling thread's kernel dispatches: the next kernel launched records start
 * when it begins, every launch until the hook is cleared (NULL, NULL) records
 * stop when it ends, so the pair spans all kernels of an operation. Returns 1
 * when a kernel launched under the pair being replaced, 0 when none did (its
 * events then hold no record of that operation). */
DAV2_API int dav2_hip_launch_events(void* start, void* stop);

/* fp32 GEMM of the fp32 precision mode: out = a . b^T + bias with the
 * epilogues ROW, ROW_GELU, ROW_LAYERSCALE, TRANSPOSED (residual, relu_output)
 * and CONVT of the int8 GEMM. a [m][lda], b [n][ldb] float32, 16-byte
 * aligned, k, lda, ldb multiples of 4 (pad columns with zeros).
 * Replaces linear_tiled.glsl / linear_vec*.glsl (src/operators.cpp:882-955),
 * the GEMM of conv2d (:1528-1676), conv_transpose_nonoverlap (:1807-1861) and
 * project_tokens (:1408-1452). */
typedef struct dav2_gemm_f32_args {
    const float* a;
    uint64_t lda;
    const float* b;
    uint64_t ldb;
    uint32_t m, n, k;
    uint32_t epilogue;      /* DAV2_GEMM_EPI_* (not RAW_I32 / ROW_COLMAX)      */
    const float* bias;      /* [n] (CONVT: [convt_channels]) or NULL = 0      */
    float* out;
    uint64_t out_row_offset;
    uint64_t out_row_stride;
    const float* residual;  /* LAYERSCALE (may alias out) or TRANSPOSED        */
    const float* gamma;
    uint32_t convt_kernel, convt_width, convt_height, convt_channels;
    uint32_t relu_output;   /* TRANSPOSED only                                 */
    /* 1: both operands rounded to binary16 before the products, which are
     * exact (subnormal operands too), fp32 accumulation: the fp16 mode's
     * cooperative-matrix linears (linear_coop_fp16.glsl,
     * src/operators.cpp:540-768). 0: fp32; from k = 64 on every product is
     * within 1.001 x 2^-24 of itself before it is summed. An output's bits
     * depend on its row of a and of b and on k alone, not on m or n. */
    uint32_t half_operands;
} dav2_gemm_f32_args;
DAV2_API int dav2_hip_gemm_f32(const dav2_gemm_f32_args* args, void* stream);
/* Native binary16 products: out = sum over k ascending of
 * float(fp16(h(a) * h(b))) in fp32 (h = round to binary16), then the ROW,
 * TRANSPOSED or CONVT epilogue (+ bias; no residual / ReLU). Replaces the
 * dot products of prepare_tokens_fp16.glsl:37-52, project_tokens_fp16.glsl
 * and conv_transpose_nonoverlap_fp16.glsl (src/operators.cpp:1211-1406,
 * :1453-1481, :1862-1906); the same bits as the CPU oracle. */
DAV2_API int dav2_hip_gemm_h16_products(const dav2_gemm_f32_args* args, void* stream);

/* fp32 im2col of conv2d (src/operators.cpp:1528-1676): out[p][c], p = oy*OW
 * + ox, c = ic*k*k + ky*k + kx, zero padding, columns C*k*k .. ld-1 zero;
 * relu != 0 takes max(input, 0) (the DPT residual units' ReLU). */
DAV2_API int dav2_hip_im2col_f32(const float* input, uint32_t input_width, uint32_t input_height,
                                 uint32_t input_channels, uint32_t output_width, uint32_t output_height,
                                 uint32_t kernel, uint32_t stride, int32_t padding, uint32_t relu, float* out,
                                 uint32_t ld, void* stream);
/* Row tiles (rows of col_absmax) of a dav2_hip_gemm_i8 call with m rows and
 * n output columns. No reference counterpart: the attention's digit packing
 * reads these maxima instead of a pass over k and v. */
DAV2_API uint32_t dav2_hip_gemm_i8_row_tiles(uint32_t m, uint32_t n, uint32_t epilogue);
/* Scratch bytes of a split-K dav2_hip_gemm_i8 call. No reference counterpart. */
DAV2_API uint64_t dav2_hip_gemm_i8_split_scratch_bytes(uint32_t m, uint32_t n, uint32_t split_k);

/* Implicit-GEMM int8 convolution: replaces the im2col_quantize_int8.glsl +
 * linear_int8_tiled.glsl pair of VulkanOperators::conv2d_int8
 * (src/operators.cpp:1735-1805) for kernel 3 / stride 1 / padding 1 and
 * kernel 1 / stride 1 / padding 0, channels % 64 == 0, out_channels % 32 == 0
 * (dav2_hip_conv2d_i8_supported). Same output bits as
 * dav2_hip_im2col_quantize_i8 followed by dav2_hip_gemm_i8 with
 * DAV2_GEMM_EPI_TRANSPOSED; the im2col matrix is never stored. The weights are
 * the GpuModel int8 rows packed by dav2_hip_conv_weights_pack: K walked
 * tap-major (k = (ky*k + kx)*channels + c holds src[n][c*k*k + ky*k + kx])
 * and cut into 16-row x 64-byte MFMA operand fragments, fragment (rows
 * 16 nb.., K step ks) at byte (nb * K/64 + ks) * 1024, lane l's 16 bytes at
 * + 16 l (row 16 nb + l % 16, K bytes 64 ks + 16 (l / 16) ..). Needs
 * out_channels % 16 == 0 and kernel*kernel*channels % 64 == 0. */
enum {
    DAV2_CONV_RELU_INPUT = 1,   /* convolve max(input, 0) (relu.glsl before the conv)  */
    DAV2_CONV_RELU_OUTPUT = 2,  /* out = max(out, 0) after the residual (relu.glsl)     */
    /* Also write the next convolution's per-pixel channel-group maxima of the
     * output into partial_out ([out_channels/32][height*width], the layout of
     * the scratch): |out| (EMIT_ABSMAX) or max(out, 0) (EMIT_RELU_MAX, for a
     * consumer that applies DAV2_CONV_RELU_INPUT). Needs out_channels / 32
     * groups that each lie in one wave's channels (dav2_hip_conv2d_i8_emits). */
    DAV2_CONV_EMIT_ABSMAX = 4,
    DAV2_CONV_EMIT_RELU_MAX = 8
};

typedef struct dav2_conv_i8_args {
    const float* input;          /* CHW [channels][height][width]                  */
    uint32_t width, height, channels;
    uint32_t kernel;             /* 1 or 3                                         */
    const int8_t* weight;        /* packed (dav2_hip_conv_weights_pack)            */
    const float* weight_scales;  /* [out_channels]                                 */
    const float* bias;           /* [out_channels] or NULL = 0                     */
    uint32_t out_channels;
    float* out;                  /* CHW [out_channels][height][width]              */
    float* scratch;              /* dav2_hip_im2col_scratch_floats() floats        */
    uint64_t scratch_floats;
    uint32_t flags;              /* DAV2_CONV_*                                    */
    const float* residual;       /* NULL, or CHW like out: out = conv + residual   */
    /* The input's channel-group maxima (|x|, or max(x, 0) with RELU_INPUT)
     * when a producer has already written them (an EMIT flag or
     * dav2_hip_bilinear_align_true_maxima); NULL: computed into scratch. */
    const float* partial_in;
    float* partial_out;          /* with an EMIT flag                              */
} dav2_conv_i8_args;

DAV2_API int dav2_hip_conv2d_i8_supported(uint32_t width, uint32_t height, uint32_t channels,
                                          uint32_t out_channels, uint32_t kernel, uint32_t stride,
                                          uint32_t padding);
/* Nonzero if a supported convolution to out_channels can also emit its
 * output's channel-group maxima (DAV2_CONV_EMIT_*). No reference
 * counterpart (a fusion of channel_group maxima into the producer). */
DAV2_API int dav2_hip_conv2d_i8_emits(uint32_t out_channels, uint32_t kernel);
DAV2_API int dav2_hip_conv_weights_pack(int8_t* dst, const int8_t* src, uint32_t out_channels,
                                            uint32_t channels, uint32_t kernel, uint64_t ldb,
                                            void* stream);
DAV2_API int dav2_hip_conv2d_i8(const dav2_conv_i8_args* args, void* stream);

/* Implicit-GEMM fp32 conv2d of the fp32 / fp16 modes (src/operators.cpp:
 * 1528-1676): kernel 3 / stride 1 / padding 1 with channels % 4 == 0, kernel 1
 * / stride 1 / padding 0 with channels % 16 == 0
 * (dav2_hip_conv2d_f32_supported). weight [out_channels][channels*k*k], 16-byte
 * aligned; flags DAV2_CONV_RELU_INPUT / RELU_OUTPUT; out must not overlap
 * input (it may be the residual). */
typedef struct dav2_conv_f32_args {
    const float* input;          /* CHW [channels][height][width]                  */
    uint32_t width, height, channels;
    uint32_t kernel;             /* 1 or 3                                         */
    const float* weight;
    const float* bias;           /* [out_channels] or NULL = 0                     */
    uint32_t out_channels;
    uint32_t flags;
    float* out;                  /* CHW [out_channels][height][width]              */
    const float* residual;       /* NULL, or CHW like out: out = conv + residual   */
} dav2_conv_f32_args;
DAV2_API int dav2_hip_conv2d_f32_supported(uint32_t width, uint32_t height, uint32_t channels,
                                           uint32_t out_channels, uint32_t kernel, uint32_t stride,
                                           uint32_t padding);
DAV2_API int dav2_hip_conv2d_f32(const dav2_conv_f32_args* args, void* stream);

/* 1x1 convolution to a few output channels (out_channels <= 4, channels <=
 * 64), the DPT head's last layer (dpt.cpp:838-855 routed through the int8
 * convolution): same bits as dav2_hip_im2col_quantize_i8 + dav2_hip_gemm_i8
 * (DAV2_GEMM_EPI_TRANSPOSED), one thread per pixel. weight is the GpuModel
 * int8 layout [out_channels][ldw]. flags as above (no residual); pre_relu
 * (optional) receives the output before DAV2_CONV_RELU_OUTPUT. */
DAV2_API int dav2_hip_conv1x1_narrow_i8(const float* input, uint32_t width, uint32_t height,
                                        uint32_t channels, const int8_t* weight, uint32_t ldw,
                                        const float* weight_scales, const float* bias,
                                        uint32_t out_channels, float* out, float* pre_relu,
                                        uint32_t flags, void* stream);

/* Elementwise kernels. Reference: gelu.glsl, add_scaled.glsl, add.glsl, relu.glsl. */
DAV2_API int dav2_hip_gelu(float* out, const float* input, uint64_t count, void* stream);
DAV2_API int dav2_hip_add_scaled(float* out, const float* residual, const float* addend,
                                 const float* scale, uint64_t count, uint32_t columns,
                                 void* stream);
DAV2_API int dav2_hip_add(float* out, const float* left, const float* right, uint64_t count,
                          void* stream);
DAV2_API int dav2_hip_relu(float* out, const float* input, uint64_t count, void* stream);
/* Each float replaced by the nearest binary16 value (round to nearest even),
 * kept as a float: the fp16 mode's half weights, the reference's float_to_half
 * (src/gpu_model.cpp:51-98) applied on the device. */
DAV2_API int dav2_hip_round_half(float* data, uint64_t count, void* stream);

/* fp32 attention, head_dim 64, fused (the fp32 precision mode's path): scores,
 * softmax and values in one kernel, no score buffer, sums in the MFMA's order. qkv and
 * out [batch*T][H*64] 16-byte aligned. */
DAV2_API int dav2_hip_attention_f32(float* out, const float* qkv, uint32_t tokens, uint32_t heads,
                                    uint32_t batch, void* stream);

/* fp32 attention, head_dim 64, on the matrix cores over materialised scores,
 * for callers that want scores or probabilities; no precision mode uses these
 * (dav2_hip_attention_f32 is 3 to 4 times as fast)
 * (src/operators.cpp:1169-1208 with bmm.glsl and
 * softmax_lastdim.glsl, sums in the MFMA's order: within tolerance of the
 * reference, not bit for bit). qkv is [batch*T][3*H*64] token-major (q | k |
 * v, head h at h*64); scores [batch][H][T][T] fp32, softmax in place,
 * dav2_hip_attention_scratch_bytes() bytes. fp16 must be 0 (binary16 is
 * dav2_hip_attention_ref_*). */
DAV2_API uint64_t dav2_hip_attention_scratch_bytes(uint32_t tokens, uint32_t heads, uint32_t batch,
                                                   int fp16);
DAV2_API int dav2_hip_attention_scores(void* scores, const float* qkv, uint32_t tokens,
                                       uint32_t heads, uint32_t batch, int fp16,
                                       void* stream);
DAV2_API int dav2_hip_softmax_rows(void* scores, uint64_t rows, uint32_t columns,
                                   uint32_t row_stride, int fp16, void* stream);
DAV2_API int dav2_hip_attention_values(float* out, const void* probabilities,
                                       const float* qkv, uint32_t tokens, uint32_t heads,
                                       uint32_t batch, int fp16, void* stream);

/* Attention in the reference shaders' own arithmetic order (VALU): fp16 = 0
 * follows bmm.glsl + softmax_lastdim.glsl (fp32 scores [batch][H][T][T]),
 * fp16 = 1 follows bmm_score_fp16.glsl + softmax_lastdim_half.glsl +
 * bmm_value_fp16.glsl (binary16 scores packed as half2 words
 * [batch][H][T][ceil(T/2)], every product rounded to binary16). Scores and
 * values sum in feature / source-token order, the softmax over 128 lanes and
 * the halving tree, exp is exp_cw, the division IEEE: the CPU oracle's
 * orc_attention_head64 modes 0 and 1 give the same bits. Reference:
 * src/operators.cpp:1098-1209. Scratch: dav2_hip_attention_ref_scratch_bytes()
 * (the reference's score buffer size). The softmax works in place on rows of
 * `columns` scores. */
DAV2_API uint64_t dav2_hip_attention_ref_scratch_bytes(uint32_t tokens, uint32_t heads, uint32_t batch, int fp16);
DAV2_API int dav2_hip_attention_ref_scores(void* scores, const float* qkv, uint32_t tokens, uint32_t heads,
                                           uint32_t batch, int fp16, void* stream);
DAV2_API int dav2_hip_attention_ref_softmax(void* scores, uint64_t rows, uint32_t columns, int fp16, void* stream);
DAV2_API int dav2_hip_attention_ref_values(float* out, const void* probabilities, const float* qkv,
                                           uint32_t tokens, uint32_t heads, uint32_t batch, int fp16,
                                           void* stream);

/* The binary16 pipeline above (bmm_score_fp16.glsl, softmax_lastdim_half.glsl,
 * bmm_value_fp16.glsl) fused per block of query rows, the same bits as the
 * three kernels: keys and values are rounded to binary16 once into the
 * scratch (dav2_hip_attention_ref16_fused_scratch_bytes() bytes; 0 above
 * 2240 tokens, where the three kernels are faster: use them), then each
 * workgroup keeps its 16 rows' binary16 scores in LDS through the softmax
 * and the value sums. No reference counterpart as one
 * kernel; reference: src/operators.cpp:1132-1167. */
DAV2_API uint64_t dav2_hip_attention_ref16_fused_scratch_bytes(uint32_t tokens, uint32_t heads, uint32_t batch);
DAV2_API int dav2_hip_attention_ref16_fused(float* out, const float* qkv, uint32_t tokens, uint32_t heads,
                                            uint32_t batch, void* scratch, uint64_t scratch_bytes, void* stream);

/* The reference's int8-mode scores on devices with cooperative_matrix_fp16
 * (src/operators.cpp:1137-1148 selects bmm_score_coop_fp16.glsl:12-33):
 * binary16(q * 0.125) and binary16(k) operands, every product exact, the fp32
 * sums in the matrix unit's order (v_mfma_f32_16x16x32_f16, two K steps of
 * 32 features), each score stored as binary16 in the packed
 * [batch][H][T][ceil(T/2)] layout of dav2_hip_attention_ref_scores (fp16 = 1);
 * the softmax and values then run as above. The shader leaves the sum order
 * to the device, so these scores are held to the oracle's mode 3 (exact
 * products summed in double, rounded to fp32 and then binary16) within one
 * binary16 rounding, not bit for bit. */
DAV2_API int dav2_hip_attention_ref_scores_coop(void* scores, const float* qkv, uint32_t tokens, uint32_t heads,
                                                uint32_t batch, void* stream);
/* dav2_hip_attention_ref16_fused with the cooperative-matrix scores above
 * (same scratch); the same bits as dav2_hip_attention_ref_scores_coop +
 * _ref_softmax + _ref_values with fp16 = 1. */
DAV2_API int dav2_hip_attention_ref16_fused_coop(float* out, const float* qkv, uint32_t tokens, uint32_t heads,
                                                 uint32_t batch, void* scratch, uint64_t scratch_bytes,
                                                 void* stream);

/* Fused attention (int8-mode default): replaces the materialised binary16
 * path of src/operators.cpp:1132-1167 (bmm_score_fp16.glsl,
 * softmax_lastdim_half.glsl, bmm_value_fp16.glsl) with an integer-exact
 * kernel: q*0.125, k and v in 15-bit block floating point split into int8
 * digit planes, every dot product an exact int32 MFMA sum, 21-bit softmax
 * numerators, one rounding of the exact quotient per output. The result does
 * not depend on summation order. qkv and out as above; scratch holds the
 * digit planes, exponents and block maxima,
 * dav2_hip_attention_fused_scratch_bytes() bytes, 16-byte aligned. */
DAV2_API uint64_t dav2_hip_attention_fused_scratch_bytes(uint32_t tokens, uint32_t heads, uint32_t batch);
DAV2_API int dav2_hip_attention_fused(float* out, const float* qkv, uint32_t tokens, uint32_t heads,
                                      uint32_t batch, void* scratch, uint64_t scratch_bytes, void* stream);
/* The same attention for one image (batch 1) when the qkv GEMM ran with
 * DAV2_GEMM_EPI_ROW_COLMAX from column heads*64 on: col_absmax holds
 * [partial_rows][2*heads*64] maxima of |k| and |v| per column and row tile,
 * so the digit packing reads qkv once. Same output bits as
 * dav2_hip_attention_fused. No reference counterpart (a fusion). */
DAV2_API int dav2_hip_attention_fused_colmax(float* out, const float* qkv, uint32_t tokens, uint32_t heads,
                                             const float* col_absmax, uint32_t partial_rows, void* scratch,
                                             uint64_t scratch_bytes, void* stream);

/* bilinear_align_true.glsl:27-63, CHW. */
DAV2_API int dav2_hip_bilinear_align_true(float* out, const float* input,
                                          uint32_t input_width, uint32_t input_height,
                                          uint32_t output_width, uint32_t output_height,
                                          uint32_t channels, void* stream);
/* The same output bits, plus the per-pixel maxima of |out| over each group of
 * 32 channels into partial ([channels/32][output plane], channels % 32 == 0):
 * the input maxima of a following dav2_hip_conv2d_i8 (partial_in). No
 * reference counterpart (a fusion). */
DAV2_API int dav2_hip_bilinear_align_true_maxima(float* out, float* partial, const float* input,
                                                 uint32_t input_width, uint32_t input_height,
                                                 uint32_t output_width, uint32_t output_height,
                                                 uint32_t channels, void* stream);

/* reduce_minmax.glsl as a two-stage grid reduction; partials must hold
 * 2*dav2_hip_minmax_partials(count) floats. range[0] = min, range[1] = max. */
DAV2_API uint32_t dav2_hip_minmax_partials(uint64_t count);
DAV2_API int dav2_hip_reduce_minmax(const float* input, uint64_t count, float* range,
                                    float* partials, void* stream);
/* normalize_relative.glsl:8-16 */
DAV2_API int dav2_hip_normalize_relative(float* depth, const float* range, uint64_t count,
                                         void* stream);

/* Host-image paths (the reference runs them on the CPU around the tensor
 * inference; here they run on the device buffers of the image).
 * preprocess_bgr8: src/image.cpp:163-270 (dav2::preprocess_bgr8) -- bgr is
 *   height rows of `stride` bytes, 3 bytes (B, G, R) per pixel; out is the
 *   normalised RGB CHW float32 [3][dst_height][dst_width] of the cubic resize.
 * preprocess_bgra8_nearest: src/image.cpp:289-339
 *   (dav2::preprocess_inferbridge_bgra8) -- 4 bytes per pixel, stride and base
 *   4-byte aligned; model channel c is byte c of the pixel.
 * normalize_span: src/dav2.cpp:787-800 -- out = (depth - range[0]) /
 *   (range[1] - range[0]), or 0 everywhere when that span is not positive;
 *   range from dav2_hip_reduce_minmax. */
DAV2_API int dav2_hip_preprocess_bgr8(const uint8_t* bgr, uint32_t width, uint32_t height, uint64_t stride,
                                      uint32_t dst_width, uint32_t dst_height, float* out, void* stream);
DAV2_API int dav2_hip_preprocess_bgra8_nearest(const uint8_t* bgra, uint32_t width, uint32_t height,
                                               uint64_t stride, uint32_t dst_width, uint32_t dst_height,
                                               float* out, void* stream);
DAV2_API int dav2_hip_normalize_span(const float* depth, const float* range, uint64_t count, float* out,
                                     void* stream);
/* preprocess_rgba.glsl (src/gpu_preprocess.cpp:41-104, the resize of the
 * GPU submit path): 32-bit pixels, rgba_order 1 = R in byte 0 (RGBA8), 0 =
 * R in byte 2 (BGRA8); stride a multiple of 4 bytes; float32 cubic resize to
 * the normalised RGB CHW [3][dst_height][dst_width]. */
DAV2_API int dav2_hip_preprocess_rgba8(const uint32_t* pixels, uint32_t width, uint32_t height,
                                       uint64_t stride_bytes, uint32_t dst_width, uint32_t dst_height,
                                       uint32_t rgba_order, float* out, void* stream);

/* position_bicubic.glsl:76-105 with the set-up of src/operators.cpp:1323-1376:
 * position is the [1370][D] pos_embed, out is CHW [D][ph][pw]. */
DAV2_API int dav2_hip_position_bicubic(float* out, const float* position,
                                       uint32_t patch_width, uint32_t patch_height,
                                       uint32_t embedding, void* stream);
/* copy_class_token.glsl + add_position.glsl (src/operators.cpp:1299-1304,
 * :1389-1405) for batch images of T = pw*ph+1 tokens each: token 0 becomes
 * class_token + position[0..D), token t > 0 gets interpolated[f*pw*ph + t-1]
 * added. */
DAV2_API int dav2_hip_finish_tokens(float* tokens, const float* interpolated,
                                    const float* position, const float* class_token,
                                    uint32_t patch_width, uint32_t patch_height,
                                    uint32_t embedding, uint32_t batch, void* stream);

/* ---- operators of a decoder behind the encoder (no reference counterpart) ----
 *
 * Element types of their activations; sums, norms and softmax statistics are
 * fp32 whatever the type. A result is rounded once; the attentions also round
 * the softmax's weights on their way into the product with the values, as each
 * says below. */
enum { DAV2_DTYPE_F32 = 0, DAV2_DTYPE_F16 = 1, DAV2_DTYPE_BF16 = 2 };

/* Which features of a head form a rotated pair: i and i + rotary_dim/2
 * (HALVES), or 2i and 2i + 1 (PAIRS). */
enum { DAV2_ROTARY_HALVES = 0, DAV2_ROTARY_PAIRS = 1 };

/* Rotary positions: the first rotary_dim features of every head turned pair
 * by pair, (a, b) -> amplitude * (a cos t - b sin t, b cos t + a sin t) with
 * t = positions[token] * frequencies[i]; the others are copied. t is formed
 * and reduced to a turn in 64 bits, so far positions keep their angle.
 * Tokens are *_stride elements apart (at least heads * head_dim), heads
 * head_dim. output may be input with the same stride; it must not overlap it
 * otherwise. head_dim <= 1024; rotary_dim even, 2 .. head_dim. frequencies is
 * device memory: dav2_ops_rotary_frequencies() fills a host table. */
typedef struct dav2_rotary_args {
    const void* input;           /* [tokens][heads][head_dim]                      */
    void* output;
    uint64_t input_stride, output_stride;
    const int32_t* positions;    /* [tokens], any sign                             */
    const double* frequencies;   /* [rotary_dim / 2] radians per position          */
    uint32_t tokens, heads, head_dim, rotary_dim;
    uint32_t layout;             /* DAV2_ROTARY_*                                  */
    uint32_t dtype;              /* DAV2_DTYPE_* of input and output               */
    float amplitude;             /* 1 for a plain rotation                         */
} dav2_rotary_args;
DAV2_API int dav2_hip_rotary(const dav2_rotary_args* args, void* stream);

/* Norm of a head: x / sqrt(mean(x^2) + epsilon) * weight (RMS), or
 * (x - mean) / sqrt(variance + epsilon) * weight (LAYER). There is no bias. The
 * squares of a head's features are summed in fp32: the sum stays below 2^128. */
enum { DAV2_QK_NORM_RMS = 0, DAV2_QK_NORM_LAYER = 1 };

/* The norm of every query head and every key head over its head_dim
 * features, then the rotation of dav2_hip_rotary, in one pass over both.
 * weight [head_dim] fp32, NULL = ones. rotary_dim 0: the norm alone
 * (positions and frequencies unused). Query and key may be parts of one
 * packed row; an output may be its input with the same stride, and must not
 * overlap any input otherwise. query_heads or key_heads may be 0. */
typedef struct dav2_qk_norm_rotary_args {
    const void* query;           /* [tokens][query_heads][head_dim]                */
    const void* key;             /* [tokens][key_heads][head_dim]                  */
    void* query_out;
    void* key_out;
    uint64_t query_stride, key_stride, query_out_stride, key_out_stride;
    const float* query_weight;
    const float* key_weight;
    const int32_t* positions;
    const double* frequencies;
    uint32_t tokens, query_heads, key_heads, head_dim, rotary_dim;
    uint32_t layout, dtype;
    uint32_t norm;               /* DAV2_QK_NORM_*                                 */
    float epsilon;               /* > 0                                            */
    float amplitude;
} dav2_qk_norm_rotary_args;
DAV2_API int dav2_hip_qk_norm_rotary(const dav2_qk_norm_rotary_args* args, void* stream);

/* A key/value cache in 8 bits: pages of page_size tokens, and in each page one
 * scale per head for its keys and one for its values; a code c stands for
 * c * scale. Values are held feature-major, so that the keys of one feature
 * are contiguous. page_size a multiple of 16 up to 256, head_dim a multiple
 * of 16 up to 128, kv_heads up to 32767; keys and values 16-byte aligned. Sequence s owns the pages
 * page_table[s][0], [1], ...: token t is slot t % page_size of page
 * page_table[s][t / page_size]. A table entry outside [0, pages) is no page:
 * nothing is stored there and its tokens are not seen. Pages need no
 * clearing before their first use. */
typedef struct dav2_cache_i8 {
    int8_t* keys;                /* [pages][kv_heads][page_size][head_dim]         */
    int8_t* values;              /* [pages][kv_heads][head_dim][page_size]         */
    float* key_scales;           /* [pages][kv_heads]                              */
    float* value_scales;         /* [pages][kv_heads]                              */
    uint32_t pages, kv_heads, page_size, head_dim;
} dav2_cache_i8;

/* Stores new tokens. Rows starts[s] .. starts[s+1] of keys and values become
 * the last tokens of sequence s, which holds lengths[s] tokens after the call.
 * A page's scale is the larger of what it was (if older tokens are in the
 * page) and max(absmax of its new rows / 127, 1e-8), codes are x / scale
 * rounded half to even, and where a scale grows the page's older codes are
 * rounded again: value = code * old scale in fp32, code = rint(value / scale).
 * Storing the same rows at the same lengths again changes nothing. A NaN or
 * infinity makes the scale of its page NaN or infinite, and with it the
 * page's values, until the page is begun anew. starts must not decrease; rows
 * outside [0, tokens) and positions outside the table are not stored. Pages
 * that get tokens must belong to one sequence only, once; a sequence without
 * new rows may name any. Other bytes of the cache are left as they were.
 * max_new 0 says that nothing is new: nothing is stored. sequences stays below
 * 2^16. */
typedef struct dav2_cache_store_i8_args {
    dav2_cache_i8 cache;
    const void* keys;            /* [tokens][kv_heads][head_dim]                   */
    const void* values;
    uint64_t key_stride, value_stride;  /* elements between tokens                 */
    const int32_t* page_table;   /* [sequences][table_pages]                       */
    const int32_t* starts;       /* [sequences + 1]                                */
    const int32_t* lengths;      /* [sequences]                                    */
    uint32_t sequences, table_pages, tokens;
    uint32_t max_new;            /* most new tokens of a sequence: sizes the launch */
    uint32_t dtype;
} dav2_cache_store_i8_args;
DAV2_API int dav2_hip_cache_store_i8(const dav2_cache_store_i8_args* args, void* stream);

/* softmax(scale * q k^T) v over a cache: query rows starts[s] .. starts[s+1] are
 * the last tokens of sequence s, of lengths[s] tokens in all. causal: row i of n
 * sees the first lengths[s] - n + 1 + i tokens; otherwise all. heads is a
 * multiple of kv_heads; head h reads head h / (heads / kv_heads) of the cache. A
 * row that sees nothing gives zeros; output rows of no sequence are left as they
 * were. Scales of pages are not negative, and a value scale below 2^-80 counts
 * as that. Scores stay below 2^127 in size, with the scale and without. A query
 * row enters its product as binary16 times a power of two (exact for f16 and
 * bf16; f32: two parts, 22 bits), a weight as binary16 (11 bits down to 2^-27 of
 * the largest) or, in f32 and where a call has few rows, as two parts (22 bits).
 * tokens * heads stays below 2^32 - 512, sequences * kv_heads below 2^23,
 * sequences below 2^16. Strides (elements between tokens) are multiples of 8,
 * query and output 16-byte aligned; output overlaps no input. max_query and
 * max_length, the most new and the most tokens of a sequence, size the launch
 * and the scratch; a sequence beyond them is still computed (max_query 0 says
 * that there are no rows: nothing is). One way of dealing out the work is chosen
 * for a call by them: prompts and single tokens over long caches are better two
 * calls, as the tokens of a mixed one walk their caches alone. scratch:
 * dav2_hip_attention_cache_i8_scratch_bytes() bytes (0: none), 16-byte aligned,
 * in use until the call's work is done. That number depends on the sizes, never
 * on the pointers. */
typedef struct dav2_attention_cache_i8_args {
    dav2_cache_i8 cache;
    const void* query;           /* [tokens][heads][head_dim]                      */
    void* output;
    uint64_t query_stride, output_stride;
    const int32_t* page_table;   /* [sequences][table_pages]                       */
    const int32_t* starts;       /* [sequences + 1]                                */
    const int32_t* lengths;      /* [sequences]                                    */
    uint32_t sequences, table_pages, tokens, heads;
    uint32_t max_query, max_length;
    uint32_t causal, dtype;
    float scale;
    void* scratch;
    uint64_t scratch_bytes;
} dav2_attention_cache_i8_args;
DAV2_API uint64_t dav2_hip_attention_cache_i8_scratch_bytes(const dav2_attention_cache_i8_args* args);
DAV2_API int dav2_hip_attention_cache_i8(const dav2_attention_cache_i8_args* args, void* stream);

/* softmax(scale * q k^T) v of queries against keys and values of another length
 * (an encoder's tokens), batch by batch. Key j of batch b is seen if j <
 * key_lengths[b] (NULL: key_tokens) and key_mask[b][j] != 0 (NULL: all); what is
 * not seen may hold anything, NaN included. A batch that sees nothing gives
 * zeros. Scores stay below 2^127 in size, with the scale and without. Weights
 * are rounded to the tensors' type for the product with the values, f16 ones to
 * 11 bits down to 2^-27 of the largest. heads is a multiple of kv_heads; head h
 * reads key head h / (heads / kv_heads). head_dim a multiple of 16 up to 128;
 * strides in elements, multiples of 8, those of the inputs between batches may
 * be 0; the four tensors 16-byte aligned; output overlaps no input, nor a
 * batch's output another's. batch stays below 2^16, batch * query_tokens * heads
 * below 2^32 - 256, batch * kv_heads below 2^23. scratch as for
 * dav2_hip_attention_cache_i8; its size goes by the sizes alone, a key mask's
 * part included. A call without a mask whose keys are not split touches none and
 * may leave it NULL. */
typedef struct dav2_cross_attention_args {
    const void* query;           /* [batch][query_tokens][heads][head_dim]         */
    const void* keys;            /* [batch][key_tokens][kv_heads][head_dim]        */
    const void* values;          /* like keys                                      */
    void* output;                /* like query                                     */
    uint64_t query_stride, key_stride, value_stride, output_stride;  /* between tokens */
    uint64_t query_batch_stride, key_batch_stride, value_batch_stride, output_batch_stride;
    const int32_t* key_lengths;  /* [batch] or NULL                                */
    const uint8_t* key_mask;     /* [batch][key_tokens] or NULL                    */
    uint32_t batch, query_tokens, key_tokens, heads, kv_heads, head_dim;
    uint32_t dtype;
    float scale;
    void* scratch;
    uint64_t scratch_bytes;
} dav2_cross_attention_args;
DAV2_API uint64_t dav2_hip_cross_attention_scratch_bytes(const dav2_cross_attention_args* args);
DAV2_API int dav2_hip_cross_attention(const dav2_cross_attention_args* args, void* stream);

/* A key/value cache in 4 bits: pages as dav2_cache_i8 has them, and one scale
 * for each token and head, for its keys and for its values. A code c of -7 .. 7
 * is held as c + 8 in half a byte and stands for c * scale (0 would be -8, which
 * is read but never stored). A key's features 2 i and 2 i + 1 are the low and
 * the high half of byte i. Values are held 16 tokens at a time, feature by
 * feature: the tokens 16 t + 2 i and 16 t + 2 i + 1 of a feature are byte i of
 * its eight. Limits as for dav2_cache_i8. */
typedef struct dav2_cache_i4 {
    uint8_t* keys;               /* [pages][kv_heads][page_size][head_dim / 2]     */
    uint8_t* values;             /* [pages][kv_heads][page_size / 16][head_dim][8] */
    float* key_scales;           /* [pages][kv_heads][page_size]                   */
    float* value_scales;         /* [pages][kv_heads][page_size]                   */
    uint32_t pages, kv_heads, page_size, head_dim;
} dav2_cache_i4;

/* Stores new tokens as dav2_hip_cache_store_i8 does, with its rules for rows,
 * positions, pages and sequences. A head of a token gets the scale
 * max(absmax / 7, 1e-8) and codes x / scale rounded half to even, quotients
 * being fp32. Older tokens keep their codes and scales: storing is exact in any
 * order and number of calls. A NaN or infinity makes the scale of its head and
 * token NaN or infinite, and with it those values and no others. Bytes of
 * other slots are left as they were. */
typedef struct dav2_cache_store_i4_args {
    dav2_cache_i4 cache;
    const void* keys;            /* [tokens][kv_heads][head_dim]                   */
    const void* values;
    uint64_t key_stride, value_stride;  /* elements between tokens                 */
    const int32_t* page_table;   /* [sequences][table_pages]                       */
    const int32_t* starts;       /* [sequences + 1]                                */
    const int32_t* lengths;      /* [sequences]                                    */
    uint32_t sequences, table_pages, tokens;
    uint32_t max_new;            /* most new tokens of a sequence: sizes the launch */
    uint32_t dtype;
} dav2_cache_store_i4_args;
DAV2_API int dav2_hip_cache_store_i4(const dav2_cache_store_i4_args* args, void* stream);

/* dav2_hip_attention_cache_i8 over a cache in 4 bits: its rules, limits, types,
 * hints and scratch, with scales of tokens in the place of scales of pages. A
 * token that a row does not see may have any scale, NaN included. A weight is
 * binary16 (11 bits) where a bf16 call has many rows, and two parts (22 bits)
 * else; with many rows of 16 bits a value's scale goes with its weight by
 * its logarithm, to 2^-20 of the weight for scales of 1e-8 to 2^32, 2^-18 for any. */
typedef struct dav2_attention_cache_i4_args {
    dav2_cache_i4 cache;
    const void* query;           /* [tokens][heads][head_dim]                      */
    void* output;
    uint64_t query_stride, output_stride;
    const int32_t* page_table;   /* [sequences][table_pages]                       */
    const int32_t* starts;       /* [sequences + 1]                                */
    const int32_t* lengths;      /* [sequences]                                    */
    uint32_t sequences, table_pages, tokens, heads;
    uint32_t max_query, max_length;
    uint32_t causal, dtype;
    float scale;
    void* scratch;
    uint64_t scratch_bytes;
} dav2_attention_cache_i4_args;
DAV2_API uint64_t dav2_hip_attention_cache_i4_scratch_bytes(const dav2_attention_cache_i4_args* args);
DAV2_API int dav2_hip_attention_cache_i4(const dav2_attention_cache_i4_args* args, void* stream);

/* What a step of a paged cache (of either width) needs, from what its sequences
 * hold and get, so that a captured step needs no host between its replays.
 *
 * added[s] >= 0: sequence s gets that many tokens, rows starts[s] .. starts[s+1]
 * of the step, rows of all sequences one after the other. Pages for them come
 * from the front of a ring of free ones: free_pages[(first + i) % pages] for i <
 * count, {first, count} = free_state, go in order to the sequences that need
 * any, in order. A sequence is served if it needs no page or if the pages that
 * it and the sequences before it need are there, if its tokens fit the table and
 * are below 2^31, and if the step's rows up to its last one fit `tokens`; one that
 * does not fit needs nothing. If served it has
 * length held[s] + added[s], and held_out[s] is that; if not, it gets no page,
 * has length 0, so that nothing is stored or seen in this step, and still holds
 * what it held. added[s] < 0: the sequence ends. Its pages go to the end of the
 * ring, for later calls (those beyond `pages` entries are dropped), its length
 * and held_out[s] are 0. Its table entries stay.
 *
 * Row r of sequence s, i-th of its new tokens: positions[r] = held[s] + i,
 * owners[r] = s, slots[r] = page * page_size + slot where it is stored, -1 where
 * it is not (not served, or the entry is no page). Rows of no sequence: 0, -1, -1.
 * starts end at `tokens` at the most. positions, owners and slots may be NULL.
 *
 * held counts below 0 are 0. free_state and the ring outside [0, pages) are
 * brought into it; a ring entry that is no page is handed out and is no page in
 * the table. The pages of a sequence belong to it alone. held_out may be held
 * and free_state_out free_state; other outputs overlap nothing. pages up to
 * 2^31 - 1, page_size 16 .. 256 in steps of 16, sequences below 2^16, tokens and
 * table_pages below 2^31; with sequences 0 nothing is written. scratch:
 * dav2_hip_cache_plan_scratch_bytes() bytes,
 * 16-byte aligned, in use until the call's work is done. */
typedef struct dav2_cache_plan_args {
    const int32_t* held;         /* [sequences]                                    */
    const int32_t* added;        /* [sequences]                                    */
    int32_t* page_table;         /* [sequences][table_pages], new pages are added  */
    int32_t* free_pages;         /* [pages]                                        */
    const int32_t* free_state;   /* [2]                                            */
    int32_t* held_out;           /* [sequences]                                    */
    int32_t* free_state_out;     /* [2]                                            */
    int32_t* starts;             /* [sequences + 1]                                */
    int32_t* lengths;            /* [sequences]                                    */
    int32_t* positions;          /* [tokens] or NULL                               */
    int32_t* owners;             /* [tokens] or NULL                               */
    int64_t* slots;              /* [tokens] or NULL                               */
    uint32_t sequences, table_pages, tokens, pages, page_size;
    void* scratch;
    uint64_t scratch_bytes;
} dav2_cache_plan_args;
DAV2_API uint64_t dav2_hip_cache_plan_scratch_bytes(const dav2_cache_plan_args* args);
DAV2_API int dav2_hip_cache_plan(const dav2_cache_plan_args* args, void* stream);

/* The residual's addition, the root-mean-square norm and rows in 8 bits:
 *   h = input + residual, rounded to the type (residual NULL: h = input);
 *   y = (h * f) * weight, f = 1 / sqrt(mean(h^2) + epsilon) over a row, formed in
 *       64 bits and rounded to fp32, each product fp32;
 *   sum = h, output = y rounded to the type;
 *   codes = y / scale rounded half to even, scale = max(absmax(y) / 127, 1e-8),
 *       as dav2_hip_quantize_rows_i8 has them, bytes [columns, code_stride) zero:
 *       the rows of dav2_hip_gemm_i8.
 * Each of sum, output and codes (with scales) is left out with NULL, not all
 * three. weight [columns] fp32, NULL = ones. A row with a NaN or infinity has NaN
 * in y; its codes mean nothing and its scale is NaN. Strides in elements, at
 * least columns; code_stride a multiple of 64, codes 16-byte aligned. sum and output
 * may each be input or residual with the same stride; they overlap nothing
 * otherwise. columns below 2^20, rows below 2^31. */
typedef struct dav2_add_rms_norm_args {
    const void* input;           /* [rows][columns]                                */
    const void* residual;        /* [rows][columns] or NULL                        */
    const float* weight;
    void* sum;                   /* [rows][columns] or NULL                        */
    void* output;                /* [rows][columns] or NULL                        */
    int8_t* codes;               /* [rows][code_stride] or NULL                    */
    float* scales;               /* [rows], with codes                             */
    uint64_t input_stride, residual_stride, sum_stride, output_stride, code_stride;
    uint32_t rows, columns;
    uint32_t dtype;              /* DAV2_DTYPE_* of input, residual, sum, output   */
    float epsilon;               /* > 0                                            */
} dav2_add_rms_norm_args;
DAV2_API int dav2_hip_add_rms_norm(const dav2_add_rms_norm_args* args, void* stream);

/* The next token of each row of logits. The tokens of a row stand in order of
 * their logits, the largest first, equal ones by index; of this order a prefix is
 * kept, its weights being e_i = exp((l_i - l_0) / temperature):
 *   min_p in (0, 1]: tokens with e_i >= min_p;
 *   top_k > 0: the first top_k;
 *   top_p < 1: of what these leave, those before which the sum of the weights
 *       is below top_p of the whole.
 * The first token always stays. The token drawn is the first at which the sum
 * of the kept weights is above uniform times the whole; its probability is its
 * weight over the whole. temperature <= 0 (or NaN) keeps the first token alone.
 * temperature NULL is 1 for all rows; top_k, top_p, min_p NULL or outside the
 * ranges above (NaN included) keep all; uniform is taken into [0, 1), NaN is 0.
 * A NaN logit counts as -infinity; such tokens are never drawn. Where +infinity is
 * the largest, tokens of it share the weight. A row without a finite logit and
 * without +infinity has token -1 and probability 0.
 *
 * Sums are integers: weights in units of 2^-s, s = min(46, 62 -
 * ceil(log2(vocabulary))), from 64-bit exponentials, so that a result does not
 * depend on their order; a token below 2^-s-1 of the first weighs nothing.
 * vocabulary 1 .. 2^20, rows below 2^16; logits of a row are contiguous, rows
 * logit_stride elements apart. scratch: dav2_hip_sample_scratch_bytes() bytes, from
 * rows, vocabulary and dtype alone, 16-byte aligned, in use until the call's work
 * is done. */
typedef struct dav2_sample_args {
    const void* logits;          /* [rows][vocabulary]                             */
    uint64_t logit_stride;
    const float* temperature;    /* [rows] or NULL                                 */
    const int32_t* top_k;        /* [rows] or NULL                                 */
    const float* top_p;          /* [rows] or NULL                                 */
    const float* min_p;          /* [rows] or NULL                                 */
    const float* uniform;        /* [rows], in [0, 1)                              */
    int32_t* tokens;             /* [rows]                                         */
    float* probabilities;        /* [rows] or NULL                                 */
    uint32_t rows, vocabulary, dtype;
    void* scratch;
    uint64_t scratch_bytes;
} dav2_sample_args;
DAV2_API uint64_t dav2_hip_sample_scratch_bytes(const dav2_sample_args* args);
DAV2_API int dav2_hip_sample(const dav2_sample_args* args, void* stream);

DAV2_API const char* dav2_hip_error_string(int error);

#ifdef __cplusplus
}
#endif

#endif /* DAV2_HIP_H */
