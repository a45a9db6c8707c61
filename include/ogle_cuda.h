/* ogle_cuda.h - C ABI of the B200 (sm_100a) backend for the OGLE graph runtime's
 * data-parallel hot path: conv2d family with fused bias/BN/activation, gemm,
 * pooling, elementwise, concat, layout conversion and the SSD box decoder and
 * post-process; and the operators of a language model's decoding step, of beam search over its paged cache, and of attention over
 * chosen pages of it.
 *
 * The reference runtime (kl456123/OGLE) has no foreign-function interface: each
 * operator's Kernel::Compute binds OpenGL textures and draws. Every entry point
 * below is what such a Compute (or a Context copy function) calls instead, and
 * its comment cites the reference code it replaces, by path inside that project.
 *
 * Conventions
 *  - All pointers are DEVICE pointers unless a name ends in _host.
 *  - Activations use ONE layout: [N][H][W][Cs] fp32 with Cs = channel stride in
 *    floats, Cs >= round_up(C,4) and Cs % 4 == 0. This is the byte layout of the
 *    reference's NHWC4 textures and of its ANY4 textures for 4-D shapes
 *    (ogl_runtime/opengl/core/tensor_format.cc:308-337). Lanes C..Cs-1 of a
 *    tensor produced here are zero unless a wider stride was requested for an
 *    in-place concat.
 *  - Every function enqueues work on `stream` and returns immediately. None
 *    allocates device memory, synchronises or aborts. Return value: OGLE_OK or
 *    a negative OgleStatus.
 *  - One host thread per device; calls for different streams/devices may run
 *    concurrently from different threads.
 */
#ifndef OGLE_CUDA_H_
#define OGLE_CUDA_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct CUstream_st* ogle_stream_t; /* == cudaStream_t */

typedef enum {
    OGLE_OK = 0,
    OGLE_ERR_INVALID = -1,     /* bad argument (shape, stride, null pointer) */
    OGLE_ERR_UNSUPPORTED = -2, /* outside what the reference defines          */
    OGLE_ERR_CUDA = -3,        /* a CUDA runtime/driver call failed            */
    OGLE_ERR_ALIGNMENT = -4,   /* pointer or stride not 16-byte aligned        */
    OGLE_ERR_DEVICE = -5,      /* not an sm_100 device / no device             */
    OGLE_ERR_TIMEOUT = -6      /* a bounded device-side wait gave up           */
} OgleStatus;

/* Arithmetic used by the dense contractions (conv2d general/pointwise, gemm). */
typedef enum {
    OGLE_MATH_FP32 = 0,   /* CUDA-core fp32 FMA                                         */
    OGLE_MATH_TF32 = 1,   /* tcgen05 kind::tf32, one pass (10-bit mantissa operands)    */
    OGLE_MATH_TF32X3 = 2  /* hi/lo operand split, three products (one TF32 pass + one BF16
                             pass of the two cross terms): fp32-grade results           */
} OgleMathMode;

typedef enum { OGLE_ACT_NONE = 0, OGLE_ACT_CLIP = 1, OGLE_ACT_RELU = 2 } OgleActivation;

const char* ogle_cuda_status_string(int status);
/* Library version and the GPU architecture it was built for ("sm_100a"). */
const char* ogle_cuda_build_info(void);
/* Number of kernels this library has launched in this process (all streams). */
uint64_t ogle_cuda_launch_count(void);
/* Last CUDA error string seen by this library on the calling thread. */
const char* ogle_cuda_last_error(void);
/* Device-side status word of the kernels that wait for copies or multiplies: 0, or the code of the first
 * bounded wait that gave up (the launch then produced no valid output). Reading
 * synchronises the device; clear resets it. */
int ogle_cuda_device_status(void);
int ogle_cuda_clear_device_status(void);
/* The raw status word: which wait gave up (1 producer, 2 MMA issuer, 3 operand split,
 * 4 epilogue, 5 accumulator hand-back; 6 depthwise, 8 direct stem or fp32 contraction,
 * 9 paged attention); 0 when none did. Synchronises the
 * device. */
int ogle_cuda_device_status_detail(void);
/* Programmatic dependent launches for the kernels launched after this call (process-wide): each kernel's
 * prologue (barrier set-up, tensor-memory allocation, descriptor prefetch) may then run while its predecessor
 * on the stream drains; every kernel waits for its predecessor's results before its first global access. Pays
 * when the launches are short (5 % at one image per step, 1-4 % up to 16), costs 1-2 % when they are long: the
 * runtime turns it on for sessions whose tensors hold less than 1 GB. The environment variable OGLE_PDL (0/1), when set, overrides it.
 * ogle_cuda_gemm_ws overlaps its product with its own packing pass whatever is set here, ogle_cuda_paged_attention
 * its second launch and those that follow; OGLE_PDL=0 keeps those apart too.
 * Captured CUDA graphs keep what was in force when they were captured. */
int ogle_cuda_set_overlapped_launches(int on);

/* How the calling thread's latest contraction with packed filters (a convolution or gemm) was laid out, for tests and reports;
 * zeros before the first. */
typedef struct {
    int form;        /* 1 whole tiles; 2 ranges of the reduction combined through memory; 3 ranges added up inside a
                        cluster; 4 tiles on pairs of SMs; 5 channels on M; 6 taps of a filter row side by side; 7 whole tiles
                        of an RGB stem, its filters kept in shared memory; 8 few rows, on the CUDA cores; 9 an RGB stem
                        whose input window is the operand */
    int ranges;      /* ranges of the reduction (1 = not split) */
    int n_tile;      /* output channels of a tile (form 8: of a warp) */
    int overlapped;  /* 1: allowed to start its set-up while the launch before it drains */
} OgleContraction;
int ogle_cuda_last_contraction(OgleContraction* out);

/* How many times a role of the tensor-core kernels polls for its turn before it gives up, or, for its operands, a thread
 * of the fp32 contraction by the copy engine, a warp of the direct RGB stem or of paged attention, for the launches that follow on any stream
 * (process-wide). polls < 0 restores the default (2^22,
 * tens of milliseconds); 0 makes every such wait give up at once. It exists to exercise the
 * give-up path without a fault: a launch whose waits run out writes no valid output, sets the
 * status word, waits for its own copies and multiplies in flight (those waits keep the full
 * bound), frees its tensor memory and returns, and the device stays usable. No counterpart in
 * the reference, whose only failure handling is glGetError -> abort (utils/macros.cc:21-28). */
int ogle_cuda_set_wait_limit(long polls);

/* ------------------------------------------------------------------ conv2d */
/* Mirrors the uniform set of Conv2DKernel::Compute,
 * ogl_runtime/opengl/nn/kernels/conv2d.cc:116-167, plus the output placement
 * fields that let a producer write straight into a concat consumer. */
typedef struct {
    int N;
    int in_hwc[3];   /* H, W, C of the input   */
    int out_hwc[3];  /* Ho, Wo, K of the output */
    int kernel, stride, pad, dilation, group;
    int has_bias;
    int act;         /* OgleActivation */
    float min_value, max_value;
    int in_channel_stride;   /* floats per input pixel; 0 = round_up(C,4)   */
    int out_channel_stride;  /* floats per output pixel; 0 = round_up(K,4)  */
    int out_channel_offset;  /* first output channel lands here (mult of 4) */
    int math_mode;           /* OgleMathMode */
    int n_tile;              /* tensor-core path: output channels per tile (a multiple of 32, at most
                                256 and round_up(K,32)); 0 = chosen by the library. Results do not
                                depend on it bit for bit (each output value sums its reduction in the
                                same order: the ranges of `split` are settled without a look at it, or at
                                sm_pair); a caller may time the candidates and keep the fastest. Many-tile 3x3
                                layers of stride 1 have tiles of 32 or 64 channels whatever is asked for, the
                                taps of a filter row side by side; layers of a few pixels (form 8 of
                                OgleContraction) have none unless split is asked for, and 5x5 and 7x7 stems of up
                                to 64 channels whose window is the operand (form 9) never: those ignore split,
                                channels_on_m and sm_pair too. */
    int split;               /* tensor-core path: ranges the reduction is split into (1 = not split, up to
                                16); 0 = chosen by the library. Two to eight ranges of a launch of few tiles
                                are added up inside a cluster of SMs; any other number, and launches of more
                                tiles than such clusters fit, need the scratch of ogle_cuda_conv2d_ws, except
                                for two ranges without an activation. A number that cannot be served is
                                replaced by the library's own. Unlike n_tile this changes the order in which a
                                value's partial sums are added. */
    int channels_on_m;       /* tensor-core path, at most 128 output channels, unsplit reduction: 2 = keep the
                                accumulator transposed (filters on the 128-row side of the multiply, 256 pixels per
                                instruction), which halves the tensor-core instructions of layers with 64-128 output
                                channels; 1 = no, 0 = chosen by the library. Ignored where it cannot run. 1 and 2 give the
                                same bits: where it could run, neither lets the taps of a 3x3 layer lie side by side. */
    int sm_pair;             /* tensor-core path: 2 = compute tiles of 256 pixels on pairs of SMs (each SM of a
                                pair loads half of the filter tile; needs n_tile a multiple of 64 and an unsplit
                                reduction - chosen or asked for by split = 1 - else ignored, as it is by layers whose taps
                                lie side by side: see n_tile), 1 = one SM per tile, 0 = chosen by the library.
                                Results do not depend on it bit for bit. */
} OgleConvParams;

/* Output size rule of Conv2DKernel::InferOutputShape (conv2d.cc:169-195).
 * Fills p->out_hwc from the other fields. */
int ogle_cuda_conv2d_infer(OgleConvParams* p);

/* Bytes of the device-side packed filter for these parameters. */
size_t ogle_cuda_conv2d_filter_bytes(const OgleConvParams* p);

/* Re-lays an OIHW filter [K][C/group][k][k] (device) into the layout the conv
 * kernels read. Replaces the NCHW->HWN4C4 upload pass,
 * ogl_runtime/opengl/core/context.cc:123-154 with nchw_to_hwn4c4.glsl. Run once
 * per model, like the reference's "ready" pre-compute (fbo_session.cc:240-245). */
int ogle_cuda_conv2d_prepack(const OgleConvParams* p, const float* w_oihw, void* packed,
                             ogle_stream_t stream);

/* y = act(conv(x, w) + bias). Variant choice follows Conv2DKernel::SelectKernel
 * (conv2d.cc:19-51): pointwise, depthwise, grouped, general. Replaces
 * conv2d.glsl, conv2d_pw.glsl, conv2d_dw.glsl, conv2d_grp.glsl and their _any4
 * twins. bias: K floats (may be NULL when has_bias == 0). */
int ogle_cuda_conv2d(const OgleConvParams* p, const float* x, const void* packed_filter,
                     const float* bias, float* y, ogle_stream_t stream);

/* y = act(conv(x, w) + bias + residual): the convolution, the Add of a residual block and the activation that
 * follows it in one pass (replaces the binary.glsl pass of nn/kernels/binary.cc and, with act != none, the relu.glsl /
 * clip.glsl pass after it; same fp32 operations in the same order as the separate passes, so the result is bit-identical
 * to them where both sum the reduction in the same ranges: always with split = 1; by itself, a convolution without an
 * activation or with scratch may split where this one does not). residual: a tensor with the output's pixels, residual_stride floats per pixel (0 = round_up(K,4)), channel c of
 * the convolution at residual[pixel * residual_stride + c]. Served by the tensor-core path only
 * (ogle_cuda_conv2d_residual_supported: math_mode TF32 or TF32X3, >= 16 input channels); OGLE_ERR_UNSUPPORTED otherwise -
 * the caller then runs ogle_cuda_conv2d and ogle_cuda_add_act. */
int ogle_cuda_conv2d_residual_supported(const OgleConvParams* p);
int ogle_cuda_conv2d_residual(const OgleConvParams* p, const float* x, const void* packed_filter, const float* bias,
                              const float* residual, int residual_stride, float* y, ogle_stream_t stream);

/* The same with scratch memory lent by the caller (device memory, 16-byte aligned, at least
 * ogle_cuda_conv2d_workspace_bytes(p), which is 0 for most layers). Layers with a long reduction
 * and few output tiles - 3x3 heads on small feature maps, the whole network at batch 1 - then split
 * their reduction over up to 16 blocks per tile: each block stores its partial tile into its own
 * slice of the scratch and a second small kernel adds the slices in a fixed order, then bias and
 * activation (bit-reproducible; any activation); or, up to eight ranges of a few tiles, the blocks of a
 * tile form a cluster and add up their partial tiles in that order by themselves, without the scratch.
 * Without scratch launches that do not fit such clusters split in two at most, and only without an activation. The scratch may be reused as soon as the stream has
 * passed this call. */
size_t ogle_cuda_conv2d_workspace_bytes(const OgleConvParams* p);
int ogle_cuda_conv2d_ws(const OgleConvParams* p, const float* x, const void* packed_filter, const float* bias,
                        float* y, void* workspace, size_t workspace_bytes, ogle_stream_t stream);

/* Name of the device kernel that ogle_cuda_conv2d (ogle_cuda_conv2d_pair, given the stacked filters' parameters) launches
 * for these parameters (for profiles and reports; "" when the parameters are invalid). "conv_tc2_kernel" stands for all
 * tensor-core forms of conv_tc2.cu and its two variants, conv_tc2_pair_kernel and conv_tc2_t_kernel, among which the scratch
 * lent decides too: OgleContraction tells those apart. */
const char* ogle_cuda_conv2d_kernel_name(const OgleConvParams* p);

/* Two convolutions that read the same input with the same window (kernel, stride,
 * pad, dilation, activation, group 1) as ONE pass over the input: the SSD box and
 * class heads, which the reference draws as two Conv2DKernel::Compute passes
 * (conv2d.cc:116-167) over the same feature map. The caller stacks the two OIHW
 * filters into one of out_hwc[2] = second_offset + K2 rows, where
 * second_offset = K1 rounded up to a multiple of 32 and the rows in between are
 * zero, packs it with ogle_cuda_conv2d_prepack under the same params, and stacks
 * the biases the same way. y_first receives channels [0, K1) as a tensor of K1
 * channels (padded to 4), y_second channels [second_offset, out_hwc[2]) as a tensor
 * of K2 channels. The arithmetic per output value is that of ogle_cuda_conv2d,
 * up to the order in which partial sums are added (the two forms may split a
 * long reduction into different numbers of ranges). Tensor-core modes only: ogle_cuda_conv2d_pair_supported says
 * whether these params are served (else run the two convolutions separately). */
int ogle_cuda_conv2d_pair_supported(const OgleConvParams* p);
int ogle_cuda_conv2d_pair(const OgleConvParams* p, const float* x, const void* packed_filter, const float* bias,
                          int first_channels, int second_offset, float* y_first, float* y_second,
                          ogle_stream_t stream);
/* ogle_cuda_conv2d_pair with scratch memory, as ogle_cuda_conv2d_ws. */
size_t ogle_cuda_conv2d_pair_workspace_bytes(const OgleConvParams* p, int first_channels, int second_offset);
int ogle_cuda_conv2d_pair_ws(const OgleConvParams* p, const float* x, const void* packed_filter, const float* bias,
                             int first_channels, int second_offset, float* y_first, float* y_second, void* workspace,
                             size_t workspace_bytes, ogle_stream_t stream);

/* -------------------------------------------------------------------- pool */
/* PoolKernel::Compute, ogl_runtime/opengl/nn/kernels/pool.cc:55-79 + pool.glsl.
 * type: 0 max (all-padding window gives 0), 1 average (divides by kernel^2,
 * padding included), 2 global average (kernel := H, requires H == W). */
typedef struct {
    int N;
    int in_hwc[3];
    int out_hwc[3];
    int kernel, stride, pad, type;
    int in_channel_stride, out_channel_stride; /* 0 = round_up(C,4) */
} OglePoolParams;
int ogle_cuda_pool_infer(OglePoolParams* p);
int ogle_cuda_pool(const OglePoolParams* p, const float* x, float* y, ogle_stream_t stream);

/* ------------------------------------------------------------- elementwise */
/* BatchNormKernel::Compute, nn/kernels/batchnorm.cc:30-78 + batchnorm.glsl:
 * (x-mean)/sqrt(var+eps)*gamma+beta, params are C floats each. */
int ogle_cuda_batchnorm(const float* x, const float* gamma, const float* beta, const float* mean,
                        const float* var, float* y, long pixels, int C, int channel_stride,
                        float eps, ogle_stream_t stream);
/* relu.glsl / clip.glsl / binary.glsl over n floats (n % 4 == 0). */
int ogle_cuda_relu(const float* x, float* y, long n, ogle_stream_t stream);
int ogle_cuda_clip(const float* x, float* y, long n, float lo, float hi, ogle_stream_t stream);
int ogle_cuda_add(const float* a, const float* b, float* y, long n, ogle_stream_t stream);
/* binary.glsl followed by relu.glsl or clip.glsl (a residual block's Add -> Relu) in one pass:
 * y = act(a + b), act an OgleActivation; bit-identical to the two passes. */
int ogle_cuda_add_act(const float* a, const float* b, float* y, long n, int act, float lo, float hi,
                      ogle_stream_t stream);

/* -------------------------------------------------------------------- gemm */
/* GemmKernel::Compute, nn/kernels/gemm.cc:25-65 + gemm.glsl:
 * Y[M,N] = alpha*A[M,K]*(transB ? B[N,K]^T : B[K,N]) + beta*C.
 * Row strides (lda, ldb, ldc, ldy, in floats) are round_up(cols,4) for the
 * reference's ANY4 layout. bias_mode: 0 none, 1 C is [M,N] (ldc), 2 C is [N]
 * broadcast over rows (the reference defines this only for M == 1). */
typedef struct {
    int M, K, N;
    int transB;
    float alpha, beta;
    int bias_mode;
    int lda, ldb, ldc, ldy;
    int math_mode; /* OgleMathMode */
} OgleGemmParams;
int ogle_cuda_gemm(const OgleGemmParams* p, const float* A, const float* B, const float* C,
                   float* Y, ogle_stream_t stream);

/* B operand re-laid for the tensor-core path: K-major [round_up(N,128)][round_up(K,32)]
 * split into hi (10 mantissa bits) and lo (remainder) halves. Like the conv filter
 * packing, it is done once for a constant B (the usual case: Gemm weights are model
 * constants) and replaces the ANY -> ANY4 upload pass of context.cc:135-141. */
size_t ogle_cuda_gemm_packed_b_bytes(const OgleGemmParams* p);
int ogle_cuda_gemm_pack_b(const OgleGemmParams* p, const float* B, void* packed, ogle_stream_t stream);
/* ogle_cuda_gemm with B given in packed form (math_mode TF32 or TF32X3; FP32 is
 * served from the raw B by ogle_cuda_gemm). */
int ogle_cuda_gemm_packed(const OgleGemmParams* p, const float* A, const void* packed_b, const float* C,
                          float* Y, ogle_stream_t stream);

/* ogle_cuda_gemm for a B that is NOT a constant (both operands produced at run
 * time): the tensor-core modes need B re-laid and split, so the caller lends
 * `workspace` (device memory, >= ogle_cuda_gemm_packed_b_bytes(p), 16-byte aligned).
 * The call packs B into it and multiplies, both on `stream`; the workspace may be
 * reused as soon as the stream has passed this call. */
int ogle_cuda_gemm_ws(const OgleGemmParams* p, const float* A, const float* B, const float* C, float* Y,
                      void* workspace, size_t workspace_bytes, ogle_stream_t stream);

/* ogle_cuda_gemm_ws with the packing scratch in a fixed device array inside the
 * library instead of a caller's workspace. It has no counterpart in the reference.
 * It allocates nothing, on any call: the scratch is a file-scope device array of
 * OGLE_GEMM_STATIC_MAX_BYTES. A problem whose packed B
 * (ogle_cuda_gemm_packed_b_bytes) is larger returns OGLE_ERR_UNSUPPORTED with the
 * sizes in ogle_cuda_last_error(); use ogle_cuda_gemm_ws then.
 * The first call on each device resolves the array's address (set-up; make it with
 * that device current and before any stream capture); later calls only launch.
 * All calls on a device share the one array: calls that may execute concurrently
 * (two streams without an event between them) race on it. Nothing in the array has
 * to be cleared between calls. */
#define OGLE_GEMM_STATIC_MAX_BYTES (8u << 20)
size_t ogle_cuda_gemm_static_max_bytes(void);
int ogle_cuda_gemm_static(const OgleGemmParams* p, const float* A, const float* B, const float* C, float* Y,
                          ogle_stream_t stream);

/* ------------------------------------------------------------------ concat */
/* ConcatKernel::Compute, nn/kernels/concat.cc:53-96 + concat_multi.glsl.
 * Shapes are 4-D (left-padded with 1s, as AmendShape does); last dimension of
 * every tensor is stored padded to a multiple of 4. One pass, each input read
 * once and written once. A NULL entry of the input array means that slice is already in
 * place (its producer wrote it there): it is neither read nor written. */
#define OGLE_MAX_CONCAT_INPUTS 16
typedef struct {
    int n_inputs;
    int axis;                                   /* 0..3 */
    int in_shapes[OGLE_MAX_CONCAT_INPUTS][4];
} OgleConcatParams;
int ogle_cuda_concat(const OgleConcatParams* p, const float* const* inputs_host_array,
                     float* y, ogle_stream_t stream);

/* -------------------------------------------------- layout / glue kernels */
/* ANY -> ANY4 / NHWC -> NHWC4 upload conversion and back
 * (Context::CopyCPUTensorToDevice / CopyDeviceTensorToCPU,
 * ogl_runtime/opengl/core/context.cc:123-185; any_to_any4.glsl, any4_to_any.glsl):
 * [rows][last] dense <-> [rows][stride] with zero fill. stride 0 = round_up(last,4). */
int ogle_cuda_pad4(const float* dense, float* padded, long rows, int last, int stride,
                   ogle_stream_t stream);
int ogle_cuda_unpad4(const float* padded, float* dense, long rows, int last, int stride,
                     ogle_stream_t stream);
/* Detector::Preprocess (examples/ssd/detector.cc:99-109) for one image: 8-bit BGR
 * (device memory, rows src_row_bytes apart) -> RGB, bilinear resize to
 * dst_h x dst_w with OpenCV's 8-bit INTER_LINEAR arithmetic (the cv::resize call
 * the reference makes), to float, minus mean_rgb; written as [dst_h][dst_w][4]
 * floats (the NHWC4 slot of one image of the network input; lane 3 = 0). */
int ogle_cuda_preprocess_bgr8(const unsigned char* bgr, int src_h, int src_w, int src_row_bytes,
                              float* dst_nhwc4, int dst_h, int dst_w, const float mean_rgb[3],
                              ogle_stream_t stream);
/* The same for n_images images in ONE launch. The images sit in one device byte buffer;
 * descs_device (device memory, n_images entries) says where each starts and how large it
 * is. Image i is written to dst_nhwc4 + i * dst_h * dst_w * 4. The sizes are not checked
 * on the device: the caller filled the table. */
typedef struct OgleImageDesc {
    long long offset;      /* byte offset of the image's first pixel in the buffer */
    int height, width;     /* pixels */
    int row_bytes;         /* distance between rows, >= 3 * width */
    int reserved;
} OgleImageDesc;
int ogle_cuda_preprocess_bgr8_batch(const unsigned char* bgr_base, const OgleImageDesc* descs_device, int n_images,
                                    float* dst_nhwc4, int dst_h, int dst_w, const float mean_rgb[3],
                                    ogle_stream_t stream);
/* NCHW dense -> NHWC4 (for callers holding NCHW images). */
int ogle_cuda_nchw_to_nhwc4(const float* nchw, float* nhwc4, int N, int C, int H, int W,
                            ogle_stream_t stream);
/* TransposeKernel (nn/kernels/transpose.cc:73-90 + transpose_any4.glsl): 4-D
 * permute, out dim i = in dim perm[i]; both sides padded on their last dim. */
int ogle_cuda_transpose(const float* x, float* y, const int in_shape[4], const int perm[4],
                        ogle_stream_t stream);
/* ReshapeKernel / FlattenKernel (nn/kernels/reshape.cc:30-46 + reshape_any4.glsl):
 * same logical element order, different padded last dimension. */
int ogle_cuda_reshape(const float* x, float* y, long n_elements, int in_last, int out_last,
                      ogle_stream_t stream);
/* The same copy with its output rows laid out for a consumer that concatenates: output row r
 * is written at y + (r / rows_per_block) * block_stride + (r % rows_per_block) * round_up(out_last,4)
 * (floats; block_stride % 4 == 0). With rows_per_block = the rows one image contributes and
 * block_stride = the floats of one image in the concatenated tensor, the copy lands in its
 * slice of that tensor and the concat pass for it (concat.cc:73-96) is not needed. */
int ogle_cuda_reshape_placed(const float* x, float* y, long n_elements, int in_last, int out_last,
                             long rows_per_block, long block_stride, ogle_stream_t stream);

/* --------------------------------------------------------------------- SSD */
/* functor::SSDBBoxDecoder (ogl_runtime/opengl/core/functor.cc:96-143 +
 * decoder.glsl): pred [N][A][4] deltas, anchors [A][4] (cx,cy,w,h) shared by all
 * images, out [N][A][4] corners (xmin,ymin,xmax,ymax). */
int ogle_cuda_ssd_decode(const float* pred, const float* anchors, float* out, int N, int A,
                         const float variances[4], ogle_stream_t stream);

/* Detector post-process (ogl_runtime/opengl/examples/ssd/detector.cc:114-228):
 * the reference does this on the CPU after reading back boxes and logits.
 * mode 0 (reference rule): softmax, best foreground class per anchor, keep
 *   score > score_thr, top_k by score over the image (ties: lower anchor
 *   first), then the reference's greedy NMS on integer pixel rectangles when
 *   nms_thr > 0. Output rows per image: top_k.
 * mode 1 (per-class, standard SSD): softmax, per foreground class keep
 *   score > score_thr and the top_k by score. Output rows per image:
 *   (C-1)*top_k. No NMS.
 * logits [N][A][logit_stride] (logit_stride >= C); boxes [N][A][4] corners.
 * Outputs (device): out_score [N][rows] (0 where empty), out_anchor [N][rows]
 * (-1 where empty), out_class [N][rows], out_box [N][rows][4] (mode 0: integer
 * pixel rect x,y,w,h as floats; mode 1: the corner box), out_count [N] (mode 0)
 * or [N][C-1] (mode 1). */
typedef struct {
    int N, A, C;
    int logit_stride;
    int mode;
    float score_thr;
    int top_k;       /* <= 256 */
    float nms_thr;   /* mode 0 only; <= 0 disables NMS */
    int image_w, image_h; /* mode 0: scale to pixels */
    /* mode 0, optional (NULL = every image is image_w x image_h): device table of n
     * entries whose width/height give the pixel size of image n's ORIGINAL frame. The
     * reference scales boxes by the raw frame it was handed, not by the network input
     * (origin_input_sizes_, detector.cc:102,179-180), so frames of different sizes in one
     * batch need their own scale. Only width and height of an entry are read. */
    const OgleImageDesc* frame_sizes;
} OgleDetectParams;
int ogle_cuda_ssd_detect(const OgleDetectParams* p, const float* logits, const float* boxes,
                         float* out_score, int* out_anchor, int* out_class, float* out_box,
                         int* out_count, ogle_stream_t stream);
/* ogle_cuda_ssd_decode followed by ogle_cuda_ssd_detect in one pass: pred [N][A][4] deltas and anchors [A][4] instead
 * of boxes. Only the boxes of selected anchors are decoded, by the same arithmetic. */
int ogle_cuda_ssd_decode_detect(const OgleDetectParams* p, const float* logits, const float* pred, const float* anchors,
                                const float variances[4], float* out_score, int* out_anchor, int* out_class,
                                float* out_box, int* out_count, ogle_stream_t stream);

/* --------------------------------------------------- language-model steps */
/* What a decoding step of a language model needs beside the products above: new keys and values into a paged cache held
 * in 8 bits, attention over that cache, and the adjustment of logits before a token is chosen. The reference, a graph
 * runtime for image networks, has no counterpart. Activations are in 32 or 16 bits with strides of their own (no padding
 * to 4). */
typedef enum { OGLE_F32 = 0, OGLE_F16 = 1, OGLE_BF16 = 2 } OgleDataType;

/* A batch of sequences and the cache their keys and values lie in.
 * Cache: e4m3 bytes, page p, key/value head h, token t of the page, element d at
 * p * page_stride + h * head_stride + t * token_stride + d (bytes; the same for keys and values; multiples of 16). One scale
 * for each page and head, a power of two, or 0: value = e4m3 * scale[p * kv_heads + h].
 * Token j of sequence b lies in page block_table[b * table_stride + j / page_tokens]. A page of a sequence that is
 * appended to belongs to that sequence alone; full pages may be shared. An entry outside [0, n_pages) names no page:
 * nothing is stored there, and its tokens are not attended.
 * Rows: sequence b has rows row_start[b] .. row_start[b + 1] of the call's q, k, v and out, the last of the kv_len[b] tokens
 * it has once they are appended: row i of n stands at position kv_len[b] - n + i. row_start NULL: one row a sequence.
 * The host gives bounds of what the device holds, so that nothing waits for it: max_rows (rows of a sequence) and
 * max_kv_len. Rows of a sequence behind its first max_rows are ignored, and tokens from position max_kv_len on: neither stored nor
 * attended; the others keep the positions that kv_len and row_start give them. Rows that no sequence has are ignored too. */
typedef struct {
    int n_seqs, n_rows;            /* sequences; rows of all of them */
    int max_rows, max_kv_len;
    int q_heads, kv_heads;         /* q_heads a multiple of kv_heads: query head h reads kv head h / (q_heads / kv_heads) */
    int head_dim;                  /* a multiple of 16, at most 256 */
    int page_tokens;               /* 16, 32, ... 1024: a power of two */
    int n_pages, table_stride;
    int dtype;                     /* OgleDataType of q, k, v and out */
    int reserved;
    long long page_stride, head_stride, token_stride;
    const int *row_start, *kv_len, *block_table;
    void *k_cache, *v_cache;
    float *k_scale, *v_scale;
} OglePagedBatch;

/* Stores the rows' keys and values in their pages and rotates keys and queries by their positions on the way.
 * Rotation of a pair (x1, x2) by row `position` of the table: (x1 c - x2 s, x2 c + x1 s), in fp32, with c = rotary[position][i],
 * s = rotary[position][rotary_dim / 2 + i]; the pairs are (x[i], x[i + rotary_dim / 2]), or neighbours with `interleaved`. Elements
 * from rotary_dim on stay as they are; rotary NULL rotates nothing.
 * A page's scale is the smallest power of two, but 2^-120 at least, with |x| <= 448 scale for what it has taken since its first slot
 * was last written, and 0 while that has been zeros alone; where a row needs a larger one, what is in the page is moved by the
 * exponent. An infinity is stored as the largest value, a NaN as NaN; neither counts for the scale.
 * q may be NULL (nothing to rotate); q_out may be q. A row that stands before the text (kv_len is less than the sequence's rows) has
 * q_out 0. Strides in elements, multiples of 16 bytes, elements side by side. */
typedef struct {
    const void *k, *v, *q;
    void* q_out;
    long long k_row, k_head, v_row, v_head, q_row, q_head, q_out_row, q_out_head;
    const float* rotary;           /* [rotary_rows][rotary_dim], rotary_rows >= max_kv_len */
    int rotary_dim;                /* a multiple of 8, at most head_dim */
    int rotary_rows;
    int interleaved;
    int reserved;
} OgleAppendParams;
int ogle_cuda_kv_append(const OglePagedBatch* batch, const OgleAppendParams* p, ogle_stream_t stream);

/* out[row][h] = sum_j softmax_j(scale q.k_j) v_j over the tokens j < kv_len of the row's sequence - with `causal` those up to the
 * row's own position, with window > 0 those after position - window. lse (may be NULL), [n_rows][q_heads]: the natural logarithm
 * of the sum of exponentials. A row without a token has out 0 and lse minus infinity. A token that a row does not attend does
 * not reach it, whatever its bytes are and however large its page's scales. Scores, statistics and sums are in fp32. Queries and
 * weights enter the products in fewer bits: as two 16-bit parts, 22 bits, for fp32 activations, and for 16-bit ones where no sequence can
 * have more than 8 rows x query heads of a kv head (max_rows); else as one, 11 bits, which a query of such a type has anyway. Of a
 * weight times its value's scale, what lies below 2^-24 of the row's largest such product may be lost; a weight below 2^-126 of the
 * row's largest is 0.
 * The caller lends `workspace` (>= ogle_cuda_paged_attention_workspace_bytes, 16-byte aligned); nothing in it has to be
 * cleared, and it may be reused once the stream has passed the call. Where no more than OGLE_ATTENTION_NO_WORKSPACE bytes are asked
 * for, nothing is read or written there. Strides in elements, multiples of 16 bytes. */
#define OGLE_ATTENTION_NO_WORKSPACE 64
typedef struct {
    const void* q;
    void* out;
    float* lse;
    long long q_row, q_head, out_row, out_head;
    float scale;
    int causal;
    int window;
    int reserved;
} OgleAttentionParams;
size_t ogle_cuda_paged_attention_workspace_bytes(const OglePagedBatch* batch, const OgleAttentionParams* p);
int ogle_cuda_paged_attention(const OglePagedBatch* batch, const OgleAttentionParams* p, void* workspace,
                              size_t workspace_bytes, ogle_stream_t stream);

/* y[r][t] from x = logits[r][t], in this order, each step rounded to fp32:
 *   x > 0 ? x / repetition[r] : x * repetition[r]      where t is among the row's tokens
 *   x - frequency[r] * n - presence[r]                  where t is n > 0 times among the row's tokens after its first prompt_len[r]
 *   x + bias_value[i]                                   where bias_token[i] == t (the last such i of the row's)
 *   minus infinity                                      where bit t % 32 of allowed[r * allowed_stride + t / 32] is 0 (a stride
 *                                                       of 0: one mask for all rows)
 * Row r's tokens are tokens[token_start[r]] .. tokens[token_start[r + 1]], its biases bias_start[r] .. bias_start[r + 1]; tokens
 * outside [0, vocab) are ignored. Any of tokens, bias_token, allowed and of the four row vectors may be NULL (no such step,
 * repetition 1, presence and frequency 0, no prompt). Row strides in elements; out may be logits where the types are the
 * same. out_dtype: dtype or OGLE_F32. */
typedef struct {
    int rows, vocab;
    int dtype, out_dtype;          /* OgleDataType */
    int n_tokens, n_biases;        /* entries of tokens and of bias_token: nothing behind them is read */
    long long logits_stride, out_stride, allowed_stride;
    const void* logits;
    void* out;
    const int *tokens, *token_start, *prompt_len;
    const float *repetition, *presence, *frequency;
    const int* bias_token;
    const float* bias_value;
    const int* bias_start;
    const unsigned* allowed;
} OgleLogitsParams;
int ogle_cuda_adjust_logits(const OgleLogitsParams* p, ogle_stream_t stream);

/* ------------------------------------------- searching over the paged cache */
/* The best continuations of a group of texts (the beams of a search) over all its beams and tokens. Row g * beams + b is beam b of group
 * g; its token t has the total
 *   scores[row] + x_t - log sum_u exp(x_u),    x = logits[row]
 * in 64 bits, where a NaN logit counts as minus infinity and plus infinity as the largest number of the logits' type. A logit of minus
 * infinity is no continuation; a beam whose score is not finite has none. scores NULL: 0 for all.
 * Of each group the `count` largest totals, in falling order, equal ones by beam, then by logit (where 64 bits have lost the difference) and
 * token, go to out_score (rounded to fp32), out_beam and out_token [n_groups][count]; behind the last there are minus infinity, -1, -1. Of
 * these the first `beams` whose token is none of ends[0 .. n_ends) go on: next_row (the parent's row, g * beams + out_beam), next_token and
 * next_score [n_groups][beams], filled up with -1, -1, minus infinity. (A count of beams * (1 + n_ends), of different end tokens, is enough
 * for all to go on.)
 * Exponentials are of fp32, but those of most rows' largest logits, and sums of 64 bits: the logarithm of a row's sum is within 2^-19 of
 * its value - that far off where thousands of equal logits far below the largest make up most of it -, most often within 2^-23. Beams of the
 * same largest logit whose logarithms are within 2^-18 of each other count as having the same sum.
 * n_groups * beams is 65535 at most. `workspace`: as above; what is in it need not outlive the call. */
typedef struct {
    int n_groups, beams, vocab, count;     /* count at most 128 */
    int dtype;                             /* OgleDataType of the logits */
    int n_ends;                            /* at most 1024 */
    long long logits_stride;
    const void* logits;
    const float* scores;
    const int* ends;
    float* out_score;
    int *out_beam, *out_token;
    int *next_row, *next_token;
    float* next_score;
} OgleBeamParams;
size_t ogle_cuda_beam_step_workspace_bytes(const OgleBeamParams* p);
int ogle_cuda_beam_step(const OgleBeamParams* p, void* workspace, size_t workspace_bytes, ogle_stream_t stream);

/* The block tables of the texts that go on, from those of the texts there were. New text i goes on from sequence parent[i] (-1, or any
 * number that is no sequence: from nothing) and is about to have tokens[i] more (tokens NULL: new_tokens each). Of its parent's
 * kv_len tokens
 *   full pages are shared;
 *   a last page that is not full stays with the first text that goes on from that parent, if refs says that nobody else has it; any other
 *   gets a page of its own, and copies[i] = (old page, new page, tokens in it) says what ogle_cuda_copy_pages has to bring there,
 * and pages are added until all its tokens have one. Entry i of copies is (-1, -1, 0) where there is nothing to copy. new_len[i] is the
 * length with the new tokens; entries of the new table behind the last page are -1. A block without a page (-1) in the parent's row
 * stays one; blocks from new_blocks on have no place in the table.
 * refs[page] counts the table entries that name a page, other tables' too; 0: free. new_refs has the counts after the old table's rows are
 * gone and the new ones are there, so that texts that end (no new one goes on from them) or were cut (kv_len is less than what the row has
 * pages for) give theirs back. Requests are served in the order of texts and blocks, the k-th with the k-th lowest page that is free in
 * refs; what a call frees the next can have. Where they run out the entry is -1.
 * state[0]: pages free in new_refs; state[1]: requests that found none. With any, the old table and refs are still good: the call can
 * be made again with fewer texts. New arrays must not overlap the old ones. Lengths below 0 count as 0. */
typedef struct {
    int n_old, n_new;
    int old_blocks, new_blocks;            /* columns */
    int page_tokens, n_pages;
    int new_tokens, reserved;
    long long old_stride, new_stride;
    const int *table, *kv_len;             /* [n_old][old_blocks], [n_old] */
    const int *parent, *tokens;            /* [n_new] */
    const int* refs;                       /* [n_pages] */
    int *new_table, *new_len, *new_refs;
    int* copies;                           /* [n_new][3] */
    int* state;                            /* [2] */
} OgleAdvanceParams;
size_t ogle_cuda_advance_pages_workspace_bytes(const OgleAdvanceParams* p);
int ogle_cuda_advance_pages(const OgleAdvanceParams* p, void* workspace, size_t workspace_bytes, ogle_stream_t stream);

/* Used pages to the front of the pool. With U pages in use (refs not 0), the k-th used page from U on moves to the k-th free one below
 * U, for the first n_copies of them: copies[k] = (page, new page, page_tokens), the rest (-1, -1, 0). The new table names the new pages
 * (new_table may be table), new_refs has their counts (it may not be refs). state[0]: U; state[1]: moves that are left. What is in the pages is
 * ogle_cuda_copy_pages' to move. Whatever names a page that moves has to be in this table. */
typedef struct {
    int n_seqs, blocks;
    int page_tokens, n_pages, n_copies, reserved;
    long long table_stride, new_stride;
    const int *table, *refs;
    int *new_table, *new_refs, *copies, *state;
} OgleCompactParams;
size_t ogle_cuda_compact_pages_workspace_bytes(const OgleCompactParams* p);
int ogle_cuda_compact_pages(const OgleCompactParams* p, void* workspace, size_t workspace_bytes, ogle_stream_t stream);

/* For each (source page, destination page, tokens) of copies, in every layer's cache: the first `tokens` tokens of all heads, keys and
 * values, and the page's scales - and bounds, where the layer has them. The other slots of the destination stay as they are. An entry that names a
 * page outside the cache is left out. No page may be the destination of two entries, or of one and the source of another.
 * Layers have their pages in the same strides (see OglePagedBatch); from a page's first byte to its last there are less than 2^36. */
typedef struct {
    void *k, *v;
    float *k_scale, *v_scale;              /* [n_pages][kv_heads] */
    signed char* bounds;                   /* [n_pages][kv_heads][2][head_dim], or NULL */
    float* bounds_scale;                   /* [n_pages][kv_heads] */
} OglePageTensors;
typedef struct {
    int n_copies, n_layers;
    int kv_heads, head_dim, page_tokens, n_pages;
    long long page_stride, head_stride, token_stride;
    const int* copies;
} OgleCopyPagesParams;
int ogle_cuda_copy_pages(const OgleCopyPagesParams* p, const OglePageTensors* layers_host_array, ogle_stream_t stream);

/* ---------------------------------- attention over chosen pages of the cache */
/* Bounds of the keys of every page that a row of the batch was appended to: bounds [n_pages][kv_heads][2][head_dim], the least and the
 * largest of the page's keys in every element as whole numbers, rounded away from each other, and their unit bounds_scale [n_pages]
 * [kv_heads]: value = bounds * bounds_scale. The unit is the page's scale times the smallest power of two t with |e4m3| <= 127 t. Of a page
 * those of its slots count that hold tokens of the sequence (positions below kv_len); a NaN does not count. To be called behind
 * ogle_cuda_kv_append, with its batch; pages that it does not touch keep their bounds. */
int ogle_cuda_page_bounds(const OglePagedBatch* batch, signed char* bounds, float* bounds_scale, ogle_stream_t stream);

/* For each row and kv head the `count` pages that its query heads attend, as blocks of the row's sequence (position / page_tokens):
 *   blocks [0, first) and the row's own block with the last - 1 before it, always (first + last at most count, last at least 1);
 *   of the others up to the row's own those with the largest scores, equal ones from the lowest.
 * chosen[row][head][0 .. count), rising, filled up with -1; a block without a page is never among them. Score of a page: the largest
 * over the head's group of query heads of
 *   sum_d (q_d > 0 ? q_d hi_d : q_d lo_d) * bounds_scale
 * where q are the row's queries as whole numbers, q / s rounded to the nearest (even) and cut at +-127, s the smallest power of two with
 * |q| <= 127 s over the group's heads (infinities and NaN count as 0). All of it is exact in fp32. For attention whose scale is positive,
 * and up to 256 query heads to a kv head. `workspace`: 16-byte aligned; nothing in it has to be cleared or kept. */
typedef struct {
    const void* q;
    long long q_row, q_head;
    const signed char* bounds;
    const float* bounds_scale;
    int* chosen;
    long long chosen_row, chosen_head;     /* strides */
    int count, first, last, reserved;
} OgleChooseParams;
size_t ogle_cuda_choose_pages_workspace_bytes(const OglePagedBatch* batch, const OgleChooseParams* p);
int ogle_cuda_choose_pages(const OglePagedBatch* batch, const OgleChooseParams* p, void* workspace, size_t workspace_bytes, ogle_stream_t stream);

/* ogle_cuda_paged_attention over chosen pages alone: a row's query heads of kv head h attend the tokens up to its position of the blocks
 * chosen[row][h][0 .. count), rising and filled up with -1 as ogle_cuda_choose_pages leaves them. p->causal is 1 and p->window 0. Results,
 * precision and workspace as there; a row that no block was chosen for has out 0 and lse minus infinity. */
typedef struct {
    const int* chosen;
    long long chosen_row, chosen_head;
    int count, reserved;
} OgleChosenPages;
size_t ogle_cuda_sparse_attention_workspace_bytes(const OglePagedBatch* batch, const OgleAttentionParams* p, const OgleChosenPages* c);
int ogle_cuda_sparse_attention(const OglePagedBatch* batch, const OgleAttentionParams* p, const OgleChosenPages* c, void* workspace,
                               size_t workspace_bytes, ogle_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* OGLE_CUDA_H_ */
