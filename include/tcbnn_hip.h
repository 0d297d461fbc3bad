/*
 * tcbnn_hip.h — C ABI of the MI355X (gfx950) binarized-network inference path.
 *
 * Every entry point replaces one piece of the CUDA reference's bit-matmul /
 * bit-convolution inference path (pnnl/TCBNN).  The citation on each
 * declaration names the reference function or method whose behaviour the
 * entry point reproduces.  The reference fuses its layers into one persistent
 * cooperative kernel (imagenet_resnet.cu:34-125); here every layer is one
 * stream-ordered launch, so a network is a host loop over *_forward calls on
 * one stream.
 *
 * Conventions
 *   - All data pointers are DEVICE pointers unless the name ends in _host.
 *   - `stream` is a hipStream_t passed as void* (NULL = the default stream).
 *   - Return value: 0 on success, a negative TCBNN_E* code otherwise.  No
 *     entry point ever calls exit(); tcbnn_last_error() returns a message for
 *     the calling thread.  (The reference prints and exits, utility.h:57-92;
 *     the C++ layer classes layered above this ABI keep that behaviour.)
 *   - Bit convention (kernel.cuh:168, param.h:60): bit = 1 <=> value >= 0
 *     (resp. >= threshold) <=> "+1"; element e of a group of 32 is bit (31-e)
 *     of its uint32 ("MSB first"); pad bits are 0 in both operands and the
 *     true K / Cin enters  K - 2*popc(a xor w).
 *
 * Engine layouts (device memory).  The batch index is innermost everywhere, so a
 * wavefront whose lanes are 64 consecutive images reads and writes contiguous runs:
 *   FC activations   : uint32 [KW128][B]          KW128 = 4*ceil(K/128) words per image
 *   conv activations : uint32 [H][W][CW][B]       CW    = ceil(C/32) words per (pixel,image)
 *   FC-ready conv out: uint32 [OH*OW*CW128][B]    feature order (y, x, c), c padded to 128
 *                                                 (kernel.cuh:798-808): an FC activation
 *   packed weights   : uint32 [NPAD32][KWTOT]     one row per output neuron/channel,
 *                                                 FC: KWTOT = KW128; conv: KWTOT = R*S*CW,
 *                                                 K index = (r*S+s)*32*CW + c; rows >= N are 0;
 *                                                 FC weights and 3x3 filters are followed by the
 *                                                 same words in the order the matrix-core kernels'
 *                                                 lanes load them (tcbnn_fc_weight_words,
 *                                                 tcbnn_conv_filter_words give the total)
 *   residual tensors : TCBNN_RES_I32: int32 [P][Q][ceil(O/4)][B][4]; TCBNN_RES_I16: int16
 *                      [P][Q][ceil(O/8)][B][8] for tensors whose values provably fit 16 bits;
 *                      TCBNN_RES_I12: per pixel and group of 16 channels uint32 [B][4] then
 *                      uint32 [B][2] (12 bits per value, 24 bytes per image) for tensors whose
 *                      values provably fit 12 bits (see "residual formats" below).  In every
 *                      format an image's group of 4 / 8 / 16 consecutive channels is one or two
 *                      contiguous pieces of 16 (or 16 + 8) bytes and consecutive images follow
 *                      each other; channels are padded to the group, not to 128
 *   fp32 stem input  : float  [B][3][H][W]        (kernel.cuh:620-625)
 * The reference's own tile-contiguous "FMT" layouts ([.../8][.../128][8][4],
 * kernel.cuh:170,222,650-660,798-815) are produced / consumed by the
 * *_to_reference_fmt / *_from_reference_fmt converters below.
 */
#ifndef TCBNN_HIP_H
#define TCBNN_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TCBNN_OK 0
#define TCBNN_EINVAL (-1)   /* bad shape / flag combination                  */
#define TCBNN_ENULL (-2)    /* required pointer is NULL (utility.h:84-92)    */
#define TCBNN_EHIP (-3)     /* HIP runtime error (utility.h:57-81)           */
#define TCBNN_EUNSUPPORTED (-4)

/* Inner-product engines.  AUTO is the process-wide default (FP4 matrix cores unless
 * changed by tcbnn_set_default_variant or the environment). */
#define TCBNN_VARIANT_AUTO 0
#define TCBNN_VARIANT_POPC 1      /* v_xor_b32 + v_bcnt_u32_b32 on the VALU   */
#define TCBNN_VARIANT_MFMA_I8 2   /* +-1 unpacked to int8, v_mfma_i32_32x32x32_i8 */
#define TCBNN_VARIANT_MFMA_F4 3   /* +-1 unpacked to FP4 E2M1, v_mfma_f32_32x32x64_f8f6f4 (exact: |sum| < 2^24) */

/* Residual storage formats.  The reference keeps residuals (pre-threshold sums, kernel.cuh:
 * 662-669, 818-824) as int32.  They are this path's dominant HBM traffic, and their magnitude
 * is bounded by construction: |first-layer sum| <= R*S*3*max|input|, and every bit
 * convolution adds at most Cin*R*S.  A tensor whose bound is <= 32767 may be stored as
 * int16 without changing a single value; the caller states the format per tensor and is
 * responsible for the bound (tcbnn_*_residual_bound compute it, the layer classes above
 * this ABI track it from the actual input data).  Producer and consumer must agree. */
#define TCBNN_RES_I32 0
#define TCBNN_RES_I16 1
/* 12 bits per value, for tensors whose bound is <= 2047 (the first layer's and the first stage's of a ResNet on
 * normalised images: they are the largest tensors of the path).  Groups of 16 channels: the 192-bit string that
 * holds value e (two's complement) at bits 12e..12e+11 is stored as words w0..w5, laid out per pixel and group as
 * uint32 [B][4] (w0..w3 of every image) followed by uint32 [B][2] (w4, w5): 24 bytes per image, pixel and group. */
#define TCBNN_RES_I12 2

/* ------------------------------------------------------------------ misc */
int tcbnn_abi_version(void);
/* Message of the last failing call on this thread ("" if none). */
const char* tcbnn_last_error(void);
/* Process-wide default for TCBNN_VARIANT_AUTO (also read once from the
 * environment variable TCBNN_VARIANT = popc | mfma_i8 | mfma_f4). */
int tcbnn_set_default_variant(int variant);
int tcbnn_get_default_variant(void);

/* ------------------------------------------------------------ geometry */
/* Derived conv geometry, identical in both reference conv constructors
 * (param.h:719-728, 897-906):
 *   pad = padding ? ((((H + s - H%s)/s - 1)*s + R - H)/2) : 0
 *   buf = padding ? ceil(H/s) : (H-R)/s + 1 ;  out = ceil(buf/pool)          */
int tcbnn_conv_pad(int in_size, int filter, int stride, int padding);
int tcbnn_conv_out(int in_size, int filter, int stride, int padding, int pool);

/* Word counts of the engine layouts above. */
size_t tcbnn_fc_act_words(int batch, int features);                    /* B*KW128          */
size_t tcbnn_conv_act_words(int height, int width, int batch, int ch); /* H*W*B*CW         */
size_t tcbnn_fc_weight_words(int in_features, int out_features);       /* NPAD32*KW128 rows + the lane-order copy, NPAD32*8*ceil(KW128/8) */
size_t tcbnn_conv_filter_words(int r, int s, int in_ch, int out_ch);   /* NPAD32*R*S*CW, x2 for 3x3 filters with
                                                                           Cin = 64/128/192/256/384/512: they carry a
                                                                           copy in MFMA lane order after the bit rows */
size_t tcbnn_inconv_filter_words(int r, int s, int in_ch, int out_ch); /* R*S*OPAD32*5     */
/* bytes of a residual tensor of `channels` channels in the given TCBNN_RES_* format */
size_t tcbnn_residual_bytes(int height, int width, int channels, int batch, int format);
/* Upper bound of |residual| of a first layer whose input satisfies |x| <= input_abs_max
 * (R*S*3 terms plus rounding slack), and of a bit convolution that adds its own
 * Cin*R*S to an injected residual bounded by injected_bound (0 if none).  INT32_MAX
 * when unknown (non-finite input_abs_max, overflow).  tcbnn_residual_format_for_bound:
 * TCBNN_RES_I16 when 0 <= bound <= 32767, else TCBNN_RES_I32.  tcbnn_residual_format_narrowest also
 * considers TCBNN_RES_I12: 0 <= bound <= 2047 and an even batch (its 128-bit pieces are then aligned).
 * tcbnn_inconv_residual_bound_of_input is the first layer's bound from the actual batch (HOST pointer,
 * float [batch][3][height][width]): the largest sum of |x| over any filter window, plus rounding slack;
 * far tighter than R*S*3*max|x| on real images, which is what lets the first stage use 12 bits. */
int tcbnn_inconv_residual_bound(int filter_height, int filter_width, float input_abs_max);
int tcbnn_inconv_residual_bound_of_input(const float* input_host, int batch, int height, int width,
                                         int filter_height, int filter_width, int stride_height,
                                         int stride_width, int padding);
/* max |x| over a HOST array (on a few host threads; +infinity if any value is NaN or infinite): the cheap first test of
 * a new first-layer batch against the recorded bound, before the window scan above. */
float tcbnn_host_abs_max(const float* values_host, size_t count);
/* Uploads of new input batches.  An uploader serves arrays of up to `bytes` bytes.  It holds pinned memory (at most
 * 64 MiB), with staged = 1 and from 4 MiB on device memory for one array, and shares a few worker threads with the
 * process's other uploaders; they end with the last one.  Where one of these cannot be had tcbnn_uploader_create returns
 * TCBNN_EHIP (a thread that cannot be started is done without), and a plain copy does the same work.  tcbnn_upload copies
 * `bytes` of HOST memory to the device, in the order of the null stream, and is complete when it returns.
 * tcbnn_upload_stage (an uploader created with staged = 1) copies an array of floats out of
 * HOST memory, takes max |x| on the way (as tcbnn_host_abs_max) and leaves the destination alone;
 * tcbnn_upload_commit then writes the staged array to `dst`.  Each call on one uploader excludes the others.  A stage and
 * its commit are two calls about the ONE array that an uploader keeps staged: the next stage replaces it from its first
 * byte on, and threads that share an uploader hold a lock of their own across the two. */
typedef struct tcbnn_uploader tcbnn_uploader;
int tcbnn_uploader_create(size_t bytes, int staged, tcbnn_uploader** out);
void tcbnn_uploader_destroy(tcbnn_uploader* uploader);
int tcbnn_upload(tcbnn_uploader* uploader, void* dst, const void* src_host, size_t bytes);
int tcbnn_upload_stage(tcbnn_uploader* uploader, const float* src_host, size_t count, float* abs_max);
int tcbnn_upload_commit(tcbnn_uploader* uploader, void* dst);
int tcbnn_conv_residual_bound(int input_channels, int filter_height, int filter_width, int injected_bound);
int tcbnn_residual_format_for_bound(int bound);
int tcbnn_residual_format_narrowest(int bound, int batch);

/* ------------------------------------------------- one-time weight packing */
/* fp32 [K][N] (param.h:58-59) -> packed [NPAD32][KW128], followed by the same words in the FP4 FC kernel's lane
 * order, uint32 [NPAD32/32][ceil(KW128/8)][64][4].  `packed` holds tcbnn_fc_weight_words(...) words; the FC and
 * output layers take only buffers written by this function.  Replaces PackFcWeight128FMT (param.h:44-63). */
int tcbnn_pack_fc_weight(const float* weight_kn, uint32_t* packed, int in_features,
                         int out_features, void* stream);
/* fp32 HWIO [R][S][C][O] (param.h:573-574) -> packed [OPAD32][R*S][CW] (+ the FP4 fragment copy
 * for the 3x3 shapes named at tcbnn_conv_filter_words).  `packed` holds
 * tcbnn_conv_filter_words(...) words.  Replaces PackFiltersByInChannels128FMT (param.h:560-581). */
int tcbnn_pack_conv_filter(const float* filter_hwio, uint32_t* packed, int r, int s, int in_ch,
                           int out_ch, void* stream);
/* fp32 HWIO [R][S][3][O] -> sign table uint32 [R*S][OPAD32][4]: entry c<3 is 0 if the
 * weight of input channel c is >= 0 and 0x80000000 otherwise (the bit the first layer
 * flips on the fp32 input, kernel.cuh:636-638); entry 3 is the sign pattern index
 * 4*neg0 + 2*neg1 + neg2.  A second table [R*S][OPAD32] follows with the patterns alone,
 * one per word.  Replaces PackFiltersByOutChannels32 (param.h:613-632). */
int tcbnn_pack_inconv_filter(const float* filter_hwio, uint32_t* packed, int r, int s, int in_ch,
                             int out_ch, void* stream);
/* fp32 +-1 matrix rows -> packed activation matrix, MSB first, batch (row) innermost:
 * out[k/32][row].  `rows` x `k` row-major input with leading dimension `ld`; k_words
 * words are written per row (zero padded).  Replaces BMMA_toBit32Row
 * (tensorcore_kernel.cu:87-97). */
int tcbnn_pack_rows(const float* src, uint32_t* packed, int rows, int k, int ld, int k_words,
                    void* stream);
/* fp32 [K][N] -> packed [N][k_words] (each column contiguous along K).  Replaces
 * BMMA_toBit32Col (tensorcore_kernel.cu:74-84). */
int tcbnn_pack_cols(const float* src, uint32_t* packed, int k, int n, int k_words, void* stream);
/* fp32 +-1 NHWC [B][H][W][C] -> packed [H][W][CW][B].  Replaces BTC_bin_input
 * (bmma_kernel.cu:73-98). */
int tcbnn_pack_conv_input_nhwc(const float* src, uint32_t* packed, int batch, int height,
                               int width, int ch, void* stream);

/* ------------------------------------------------------------ layer forward */
/* In128LayerFMT (kernel.cuh:153-172), descriptor fields of In128LayerParam
 * (param.h:210-218): fp32 [B][K] -> sign bits, FC activation layout. */
typedef struct tcbnn_in128_desc {
    const float* input;   /* [input_height][input_width] */
    uint32_t* output;     /* [KW128][B] */
    int input_height;     /* batch */
    int input_width;      /* features */
} tcbnn_in128_desc;
int tcbnn_in128_forward(const tcbnn_in128_desc* d, void* stream);

/* Fc128LayerFMT (kernel.cuh:174-226), fields of Fc128LayerParam (param.h:362-384):
 * bit[b][n] = ((float)K - 2*(float)popc(a_b xor w_n) >= bn[n]). */
typedef struct tcbnn_fc128_desc {
    const uint32_t* input;   /* [KW128(input_width)][B] */
    const uint32_t* weight;  /* tcbnn_pack_fc_weight output */
    const float* bn;         /* [weight_width] thresholds */
    uint32_t* output;        /* [KW128(weight_width)][B] */
    int input_height;        /* batch */
    int input_width;         /* K */
    int weight_width;        /* N */
    int variant;             /* TCBNN_VARIANT_* */
    int32_t* workspace;      /* optional int32 [NPAD32][B] scratch: lets small-batch layers
                                split K over workgroups; NULL = never split */
    size_t workspace_words;
} tcbnn_fc128_desc;
int tcbnn_fc128_forward(const tcbnn_fc128_desc* d, void* stream);
/* The same layer for callers that can neither allocate device memory nor hand over a workspace (code under
 * HIP graph capture, tight serving loops, harnesses that forbid hipMalloc).  NO counterpart in the
 * reference.  The split-K partial sums go to a buffer built into the library's code object (4 MiB of device
 * memory per GPU, held until the process ends); d->workspace and d->workspace_words are ignored.  The call
 * allocates and frees nothing, clears what it accumulates into with a fill kernel (no memset node), and gives
 * the same bits as tcbnn_fc128_forward.  Limits: PAD32(weight_width) * input_height <= 1048576 words, else
 * TCBNN_EINVAL; all calls on one GPU share the one buffer, so calls that overlap in time on one GPU (different
 * streams or threads) race - serialise them.  The buffer's device address is looked up on the first call per
 * device (hipGetSymbolAddress, which allocates nothing): make that first call outside a stream capture. */
int tcbnn_fc128_forward_static_scratch(const tcbnn_fc128_desc* d, void* stream);

/* Out128LayerFMT (kernel.cuh:230-280), fields of Out128LayerParam (param.h:506-530):
 * y[b][n] = ((float)K - (float)popc*2.0f)*bn_scale[n] + bn_bias[n], fp32 row major. */
typedef struct tcbnn_out128_desc {
    const uint32_t* input;
    const uint32_t* weight;
    const float* bn_scale;
    const float* bn_bias;
    float* output;           /* [B][weight_width] */
    int input_height, input_width, weight_width;
    int variant;
} tcbnn_out128_desc;
int tcbnn_out128_forward(const tcbnn_out128_desc* d, void* stream);

/* In128 (or NULL), n_fc Fc128 layers and Out128 (or NULL), one after the other: the same results, in every layer's
 * output, as the calls above in this order.  Layers that follow one another (each reads the output of the one before,
 * same batch, at most 2048 inputs and outputs, the FP4 engine) go in one launch, unless an output lies where another
 * layer of the run reads or writes: what shares memory is launched one by one.  Allocates nothing and needs no
 * workspace.  No counterpart in the reference (its network kernel runs all layers, kernel.cuh:153-280). */
int tcbnn_fc_chain_forward(const tcbnn_in128_desc* in, const tcbnn_fc128_desc* fc, int n_fc, const tcbnn_out128_desc* out,
                           void* stream);
/* The launches that tcbnn_fc_chain_forward makes of such a run: their number, and how many layers each takes (n_fc + 2
 * entries at most).  Several layers are joined where that is faster.  Launches nothing. */
int tcbnn_fc_chain_plan(const tcbnn_in128_desc* in, const tcbnn_fc128_desc* fc, int n_fc, const tcbnn_out128_desc* out,
                        int* layers, int* n_launches);

/* InConv128LayerFMT (kernel.cuh:578-672), fields of InConv128LayerParam
 * (param.h:841-869).  fp32 NCHW 3-channel input, +-1 filters, fp32 adds in the
 * reference order  acc += ((+-f0) + (+-f1)) + (+-f2)  per in-frame tap in (r,s)
 * raster order; bit = !((float)acc < bn[o]); OR-pool; residual = (int)acc.
 * save_residual requires pool 1x1 (the reference index by*output_width+bx,
 * kernel.cuh:666, is only meaningful then). */
#define TCBNN_INCONV_INPUT_NCHW 0   /* float [batch][3][H][W], the reference's device layout (kernel.cuh:620-625) */
#define TCBNN_INCONV_INPUT_PACKED 1 /* float [Hp][Wp][batch][3], zero-padded: see tcbnn_inconv_pack_input */
typedef struct tcbnn_inconv128_desc {
    const float* input;        /* device, in the layout `input_layout` names */
    const uint32_t* filter;    /* tcbnn_pack_inconv_filter output */
    const float* bn;           /* [output_channels] */
    uint32_t* output;          /* [OH][OW][CW(output_channels)][B] */
    int32_t* output_residual;  /* residual tensor in `residual_format`, or NULL */
    int input_height, input_width, input_channels;
    int filter_height, filter_width;
    int output_channels, batch;
    int stride_height, stride_width;
    int padding;               /* bool */
    int pool_height, pool_width;
    int save_residual;         /* bool */
    int residual_format;       /* TCBNN_RES_* of output_residual */
    int input_layout;          /* TCBNN_INCONV_INPUT_*; PACKED needs pool 1x1 */
} tcbnn_inconv128_desc;
int tcbnn_inconv128_forward(const tcbnn_inconv128_desc* d, void* stream);
/* The engine's own layout of the first layer's input: batch innermost like every other tensor, and zero-padded, so
 * that a lane (= image) reads the three channels of an input pixel as 12 contiguous bytes, a wavefront 768, and no
 * tap needs a test for the frame: float [Hp][Wp][batch][3] with Hp = (P - 1) * stride_height + filter_height,
 * Wp = (Q - 1) * stride_width + filter_width (P x Q = tcbnn_conv_out of the two dimensions, pool 1) and the frame's
 * pixel (0, 0) at (tcbnn_conv_pad(height...), tcbnn_conv_pad(width...)).  The reference reads [batch][3][H][W]
 * directly (kernel.cuh:620-625) and has no such step; here it belongs to the upload of an input
 * (InConv128LayerParam::initialize / set_input), not to the forward pass.  Both pointers are device pointers. */
size_t tcbnn_inconv_packed_input_floats(int batch, int height, int width, int filter_height, int filter_width,
                                        int stride_height, int stride_width, int padding);
int tcbnn_inconv_pack_input(const float* input, float* packed, int batch, int height, int width, int filter_height,
                            int filter_width, int stride_height, int stride_width, int padding, void* stream);

/* Conv128LayerFMT (kernel.cuh:676-827), fields of Conv128LayerParam (param.h:1028-1064).
 *   res = Cin*R*S - exclude*Cin - 2*popc                      (kernel.cuh:766-768)
 *   if inject_residual && o < residual_channels:
 *        res += residual_pool ? max_{i,j in {0,1}} Rin[2y+i][2x+j][b][o] : Rin[y][x][b][o]
 *                                                              (kernel.cuh:770-794)
 *   bit = !((float)res < bn[o]); OR over the pool window      (kernel.cuh:795-816)
 *   if save_residual: Rout[y][x][b][o] = res                  (kernel.cuh:818-824)
 * Channels o >= input_residual_channels of the source read as 0 (the reference
 * gets the same effect from its zero-filled 128-channel padding, param.h:979-980).
 * save_residual / inject_residual require pool 1x1, residual_pool requires the
 * source to be exactly twice the output size (as the reference indexing assumes).
 * output_residual_pool = 2 (no counterpart in the reference): Rout holds, per 2x2 window of output
 * pixels, the element-wise maximum of `res`: a P/2 x Q/2 x O tensor, i.e. exactly what a consumer
 * with residual_pool computes from the full tensor before it adds it (kernel.cuh:775-782), so that
 * consumer then injects it with residual_pool = 0.  A quarter of the bytes are written and read;
 * meant for a tensor whose every consumer pools.  Available where
 * tcbnn_conv128_pooled_save_supported says so (TCBNN_EUNSUPPORTED otherwise). */
typedef struct tcbnn_conv128_desc {
    const uint32_t* input;         /* [H][W][CW(input_channels)][B] */
    const uint32_t* filter;        /* tcbnn_pack_conv_filter output */
    const float* bn;               /* [output_channels] */
    uint32_t* output;              /* [OH][OW][CW(O)][B]; ahead_fc: [OH][OW][CW128(O)][B] */
    const int32_t* input_residual; /* source tensor (Hr x Wr x input_residual_channels) or NULL */
    int32_t* output_residual;      /* P x Q x O tensor or NULL */
    int input_height, input_width, input_channels;
    int filter_height, filter_width;
    int output_channels, batch;
    int stride_height, stride_width;
    int padding;
    int pool_height, pool_width;
    int ahead_fc, save_residual, inject_residual;
    int residual_channels;         /* inject only into o < residual_channels */
    int residual_pool;
    int input_residual_channels;   /* channel count of the source tensor */
    int variant;
    int input_residual_format;     /* TCBNN_RES_* of input_residual */
    int output_residual_format;    /* TCBNN_RES_* of output_residual */
    int output_residual_pool;      /* 0: P x Q x O tensor; 2: its 2x2 maximum, P/2 x Q/2 x O */
} tcbnn_conv128_desc;
int tcbnn_conv128_forward(const tcbnn_conv128_desc* d, void* stream);
/* 1 if the layer `d` describes can be run with output_residual_pool = 2 (whatever d->output_residual_pool says; no
 * pointer is dereferenced): the FP4 engine's 3x3 kernel on an un-pooled layer with even P and Q, output channels a
 * multiple of 64, a 12- or 16-bit injected residual whose channel limit is a multiple of 32, and a 12- or 16-bit
 * output format.  0 otherwise.  No counterpart in the reference. */
int tcbnn_conv128_pooled_save_supported(const tcbnn_conv128_desc* d);

/* Name of the device kernel (as a profiler lists it, template arguments included) that
 * the corresponding *_forward call would launch for this descriptor; no
 * launch happens and no pointer is dereferenced.  No counterpart in the reference
 * (its layers are inlined device functions of one network kernel); used to match
 * per-launch timings with profiler output. */
int tcbnn_conv128_kernel_name(const tcbnn_conv128_desc* d, char* buf, size_t len);
int tcbnn_fc128_kernel_name(const tcbnn_fc128_desc* d, char* buf, size_t len);
int tcbnn_out128_kernel_name(const tcbnn_out128_desc* d, char* buf, size_t len);
int tcbnn_inconv128_kernel_name(const tcbnn_inconv128_desc* d, char* buf, size_t len);

/* Measurement aid (no counterpart in the reference): one wavefront counts shader clock cycles over `microseconds` of
 * the device's constant-rate wall clock, on `stream`, while whatever else is queued on other streams runs beside it.
 * After the stream has been synchronised, counts[0] = shader cycles, counts[1] = wall-clock ticks (DEVICE pointer to
 * two 64-bit words); *wall_clock_khz = ticks per millisecond.  Shader MHz = counts[0] / counts[1] * khz / 1000. */
int tcbnn_shader_clock_probe(unsigned long long* counts, int microseconds, int* wall_clock_khz, void* stream);

/* ------------------------------------------------ layers of the textbook ResNet wiring */
/* The reference wires ResNet-18 without a pooling layer after the first convolution, without
 * convolutional shortcuts and without an average-pooling head (imagenet_resnet.cu:223-325).  The two
 * layers below have NO counterpart in the reference; together with a Conv128 layer of filter 1x1,
 * stride 2 and save_residual (the downsample shortcut) they let the same engine run the textbook wiring
 * (7x7/2 first layer + 3x3/2 max-pool, 1x1/2 shortcut convolutions, global average pool + fp32 FC).
 *
 * Overlapping pooling on a packed activation tensor and, optionally, its residual: every output bit is
 * the OR of the bits of its window (the maximum of the +-1 values), every output residual value the
 * maximum of the window's values; taps outside the frame are ignored.  Output size per dimension:
 * (in + 2*padding - window) / stride + 1.  The output residual has the input's format. */
typedef struct tcbnn_pool128_desc {
    const uint32_t* input;          /* device, conv activation layout [H][W][CW][B]                 */
    uint32_t* output;               /* device, [OH][OW][CW][B]                                      */
    const int32_t* input_residual;  /* device, residual layout with `channels` channels, or NULL    */
    int32_t* output_residual;       /* device, residual layout [OH][OW]..., or NULL                 */
    int input_height, input_width, channels, batch;
    int window, stride, padding;    /* square window; padding < window                              */
    int residual_format;            /* TCBNN_RES_* of both residual tensors                         */
} tcbnn_pool128_desc;
int tcbnn_pool_out(int in_size, int window, int stride, int padding);
int tcbnn_pool128_forward(const tcbnn_pool128_desc* d, void* stream);

/* Global average pool over the pixels of a residual tensor, then an fp32 fully connected layer:
 * mean[b][c] = (float)(sum over pixels of residual[p][c][b]) / (float)(height*width) (the sum is an exact
 * integer), out[b][n] = bias[n] + sum over c, in ascending order with fused multiply-add, of
 * mean[b][c] * weight[c][n].  channels <= 512. */
typedef struct tcbnn_avgpool_fc_desc {
    const int32_t* input_residual;  /* device, residual layout [H][W]... with `channels` channels   */
    const float* weight;            /* device, fp32 [channels][out_features] row major              */
    const float* bias;              /* device, fp32 [out_features]                                  */
    float* output;                  /* device, fp32 [batch][out_features] row major                 */
    int input_height, input_width, channels, batch, out_features;
    int residual_format;            /* TCBNN_RES_* of input_residual                                */
} tcbnn_avgpool_fc_desc;
int tcbnn_avgpool_fc_forward(const tcbnn_avgpool_fc_desc* d, void* stream);

/* ------------------------------------------------ float head of a network */
/* What a network computes in floating point after (or between) its binary layers, forward and backward: linear layers,
 * layer norms, and the log probabilities of its answers.  The library has no optimizer: a step on the gradients is the
 * caller's.  NO counterpart in the reference.
 *
 * Matrices are row major, `*_ld` elements from one row to the next (0: rows without gaps); pointers need the alignment of
 * one element.  Activations, weights and logits have the type `dtype` names; bias, gamma, beta, statistics, log
 * probabilities and the gradients of bias, gamma and beta are fp32.  Sums are held in fp32 and every output is rounded
 * once.  A call with rows = 0 launches nothing (the gradients of parameters become 0); other sizes are positive.
 * Outputs may not overlap inputs or each other except where noted.  Results do not depend on what else runs: the
 * same sums in the same order in every call of the same sizes and workspace. */
#define TCBNN_F32 0
#define TCBNN_BF16 1
#define TCBNN_F16 2

#define TCBNN_ACT_NONE 0
#define TCBNN_ACT_RELU 1 /* max(z, 0)                                     */
#define TCBNN_ACT_GELU 2 /* z * (1 + erf(z / sqrt(2))) / 2                */
#define TCBNN_ACT_SILU 3 /* z / (1 + exp(-z))                             */

/* z = input * weight^T + bias;  output = act(z) + residual.  `output` may be `residual` (same pointer and stride).
 * `preact` receives z, rounded to dtype: what tcbnn_linear_backward needs of a layer with an activation.
 * `workspace` (tcbnn_linear_workspace_bytes; may be NULL) lets products of few rows and outputs share a long sum over
 * inputs among workgroups.  rows <= 2^31 - 2^22, in_features <= 1048576, out_features <= 2^28. */
typedef struct tcbnn_linear_desc {
    const void* input;     /* [rows][in_features]                     */
    const void* weight;    /* [out_features][in_features]             */
    const float* bias;     /* [out_features], or NULL                 */
    const void* residual;  /* [rows][out_features], or NULL           */
    void* output;          /* [rows][out_features]                    */
    void* preact;          /* [rows][out_features], or NULL           */
    int rows, in_features, out_features;
    int dtype;             /* TCBNN_F32 / BF16 / F16                  */
    int activation;        /* TCBNN_ACT_*                             */
    long long input_ld, weight_ld, residual_ld, output_ld, preact_ld;
    void* workspace;
    size_t workspace_bytes;
} tcbnn_linear_desc;
size_t tcbnn_linear_workspace_bytes(int rows, int in_features, int out_features, int dtype);
int tcbnn_linear_forward(const tcbnn_linear_desc* d, void* stream);
/* Name of the kernel that tcbnn_linear_forward launches for this descriptor; nothing is launched, no pointer followed. */
int tcbnn_linear_kernel_name(const tcbnn_linear_desc* d, char* buf, size_t len);

/* With dz = grad_output * act'(z):  grad_input = dz * weight, grad_weight = dz^T * input, grad_bias = sums of dz over the
 * rows (the gradient of `residual` is grad_output itself).  Each of the three may be NULL; what is given is overwritten.
 * `preact` is z as the forward call wrote it (NULL without an activation); relu'(0) = 0.  In 16-bit types dz is rounded
 * to dtype before the two products, as their results are after them; grad_bias sums it unrounded.
 * `workspace` holds tcbnn_linear_grad_workspace_bytes (a NULL one is refused where that is not 0). */
typedef struct tcbnn_linear_grad_desc {
    const void* input;        /* [rows][in_features]; NULL where grad_weight is         */
    const void* weight;       /* [out_features][in_features]; NULL where grad_input is  */
    const void* preact;       /* [rows][out_features]                                   */
    const void* grad_output;  /* [rows][out_features]                                   */
    void* grad_input;         /* [rows][in_features]                                    */
    void* grad_weight;        /* [out_features][in_features]                            */
    float* grad_bias;         /* [out_features]                                         */
    int rows, in_features, out_features;
    int dtype;
    int activation;
    long long input_ld, weight_ld, preact_ld, grad_output_ld, grad_input_ld, grad_weight_ld;
    void* workspace;
    size_t workspace_bytes;
} tcbnn_linear_grad_desc;
size_t tcbnn_linear_grad_workspace_bytes(int rows, int in_features, int out_features, int dtype);
int tcbnn_linear_backward(const tcbnn_linear_grad_desc* d, void* stream);

/* mean and rstd = 1 / sqrt(variance + eps) of every row (the variance about the mean, over all features);
 * output = (input - mean) * rstd * gamma + beta.  `output` may be `input` (same pointer and stride).  `mean` and `rstd`
 * may be NULL; tcbnn_layernorm_backward needs them.  features <= 65536. */
typedef struct tcbnn_layernorm_desc {
    const void* input;   /* [rows][features]          */
    const float* gamma;  /* [features], or NULL (1)   */
    const float* beta;   /* [features], or NULL (0)   */
    void* output;        /* [rows][features]          */
    float* mean;         /* [rows], or NULL           */
    float* rstd;         /* [rows], or NULL           */
    int rows, features;
    int dtype;
    float eps;           /* >= 0                      */
    long long input_ld, output_ld;
} tcbnn_layernorm_desc;
int tcbnn_layernorm_forward(const tcbnn_layernorm_desc* d, void* stream);

/* With xh = (input - mean) * rstd and g = grad_output * gamma:
 * grad_input = rstd * (g - mean of g - xh * mean of g * xh) (means over a row's features), grad_gamma = sums of
 * grad_output * xh over the rows, grad_beta = sums of grad_output.  Each of the three may be NULL.  `grad_input` may be
 * `grad_output` (same pointer and stride).  `workspace` holds tcbnn_layernorm_grad_workspace_bytes where grad_gamma or
 * grad_beta is asked for. */
typedef struct tcbnn_layernorm_grad_desc {
    const void* input;        /* [rows][features]         */
    const float* gamma;       /* [features], or NULL (1)  */
    const float* mean;        /* [rows]                   */
    const float* rstd;        /* [rows]                   */
    const void* grad_output;  /* [rows][features]         */
    void* grad_input;         /* [rows][features]         */
    float* grad_gamma;        /* [features]               */
    float* grad_beta;         /* [features]               */
    int rows, features;
    int dtype;
    long long input_ld, grad_output_ld, grad_input_ld;
    void* workspace;
    size_t workspace_bytes;
} tcbnn_layernorm_grad_desc;
size_t tcbnn_layernorm_grad_workspace_bytes(int rows, int features);
int tcbnn_layernorm_backward(const tcbnn_layernorm_grad_desc* d, void* stream);

/* The norms after and before a block, with its gate, its scale and the residual stream between them:
 *   u = norm_after(block);  stream_out = stream_in + scale * gate * u;  output = norm_before(stream_out)
 * norm(x) = (x - mean) * rstd * gamma + beta with the mean and variance of a row's features (TCBNN_NORM_LAYER), x * rstd * gamma with
 * the mean of x^2 for the variance (TCBNN_NORM_RMS), x (TCBNN_NORM_NONE); rstd = 1 / sqrt(variance + eps).  Nothing is rounded between
 * the two norms.  Without a `block` the stream is stream_in (after = TCBNN_NORM_NONE, no gate).  `stream_out` may be `stream_in` or
 * `block`, `output` any of the three that is not wanted afterwards (same pointer and stride).  A beta belongs to a layer norm, a gamma to either.
 * The statistics may be NULL; tcbnn_blocknorm_backward needs them.  features <= 65536. */
#define TCBNN_NORM_NONE 0
#define TCBNN_NORM_RMS 1
#define TCBNN_NORM_LAYER 2
typedef struct tcbnn_blocknorm_desc {
    const void* stream_in;     /* [rows][features]                         */
    const void* block;         /* [rows][features], or NULL                */
    const float* gate;         /* [features], or NULL (1)                  */
    const float* after_gamma;  /* [features], or NULL (1)                  */
    const float* after_beta;   /* [features], or NULL (0)                  */
    const float* before_gamma; /* [features], or NULL (1)                  */
    const float* before_beta;  /* [features], or NULL (0)                  */
    void* stream_out;          /* [rows][features], or NULL                */
    void* output;              /* [rows][features]; NULL without a norm before */
    float* after_mean;         /* [rows] each, or NULL; means of layer norms only */
    float* after_rstd;
    float* before_mean;
    float* before_rstd;
    int rows, features;
    int dtype;
    int after, before;         /* TCBNN_NORM_*                             */
    float scale;
    float eps;                 /* >= 0                                     */
    long long stream_in_ld, block_ld, stream_out_ld, output_ld;
} tcbnn_blocknorm_desc;
int tcbnn_blocknorm_forward(const tcbnn_blocknorm_desc* d, void* stream);

/* With g = grad_output * before_gamma, xh = (stream_out - mean) * rstd:
 *   grad_stream_in = grad_stream_out + rstd * (g - mean of g - xh * mean of g * xh)   (no mean of g in an RMS norm),
 *   grad_u = scale * gate * grad_stream_in, and grad_block from it through norm_after in the same way;
 *   grad_gate = sums over the rows of scale * grad_stream_in * u, grad_after_gamma and _beta of grad_u * yh and grad_u (yh: the block's
 *   output, normed), grad_before_gamma and _beta of grad_output * xh and grad_output.
 * grad_stream_in is rounded where it is written only.  Any gradient that is written may be NULL; grad_output or grad_stream_out may be NULL (0).
 * grad_stream_in may be grad_output or grad_stream_out, grad_block one of them or `block` (same pointer and stride, and not both the same).
 * The stream and the statistics are the forward call's.  `workspace` holds tcbnn_blocknorm_grad_workspace_bytes. */
typedef struct tcbnn_blocknorm_grad_desc {
    const void* stream_out;       /* [rows][features]; NULL without a norm before         */
    const void* block;            /* [rows][features], or NULL                            */
    const float* gate;            /* [features], or NULL (1)                              */
    const float* after_gamma;     /* [features], or NULL (1)                              */
    const float* after_beta;      /* [features], or NULL (0)                              */
    const float* before_gamma;    /* [features], or NULL (1)                              */
    const float* after_mean;      /* [rows] each, where the norm has them                 */
    const float* after_rstd;
    const float* before_mean;
    const float* before_rstd;
    const void* grad_output;      /* [rows][features], or NULL                            */
    const void* grad_stream_out;  /* [rows][features], or NULL                            */
    void* grad_stream_in;         /* [rows][features]                                     */
    void* grad_block;             /* [rows][features]                                     */
    float* grad_gate;             /* [features] each                                      */
    float* grad_after_gamma;
    float* grad_after_beta;
    float* grad_before_gamma;
    float* grad_before_beta;
    int rows, features;
    int dtype;
    int after, before;
    float scale;
    long long stream_out_ld, block_ld, grad_output_ld, grad_stream_out_ld, grad_stream_in_ld, grad_block_ld;
    void* workspace;
    size_t workspace_bytes;
} tcbnn_blocknorm_grad_desc;
size_t tcbnn_blocknorm_grad_workspace_bytes(int rows, int features, int dtype);
int tcbnn_blocknorm_backward(const tcbnn_blocknorm_grad_desc* d, void* stream);

/* A gated feed-forward product: z = input * weight^T + bias with 2 * features columns, the gate's first;
 * output = act(z of the gate) * (z of the rest).  `preact` receives z, rounded to dtype: what tcbnn_gated_backward needs.
 * `workspace` (tcbnn_gated_workspace_bytes; may be NULL) is for copies of operands whose rows do not lie at whole 16 bytes, where these are
 * faster.  rows <= 2^31 - 2^22, in_features <= 1048576, features <= 2^27. */
typedef struct tcbnn_gated_desc {
    const void* input;   /* [rows][in_features]         */
    const void* weight;  /* [2 * features][in_features] */
    const float* bias;   /* [2 * features], or NULL     */
    void* output;        /* [rows][features]            */
    void* preact;        /* [rows][2 * features], or NULL */
    int rows, in_features, features;
    int dtype;
    int activation;      /* TCBNN_ACT_*                 */
    long long input_ld, weight_ld, output_ld, preact_ld;
    void* workspace;
    size_t workspace_bytes;
} tcbnn_gated_desc;
size_t tcbnn_gated_workspace_bytes(int rows, int in_features, int features, int dtype);
int tcbnn_gated_forward(const tcbnn_gated_desc* d, void* stream);
/* Name of the kernel that tcbnn_gated_forward launches for this descriptor; nothing is launched, no pointer followed. */
int tcbnn_gated_kernel_name(const tcbnn_gated_desc* d, char* buf, size_t len);

/* With z as the forward call wrote it, dz of the gate = grad_output * (z of the rest) * act'(z of the gate), dz of the rest =
 * grad_output * act(z of the gate):  grad_input = dz * weight, grad_weight = dz^T * input, grad_bias = sums of dz over the rows.  Each of
 * the three may be NULL; what is given is overwritten.  relu'(0) = 0.  In 16-bit types dz is rounded to dtype before the two products (f16: a dz
 * beyond 65504 is infinite there); grad_bias sums it unrounded.  `workspace` holds tcbnn_gated_grad_workspace_bytes; with `anywhere` these are enough for copies of operands whose
 * rows do not lie at whole 16 bytes, where these are faster (without, such operands are read as they lie). */
typedef struct tcbnn_gated_grad_desc {
    const void* input;        /* [rows][in_features]; NULL where grad_weight is          */
    const void* weight;       /* [2 * features][in_features]; NULL where grad_input is   */
    const void* preact;       /* [rows][2 * features]                                    */
    const void* grad_output;  /* [rows][features]                                        */
    void* grad_input;         /* [rows][in_features]                                     */
    void* grad_weight;        /* [2 * features][in_features]                             */
    float* grad_bias;         /* [2 * features]                                          */
    int rows, in_features, features;
    int dtype;
    int activation;
    long long input_ld, weight_ld, preact_ld, grad_output_ld, grad_input_ld, grad_weight_ld;
    void* workspace;
    size_t workspace_bytes;
} tcbnn_gated_grad_desc;
size_t tcbnn_gated_grad_workspace_bytes(int rows, int in_features, int features, int dtype, int anywhere);
int tcbnn_gated_backward(const tcbnn_gated_grad_desc* d, void* stream);

/* Of every row of logits x: logsumexp = log(sum exp(x_j)); logprob = x_t - logsumexp of the given class t = targets[row];
 * entropy = -sum p_j log p_j with p_j = exp(x_j - logsumexp) (in nats); rank = the number of classes before t in the order
 * "larger logit first, lower index among equals" (0: t is the best); top_index, top_logprob = the first `top` classes of
 * that order.  Any output may be NULL; targets only where logprob and rank are.
 *   t < 0        : a row without a given class: logprob 0, rank -1.   t >= classes: logprob NaN, rank -1.
 *   x_j = -inf   : a forbidden class: p_j = 0, no share in the entropy, log probability -inf.
 *   all -inf     : logsumexp -inf, every log probability -inf, entropy 0.
 *   NaN, +inf    : the row's logsumexp, log probabilities and entropy are NaN; NaN goes before every number in the order.
 * top <= 64 and <= classes.  `workspace` (tcbnn_logprobs_workspace_bytes; a NULL one is refused where that is not 0) joins
 * rows that several workgroups share. */
typedef struct tcbnn_logprobs_desc {
    const void* logits;      /* [rows][classes]           */
    const int32_t* targets;  /* [rows]                    */
    float* logprob;          /* [rows]                    */
    float* entropy;          /* [rows]                    */
    float* logsumexp;        /* [rows]                    */
    int32_t* rank;           /* [rows]                    */
    int32_t* top_index;      /* [rows][top]               */
    float* top_logprob;      /* [rows][top]               */
    int rows, classes, top;
    int dtype;
    long long logits_ld;
    void* workspace;
    size_t workspace_bytes;
} tcbnn_logprobs_desc;
size_t tcbnn_logprobs_workspace_bytes(int rows, int classes, int top, int dtype);
int tcbnn_logprobs_forward(const tcbnn_logprobs_desc* d, void* stream);

/* The gradient of sum over rows of grad_logprob * logprob + grad_entropy * entropy:
 * grad_logits_j = grad_logprob * ([j = t] - p_j) - grad_entropy * p_j * (log p_j + entropy).  `logsumexp` and `entropy`
 * are the forward call's; grad_logprob or grad_entropy may be NULL (0).  Without a given class (t < 0) grad_logprob
 * counts as 0; with t >= classes the row is NaN unless grad_logprob is NULL; a row whose classes are all forbidden gets 0.
 * p_j carries the rounding of `logsumexp` to fp32, |logsumexp| 2^-24 of it: rows of very large logits are better shifted first
 * (the forward call's log probabilities and entropy do not depend on it).
 * The mean cross entropy of n rows is grad_logprob = -1 / n.  `grad_logits` may be `logits` (same pointer and stride). */
typedef struct tcbnn_logprobs_grad_desc {
    const void* logits;         /* [rows][classes]           */
    const int32_t* targets;     /* [rows]; NULL where grad_logprob is */
    const float* logsumexp;     /* [rows]                    */
    const float* entropy;       /* [rows]; NULL where grad_entropy is */
    const float* grad_logprob;  /* [rows], or NULL           */
    const float* grad_entropy;  /* [rows], or NULL           */
    void* grad_logits;          /* [rows][classes]           */
    int rows, classes;
    int dtype;
    long long logits_ld, grad_logits_ld;
} tcbnn_logprobs_grad_desc;
int tcbnn_logprobs_backward(const tcbnn_logprobs_grad_desc* d, void* stream);

/* The softmax cross entropy of a linear classifier, which keeps no logits: z = input * weight^T + bias, of every row logsumexp =
 * log(sum exp(z_j)) and loss = logsumexp - z_t of the given class t = targets[row].  Logits are in fp32 and are not rounded.
 *   t < 0        : a row without a class: loss 0.   t >= classes: loss NaN.
 *   bias_j = -inf: a forbidden class; z_t = -inf: loss +inf; every z_j = -inf: logsumexp -inf.
 *   NaN, +inf    : the row's logsumexp and loss are NaN.
 * Finite masks, the type's lowest value too, are logits like others.  Rows of either operand are less than 2^31 / 256 bytes apart.
 * `workspace` holds tcbnn_linear_loss_workspace_bytes; with `anywhere` these are enough for copies of operands whose rows do not lie at whole 16
 * bytes, where these are faster (without, such operands are read as they lie).  rows <= 2^31 - 2^22, in_features <= 1048576, classes <= 2^28. */
typedef struct tcbnn_linear_loss_desc {
    const void* input;       /* [rows][in_features]      */
    const void* weight;      /* [classes][in_features]   */
    const float* bias;       /* [classes], or NULL       */
    const int32_t* targets;  /* [rows]; NULL where loss is */
    float* loss;             /* [rows], or NULL          */
    float* logsumexp;        /* [rows], or NULL          */
    int rows, in_features, classes;
    int dtype;
    long long input_ld, weight_ld;
    void* workspace;
    size_t workspace_bytes;
    float* logsumexp_rest;   /* [rows], or NULL: what rounding to fp32 left of logsumexp */
} tcbnn_linear_loss_desc;
size_t tcbnn_linear_loss_workspace_bytes(int rows, int in_features, int classes, int dtype, int anywhere);
int tcbnn_linear_loss_forward(const tcbnn_linear_loss_desc* d, void* stream);

/* The gradient of sum over rows of grad_loss * loss.  With d_j = grad_loss * (exp(z_j - logsumexp) - [j = t]), and d = 0 in rows without
 * a class and in rows whose classes are all forbidden (t >= classes: NaN):  grad_input = d * weight, grad_weight = d^T * input,
 * grad_bias = sums of d over the rows.  Each of the three may be NULL; what is given is overwritten.  The logits are made again, a piece
 * of the classes at a time; in 16-bit types d is rounded to dtype before the two products (in f16 times a power of two that keeps small
 * ones from getting lost); grad_bias sums it unrounded.  `logsumexp` and `logsumexp_rest` are the forward call's; without the rest exp carries logsumexp's
 * rounding, a relative |logsumexp| 2^-24 (of rows whose logits are all far beyond 2^24 logsumexp is the largest one, and exp of it 1 however many
 * classes have it).  With the forward call's `loss` the given class' d is grad_loss * (exp(-loss) - 1) instead, which is good where the class is nearly certain.
 * A row without a class still has to hold finite inputs: grad_weight sums 0 times them.  `workspace` holds
 * tcbnn_linear_loss_grad_workspace_bytes, `anywhere` as in the forward call. */
typedef struct tcbnn_linear_loss_grad_desc {
    const void* input;       /* [rows][in_features]      */
    const void* weight;      /* [classes][in_features]   */
    const float* bias;       /* [classes], or NULL       */
    const int32_t* targets;  /* [rows]                   */
    const float* logsumexp;  /* [rows]                   */
    const float* loss;       /* [rows], or NULL          */
    const float* grad_loss;  /* [rows]                   */
    void* grad_input;        /* [rows][in_features]      */
    void* grad_weight;       /* [classes][in_features]   */
    float* grad_bias;        /* [classes]                */
    int rows, in_features, classes;
    int dtype;
    long long input_ld, weight_ld, grad_input_ld, grad_weight_ld;
    void* workspace;
    size_t workspace_bytes;
    const float* logsumexp_rest; /* [rows], or NULL (0)  */
} tcbnn_linear_loss_grad_desc;
size_t tcbnn_linear_loss_grad_workspace_bytes(int rows, int in_features, int classes, int dtype, int anywhere);
int tcbnn_linear_loss_backward(const tcbnn_linear_loss_grad_desc* d, void* stream);

/* ------------------------------------------------ standalone GEMM / conv */
/* C[m][n] = K - 2*popc(A[m,:] xor B[n,:]), int32 row major [M][N].  A: [K/32][M]
 * (tcbnn_pack_rows output), B: [N][K/32] (tcbnn_pack_cols output: each column of the
 * logical K x N matrix contiguous along K); K % 32 == 0, N % 32 == 0.  Replaces
 * BMMAS / BMMAS_new (tensorcore_kernel.cu:305-356). */
int tcbnn_bmm(const uint32_t* a, const uint32_t* b, int32_t* c, int m, int n, int k, int variant,
              void* stream);
/* out[b][p][q][o] = Cin*R*S - exclude*Cin - 2*popc  (bmma_kernel.cu:154-159), int32
 * [N][P][Q][O] (the layout BTC_trans_output produces, bmma_kernel.cu:247-263).
 * input: [H][W][CW][B]; filter: tcbnn_pack_conv_filter output.  Replaces
 * BTC_Conv2d_balance[_128] (bmma_kernel.cu:101-165, 326-392). */
int tcbnn_bconv(const uint32_t* input, const uint32_t* filter, int32_t* output, int batch,
                int height, int width, int in_ch, int out_ch, int r, int s, int stride_h,
                int stride_w, int pad_h, int pad_w, int out_h, int out_w, int variant,
                void* stream);

/* -------------------------------------------------- unpack / interop */
/* bits -> +-1.0f, [B][N] row major.  Replaces UnPackFcOutput128FMT (param.h:87-104). */
int tcbnn_unpack_fc_output(const uint32_t* packed, float* out, int batch, int features,
                           void* stream);
/* bits -> +-1.0f, NHWC [B][H][W][C].  Replaces UnpackConvOutput32FMT (param.h:661-688). */
int tcbnn_unpack_conv_output(const uint32_t* packed, float* out, int height, int width, int ch,
                             int batch, void* stream);
/* Engine FC activation layout <-> reference [ceil(B/8)][ceil(K/128)][8][4] tiles
 * (kernel.cuh:170,222-223).  fmt holds PAD8(B)*ceil(K/128)*4 words. */
int tcbnn_fc_to_reference_fmt(const uint32_t* packed, uint32_t* fmt, int batch, int features,
                              void* stream);
int tcbnn_fc_from_reference_fmt(const uint32_t* fmt, uint32_t* packed, int batch, int features,
                                void* stream);
/* Engine conv activation layout <-> reference [H][W][PAD8(B)/8][ceil(C/128)][8][4]
 * (kernel.cuh:650-660, 811-815). */
int tcbnn_conv_to_reference_fmt(const uint32_t* packed, uint32_t* fmt, int height, int width,
                                int batch, int ch, void* stream);
int tcbnn_conv_from_reference_fmt(const uint32_t* fmt, uint32_t* packed, int height, int width,
                                  int batch, int ch, void* stream);
/* Engine residual (either format) -> reference int32 [P][Q][PAD8(B)][PAD128(O)] with
 * zero fill (kernel.cuh:666-668, 820-823). */
int tcbnn_residual_to_reference(const int32_t* res, int32_t* ref, int height, int width,
                                int batch, int ch, int format, void* stream);
/* The reverse: a residual in the reference layout -> the engine layout `format`
 * (tcbnn_residual_bytes(...) bytes), for a Conv128 layer that injects a residual a
 * reference-layout producer saved (read at kernel.cuh:760-791).  TCBNN_RES_I16 keeps the low
 * 16 bits: only for values the caller knows to fit. */
int tcbnn_residual_from_reference(const int32_t* ref, int32_t* res, int height, int width,
                                  int batch, int ch, int format, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* TCBNN_HIP_H */
