/*
 * Operator registry and parameter descriptors of the htp-ops dispatch surface.
 *
 * Wire-compatible restatement of the reference's include/op_reg.h (enum at :5-13,
 * RpcmemBufAddr :15-18, RmsNormF32Params :20-25, MatMulParams :27-34, FlashAttnParams
 * :36-47): same names, same enumerator values 0..5, same packed sizes (8/24/36/60 B).
 *
 * Additions, all AFTER the reference's six indices so their values never move:
 *   - fp16-activation quantised matmuls (the reference registry only has fp32-activation
 *     "A32" ops, but the lm_head / prefill workloads feed fp16 activations);
 *   - HTP_OPS_COUNT therefore grows from 6 to 8; HTP_OPS_REFERENCE_COUNT keeps the old value.
 *
 * Weight layout consumed by indices 2, 3, 4, 6, 7 in this library: standard ggml block_q4_0 /
 * block_q8_0 (quants.h; index 4 = the Q4_0 block with the IQ4_NL value table), N rows of K/32
 * consecutive blocks, the layout walked by the reference's dequantize_common_weight_* routines
 * (src/dsp/ops/mat_mul.c:572-640); with the library option "permuted_weights" indices 2, 3, 4 read the
 * reference-private permuted super-blocks instead.  Index 1 reads fp16 weights in the reference's
 * 32 x 32 tile order (src/host/test.c:303-313).  Index 0 is RMSNorm.  Index 5 (FlashAttention) is
 * not built: the dispatcher answers -1; attention over this library's own 8-bit cache is index 17, among the
 * operators around a decoder's matmuls that enum HtpOpsDecoderIndex names.
 */
#ifndef HTP_OPS_OP_REG_H
#define HTP_OPS_OP_REG_H

#include <stdint.h>

enum HtpOpsIndex {
  HTP_OPS_RMS_NORM_F32                     = 0,
  HTP_OPS_MAT_MUL_PERMUTED_W16A32          = 1,
  HTP_OPS_MAT_MUL_PERMUTED_W4D16A32        = 2, /* Q4_0 weights, fp16 scale, fp32 activations */
  HTP_OPS_MAT_MUL_PERMUTED_W8D16A32        = 3, /* Q8_0 weights, fp16 scale, fp32 activations */
  HTP_OPS_MAT_MUL_PERMUTED_W4D16A32_IQ4_NL = 4,
  HTP_OPS_FLASH_ATTN_QO_F32_KV_F16         = 5,
  /* ---- appended by the B200 library ---- */
  HTP_OPS_MAT_MUL_W4D16A16                 = 6, /* Q4_0 weights, fp16 activations, fp32 output */
  HTP_OPS_MAT_MUL_W8D16A16                 = 7, /* Q8_0 weights, fp16 activations, fp32 output */
  HTP_OPS_COUNT,
};

#define HTP_OPS_REFERENCE_COUNT 6

/* The operators around a decoder's matmuls (htp_ops_b200.h says what they compute), from 16 on: the indices in
 * between stay free for the registry above. */
enum HtpOpsDecoderIndex {
  HTP_OPS_KV_APPEND      = 16,
  HTP_OPS_ATTN_PAGED     = 17,
  HTP_OPS_ADD_RMS_NORM   = 18,
  HTP_OPS_LOGITS_PROCESS = 19,
};

#define HTP_OPS_PACKED __attribute__((packed))

/* A buffer is named by the handle the buffer table gave out (the reference's rpcmem fd)
 * plus a byte offset into it. */
struct RpcmemBufAddr {
  int32_t fd;
  int32_t offset;
} HTP_OPS_PACKED;

struct RmsNormF32Params {
  struct RpcmemBufAddr dst;
  struct RpcmemBufAddr src;
  int32_t ne0; /* row length  */
  int32_t ne1; /* row count   */
} HTP_OPS_PACKED;

/* output[m][n] (fp32) = activation[m][k] * weight[n][k]^T */
struct MatMulParams {
  struct RpcmemBufAddr output;
  struct RpcmemBufAddr activation;
  struct RpcmemBufAddr weight;
  int32_t m;
  int32_t k;
  int32_t n;
} HTP_OPS_PACKED;

struct FlashAttnParams {
  struct RpcmemBufAddr o;
  struct RpcmemBufAddr q;
  struct RpcmemBufAddr k;
  struct RpcmemBufAddr v;
  struct RpcmemBufAddr mask;
  int32_t qo_len;
  int32_t kv_len;
  int32_t n_heads;
  int32_t n_kv_heads;
  int32_t head_dim;
} HTP_OPS_PACKED;

/* ---- operators 16 .. 19: the arguments of the functions in htp_ops_b200.h, buffers by handle.  A buffer with
 * fd <= 0 is absent (NULL there).  Strides count elements. ---- */
struct PagedKvParams {
  struct RpcmemBufAddr k_codes, v_codes, k_scale, v_scale, page_table, q_start, ctx_len;
  int32_t              n_pages, page_size, n_kv_heads, head_dim, kv_type, n_seqs, table_stride, n_rows;
} HTP_OPS_PACKED;

struct KvAppendParams {
  struct PagedKvParams kv;
  struct RpcmemBufAddr k, v, q, q_out, rope_table, positions;
  int32_t              k_stride, v_stride, q_stride, q_out_stride;
  int32_t              n_heads, act_type, q_out_type;
  int32_t              rope_mode, rot_dim, table_len;
} HTP_OPS_PACKED;

struct AttnPagedParams {
  struct PagedKvParams kv;
  struct RpcmemBufAddr out, q, workspace;
  int32_t              workspace_bytes;
  int32_t              out_stride, q_stride;
  int32_t              n_heads, act_type;
  float                scale;
  int32_t              window, max_q, max_ctx;
} HTP_OPS_PACKED;

struct AddRmsNormParams {
  struct RpcmemBufAddr h_out, norm_out, x, block, post_weight, gate, weight;
  int32_t              gate_stride;
  float                block_scale, eps;
  int32_t              n, rows, norm_type;
} HTP_OPS_PACKED;

struct LogitsProcessParams {
  struct RpcmemBufAddr dst, src;
  struct RpcmemBufAddr history, history_start, prompt_len, repetition, presence, frequency;
  struct RpcmemBufAddr bias_token, bias_value, bias_start, mask, mask_row;
  int32_t              stride, rows, vocab, n_history, n_bias, n_mask_rows;
} HTP_OPS_PACKED;

#if defined(__cplusplus)
static_assert(sizeof(struct PagedKvParams) == 88 && sizeof(struct KvAppendParams) == 176 &&
                sizeof(struct AttnPagedParams) == 148 && sizeof(struct AddRmsNormParams) == 80 &&
                sizeof(struct LogitsProcessParams) == 128,
              "wire size");
static_assert(sizeof(struct RpcmemBufAddr) == 8, "wire size");
static_assert(sizeof(struct RmsNormF32Params) == 24, "wire size");
static_assert(sizeof(struct MatMulParams) == 36, "wire size");
static_assert(sizeof(struct FlashAttnParams) == 60, "wire size");
#else
_Static_assert(sizeof(struct PagedKvParams) == 88 && sizeof(struct KvAppendParams) == 176 &&
                 sizeof(struct AttnPagedParams) == 148 && sizeof(struct AddRmsNormParams) == 80 &&
                 sizeof(struct LogitsProcessParams) == 128,
               "wire size");
_Static_assert(sizeof(struct RpcmemBufAddr) == 8, "wire size");
_Static_assert(sizeof(struct RmsNormF32Params) == 24, "wire size");
_Static_assert(sizeof(struct MatMulParams) == 36, "wire size");
_Static_assert(sizeof(struct FlashAttnParams) == 60, "wire size");
#endif

#endif /* HTP_OPS_OP_REG_H */
