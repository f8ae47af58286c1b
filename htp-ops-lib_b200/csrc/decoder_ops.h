// Kernels of the operators around a decoder's matmuls: what the checked entry points (decoder_ops.cu)
// hand to the launchers.  Layouts and formulas: include/htp_ops_b200.h.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace htp {

// error codes a kernel may record (htp_b200_stream_status)
constexpr int kErrPage     = 301;
constexpr int kErrSequence = 302;
constexpr int kErrPosition = 303;
constexpr int kErrRange    = 304;
constexpr int kErrMaskRow  = 305;
constexpr int kErrWait     = 311;  // a bounded wait inside attention ran out

constexpr float kKvMinScale = 0x1p-100f;  // scale of a block of zeros

struct KvView {
  uint8_t       *k_codes, *v_codes;
  float         *k_scale, *v_scale;
  const int32_t *page_table, *q_start, *ctx_len;
  int            n_pages, page_size, page_shift, n_kv_heads, n_seqs, table_stride, n_rows;
};

struct KvAppendArgs {
  KvView         kv;
  const void    *k, *v, *q;
  void          *q_out;
  long long      k_stride, v_stride, q_stride, q_out_stride;
  const float   *rope_table;
  const int32_t *positions;
  int            table_len, rot_dim, mode, n_heads;
  long long      kv_slots;  // page slots of the grid: n_rows / page_size + 2 * n_seqs
  int           *err;
};
cudaError_t kv_append_launch(const KvAppendArgs &a, int head_dim, int kv_type, bool a16, bool q_out16, bool pdl,
                             cudaStream_t stream);

struct AttnArgs {
  KvView      kv;
  const void *q;
  void       *out;
  long long   q_stride, out_stride;
  float      *part;     // workspace: partial results of the groups of splits (groups > 1)
  int         n_heads, group;  // group = query heads of one key/value head
  float       scale_log2;      // scale * log2(e)
  int         window, max_q, max_ctx;
  int         col_groups, splits, groups;  // splits = CTAs of a cluster, groups = clusters (CTAs) over one context
  long long   row_slots;       // attn_prompt.cu: blocks of rows of the grid
  int        *err;
};
// How a step is cut: columns of query rows x heads of a key/value head per CTA, CTAs of a cluster and
// clusters over one context.
struct AttnPlan {
  bool      tile;           // the kernel for many rows (attn_prompt.cu)
  bool      two_row_tiles;  // of it: two tiles of rows per CTA
  long long row_slots;      // of it: blocks of rows, bounded by what n_rows and n_seqs allow
  int       col_tiles;      // 8-column tiles per CTA
  int       col_groups, splits, groups;
};
AttnPlan    attn_plan(int sm_count, int n_seqs, int n_rows, int n_kv_heads, int group, bool f32, int max_q, int max_ctx,
                      size_t workspace_bytes, int head_dim);
size_t      attn_part_bytes(int n_seqs, int max_q, int n_heads, int head_dim, int groups);
cudaError_t attn_decode_launch(const AttnArgs &a, const AttnPlan &p, int head_dim, int kv_type, bool a16, bool pdl,
                               cudaStream_t stream);

cudaError_t attn_prompt_launch(const AttnArgs &a, const AttnPlan &p, int head_dim, int kv_type, bool a16, bool pdl,
                               cudaStream_t stream);
// joins the results of the groups (attn_decode.cu)
cudaError_t attn_join_launch(const AttnArgs &a, int head_dim, bool a16, bool pdl, cudaStream_t stream);

struct AddRmsNormArgs {
  float       *h_out;
  void        *norm_out;
  const float *x, *block, *post_weight, *gate, *weight;
  long long    gate_stride;
  float        block_scale, eps;
  int          n, rows;
};
cudaError_t add_rms_norm_launch(const AddRmsNormArgs &a, bool norm16, bool pdl, cudaStream_t stream);

struct LogitsArgs {
  float          *dst;
  const float    *src;
  long long       stride;
  int             rows, vocab;
  const int32_t  *history, *history_start, *prompt_len;
  const float    *repetition, *presence, *frequency;
  const int32_t  *bias_token, *bias_start;
  const float    *bias_value;
  const uint32_t *mask;
  const int32_t  *mask_row;
  int             n_history, n_bias, n_mask_rows;
  int            *err;
};
cudaError_t logits_process_launch(const LogitsArgs &a, int sm_count, bool pdl, cudaStream_t stream);

// Dynamic shared memory of a kernel on the current device, set once per kernel and device (decoder_ops.cu).
cudaError_t allow_smem(const void *kernel, int bytes);

// Launch with or without programmatic stream serialisation, in clusters of `cluster` CTAs.
template <typename Kernel, typename Args>
inline cudaError_t launch_decoder_kernel(Kernel kernel, const Args &args, unsigned grid, unsigned threads, size_t smem,
                                         bool pdl, unsigned cluster, cudaStream_t stream) {
  cudaLaunchConfig_t  cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim          = dim3(grid);
  cfg.blockDim         = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream           = stream;
  cfg.attrs            = attr;
  if (pdl) {
    attr[cfg.numAttrs].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[cfg.numAttrs].id                 = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x   = cluster;
    attr[cfg.numAttrs].val.clusterDim.y   = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  return cudaLaunchKernelEx(&cfg, kernel, args);
}

}  // namespace htp
