// Checked entry points of the operators around a decoder's matmuls (include/htp_ops_b200.h): argument
// checks, kernel choice, launch.  Nothing here allocates device memory or keeps state between calls, apart from one
// error word per device.
#include "decoder_ops.h"

#include <cmath>
#include <map>
#include <mutex>
#include <set>
#include <utility>

#include "device_ctx.h"
#include "htp_ops_b200.h"

namespace htp {

namespace {

std::mutex           g_err_mu;
std::map<int, int *> g_err_words;

constexpr int kMaxLength = 1 << 30;

bool aligned(const void *p, uintptr_t n) {
  return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0;
}

size_t act_size(int type) {
  return type == HTP_B200_ACT_F16 ? 2 : 4;
}

bool is_act(int type) {
  return type == HTP_B200_ACT_F32 || type == HTP_B200_ACT_F16;
}

// rows of `width` elements, `stride` apart: 16-byte aligned base and rows, no overlap of rows
bool rows_ok(const void *p, int64_t stride, int64_t width, int type) {
  return p && aligned(p, 16) && stride >= width && stride <= (int64_t) 1 << 40 && stride * act_size(type) % 16 == 0;
}

// bytes from the first to the last element of `rows` rows
size_t extent(int64_t rows, int64_t stride, int64_t width, size_t size) {
  return (size_t) ((rows - 1) * stride + width) * size;
}

bool overlap(const void *a, size_t na, const void *b, size_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a && b && x < y + nb && y < x + na;
}

// the sizes of a cache, its pointers apart
bool sizes_ok(const HtpB200PagedKv *kv) {
  return kv && kv->n_pages > 0 && (kv->page_size == 16 || kv->page_size == 32 || kv->page_size == 64 || kv->page_size == 128) &&
         kv->n_kv_heads > 0 && kv->n_kv_heads <= 65536 && (kv->head_dim == 64 || kv->head_dim == 128) &&
         (kv->kv_type == HTP_B200_KV_I8 || kv->kv_type == HTP_B200_KV_E4M3) && kv->n_seqs > 0 && kv->table_stride > 0 &&
         kv->n_rows > 0 && kv->n_rows <= kMaxLength && kv->n_seqs <= kMaxLength &&
         (int64_t) kv->n_pages * kv->n_kv_heads <= 0x7fffffff / kv->page_size;
}

bool view_of(const HtpB200PagedKv *kv, KvView *v) {
  if (!sizes_ok(kv) || !kv->k_codes || !kv->v_codes || !kv->k_scale || !kv->v_scale || !kv->page_table || !kv->q_start ||
      !kv->ctx_len) {
    return false;
  }
  if (!aligned(kv->k_codes, 16) || !aligned(kv->v_codes, 16) || !aligned(kv->k_scale, 4) || !aligned(kv->v_scale, 4) ||
      !aligned(kv->page_table, 4) || !aligned(kv->q_start, 4) || !aligned(kv->ctx_len, 4)) {
    return false;
  }
  v->k_codes = static_cast<uint8_t *>(kv->k_codes), v->v_codes = static_cast<uint8_t *>(kv->v_codes);
  v->k_scale = kv->k_scale, v->v_scale = kv->v_scale;
  v->page_table = kv->page_table, v->q_start = kv->q_start, v->ctx_len = kv->ctx_len;
  v->n_pages = kv->n_pages, v->page_size = kv->page_size, v->n_kv_heads = kv->n_kv_heads;
  v->n_seqs = kv->n_seqs, v->table_stride = kv->table_stride, v->n_rows = kv->n_rows;
  v->page_shift = kv->page_size == 16 ? 4 : (kv->page_size == 32 ? 5 : (kv->page_size == 64 ? 6 : 7));
  return true;
}

size_t codes_bytes(const HtpB200PagedKv *kv) {
  return (size_t) kv->n_pages * kv->n_kv_heads * kv->page_size * kv->head_dim;
}

// queries and outputs of attention against what a plan needs
bool step_ok(const HtpB200PagedKv *kv, int n_heads, int act_type, int max_q, int max_ctx) {
  return sizes_ok(kv) && n_heads > 0 && n_heads <= 65536 && n_heads % kv->n_kv_heads == 0 && is_act(act_type) && max_q > 0 &&
         max_q <= kv->n_rows && max_ctx > 0 && (int64_t) max_ctx <= (int64_t) kv->table_stride * kv->page_size;
}

int done(cudaError_t e, int launches) {
  if (e != cudaSuccess) {
    cudaGetLastError();
    return -2;
  }
  count_launch(launches);
  return 0;
}

}  // namespace

int *device_error_word(DeviceCtx *ctx) {
  std::lock_guard<std::mutex> lk(g_err_mu);
  auto                        it = g_err_words.find(ctx->device);
  if (it != g_err_words.end()) {
    return it->second;
  }
  // (a capture in progress on this thread forbids allocations unless it is told that this one is no part of it)
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) {
    cudaGetLastError();
    return nullptr;
  }
  void             *p = nullptr, *dp = nullptr;
  const cudaError_t e = cudaHostAlloc(&p, 64, cudaHostAllocMapped | cudaHostAllocPortable);
  const bool        ok = e == cudaSuccess && cudaHostGetDevicePointer(&dp, p, 0) == cudaSuccess && dp == p;
  cudaThreadExchangeStreamCaptureMode(&mode);
  if (!ok) {
    cudaGetLastError();
    return nullptr;
  }
  *static_cast<int *>(p) = 0;
  return g_err_words[ctx->device] = static_cast<int *>(p);
}

cudaError_t allow_smem(const void *kernel, int bytes) {
  int device = -1;
  if (const cudaError_t e = cudaGetDevice(&device); e != cudaSuccess) {
    return e;
  }
  static std::mutex                                mu;
  static std::set<std::pair<int, const void *>>    done_for;
  std::lock_guard<std::mutex>                      lk(mu);
  if (done_for.count({ device, kernel })) {
    return cudaSuccess;
  }
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) {
    done_for.insert({ device, kernel });
  }
  return e;
}

int take_device_error(DeviceCtx *ctx) {
  std::lock_guard<std::mutex> lk(g_err_mu);
  auto                        it = g_err_words.find(ctx->device);
  return it == g_err_words.end() ? 0 : __atomic_exchange_n(it->second, 0, __ATOMIC_ACQ_REL);
}

}  // namespace htp

using namespace htp;

extern "C" {

int htp_b200_kv_append(const struct HtpB200PagedKv *kv, const struct HtpB200Rope *rope, const void *k, int64_t k_stride,
                       const void *v, int64_t v_stride, const void *q, int64_t q_stride, void *q_out,
                       int64_t q_out_stride, int n_heads, int act_type, int q_out_type, void *stream) {
  KvAppendArgs a = {};
  if (!view_of(kv, &a.kv) || !is_act(act_type)) {
    return -1;
  }
  const int64_t wide = (int64_t) kv->n_kv_heads * kv->head_dim;
  const size_t  n_scale = (size_t) kv->n_pages * kv->n_kv_heads * sizeof(float);
  if (overlap(kv->k_codes, codes_bytes(kv), kv->v_codes, codes_bytes(kv)) || overlap(kv->k_scale, n_scale, kv->v_scale, n_scale)) {
    return -1;  // keys and values are written by different CTAs
  }
  if (!rows_ok(k, k_stride, wide, act_type) || !rows_ok(v, v_stride, wide, act_type)) {
    return -1;
  }
  for (const void *codes : { kv->k_codes, kv->v_codes }) {
    if (overlap(k, extent(kv->n_rows, k_stride, wide, act_size(act_type)), codes, codes_bytes(kv)) ||
        overlap(v, extent(kv->n_rows, v_stride, wide, act_size(act_type)), codes, codes_bytes(kv))) {
      return -1;
    }
  }
  if (q) {
    const int64_t q_wide = (int64_t) n_heads * kv->head_dim;
    if (n_heads <= 0 || n_heads > 65536 || !is_act(q_out_type) || !rows_ok(q, q_stride, q_wide, act_type) ||
        !rows_ok(q_out, q_out_stride, q_wide, q_out_type)) {
      return -1;
    }
    const size_t out_bytes = extent(kv->n_rows, q_out_stride, q_wide, act_size(q_out_type));
    const bool   in_place  = q_out == q && q_out_type == act_type && q_out_stride == q_stride;
    if ((!in_place && overlap(q_out, out_bytes, q, extent(kv->n_rows, q_stride, q_wide, act_size(act_type)))) ||
        (!in_place && (overlap(q_out, out_bytes, k, extent(kv->n_rows, k_stride, wide, act_size(act_type))) ||
                       overlap(q_out, out_bytes, v, extent(kv->n_rows, v_stride, wide, act_size(act_type))))) ||
        overlap(q_out, out_bytes, kv->k_codes, codes_bytes(kv)) || overlap(q_out, out_bytes, kv->v_codes, codes_bytes(kv))) {
      return -1;
    }
    a.q = q, a.q_out = q_out, a.q_stride = q_stride, a.q_out_stride = q_out_stride, a.n_heads = n_heads;
  }
  if (rope && rope->mode != HTP_B200_ROPE_NONE) {
    if ((rope->mode != HTP_B200_ROPE_PAIRS && rope->mode != HTP_B200_ROPE_HALVES) || !rope->table || !aligned(rope->table, 16) ||
        rope->table_len <= 0 || rope->rot_dim <= 0 || rope->rot_dim % 8 != 0 || rope->rot_dim > kv->head_dim ||
        !aligned(rope->positions, 4)) {
      return -1;
    }
    a.rope_table = rope->table, a.positions = rope->positions, a.table_len = rope->table_len;
    a.rot_dim = rope->rot_dim, a.mode = rope->mode;
  }
  DeviceCtx *ctx = current_device_ctx();
  if (!ctx || !(a.err = device_error_word(ctx))) {
    return -2;
  }
  a.k = k, a.v = v, a.k_stride = k_stride, a.v_stride = v_stride;
  a.kv_slots = (long long) kv->n_rows / kv->page_size + 2ll * kv->n_seqs;
  return done(kv_append_launch(a, kv->head_dim, kv->kv_type, act_type == HTP_B200_ACT_F16, q_out_type == HTP_B200_ACT_F16,
                               g_opt_pdl != 0, static_cast<cudaStream_t>(stream)),
              1);
}

size_t htp_b200_attn_workspace(const struct HtpB200PagedKv *kv, int n_heads, int act_type, int max_q, int max_ctx) {
  if (!step_ok(kv, n_heads, act_type, max_q, max_ctx)) {
    return (size_t) -1;
  }
  DeviceCtx     *ctx = current_device_ctx();
  const AttnPlan p   = attn_plan(ctx ? ctx->sm_count : 148, kv->n_seqs, kv->n_rows, kv->n_kv_heads, n_heads / kv->n_kv_heads,
                                 act_type == HTP_B200_ACT_F32, max_q, max_ctx, (size_t) -1, kv->head_dim);
  return attn_part_bytes(kv->n_seqs, max_q, n_heads, kv->head_dim, p.groups);
}

int htp_b200_attn_paged(void *out, int64_t out_stride, const void *q, int64_t q_stride, const struct HtpB200PagedKv *kv,
                        int n_heads, int act_type, float scale, int window, int max_q, int max_ctx, void *workspace,
                        size_t workspace_bytes, void *stream) {
  AttnArgs a = {};
  if (!step_ok(kv, n_heads, act_type, max_q, max_ctx) || !view_of(kv, &a.kv)) {
    return -1;
  }
  const int64_t wide = (int64_t) n_heads * kv->head_dim;
  if (!rows_ok(q, q_stride, wide, act_type) || !rows_ok(out, out_stride, wide, act_type) || window < 0 ||
      !(scale >= 1e-20f && scale <= 1e20f) || !aligned(workspace, 16)) {
    return -1;
  }
  const size_t out_bytes = extent(kv->n_rows, out_stride, wide, act_size(act_type));
  if (!workspace) {
    workspace_bytes = 0;
  }
  if (overlap(out, out_bytes, q, extent(kv->n_rows, q_stride, wide, act_size(act_type))) ||
      overlap(out, out_bytes, kv->k_codes, codes_bytes(kv)) || overlap(out, out_bytes, kv->v_codes, codes_bytes(kv)) ||
      overlap(out, out_bytes, workspace, workspace_bytes)) {
    return -1;
  }
  DeviceCtx *ctx = current_device_ctx();
  if (!ctx || !(a.err = device_error_word(ctx))) {
    return -2;
  }
  a.group          = n_heads / kv->n_kv_heads;
  const AttnPlan p = attn_plan(ctx->sm_count, kv->n_seqs, kv->n_rows, kv->n_kv_heads, a.group, act_type == HTP_B200_ACT_F32, max_q,
                               max_ctx, workspace_bytes, kv->head_dim);
  a.q = q, a.out = out, a.q_stride = q_stride, a.out_stride = out_stride;
  a.part       = static_cast<float *>(workspace);
  a.n_heads    = n_heads;
  a.scale_log2 = scale * 1.44269504088896340736f;
  a.window = window, a.max_q = max_q, a.max_ctx = max_ctx;
  a.col_groups = p.col_groups, a.splits = p.splits, a.groups = p.groups, a.row_slots = p.row_slots;
  const auto launch = p.tile ? attn_prompt_launch : attn_decode_launch;
  return done(launch(a, p, kv->head_dim, kv->kv_type, act_type == HTP_B200_ACT_F16, g_opt_pdl != 0,
                     static_cast<cudaStream_t>(stream)),
              p.groups > 1 ? 2 : 1);
}

int htp_b200_add_rms_norm(float *h_out, void *norm_out, const float *x, const float *block, const float *post_weight,
                          const float *gate, int64_t gate_stride, const float *weight, float block_scale, float eps,
                          int n, int rows, int norm_type, void *stream) {
  if (!x || (!h_out && !norm_out) || n <= 0 || n > kMaxLength || rows <= 0 || rows > kMaxLength || !is_act(norm_type) ||
      !(eps >= 0.f && eps <= 1e30f) || !std::isfinite(block_scale)) {
    return -1;
  }
  if (!block && (post_weight || gate)) {
    return -1;
  }
  if (gate && gate_stride != 0 && gate_stride < n) {
    return -1;
  }
  if (!aligned(x, 4) || !aligned(block, 4) || !aligned(h_out, 4) || !aligned(post_weight, 4) || !aligned(gate, 4) ||
      !aligned(weight, 4) || !aligned(norm_out, act_size(norm_type))) {
    return -1;
  }
  const size_t bytes = (size_t) rows * n * sizeof(float), norm_bytes = (size_t) rows * n * act_size(norm_type);
  const size_t gate_bytes = gate ? extent(gate_stride ? rows : 1, gate_stride, n, sizeof(float)) : 0;
  const size_t row_bytes  = (size_t) n * sizeof(float);
  auto         clash      = [&](const void *out, size_t out_bytes, bool may_equal) {
    auto inside = [&](const void *in) { return overlap(out, out_bytes, in, bytes) && !(may_equal && out == in); };
    return inside(x) || inside(block) || overlap(out, out_bytes, gate, gate_bytes) ||
           overlap(out, out_bytes, post_weight, row_bytes) || overlap(out, out_bytes, weight, row_bytes);
  };
  if (clash(h_out, bytes, true) || clash(norm_out, norm_bytes, norm_type == HTP_B200_ACT_F32) ||
      overlap(h_out, bytes, norm_out, norm_bytes)) {
    return -1;
  }
  if (!current_device_ctx()) {
    return -2;
  }
  AddRmsNormArgs a = {};
  a.h_out = h_out, a.norm_out = norm_out, a.x = x, a.block = block, a.post_weight = post_weight, a.gate = gate;
  a.gate_stride = gate ? gate_stride : 0, a.weight = weight, a.block_scale = block_scale, a.eps = eps, a.n = n, a.rows = rows;
  return done(add_rms_norm_launch(a, norm_type == HTP_B200_ACT_F16, g_opt_pdl != 0, static_cast<cudaStream_t>(stream)), 1);
}

int htp_b200_logits_process(float *dst, const float *src, int64_t stride, int rows, int vocab,
                            const struct HtpB200LogitsParams *p, void *stream) {
  if (!dst || !src || !p || !aligned(dst, 16) || !aligned(src, 16) || rows <= 0 || vocab <= 0 || vocab > kMaxLength ||
      stride < vocab || stride > (int64_t) 1 << 40) {
    return -1;
  }
  if ((p->history != nullptr) != (p->history_start != nullptr) || (p->prompt_len && !p->history)) {
    return -1;
  }
  if ((p->bias_token != nullptr) != (p->bias_start != nullptr) || (p->bias_token != nullptr) != (p->bias_value != nullptr)) {
    return -1;
  }
  if ((p->history && p->n_history < 0) || (p->bias_token && p->n_bias < 0) || (p->mask && p->n_mask_rows <= 0) ||
      (p->mask_row && !p->mask) || (p->mask && !p->mask_row && p->n_mask_rows < rows)) {
    return -1;
  }
  const void *ints[] = { p->history, p->history_start, p->prompt_len, p->repetition, p->presence, p->frequency,
                         p->bias_token, p->bias_value, p->bias_start, p->mask, p->mask_row };
  for (const void *q : ints) {
    if (!aligned(q, 4)) {
      return -1;
    }
  }
  const size_t bytes = extent(rows, stride, vocab, sizeof(float));
  if (dst != src && overlap(dst, bytes, src, bytes)) {
    return -1;
  }
  DeviceCtx *ctx = current_device_ctx();
  LogitsArgs a   = {};
  if (!ctx || !(a.err = device_error_word(ctx))) {
    return -2;
  }
  a.dst = dst, a.src = src, a.stride = stride, a.rows = rows, a.vocab = vocab;
  a.history = p->history, a.history_start = p->history_start, a.prompt_len = p->prompt_len;
  a.repetition = p->repetition, a.presence = p->presence, a.frequency = p->frequency;
  a.bias_token = p->bias_token, a.bias_start = p->bias_start, a.bias_value = p->bias_value;
  a.mask = p->mask, a.mask_row = p->mask_row;
  a.n_history = p->n_history, a.n_bias = p->n_bias, a.n_mask_rows = p->n_mask_rows;
  return done(logits_process_launch(a, ctx->sm_count, g_opt_pdl != 0, static_cast<cudaStream_t>(stream)), 1);
}

}  // extern "C"
