// Append of a step's keys and values to the paged 8-bit cache, with the position rotation of keys and
// queries on the way (formulas and rounding rules: include/htp_ops_b200.h, htp_b200_kv_append).
//
// One launch, two kinds of CTAs.  A cache CTA owns one (page, head, keys or values) that the step writes
// to: the new elements are read once into registers, rotated there, their largest magnitude gives the
// page's scale, older codes follow a grown scale, the new codes are stored 8 bytes a thread - whole pages
// leave as contiguous runs, [page][head][token][dim].  A query CTA rotates one row.  Every arithmetic step is
// an explicitly rounded fp32 operation (no contraction), so the bytes are the same whatever the compiler does.
//
// Bound: HBM for prompts (each element is read once, codes and queries written once: 279 MB of 6.5 k rows with 32 + 8
// + 8 heads of 128 in 51.8 us = 0.82 of the measured copy rate), latency of the dependent loads (lengths -> page ->
// scale) for single tokens (2.8 us for one, 7.0 us for 64).
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "decoder_common.cuh"
#include "ptx.cuh"

namespace htp {

namespace {

constexpr int kThreads = 256;

constexpr int kRopeHalves = 2;  // HTP_B200_ROPE_HALVES

// First elements of the two groups of four that thread part j (0 .. D / 8 - 1) of a head holds: with
// halves rotated against each other the partner group lies rot_dim / 2 further on.
__device__ __forceinline__ void part_dims(int j, int mode, int rot_dim, int &lo, int &hi) {
  if (mode == kRopeHalves && 8 * j < rot_dim) {
    lo = 4 * j;
    hi = lo + (rot_dim >> 1);
  } else {
    lo = 8 * j;
    hi = lo + 4;
  }
}

template <bool A16>
__device__ __forceinline__ void load4(const void *row, int at, float *x) {
  if constexpr (A16) {
    const uint2  u = *reinterpret_cast<const uint2 *>(static_cast<const __half *>(row) + at);
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&u.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
  } else {
    const float4 u = *reinterpret_cast<const float4 *>(static_cast<const float *>(row) + at);
    x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
  }
}

__device__ __forceinline__ void turn(float &a, float &b, float c, float s) {
  const float y = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  b             = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
  a             = y;
}

// Rotates the eight elements of part j with the table row of their position.
__device__ __forceinline__ void rotate8(float (&x)[8], const float *row, int j, int mode, int rot_dim) {
  if (8 * j >= rot_dim) {
    return;
  }
  const float4 c = *reinterpret_cast<const float4 *>(row + 4 * j);
  const float4 s = *reinterpret_cast<const float4 *>(row + (rot_dim >> 1) + 4 * j);
  if (mode == kRopeHalves) {
    turn(x[0], x[4], c.x, s.x), turn(x[1], x[5], c.y, s.y), turn(x[2], x[6], c.z, s.z), turn(x[3], x[7], c.w, s.w);
  } else {
    turn(x[0], x[1], c.x, s.x), turn(x[2], x[3], c.y, s.y), turn(x[4], x[5], c.z, s.z), turn(x[6], x[7], c.w, s.w);
  }
}

// Four values times `by` as codes, lowest byte first.
template <int KVT>
__device__ __forceinline__ uint32_t to_codes4(const float *x, float by) {
  if constexpr (KVT == kKvI8) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      int q = __float2int_rn(__fmul_rn(x[i], by));  // ties to even; NaN: 0
      q     = q < -127 ? -127 : (q > 127 ? 127 : q);
      w |= (uint32_t) (q & 0xff) << (8 * i);
    }
    return w;
  } else {
    // (NaN: 0, as in signed bytes - a code that is no number would reach rows that do not see its token)
    auto         c = [&](float v) { return v == v ? __fmul_rn(v, by) : 0.f; };
    const float2 a = make_float2(c(x[0]), c(x[1]));
    const float2 b = make_float2(c(x[2]), c(x[3]));
    return (uint32_t) __nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3) |
           (uint32_t) __nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3) << 16;
  }
}

template <int KVT>
__device__ __forceinline__ void from_codes4(uint32_t w, float *x) {
  if constexpr (KVT == kKvI8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = (float) (int8_t) (w >> (8 * i));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t) (w >> (16 * i)), __NV_E4M3);
      const float2      f = __half22float2(__half2(h));
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
}

// One page of one head: `passes` = tokens of a page / tokens that the CTA covers at a time.
template <int D, int KVT, bool A16, int PASSES>
__device__ __forceinline__ void append_page(const KvAppendArgs &a, int b, int page_no, int head, bool keys) {
  __shared__ float red[kThreads / 32];
  constexpr int PARTS  = D / 8;               // threads of a token
  constexpr int TOKENS = kThreads / PARTS;    // tokens of a pass
  const KvView &kv = a.kv;
  int           q0, q_len, ctx;
  if (!sequence_of(kv, b, kv.n_rows, 0x7fffffff, q0, q_len, ctx) || ctx < q_len) {
    if (threadIdx.x == 0) {
      record_error(a.err, kErrSequence);
    }
    return;
  }
  const int first = ctx - q_len;  // the first new token
  const int page0 = (page_no + (first >> kv.page_shift)) << kv.page_shift;
  if (q_len == 0 || page_no < 0 || page0 >= ctx) {
    return;
  }
  const int from = (first > page0 ? first : page0) - page0, to = (ctx < page0 + kv.page_size ? ctx : page0 + kv.page_size) - page0;
  const int page = kv.page_table[(long long) b * kv.table_stride + (page0 >> kv.page_shift)];
  const int j    = threadIdx.x % PARTS;
  int       lo, hi;
  part_dims(j, keys ? a.mode : 0, a.rot_dim, lo, hi);
  const uint8_t  *src    = static_cast<const uint8_t *>(keys ? a.k : a.v);
  const long long stride = keys ? a.k_stride : a.v_stride;
  float           x[PASSES][8];
  float           amax = 0.f;
  bool            bad  = page < 0 || page >= kv.n_pages, bad_pos = false;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int slot = p * TOKENS + threadIdx.x / PARTS;
    if (slot < from || slot >= to) {
      continue;
    }
    const long long row = (long long) q0 + page0 + slot - first;
    const void     *at  = src + (row * stride + head * D) * (A16 ? 2 : 4);
    load4<A16>(at, lo, x[p]);
    load4<A16>(at, hi, x[p] + 4);
    if (keys && a.mode) {
      const int pos = a.positions ? a.positions[row] : page0 + slot;
      if (pos < 0 || pos >= a.table_len) {
        bad_pos = true;
      } else {
        rotate8(x[p], a.rope_table + (long long) pos * a.rot_dim, j, a.mode, a.rot_dim);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float m = fabsf(x[p][i]);
      amax          = m <= 3.402823466e38f ? fmaxf(amax, m) : amax;  // (infinities and NaN do not count)
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  }
  if ((threadIdx.x & 31) == 0) {
    red[threadIdx.x >> 5] = amax;
  }
  bad_pos = __syncthreads_or(bad_pos);
  if (bad || bad_pos) {
    if (threadIdx.x == 0) {
      record_error(a.err, bad ? kErrPage : kErrPosition);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) {
    amax = fmaxf(amax, red[i]);
  }
  const long long block  = (long long) page * kv.n_kv_heads + head;
  uint8_t        *codes  = (keys ? kv.k_codes : kv.v_codes) + (block << kv.page_shift) * D;
  float          *scales = (keys ? kv.k_scale : kv.v_scale) + block;
  float           scale  = fmaxf(__fdiv_rn(amax, KVT == kKvI8 ? 127.f : 448.f), kKvMinScale);
  if (from > 0) {
    const float before = *scales;
    scale              = fmaxf(scale, before);
    __syncthreads();  // every thread has read the old scale
    if (scale > before) {
      const float ratio = __fdiv_rn(before, scale);
      for (int i = threadIdx.x; i < from * (D / 8); i += kThreads) {
        uint2 *at = reinterpret_cast<uint2 *>(codes) + i;
        uint2  w  = *at;
        float  c[8];
        from_codes4<KVT>(w.x, c);
        from_codes4<KVT>(w.y, c + 4);
        w.x = to_codes4<KVT>(c, ratio);
        w.y = to_codes4<KVT>(c + 4, ratio);
        *at = w;
      }
    }
  }
  if (threadIdx.x == 0) {
    *scales = scale;
  }
  const float by = __frcp_rn(scale);
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int slot = p * TOKENS + threadIdx.x / PARTS;
    if (slot < from || slot >= to) {
      continue;
    }
    uint8_t *at = codes + slot * D;
    *reinterpret_cast<uint32_t *>(at + lo) = to_codes4<KVT>(x[p], by);
    *reinterpret_cast<uint32_t *>(at + hi) = to_codes4<KVT>(x[p] + 4, by);
  }
}

template <int D, bool A16, bool O16>
__device__ __forceinline__ void rotate_row(const KvAppendArgs &a, int row) {
  constexpr int PARTS = D / 8, BATCH = 2;
  const KvView &kv    = a.kv;
  const uint8_t *src  = static_cast<const uint8_t *>(a.q) + row * a.q_stride * (A16 ? 2 : 4);
  uint8_t       *dst  = static_cast<uint8_t *>(a.q_out) + row * a.q_out_stride * (O16 ? 2 : 4);
  const int      items = a.n_heads * PARTS;
  float          x[BATCH][8];
  auto           load = [&](int i0) {
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int i = i0 + k * kThreads;
      if (i < items) {
        int lo, hi;
        part_dims(i % PARTS, a.mode, a.rot_dim, lo, hi);
        load4<A16>(src, i / PARTS * D + lo, x[k]);
        load4<A16>(src, i / PARTS * D + hi, x[k] + 4);
      }
    }
  };
  load(threadIdx.x);  // (on its way while the row's position is looked up)
  if (row >= kv.q_start[kv.n_seqs]) {
    return;  // behind the last sequence
  }
  int pos = 0;
  if (a.mode) {
    if (a.positions) {
      pos = a.positions[row];
    } else {
      const int b = interval_of(kv.n_seqs, row, [&](int i) { return (long long) kv.q_start[i]; });
      int       q0, q_len, ctx;
      if (b >= kv.n_seqs || !sequence_of(kv, b, kv.n_rows, 0x7fffffff, q0, q_len, ctx) || ctx < q_len) {
        if (threadIdx.x == 0) {
          record_error(a.err, kErrSequence);
        }
        return;
      }
      pos = ctx - q_len + row - q0;
    }
    if (pos < 0 || pos >= a.table_len) {
      if (threadIdx.x == 0) {
        record_error(a.err, kErrPosition);
      }
      return;
    }
  }
  const float *table = a.rope_table + (long long) pos * a.rot_dim;
  for (int i0 = threadIdx.x; i0 < items; i0 += BATCH * kThreads) {
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int i = i0 + k * kThreads;
      if (i >= items) {
        continue;
      }
      const int head = i / PARTS, j = i % PARTS;
      int       lo, hi;
      part_dims(j, a.mode, a.rot_dim, lo, hi);
      if (a.mode) {
        rotate8(x[k], table, j, a.mode, a.rot_dim);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int    at = head * D + (h ? hi : lo);
        const float *y  = x[k] + 4 * h;
        if constexpr (O16) {
          const __half2 u = __floats2half2_rn(y[0], y[1]), w = __floats2half2_rn(y[2], y[3]);
          uint2         o;
          o.x = *reinterpret_cast<const uint32_t *>(&u);
          o.y = *reinterpret_cast<const uint32_t *>(&w);
          *reinterpret_cast<uint2 *>(reinterpret_cast<__half *>(dst) + at) = o;
        } else {
          *reinterpret_cast<float4 *>(reinterpret_cast<float *>(dst) + at) = make_float4(y[0], y[1], y[2], y[3]);
        }
      }
    }
    load(i0 + BATCH * kThreads);
  }
}

template <int D, int KVT, bool A16, bool O16, int PASSES>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const __grid_constant__ KvAppendArgs a) {
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const KvView   &kv     = a.kv;
  const long long caches = a.kv_slots * kv.n_kv_heads * 2;
  if (blockIdx.x >= caches) {
    rotate_row<D, A16, O16>(a, (int) (blockIdx.x - caches));
    return;
  }
  // Page slots: sequence b has those from q_start[b] / page_size + 2 b on, at least as many as its rows can
  // touch pages - the host need not know the lengths.
  const bool      keys = blockIdx.x & 1;
  const int       head = (int) ((blockIdx.x >> 1) % kv.n_kv_heads);
  const long long slot = (blockIdx.x >> 1) / kv.n_kv_heads;
  auto            at   = [&](int i) { return (long long) (kv.q_start[i] >> kv.page_shift) + 2ll * i; };
  const int       b    = interval_of(kv.n_seqs, slot, at);
  if (b >= kv.n_seqs) {
    return;
  }
  append_page<D, KVT, A16, PASSES>(a, b, (int) (slot - at(b)), head, keys);
}

template <int D, int KVT, bool A16, bool O16>
cudaError_t launch_passes(const KvAppendArgs &a, bool pdl, cudaStream_t st) {
  const long long grid   = a.kv_slots * a.kv.n_kv_heads * 2 + (a.q ? a.kv.n_rows : 0);
  const int       passes = a.kv.page_size * (D / 8) / kThreads;
  if (grid > 0x7fffffffll) {
    return cudaErrorInvalidConfiguration;
  }
  switch (passes) {
    case 0:
    case 1: return launch_decoder_kernel(kv_append_kernel<D, KVT, A16, O16, 1>, a, (unsigned) grid, kThreads, 0, pdl, 1, st);
    case 2: return launch_decoder_kernel(kv_append_kernel<D, KVT, A16, O16, 2>, a, (unsigned) grid, kThreads, 0, pdl, 1, st);
    case 4: return launch_decoder_kernel(kv_append_kernel<D, KVT, A16, O16, 4>, a, (unsigned) grid, kThreads, 0, pdl, 1, st);
    default: return launch_decoder_kernel(kv_append_kernel<D, KVT, A16, O16, 8>, a, (unsigned) grid, kThreads, 0, pdl, 1, st);
  }
}

template <int D, int KVT>
cudaError_t launch_types(const KvAppendArgs &a, bool a16, bool o16, bool pdl, cudaStream_t st) {
  if (a16) {
    return o16 ? launch_passes<D, KVT, true, true>(a, pdl, st) : launch_passes<D, KVT, true, false>(a, pdl, st);
  }
  return o16 ? launch_passes<D, KVT, false, true>(a, pdl, st) : launch_passes<D, KVT, false, false>(a, pdl, st);
}

}  // namespace

cudaError_t kv_append_launch(const KvAppendArgs &a, int head_dim, int kv_type, bool a16, bool q_out16, bool pdl,
                             cudaStream_t st) {
  if (head_dim == 64) {
    return kv_type == kKvI8 ? launch_types<64, kKvI8>(a, a16, q_out16, pdl, st) : launch_types<64, kKvE4m3>(a, a16, q_out16, pdl, st);
  }
  return kv_type == kKvI8 ? launch_types<128, kKvI8>(a, a16, q_out16, pdl, st) : launch_types<128, kKvE4m3>(a, a16, q_out16, pdl, st);
}

}  // namespace htp
