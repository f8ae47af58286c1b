// Logits processing before a token is chosen (formula: include/htp_ops_b200.h, htp_b200_logits_process).
//
// A CTA owns a run of kChunk tokens of one row.  It walks the row's history and biases and counts, in shared
// memory, those that fall into its run (integer counts: their order does not matter; biases are added by
// one warp in list order), then streams the run once: 16-byte loads and stores, the few tokens with a
// penalty or bias fixed on the way, the mask's bits applied.  In place only what changes is touched.
// Bound: HBM, 8 bytes a logit (out of place); the history is read once per run, from L2.
#include <math_constants.h>

#include "decoder_common.cuh"
#include "ptx.cuh"

namespace htp {

namespace {

constexpr int      kThreads = 256;
constexpr uint32_t kSeen    = 0x80000000u;  // in the history; low bits: times in the answer

template <int CHUNK>
__global__ void __launch_bounds__(kThreads) logits_process_kernel(const __grid_constant__ LogitsArgs a) {
  __shared__ __align__(16) uint32_t count[CHUNK];
  __shared__ __align__(16) float    bias[CHUNK];
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  // Runs are cut at multiples of 16 bytes from the (aligned) start of the buffer: `shift` elements of the
  // row's first group belong to what lies before it.
  const int       chunks = (a.vocab + 3 + CHUNK - 1) / CHUNK;
  const long long row    = blockIdx.x / chunks;
  const long long base   = row * a.stride;
  const int       shift  = (int) (base & 3);
  const int       v0     = (int) (blockIdx.x % chunks) * CHUNK;  // first element of the run, counted from base - shift
  const int       t0     = v0 - shift;                           // its token
  if (t0 >= a.vocab) {
    return;
  }
  for (int i = threadIdx.x; i < CHUNK / 4; i += kThreads) {
    reinterpret_cast<uint4 *>(count)[i]  = make_uint4(0, 0, 0, 0);
    reinterpret_cast<float4 *>(bias)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __syncthreads();
  bool touched = false;
  if (a.history) {
    const int h0 = a.history_start[row], h1 = a.history_start[row + 1];
    const int split = a.prompt_len ? a.prompt_len[row] : 0;
    if (h0 < 0 || h1 < h0 || h1 > a.n_history) {
      if (threadIdx.x == 0) {
        record_error(a.err, kErrRange);
      }
    } else {
      for (long long i = (long long) h0 + threadIdx.x; i < h1; i += kThreads) {
        const int t = a.history[i];
        if (t >= 0 && t < a.vocab && t >= t0 && t - t0 < CHUNK) {
          touched = true;
          if (i - h0 >= split) {
            atomicAdd(count + (t - t0), 1u);
          }
          atomicOr(count + (t - t0), kSeen);
        }
      }
    }
  }
  if (a.bias_token && threadIdx.x < 32) {
    const int b0 = a.bias_start[row], b1 = a.bias_start[row + 1];
    if (b0 < 0 || b1 < b0 || b1 > a.n_bias) {
      if (threadIdx.x == 0) {
        record_error(a.err, kErrRange);
      }
    } else {
      for (long long i = b0; i < b1; i += 32) {
        const long long j = i + threadIdx.x;
        const int       t = j < b1 ? a.bias_token[j] : -1;
        const bool here = t >= 0 && t < a.vocab && t >= t0 && t - t0 < CHUNK;
        // lanes that name the same token add one after the other, in list order
        const uint32_t same = __match_any_sync(0xffffffffu, here ? t : -1 - (int) threadIdx.x);
        const int      rank = __popc(same & ((1u << threadIdx.x) - 1));
        const int      most = __reduce_max_sync(0xffffffffu, here ? rank : -1);
        const float    v    = here ? a.bias_value[j] : 0.f;
        for (int r = 0; r <= most; ++r) {
          if (here && rank == r) {
            bias[t - t0] += v;
          }
          __syncwarp();
        }
        touched = touched || here;
      }
    }
  }
  const bool      any = __syncthreads_or(touched);
  const uint32_t *mask = nullptr;
  if (a.mask) {
    const int m = a.mask_row ? a.mask_row[row] : (int) row;
    if (m >= a.n_mask_rows || m < -1) {
      if (threadIdx.x == 0) {
        record_error(a.err, kErrMaskRow);
      }
    } else if (m >= 0) {
      mask = a.mask + (long long) m * ((a.vocab + 31) / 32);
    }
  }
  const bool in_place = a.dst == a.src;
  if (in_place && !any && !mask) {
    return;
  }
  const float rep  = a.repetition ? a.repetition[row] : 1.f;
  const float pres = a.presence ? a.presence[row] : 0.f;
  const float freq = a.frequency ? a.frequency[row] : 0.f;
  auto        fixed = [&](float y, int i) {
    const uint32_t c = count[i];
    if (c & kSeen) {
      const uint32_t n = c & ~kSeen;
      y                = y > 0.f ? y / rep : y * rep;
      y -= freq * (float) n;
      y -= n ? pres : 0.f;
    }
    return y + bias[i];
  };
  const float *src = a.src + (base - shift) + v0;
  float       *dst = a.dst + (base - shift) + v0;
  for (int i = 4 * threadIdx.x; i < CHUNK; i += 4 * kThreads) {
    const int t = t0 + i;
    if (t >= a.vocab) {
      break;
    }
    uint32_t allowed = 0xf;  // of tokens t .. t + 3
    if (mask) {
      if (t >= 0) {
        const uint32_t lo = mask[t >> 5];
        const uint32_t hi = (t & 31) > 28 && (t >> 5) + 1 < (a.vocab + 31) / 32 ? mask[(t >> 5) + 1] : 0u;
        allowed           = __funnelshift_r(lo, hi, t & 31) & 0xf;
      } else {
        allowed = mask[0] << -t & 0xf;
      }
    }
    uint32_t changes = 0;
    if (any) {
      const uint4  c = *reinterpret_cast<const uint4 *>(count + i);
      const float4 b = *reinterpret_cast<const float4 *>(bias + i);
      changes        = ((c.x != 0) | (b.x != 0.f)) | ((c.y != 0) | (b.y != 0.f)) << 1 | ((c.z != 0) | (b.z != 0.f)) << 2 |
                ((c.w != 0) | (b.w != 0.f)) << 3;
    }
    if (t >= 0 && t + 4 <= a.vocab && !in_place) {
      float4 y = __ldcs(reinterpret_cast<const float4 *>(src + i));
      if (changes) {
        y.x = fixed(y.x, i), y.y = fixed(y.y, i + 1), y.z = fixed(y.z, i + 2), y.w = fixed(y.w, i + 3);
      }
      if (allowed != 0xf) {
        y.x = allowed & 1 ? y.x : -CUDART_INF_F;
        y.y = allowed & 2 ? y.y : -CUDART_INF_F;
        y.z = allowed & 4 ? y.z : -CUDART_INF_F;
        y.w = allowed & 8 ? y.w : -CUDART_INF_F;
      }
      __stcs(reinterpret_cast<float4 *>(dst + i), y);
    } else if (t >= 0 && t + 4 <= a.vocab && allowed == 0) {
      __stcs(reinterpret_cast<float4 *>(dst + i), make_float4(-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (t + e < 0 || t + e >= a.vocab) {
          continue;
        }
        const bool ok = allowed >> e & 1, change = changes >> e & 1;
        if (!ok) {
          dst[i + e] = -CUDART_INF_F;
        } else if (change || !in_place) {
          dst[i + e] = change ? fixed(src[i + e], i + e) : src[i + e];
        }
      }
    }
  }
}

template <int CHUNK>
cudaError_t launch_chunks(const LogitsArgs &a, bool pdl, cudaStream_t st) {
  const long long chunks = ((long long) a.vocab + 3 + CHUNK - 1) / CHUNK, grid = chunks * a.rows;
  if (grid > 0x7fffffffll) {
    return cudaErrorInvalidConfiguration;
  }
  return launch_decoder_kernel(logits_process_kernel<CHUNK>, a, (unsigned) grid, kThreads, 0, pdl, 1, st);
}

}  // namespace

cudaError_t logits_process_launch(const LogitsArgs &a, int sm_count, bool pdl, cudaStream_t st) {
  // long runs read the history less often, short ones keep every SM busy with few rows
  if ((long long) a.rows * a.vocab / 4096 >= 4ll * sm_count) {
    return launch_chunks<4096>(a, pdl, st);
  }
  return launch_chunks<1024>(a, pdl, st);
}

}  // namespace htp
