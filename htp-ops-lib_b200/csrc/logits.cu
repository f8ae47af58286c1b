// Logits processing before a token is chosen (formula: include/htp_ops_b200.h, htp_b200_logits_process).
//
// A CTA owns a run of CHUNK tokens of one row.  It walks the row's history and biases and counts, in shared
// memory, those that fall into its run (integer counts: their order does not matter; biases are added in
// list order), while the run's logits are already on their way to its registers, and stores them with the few
// tokens that have a penalty or bias fixed and the mask's bits applied: 16-byte loads and stores.  In place
// only what changes is touched.
// Bound: HBM, 8 bytes a logit (out of place), and the phases of short CTAs: 200 rows of 128256 take 57 us against 31.5 of
// HBM time (a copy through the same CTAs 40 us; history 10, biases 4, mask 3 more); one row 4.9 us.  The history
// is read once per run, from L2; runs of 8192 tokens with 512 threads halve that and lose as much to fewer CTAs.
#include <math_constants.h>

#include "decoder_common.cuh"
#include "ptx.cuh"

namespace htp {

namespace {

constexpr int      kListed  = 256;  // biases of a run that are added up by their first ones
constexpr uint32_t kSeen    = 0x80000000u;  // in the history; low bits: times in the answer

template <int CHUNK>
struct Counts {
  uint32_t count[CHUNK];
  float    bias[CHUNK];
  uint32_t touched[CHUNK / 32];  // tokens of the run with a count or a bias
  int2     listed[kListed];
};

// Adds up the biases of a run whose list overflowed: one warp, in list order.
__device__ __noinline__ void add_biases(const LogitsArgs &a, int b0, int n, int t0, int t1, float *bias) {
  const int lane = threadIdx.x & 31;
  for (long long i = 0; i < n; i += 32) {
    const long long j    = i + lane;
    const int       t    = j < n ? a.bias_token[b0 + j] : -1;
    const bool      here = t >= t0 && t < t1;
    // lanes that name the same token add one after the other
    const uint32_t same = __match_any_sync(0xffffffffu, here ? t : -1 - lane);
    const int      rank = __popc(same & ((1u << lane) - 1));
    const int      last = __reduce_max_sync(0xffffffffu, here ? rank : -1);
    const float    v    = here ? a.bias_value[b0 + j] : 0.f;
    for (int r = 0; r <= last; ++r) {
      if (here && rank == r) {
        bias[t - t0] += v;
      }
      __syncwarp();
    }
  }
}

template <int CHUNK, int kThreads>
__global__ void __launch_bounds__(kThreads, 1536 / kThreads) logits_process_kernel(const __grid_constant__ LogitsArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Counts<CHUNK> &sm = *reinterpret_cast<Counts<CHUNK> *>(smem_raw);
  uint32_t      *count = sm.count, *touched = sm.touched;
  float         *bias   = sm.bias;
  int2          *listed = sm.listed;
  __shared__ int n_listed;
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  // Runs are cut at multiples of 16 bytes from the (aligned) start of the buffer: `shift` elements of the
  // row's first group belong to what lies before it.
  const unsigned  chunks = (a.vocab + 3 + CHUNK - 1) / CHUNK;
  const int       row    = (int) (blockIdx.x / chunks);
  const long long base   = row * a.stride;
  const int       shift  = (int) (base & 3);
  const int       v0     = (int) (blockIdx.x % chunks) * CHUNK;  // first element of the run, counted from base - shift
  const int       t0     = v0 - shift;                           // its token
  if (t0 >= a.vocab) {
    return;
  }
  const int    t1       = t0 + CHUNK < a.vocab ? t0 + CHUNK : a.vocab;
  const bool   in_place = a.dst == a.src;
  const float *src      = a.src + (base - shift) + v0;
  float       *dst      = a.dst + (base - shift) + v0;
  // Everything is asked for before anything waits: what the row has beside its logits, ...
  int h0 = 0, h1 = 0, split = 0, b0 = 0, b1 = 0, m = -1;
  if (a.history) {
    h0 = a.history_start[row], h1 = a.history_start[row + 1];
    split = a.prompt_len ? a.prompt_len[row] : 0;
  }
  if (a.bias_token) {
    b0 = a.bias_start[row], b1 = a.bias_start[row + 1];
  }
  if (a.mask) {
    m = a.mask_row ? a.mask_row[row] : row;
  }
  const float rep  = a.repetition ? a.repetition[row] : 1.f;
  const float pres = a.presence ? a.presence[row] : 0.f;
  const float freq = a.frequency ? a.frequency[row] : 0.f;
  // ... the run's logits (in place only those that change are read), ...
  constexpr int V = CHUNK / (4 * kThreads);
  float4        held[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int i = 4 * (threadIdx.x + k * kThreads), t = t0 + i;
    if (!in_place && t >= 0 && t + 4 <= a.vocab) {
      held[k] = __ldcs(reinterpret_cast<const float4 *>(src + i));
    }
  }
  if (h0 < 0 || h1 < h0 || h1 > a.n_history || b0 < 0 || b1 < b0 || b1 > a.n_bias || m < -1 || (m >= a.n_mask_rows && a.mask)) {
    if (threadIdx.x == 0) {
      record_error(a.err, m < -1 || (m >= a.n_mask_rows && a.mask) ? kErrMaskRow : kErrRange);
    }
    h1 = h0 < 0 || h1 < h0 || h1 > a.n_history ? (h0 = 0) : h1;
    b1 = b0 < 0 || b1 < b0 || b1 > a.n_bias ? (b0 = 0) : b1;
    m  = m < -1 || m >= a.n_mask_rows ? -1 : m;
  }
  // ... and the first tokens of history and biases
  const int      n_hist = h1 - h0, n_bias = b1 - b0;
  const int32_t *history = a.history + h0, *bias_token = a.bias_token + b0;
  int            token[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const unsigned i = threadIdx.x + k * kThreads;
    token[k]         = i < (unsigned) n_hist ? history[i] : -1;
  }
  int bias_of = threadIdx.x < (unsigned) n_bias ? bias_token[threadIdx.x] : -1;
#pragma unroll
  for (int i = threadIdx.x; i < CHUNK / 4; i += kThreads) {
    reinterpret_cast<uint4 *>(count)[i] = make_uint4(0, 0, 0, 0);
    reinterpret_cast<float4 *>(bias)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  if (threadIdx.x < CHUNK / 32) {
    touched[threadIdx.x] = 0;
  }
  if (threadIdx.x == 0) {
    n_listed = 0;
  }
  __syncthreads();
  bool any = false;
  auto mark = [&](int t) {
    any = true;
    atomicOr(touched + ((t - t0) >> 5), 1u << ((t - t0) & 31));
  };
  for (unsigned i0 = threadIdx.x; i0 < (unsigned) n_hist; i0 += 4 * kThreads) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int t = token[k];
      if (t >= 0 && t >= t0 && t < t1) {
        mark(t);
        if ((int) (i0 + k * kThreads) >= split) {
          atomicAdd(count + (t - t0), 1u);
        }
        atomicOr(count + (t - t0), kSeen);
      }
      const unsigned i = i0 + (4 + k) * kThreads;
      token[k]         = i < (unsigned) n_hist ? history[i] : -1;
    }
  }
  // Biases: those of this run go to a list, in no order, with their places in the row's list; the first one of
  // each token then adds them up in that order.  A list that overflows is walked by one warp instead.
  for (unsigned i = threadIdx.x; i < (unsigned) n_bias; i += kThreads) {
    const int t = bias_of;
    if (t >= 0 && t >= t0 && t < t1) {
      mark(t);
      const int e = atomicAdd(&n_listed, 1);
      if (e < kListed) {
        listed[e] = make_int2(t - t0, (int) i);
      }
    }
    bias_of = i + kThreads < (unsigned) n_bias ? bias_token[i + kThreads] : -1;
  }
  any = __syncthreads_or(any);
  if (n_listed > kListed) {
    if (threadIdx.x < 32) {
      add_biases(a, b0, n_bias, t0 < 0 ? 0 : t0, t1, bias + (t0 < 0 ? -t0 : 0));
    }
    __syncthreads();
  } else if (n_listed > 0) {
    if ((int) threadIdx.x < n_listed) {
      const int2 mine = listed[threadIdx.x];
      int        at   = mine.y;
      for (int e = 0; e < n_listed; ++e) {
        at = listed[e].x == mine.x && listed[e].y < at ? listed[e].y : at;
      }
      if (at == mine.y) {  // the token's first: it and then the next one of them, and so on
        float sum = 0.f;
        while (at != 0x7fffffff) {
          sum += a.bias_value[(long long) b0 + at];
          int next = 0x7fffffff;
          for (int e = 0; e < n_listed; ++e) {
            next = listed[e].x == mine.x && listed[e].y > at && listed[e].y < next ? listed[e].y : next;
          }
          at = next;
        }
        bias[mine.x] = sum;
      }
    }
    __syncthreads();
  }
  if (in_place && !any && m < 0) {
    return;
  }
  const int       words = (a.vocab + 31) / 32;
  const uint32_t *mask  = m >= 0 ? a.mask + (long long) m * words : nullptr;
  auto            fixed = [&](float y, int i) {
    const uint32_t c = count[i];
    if (c & kSeen) {
      const uint32_t n = c & ~kSeen;
      y                = y > 0.f ? y / rep : y * rep;
      y -= freq * (float) n;
      y -= n ? pres : 0.f;
    }
    return y + bias[i];
  };
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int i = 4 * (threadIdx.x + k * kThreads), t = t0 + i;
    if (t >= a.vocab) {
      break;
    }
    uint32_t allowed = 0xf;  // of tokens t .. t + 3
    if (mask) {
      const int at = t < 0 ? 0 : t, w = at >> 5;
      allowed = __funnelshift_r(mask[w], mask[w + 1 < words ? w + 1 : w], at & 31) << (at - t) & 0xf;
    }
    const uint32_t changes = touched[i >> 5] >> (i & 31) & 0xf;
    if (t >= 0 && t + 4 <= a.vocab && !in_place) {
      float4 y = held[k];
      if (changes) {
#pragma unroll 1
        for (int e = 0; e < 4; ++e) {  // (each element in turn comes to the front and leaves at the back)
          const float z = changes >> e & 1 ? fixed(y.x, i + e) : y.x;
          y             = make_float4(y.y, y.z, y.w, z);
        }
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
    } else if (!in_place || changes || allowed != 0xf) {
#pragma unroll 1
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

template <int CHUNK, int THREADS>
cudaError_t launch_chunks(const LogitsArgs &a, bool pdl, cudaStream_t st) {
  const long long chunks = ((long long) a.vocab + 3 + CHUNK - 1) / CHUNK, grid = chunks * a.rows;
  if (grid > 0x7fffffffll) {
    return cudaErrorInvalidConfiguration;
  }
  const cudaError_t e = allow_smem(reinterpret_cast<const void *>(logits_process_kernel<CHUNK, THREADS>), (int) sizeof(Counts<CHUNK>));
  return e != cudaSuccess ? e : launch_decoder_kernel(logits_process_kernel<CHUNK, THREADS>, a, (unsigned) grid, THREADS, sizeof(Counts<CHUNK>), pdl, 1, st);
}

}  // namespace

cudaError_t logits_process_launch(const LogitsArgs &a, int sm_count, bool pdl, cudaStream_t st) {
  // long runs read the history less often, short ones keep every SM busy with few rows
  if ((long long) a.rows * a.vocab / 4096 >= 4ll * sm_count) {
    return launch_chunks<4096, 256>(a, pdl, st);
  }
  return launch_chunks<1024, 256>(a, pdl, st);
}

}  // namespace htp
