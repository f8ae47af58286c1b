// Residual and norms between two blocks of a decoder (formula: include/htp_ops_b200.h,
// htp_b200_add_rms_norm): one CTA per row, the row kept in registers between the two sums of squares, so that
// x, block and gate are read once and h and the norm written once - HBM-bound, 16 bytes or more an element
// against a handful of operations (8191 x 4096 with a gate per row: 671 MB in 105 us = 0.97 of the measured copy rate; 8
// rows 2.8 us).  Sums are added in a fixed order (per-thread strided partial sums, warp
// tree, warps in order): results do not depend on the launch.
#include <cuda_fp16.h>

#include "decoder_common.cuh"
#include "ptx.cuh"

namespace htp {

namespace {

constexpr int kMaxThreads = 1024;
constexpr int kManyThreads = 512;

__device__ __forceinline__ float cta_sum(float v, float *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  if ((threadIdx.x & 31) == 0) {
    red[threadIdx.x >> 5] = v;
  }
  __syncthreads();
  const int lane = threadIdx.x & 31;
  v              = lane < (int) blockDim.x / 32 ? red[lane] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return v;
}

template <int W>
__device__ __forceinline__ void ld(const float *p, float (&x)[W]) {
  if constexpr (W == 4) {
    const float4 v = *reinterpret_cast<const float4 *>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    x[0] = *p;
  }
}
// read once: not kept
template <int W>
__device__ __forceinline__ void ld_row(const float *p, float (&x)[W]) {
  if constexpr (W == 4) {
    const float4 v = __ldcs(reinterpret_cast<const float4 *>(p));
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    x[0] = __ldcs(p);
  }
}
template <int W>
__device__ __forceinline__ void st(float *p, const float (&x)[W]) {
  if constexpr (W == 4) {
    *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
    *p = x[0];
  }
}
template <int W>
__device__ __forceinline__ void st(__half *p, const float (&x)[W]) {
  if constexpr (W == 4) {
    const __half2 a = __floats2half2_rn(x[0], x[1]), b = __floats2half2_rn(x[2], x[3]);
    uint2         o;
    o.x = *reinterpret_cast<const uint32_t *>(&a);
    o.y = *reinterpret_cast<const uint32_t *>(&b);
    *reinterpret_cast<uint2 *>(p) = o;
  } else {
    *p = __float2half_rn(x[0]);
  }
}

// V groups of W elements a thread in registers; V = 0: rows longer than the registers take, walked three
// times (the sums of squares of the block and of h, then the norm; h is recomputed or read back).
template <int W, int V, typename Out>
__global__ void __launch_bounds__(kMaxThreads) add_rms_norm_kernel(const __grid_constant__ AddRmsNormArgs a) {
  __shared__ float red[2][kMaxThreads / 32];
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const long long row   = blockIdx.x;
  const float    *x     = a.x + row * a.n;
  const float    *block = a.block ? a.block + row * a.n : nullptr;
  const float    *gate  = a.gate ? a.gate + row * a.gate_stride : nullptr;
  float          *h_out = a.h_out ? a.h_out + row * a.n : nullptr;
  Out            *out   = a.norm_out ? static_cast<Out *>(a.norm_out) + row * a.n : nullptr;
  const int       step  = blockDim.x * W;
  // b of this element after the post norm's scale, the gate and the residual
  auto residual = [&](int i, float post, float (&h)[W], const float (&bv)[W]) {
    float w[W], g[W];
    if (a.post_weight) {
      ld<W>(a.post_weight + i, w);
    }
    if (gate) {
      ld<W>(gate + i, g);
    }
#pragma unroll
    for (int e = 0; e < W; ++e) {
      float b = bv[e];
      if (a.post_weight) {
        b = b * post * w[e];
      }
      if (gate) {
        b *= g[e];
      }
      h[e] = fmaf(a.block_scale, b, h[e]);
    }
  };
  if constexpr (V > 0) {
    // every operand is asked for before the first sum waits for its row (the longest rows leave no registers for
    // that: gate and weights are read where they are used)
    constexpr bool EARLY = V <= 2;
    float h[V][W], bv[V][W], pw[V][W], g[V][W], w[V][W];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = threadIdx.x * W + v * step;
      if (i < a.n) {
        ld_row<W>(x + i, h[v]);
        if (block) {
          ld_row<W>(block + i, bv[v]);
        }
        if (EARLY && gate) {
          ld<W>(gate + i, g[v]);
        }
        if (EARLY && a.post_weight) {
          ld<W>(a.post_weight + i, pw[v]);
        }
        if (EARLY && a.weight) {
          ld<W>(a.weight + i, w[v]);
        }
      }
    }
    float ss = 0.f, post = 1.f;
    if (a.post_weight) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (threadIdx.x * W + v * step < a.n) {
#pragma unroll
          for (int e = 0; e < W; ++e) {
            ss = fmaf(bv[v][e], bv[v][e], ss);
          }
        }
      }
      post = 1.0f / sqrtf(cta_sum(ss, red[0]) / (float) a.n + a.eps);
    }
    ss = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = threadIdx.x * W + v * step;
      if (i < a.n) {
        if (!EARLY && gate) {
          ld<W>(gate + i, g[v]);
        }
        if (!EARLY && a.post_weight) {
          ld<W>(a.post_weight + i, pw[v]);
        }
#pragma unroll
        for (int e = 0; e < W; ++e) {
          if (block) {
            float b = bv[v][e];
            b       = a.post_weight ? b * post * pw[v][e] : b;
            b       = gate ? b * g[v][e] : b;
            h[v][e] = fmaf(a.block_scale, b, h[v][e]);
          }
          ss = fmaf(h[v][e], h[v][e], ss);
        }
        if (h_out) {
          st<W>(h_out + i, h[v]);
        }
      }
    }
    if (!out) {
      return;
    }
    const float scale = 1.0f / sqrtf(cta_sum(ss, red[1]) / (float) a.n + a.eps);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = threadIdx.x * W + v * step;
      if (i < a.n) {
        if (!EARLY && a.weight) {
          ld<W>(a.weight + i, w[v]);
        }
#pragma unroll
        for (int e = 0; e < W; ++e) {
          h[v][e] = a.weight ? h[v][e] * scale * w[v][e] : h[v][e] * scale;
        }
        st<W>(out + i, h[v]);
      }
    }
  } else {
    float ss = 0.f, post = 1.f;
    if (block && a.post_weight) {
      for (int i = threadIdx.x * W; i < a.n; i += step) {
        float b[W];
        ld<W>(block + i, b);
#pragma unroll
        for (int e = 0; e < W; ++e) {
          ss = fmaf(b[e], b[e], ss);
        }
      }
      post = 1.0f / sqrtf(cta_sum(ss, red[0]) / (float) a.n + a.eps);
    }
    auto h_at = [&](int i, float (&h)[W]) {
      ld<W>(x + i, h);
      if (block) {
        float b[W];
        ld<W>(block + i, b);
        residual(i, post, h, b);
      }
    };
    ss = 0.f;
    for (int i = threadIdx.x * W; i < a.n; i += step) {
      float h[W];
      h_at(i, h);
      if (h_out) {
        st<W>(h_out + i, h);
      }
#pragma unroll
      for (int e = 0; e < W; ++e) {
        ss = fmaf(h[e], h[e], ss);
      }
    }
    if (!out) {
      return;
    }
    const float scale = 1.0f / sqrtf(cta_sum(ss, red[1]) / (float) a.n + a.eps);
    for (int i = threadIdx.x * W; i < a.n; i += step) {
      float h[W], w[W];
      if (h_out) {
        ld<W>(h_out + i, h);  // (h_out may be x or block: what this thread wrote above)
      } else {
        h_at(i, h);
      }
      if (a.weight) {
        ld<W>(a.weight + i, w);
      }
#pragma unroll
      for (int e = 0; e < W; ++e) {
        h[e] = a.weight ? h[e] * scale * w[e] : h[e] * scale;
      }
      st<W>(out + i, h);
    }
  }
}

template <int W, typename Out>
cudaError_t launch_width(const AddRmsNormArgs &a, bool pdl, cudaStream_t st) {
  const long long groups  = ((long long) a.n + W - 1) / W;
  // Few rows: as many threads as there are groups, for the latency.  Many: fewer threads with more groups each, so
  // that more rows are on an SM at once.
  const int       most    = a.rows > 296 ? kManyThreads : kMaxThreads;
  const long long t1      = (groups + 31) / 32 * 32;
  const unsigned  threads = (unsigned) (t1 < most ? t1 : (groups > 4ll * most ? kMaxThreads : most));
  const long long per     = (groups + threads - 1) / threads;
  const unsigned  grid    = (unsigned) a.rows;
  if (per <= 1) {
    return launch_decoder_kernel(add_rms_norm_kernel<W, 1, Out>, a, grid, threads, 0, pdl, 1, st);
  }
  if (per <= 2) {
    return launch_decoder_kernel(add_rms_norm_kernel<W, 2, Out>, a, grid, threads, 0, pdl, 1, st);
  }
  if (per <= 4) {
    return launch_decoder_kernel(add_rms_norm_kernel<W, 4, Out>, a, grid, threads, 0, pdl, 1, st);
  }
  return launch_decoder_kernel(add_rms_norm_kernel<W, 0, Out>, a, grid, threads, 0, pdl, 1, st);
}

}  // namespace

cudaError_t add_rms_norm_launch(const AddRmsNormArgs &a, bool norm16, bool pdl, cudaStream_t st) {
  // four elements at a time when every row of every operand is 16-byte aligned (fp16 norms: 8)
  const uintptr_t all = (uintptr_t) a.x | (uintptr_t) a.block | (uintptr_t) a.h_out | (uintptr_t) a.post_weight |
                        (uintptr_t) a.gate | (uintptr_t) a.weight | (norm16 ? (uintptr_t) a.norm_out << 1 : (uintptr_t) a.norm_out);
  const bool wide = a.n % 4 == 0 && (all & 15) == 0 && a.gate_stride % 4 == 0;
  if (norm16) {
    return wide ? launch_width<4, __half>(a, pdl, st) : launch_width<1, __half>(a, pdl, st);
  }
  return wide ? launch_width<4, float>(a, pdl, st) : launch_width<1, float>(a, pdl, st);
}

}  // namespace htp
