// Attention over the paged 8-bit cache for few rows per sequence (formula: include/htp_ops_b200.h,
// htp_b200_attn_paged).
//
// All query rows and heads that read one key/value head are the COLUMNS of one tile (8 or 16 of them), so
// every code is fetched from HBM once and the warp-level tensor-core instructions work on full tiles:
//   S^T[token][column] = K[token][d] . Q^T[d][column]     A = 16 tokens of codes, B = the queries
//   O^T[d][column]    += V^T[d][token] . P^T[token][column]
// Codes become fp16 exactly (signed bytes and e4m3 both fit) on their way from shared memory to the A
// fragments, in registers: the order of d inside a fragment is free as long as K and Q (or V^T and O^T)
// agree, so each lane loads 16 contiguous bytes of a row.  P^T comes from S^T by an 8 x 8 transpose in the
// warp.  fp32 queries and weights are two fp16 terms each (hi + lo), two MMAs into the same accumulator.
//
// Scales never touch the codes.  With x = s * (k_scale * scale * log2 e) + log2(v_scale) the weight
// n = 2^(x - M) carries the value block's scale (M: running maximum of x, raised only when x leaves it more
// than kSlack behind), O sums n * code, and the softmax denominator sums n / v_scale per block: one running
// maximum, one FMA and one exponential per score, everything in fp32.
//
// Work: CTA = 4 warps; a warp walks 32-token steps of its CTA's share of the context, the next steps
// on their way to its ring in shared memory meanwhile: tiled copies of 16 tokens (2 KB runs in
// HBM; 64- and 128-byte pieces fetched by the lanes themselves reached 4.4 of 6.5 TB/s with nothing computed).
// Two steps a warp leave room for three CTAs on an SM; three steps and two CTAs were 9 % slower.
// Few short contexts are shared by the CTAs of a cluster, whose results meet in distributed shared memory in rank
// order; otherwise by independent CTAs whose results meet in the workspace and a second small launch
// (attn_plan).  No atomics: results do not depend on scheduling.
//
// Bound: HBM; 64 contexts of up to 8192 tokens, fp16 and e4m3: 97 us for 539 MB = 0.85 of the measured copy rate (the
// copies alone 85 us, the arithmetic alone 78); fp32 doubles the products: 2 contexts of 131072, 8 columns, 114 us.
#include <cooperative_groups.h>
#include <cuda.h>
#include <cuda_fp16.h>

#include "attn_common.cuh"
#include "ptx.cuh"

namespace cg = cooperative_groups;

namespace htp {

namespace {

constexpr int   kWarps   = 4;
constexpr int   kThreads = kWarps * 32;
constexpr int   kStep    = 32;  // tokens of a warp's step: two 16-token MMA tiles
constexpr int   kStages  = 2;   // steps of a warp in shared memory or on their way
constexpr int   kChain   = 6;   // fp32: steps after which the running sums are put aside
// One step of a warp: two 16-token tiles of keys and of values as the copy engine lays them down, rows of D bytes
// with their 16-byte chunks swizzled by the row (128 or 64 bytes wide).
template <int D>
struct alignas(1024) DecodeStage {
  uint8_t k[2][16 * D], v[2][16 * D];
};
// byte offset of the 16-byte chunk c of row r
template <int D>
__device__ __forceinline__ int swizzled(int r, int c) {
  return D == 128 ? r * 128 + ((c ^ (r & 7)) << 4) : r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
}
// Token of MMA row (and of position k of the second product) i, 0 .. 7; rows 8 .. 15 are its tokens plus 8.
// Rows of one 8-lane phase then differ in bits 0 and 2, the rows of one lane group in bits 1 and 2: no two
// lanes of a phase meet on a bank, whether they read keys by rows or values by columns.
__device__ __forceinline__ int token_of(int i) {
  return i & 1 ? (i - 1) ^ 5 : i;
}

struct DecodeArgs {
  AttnArgs    a;
  CUtensorMap kmap, vmap;  // codes as rows of head_dim bytes, boxes of 16 rows
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <int KVT, int D, int NT, bool F32>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 3 : 2) attn_decode_kernel(const __grid_constant__ DecodeArgs args) {
  const AttnArgs &a = args.a;
  constexpr int NC    = NT * 8;
  constexpr int KI    = D / 64;          // 16-byte pieces of a key row per lane
  constexpr int MT    = D / 16;          // 16-row tiles of O^T
  constexpr int VW    = D / 32;          // words of a value row per lane (8 lanes x VW words = a row)
  constexpr int TERMS = F32 ? 2 : 1;
  constexpr int QP    = D + 8;           // pitch of a query column in shared memory (halves): conflict-free 16-byte reads
  constexpr int OP    = D + 4;           // pitch of an output column (floats)
  using Stage = DecodeStage<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + (-smem_u32(smem_raw) & 1023u);  // (the same in every CTA of a cluster)
  Stage   *ring = reinterpret_cast<Stage *>(smem) + (threadIdx.x >> 5) * kStages;  // this warp's
  // the warps' results take the rings' place
  float(*sm_o)[NC][OP] = reinterpret_cast<float(*)[NC][OP]>(smem);
  static_assert(sizeof(float) * kWarps * NC * OP <= sizeof(Stage) * kWarps * kStages, "room for the results");
  __shared__ __align__(16) __half sm_q[TERMS][NC][QP];
  __shared__ float ml[kWarps][2][NC];
  __shared__ float q_unit[NC];  // fp32 queries: the power of two that a column was divided by
  __shared__ uint64_t bars[kWarps][kStages];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bars[warp][i], 1);
    }
    mbar_fence_init();
    tma_prefetch_descriptor(&args.kmap);
    tma_prefetch_descriptor(&args.vmap);
  }
  __syncwarp();
  pdl_launch_dependents();
  pdl_wait_prior_grids();

  const KvView &kv = a.kv;
  unsigned      id    = blockIdx.x;
  const int     split = id % a.splits;
  id /= a.splits;
  const int grp = id % a.groups;
  id /= a.groups;
  const int head = id % kv.n_kv_heads;
  id /= kv.n_kv_heads;
  const int cols0 = (int) (id % a.col_groups) * NC;
  const int b     = id / a.col_groups;

  int q0, q_len, ctx;
  if (!sequence_of(kv, b, a.max_q, a.max_ctx, q0, q_len, ctx)) {
    if (threadIdx.x == 0) {
      record_error(a.err, kErrSequence);
    }
    return;  // (every CTA of the cluster leaves here)
  }
  const int n_cols = q_len * a.group - cols0 < NC ? q_len * a.group - cols0 : NC;  // columns in use
  if (n_cols <= 0) {
    return;
  }
  const int past = ctx - q_len;  // token number of row 0 (negative: the first rows see nothing)
  const int r0 = cols0 / a.group, r1 = (cols0 + n_cols - 1) / a.group;
  int       hi = past + r1 + 1, lo = 0;
  hi = hi < 0 ? 0 : hi;
  if (a.window > 0 && past + r0 - a.window + 1 > 0) {
    lo = past + r0 - a.window + 1;
  }
  const int s0 = lo / kStep, steps = hi > lo ? (hi + kStep - 1) / kStep - s0 : 0;
  const int parts = a.splits * a.groups, part = grp * a.splits + split;
  const int begin = s0 + (int) ((long long) steps * part / parts), end = s0 + (int) ((long long) steps * (part + 1) / parts);

  // queries -> shared memory, unused columns as zeros.  fp32 columns are divided by the power of two that
  // brings their largest magnitude into [2^13, 2^14): nothing overflows fp16 and the second term keeps its bits.
  for (int i = threadIdx.x; i < NC * (D / 4); i += kThreads) {
    const int c = i / (D / 4), d = i % (D / 4) * 4;
    float4    v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c < n_cols) {
      const int       r  = (cols0 + c) / a.group, h = head * a.group + (cols0 + c) % a.group;
      const long long at = (long long) (q0 + r) * a.q_stride + h * D + d;
      if constexpr (F32) {
        v = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + at);
      } else {
        *reinterpret_cast<uint2 *>(&sm_q[0][c][d]) = *reinterpret_cast<const uint2 *>(static_cast<const __half *>(a.q) + at);
        continue;
      }
    }
    if constexpr (F32) {
      float m = fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
#pragma unroll
      for (int o = D / 8; o > 0; o >>= 1) {  // (the D / 4 lanes of a column: a warp, or half of one)
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      }
      float unit, f;
      query_unit(m, unit, f);
      v.x *= f, v.y *= f, v.z *= f, v.w *= f;
      if (d == 0) {
        q_unit[c] = unit;
      }
    }
    uint2 h, l;
    split_h2(v.x, v.y, h.x, l.x);
    split_h2(v.z, v.w, h.y, l.y);
    *reinterpret_cast<uint2 *>(&sm_q[0][c][d]) = h;
    if constexpr (F32) {
      *reinterpret_cast<uint2 *>(&sm_q[TERMS - 1][c][d]) = l;
    }
  }
  // what the lane's columns (2 t, 2 t + 1 of each 8) see: tokens first[] .. last[]
  int last[NT][2], first[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int c = cols0 + n * 8 + 2 * t + j;
      last[n][j]  = past + c / a.group;
      first[n][j] = a.window > 0 ? last[n][j] - a.window + 1 : 0;
    }
  }
  const int all_from = a.window > 0 ? past + r1 - a.window + 1 : 0, all_to = past + r0;  // seen by every column

  const int       P = kv.page_size;
  const int      *table = kv.page_table + (long long) b * kv.table_stride;
  // page numbers of a step's two tiles as they stand in the table (-1 where there is nothing to read)
  auto ask = [&](int step, int (&raw)[2]) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int tok = step * kStep + m * 16;
      raw[m]        = step < end && tok < hi && tok + 16 > lo ? table[tok >> kv.page_shift] : -1;
    }
  };
  // Asks for a step: four tiled copies on one barrier, and per lane the scales of tile lane & 1.  raw: checked
  // on the way, -1 for a bad entry.
  const uint64_t policy = l2_policy_evict_first();
  auto fetch = [&](int step, int slot, int (&raw)[2], float (&scale)[2]) {
    int tiles = 0;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int tok = step * kStep + m * 16;
      if (raw[m] < 0 || raw[m] >= kv.n_pages) {
        if (lane == 0 && step < end && tok < hi && tok + 16 > lo) {
          record_error(a.err, kErrPage);
        }
        raw[m] = -1;
      } else {
        ++tiles;
      }
    }
    if (lane == 0) {
      uint64_t *bar = &bars[warp][slot];
      mbar_arrive_expect_tx(bar, tiles * 2 * 16 * D);
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        if (raw[m] >= 0) {
          // (the entry points see to it that a cache has fewer than 2^31 rows)
          const int row = (((raw[m] * kv.n_kv_heads) + head) << kv.page_shift) + ((step * kStep + m * 16) & (P - 1));
          tma_load_2d(ring[slot].k[m], &args.kmap, 0, row, bar, policy);
          tma_load_2d(ring[slot].v[m], &args.vmap, 0, row, bar, policy);
        }
      }
    }
    const int mine = lane & 1 ? raw[1] : raw[0];
    if (mine >= 0) {
      const long long block = (long long) mine * kv.n_kv_heads + head;
      scale[0] = kv.k_scale[block], scale[1] = kv.v_scale[block];
    }
  };

  float o[NT][MT][4], l[NT][2], mx[NT][2];
  // fp32: the matrix instructions' sums are cut at their last bit, not rounded; every kChain steps they are added to sums
  // that are (where the registers allow it: 10727 tokens in two shares 1.5e-6 off without, plain fp32 sums 0.8e-6)
  constexpr bool CHAINS = F32 && NT * MT <= 8;
  float          done[CHAINS ? NT : 1][CHAINS ? MT : 1][4] = {};
  int            chain = 0;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    l[n][0] = l[n][1] = 0.f;
    mx[n][0] = mx[n][1] = kFloor;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    }
  }
  bool huge = false;
  int  step = begin + warp;
  int   pg[kStages][2], ahead[2];  // pages of the steps in the ring, and of the one after them
  float scale[kStages][2];         // and scales
#pragma unroll
  for (int i = 0; i < kStages; ++i) {
    ask(step + i * kWarps, pg[i]);
  }
#pragma unroll
  for (int i = 0; i < kStages; ++i) {
    fetch(step + i * kWarps, i, pg[i], scale[i]);
  }
  ask(step + kStages * kWarps, ahead);
  int      slot   = 0;
  uint32_t parity = 0;
  __syncthreads();  // the queries are in place
  float unit[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      unit[n][j] = F32 ? q_unit[n * 8 + 2 * t + j] : 1.f;
    }
  }

#pragma unroll 1
  for (; step < end; step += kWarps) {
    Stage &st = ring[slot];
    if (!__all_sync(0xffffffffu, mbar_wait(&bars[warp][slot], parity))) {
      record_error(a.err, kErrWait);
      break;
    }
    // ---- scores
    float s[2][NT][4], s2[2][NT][4];  // (fp32: what the second terms make, apart: it is lost in no large sum)
    float by[2], up[2], inv[2];
    block_scales(scale[0][0], scale[0][1], a.scale_log2, by[0], up[0], inv[0]);  // (of the lane's tile)
#pragma unroll
    for (int m = 1; m >= 0; --m) {
      by[m]  = __shfl_sync(0xffffffffu, by[0], m);
      up[m]  = __shfl_sync(0xffffffffu, up[0], m);
      inv[m] = __shfl_sync(0xffffffffu, inv[0], m);
      if (pg[0][m] < 0) {
        by[m] = 1.f, up[m] = inv[m] = 0.f;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        s[m][n][0] = s[m][n][1] = s[m][n][2] = s[m][n][3] = 0.f;
        s2[m][n][0] = s2[m][n][1] = s2[m][n][2] = s2[m][n][3] = 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < KI; ++i) {
#pragma unroll
      for (int w2 = 0; w2 < 2; ++w2) {
        uint4 qf[NT][TERMS];  // two words of codes against 8 halves of the lane's column
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int x = 0; x < TERMS; ++x) {
            qf[n][x] = *reinterpret_cast<const uint4 *>(&sm_q[x][n * 8 + g][i * 64 + t * 16 + w2 * 8]);
          }
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const uint2 k0 = *reinterpret_cast<const uint2 *>(st.k[m] + swizzled<D>(token_of(g), 4 * i + t) + 8 * w2);
          const uint2 k1 = *reinterpret_cast<const uint2 *>(st.k[m] + swizzled<D>(token_of(g) + 8, 4 * i + t) + 8 * w2);
#pragma unroll
          for (int w1 = 0; w1 < 2; ++w1) {
            const uint32_t c0 = w1 ? k0.y : k0.x, c1 = w1 ? k1.y : k1.x;
            uint32_t       h0[2], h1[2];
            codes_to_h2<KVT>(c0, h0);
            codes_to_h2<KVT>(c1, h1);
            const uint32_t af[4] = { h0[0], h1[0], h0[1], h1[1] };
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
              for (int x = 0; x < TERMS; ++x) {
                mma_16816(x ? s2[m][n] : s[m][n], af, w1 ? qf[n][x].z : qf[n][x].x, w1 ? qf[n][x].w : qf[n][x].y);
              }
            }
          }
        }
      }
    }
    if constexpr (F32) {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[m][n][e] += s2[m][n][e];
          }
        }
      }
    }
    const int live[2] = { pg[0][0], pg[0][1] };
    // ---- weights
    const int  tok0 = step * kStep;
    const bool full = live[0] >= 0 && live[1] >= 0 && tok0 >= all_from && tok0 + kStep - 1 <= all_to;
    if (!full) {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int tok = tok0 + m * 16 + token_of(g) + (e >> 1) * 8;
            if (live[m] < 0 || tok > last[n][e & 1] || tok < first[n][e & 1]) {
              s[m][n][e] = -INFINITY;
            }
          }
        }
      }
    }
    auto exponent = [&](int m, int n, int e) {
      const float b = by[m] * unit[n][e & 1], x = mx[n][e & 1];
      return huge ? fmaf(s[m][n][e], b, up[m]) - x + kLift : fmaf(s[m][n][e], b, up[m] - x + kLift);
    };
    float y[2][NT][4];
    float top = -INFINITY;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[m][n][e] = exponent(m, n, e);
          top        = fmaxf(top, y[m][n][e]);
        }
      }
    }
    if (__any_sync(0xffffffffu, top > kLift + kSlack)) {
      bool far = false;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float x = kFloor;
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            x = fmaxf(x, fmaxf(fmaf(s[m][n][j], by[m] * unit[n][j], up[m]), fmaf(s[m][n][j + 2], by[m] * unit[n][j], up[m])));
          }
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          x = fmaxf(x, mx[n][j]);
          const float f = exp2_approx(mx[n][j] - x);
          mx[n][j]      = x;
          l[n][j] *= f;
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            o[n][i][j] *= f;
            o[n][i][j + 2] *= f;
            if constexpr (CHAINS) {
              done[n][i][j] *= f;
              done[n][i][j + 2] *= f;
            }
          }
        }
        far = far || (fabsf(mx[n][0]) > kHuge && mx[n][0] != kFloor) || (fabsf(mx[n][1]) > kHuge && mx[n][1] != kFloor);
      }
      huge = __any_sync(0xffffffffu, far);
#pragma unroll
      for (int m = 0; m < 2; ++m) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[m][n][e] = exponent(m, n, e);
          }
        }
      }
    }
    uint32_t pf[2][NT][TERMS][2];  // B fragments: tokens 2 t, 2 t + 1 and 2 t + 8, 2 t + 9 of column g
#pragma unroll
    for (int m = 0; m < 2; ++m) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[m][n][e] = exp2_approx(y[m][n][e]);
        }
        l[n][0] = fmaf(y[m][n][0] + y[m][n][2], inv[m], l[n][0]);
        l[n][1] = fmaf(y[m][n][1] + y[m][n][3], inv[m], l[n][1]);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if constexpr (F32) {
            uint32_t h, lo16;
            split_h2(y[m][n][2 * r], y[m][n][2 * r + 1], h, lo16);
            pf[m][n][0][r]         = transpose8x8(h);
            pf[m][n][TERMS - 1][r] = transpose8x8(lo16);
          } else {
            pf[m][n][0][r] = transpose8x8(pack_h2(y[m][n][2 * r], y[m][n][2 * r + 1]));
          }
        }
      }
    }
    // ---- O^T += V^T P^T
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      uint32_t vr[4][VW];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = token_of(2 * t + (r & 1)) + (r >> 1) * 8;  // positions 2 t, 2 t + 1, 2 t + 8, 2 t + 9
        if constexpr (VW == 4) {
          const uint4 v = *reinterpret_cast<const uint4 *>(st.v[m] + swizzled<D>(row, g));
          vr[r][0] = v.x, vr[r][1] = v.y, vr[r][2] = v.z, vr[r][3] = v.w;
        } else {
          const uint2 v = *reinterpret_cast<const uint2 *>(st.v[m] + swizzled<D>(row, g >> 1) + (g & 1) * 8);
          vr[r][0] = v.x, vr[r][1] = v.y;
        }
        // (codes behind the context may be no numbers: their weight 0 would not hide them)
        const int tok = tok0 + m * 16 + row;
        if (!full && (live[m] < 0 || tok >= hi || tok < lo)) {
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            vr[r][w] = 0;
          }
        }
      }
#pragma unroll
      for (int w = 0; w < VW; ++w) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          // codes (token A, token B) of d = 4 w + 2 half and of the one after it, side by side
          const uint32_t sel = half ? 0x7362 : 0x5140;
          uint32_t       ab[2], cd[2];
          codes_to_h2<KVT>(__byte_perm(vr[0][w], vr[1][w], sel), ab);
          codes_to_h2<KVT>(__byte_perm(vr[2][w], vr[3][w], sel), cd);
          const uint32_t af[4] = { ab[0], ab[1], cd[0], cd[1] };
#pragma unroll
          for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int x = 0; x < TERMS; ++x) {
              mma_16816(o[n][2 * w + half], af, pf[m][n][x][0], pf[m][n][x][1]);
            }
          }
        }
      }
    }
    if constexpr (CHAINS) {
      if (++chain == kChain || step + kWarps >= end) {
        chain = 0;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int i = 0; i < MT; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              done[n][i][e] += o[n][i][e];
              o[n][i][e] = step + kWarps >= end ? done[n][i][e] : 0.f;
            }
          }
        }
      }
    }
    // the slot takes the step after those in the ring
    __syncwarp();  // (everybody has used what lay there)
#pragma unroll
    for (int i = 0; i + 1 < kStages; ++i) {
      pg[i][0] = pg[i + 1][0], pg[i][1] = pg[i + 1][1];
      scale[i][0] = scale[i + 1][0], scale[i][1] = scale[i + 1][1];
    }
    fetch(step + kStages * kWarps, slot, ahead, scale[kStages - 1]);
    pg[kStages - 1][0] = ahead[0], pg[kStages - 1][1] = ahead[1];
    ask(step + (kStages + 1) * kWarps, ahead);
    if (++slot == kStages) {
      slot = 0, parity ^= 1;
    }
  }

  // ---- the warps' results, in warp order
  __syncthreads();  // the rings are no longer needed
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int c = n * 8 + 2 * t + j;
      float     x = l[n][j];
      x += __shfl_xor_sync(0xffffffffu, x, 4);
      x += __shfl_xor_sync(0xffffffffu, x, 8);
      x += __shfl_xor_sync(0xffffffffu, x, 16);
      if (g == 0) {
        ml[warp][0][c] = mx[n][j];
        ml[warp][1][c] = x;
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        *reinterpret_cast<float2 *>(&sm_o[warp][c][g * (D / 8) + 2 * i]) = make_float2(o[n][i][j], o[n][i][j + 2]);
      }
    }
  }
  __syncthreads();
  constexpr int PER = NC * (D / 4) / kThreads;  // groups of four outputs a thread adds
  float         m_cta[PER], l_cta[PER];
  float4        acc[PER];
#pragma unroll
  for (int p = 0; p < PER; ++p) {
    const int i = threadIdx.x + p * kThreads, c = i / (D / 4), d = i % (D / 4) * 4;
    float     m = kFloor, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      m = fmaxf(m, ml[w][0][c]);
    }
    acc[p] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float  f = exp2_approx(ml[w][0][c] - m);
      const float4 v = *reinterpret_cast<const float4 *>(&sm_o[w][c][d]);
      sum            = fmaf(f, ml[w][1][c], sum);
      acc[p].x = fmaf(f, v.x, acc[p].x), acc[p].y = fmaf(f, v.y, acc[p].y);
      acc[p].z = fmaf(f, v.z, acc[p].z), acc[p].w = fmaf(f, v.w, acc[p].w);
    }
    m_cta[p] = m, l_cta[p] = sum;
  }

  // ---- the cluster's results, in rank order: every CTA leaves its sums in warp slot 0, then each thread of
  // rank r adds the groups i with i % splits == r
  if (a.splits > 1) {
    __syncthreads();
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int i = threadIdx.x + p * kThreads, c = i / (D / 4), d = i % (D / 4) * 4;
      *reinterpret_cast<float4 *>(&sm_o[0][c][d]) = acc[p];
      if (d == 0) {
        ml[0][0][c] = m_cta[p], ml[0][1][c] = l_cta[p];
      }
    }
    cg::this_cluster().sync();
  }
  auto finish = [&](int c, int d, float m, float sum, float4 v) {
    if (c >= n_cols) {
      return;
    }
    const int r = (cols0 + c) / a.group, h = head * a.group + (cols0 + c) % a.group;
    if (a.groups > 1) {
      // partial results, [cluster][sequence][row][head]: D sums, then maximum and denominator
      const long long at = (((long long) grp * kv.n_seqs + b) * a.max_q + r) * a.n_heads + h;
      float          *to = a.part + at * (D + 4);
      *reinterpret_cast<float4 *>(to + d) = v;
      if (d == 0) {
        *reinterpret_cast<float2 *>(to + D) = make_float2(m, sum);
      }
      return;
    }
    const float     f  = sum > 0.f ? 1.f / sum : 0.f;
    const long long at = (long long) (q0 + r) * a.out_stride + h * D + d;
    if constexpr (F32) {
      *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + at) = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
    } else {
      uint2 u;
      u.x = pack_h2(v.x * f, v.y * f);
      u.y = pack_h2(v.z * f, v.w * f);
      *reinterpret_cast<uint2 *>(static_cast<__half *>(a.out) + at) = u;
    }
  };
  if (a.splits == 1) {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int i = threadIdx.x + p * kThreads;
      finish(i / (D / 4), i % (D / 4) * 4, m_cta[p], l_cta[p], acc[p]);
    }
    return;
  }
  cg::cluster_group cluster = cg::this_cluster();
  for (int i = threadIdx.x * a.splits + split; i < NC * (D / 4); i += kThreads * a.splits) {
    const int c = i / (D / 4), d = i % (D / 4) * 4;
    float     m = kFloor, sum = 0.f;
    float4    v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int r = 0; r < a.splits; ++r) {
      m = fmaxf(m, *cluster.map_shared_rank(&ml[0][0][c], r));
    }
    for (int r = 0; r < a.splits; ++r) {
      const float  f = exp2_approx(*cluster.map_shared_rank(&ml[0][0][c], r) - m);
      const float4 x = *reinterpret_cast<const float4 *>(cluster.map_shared_rank(&sm_o[0][c][d], r));
      sum            = fmaf(f, *cluster.map_shared_rank(&ml[0][1][c], r), sum);
      v.x = fmaf(f, x.x, v.x), v.y = fmaf(f, x.y, v.y), v.z = fmaf(f, x.z, v.z), v.w = fmaf(f, x.w, v.w);
    }
    finish(c, d, m, sum, v);
  }
  cluster.sync();  // nobody leaves while others read its shared memory
}

// The clusters' results of one (sequence, row, head) per warp, in cluster order.
template <int D, bool F32>
__global__ void __launch_bounds__(128) attn_join_kernel(const __grid_constant__ AttnArgs a) {
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const long long id   = (long long) blockIdx.x * 4 + (threadIdx.x >> 5);
  const int       lane = threadIdx.x & 31;
  const int       h = (int) (id % a.n_heads), r = (int) (id / a.n_heads % a.max_q), b = (int) (id / a.n_heads / a.max_q);
  int             q0, q_len, ctx;
  if (b >= a.kv.n_seqs || !sequence_of(a.kv, b, a.max_q, a.max_ctx, q0, q_len, ctx) || r >= q_len) {
    return;
  }
  const long long each = (long long) a.kv.n_seqs * a.max_q * a.n_heads * (D + 4);
  const float    *from = a.part + id * (D + 4);
  float           m = kFloor, sum = 0.f, v[D / 32] = {};
  for (int k = 0; k < a.groups; ++k) {
    m = fmaxf(m, from[k * each + D]);
  }
  for (int k = 0; k < a.groups; ++k) {
    const float f = exp2_approx(from[k * each + D] - m);
    sum           = fmaf(f, from[k * each + D + 1], sum);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      v[i] = fmaf(f, from[k * each + lane * (D / 32) + i], v[i]);
    }
  }
  const float     f  = sum > 0.f ? 1.f / sum : 0.f;
  const long long at = (long long) (q0 + r) * a.out_stride + h * D + lane * (D / 32);
#pragma unroll
  for (int i = 0; i < D / 32; i += 2) {
    if constexpr (F32) {
      *reinterpret_cast<float2 *>(static_cast<float *>(a.out) + at + i) = make_float2(v[i] * f, v[i + 1] * f);
    } else {
      *reinterpret_cast<uint32_t *>(static_cast<__half *>(a.out) + at + i) = pack_h2(v[i] * f, v[i + 1] * f);
    }
  }
}

// codes as rows of d bytes, fetched 16 rows at a time with 16-byte chunks swizzled over the row
bool codes_map(CUtensorMap *map, const uint8_t *codes, long long rows, int d) {
  using EncodeTiledFn = decltype(&cuTensorMapEncodeTiled);
  static EncodeTiledFn enc = [] {
    void                           *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      p = nullptr;
    }
    return reinterpret_cast<EncodeTiledFn>(p);
  }();
  const cuuint64_t dim[2] = { (cuuint64_t) d, (cuuint64_t) rows }, stride[1] = { (cuuint64_t) d };
  const cuuint32_t box[2] = { (cuuint32_t) d, 16 }, step[2] = { 1, 1 };
  return enc && enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(codes), dim, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    d == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int KVT, int D, bool F32>
cudaError_t launch_tiles(const AttnArgs &a, const AttnPlan &p, bool pdl, cudaStream_t st) {
  const long long grid = (long long) a.kv.n_seqs * p.col_groups * a.kv.n_kv_heads * p.groups * p.splits;
  if (grid > 0x7fffffffll) {
    return cudaErrorInvalidConfiguration;
  }
  constexpr int smem = (int) sizeof(DecodeStage<D>) * kWarps * kStages + 1024;
  DecodeArgs    args;
  args.a               = a;
  const long long rows = (long long) a.kv.n_pages * a.kv.n_kv_heads * a.kv.page_size;
  if (!codes_map(&args.kmap, a.kv.k_codes, rows, D) || !codes_map(&args.vmap, a.kv.v_codes, rows, D)) {
    return cudaErrorInvalidValue;
  }
  auto launch = [&](auto kernel) {
    const cudaError_t e = allow_smem(reinterpret_cast<const void *>(kernel), smem);
    return e != cudaSuccess ? e : launch_decoder_kernel(kernel, args, (unsigned) grid, kThreads, smem, pdl, p.splits, st);
  };
  const cudaError_t e = p.col_tiles == 1 ? launch(attn_decode_kernel<KVT, D, 1, F32>) : launch(attn_decode_kernel<KVT, D, 2, F32>);
  return e != cudaSuccess || p.groups == 1 ? e : attn_join_launch(a, D, !F32, pdl, st);
}

}  // namespace

cudaError_t attn_join_launch(const AttnArgs &a, int head_dim, bool a16, bool pdl, cudaStream_t st) {
  const long long rows = (long long) a.kv.n_seqs * a.max_q * a.n_heads, grid = (rows + 3) / 4;
  if (grid > 0x7fffffffll) {
    return cudaErrorInvalidConfiguration;
  }
  if (head_dim == 64) {
    return a16 ? launch_decoder_kernel(attn_join_kernel<64, false>, a, (unsigned) grid, 128, 0, pdl, 1, st)
               : launch_decoder_kernel(attn_join_kernel<64, true>, a, (unsigned) grid, 128, 0, pdl, 1, st);
  }
  return a16 ? launch_decoder_kernel(attn_join_kernel<128, false>, a, (unsigned) grid, 128, 0, pdl, 1, st)
             : launch_decoder_kernel(attn_join_kernel<128, true>, a, (unsigned) grid, 128, 0, pdl, 1, st);
}

size_t attn_part_bytes(int n_seqs, int max_q, int n_heads, int head_dim, int groups) {
  return groups > 1 ? (size_t) groups * n_seqs * max_q * n_heads * (head_dim + 4) * sizeof(float) : 0;
}

AttnPlan attn_plan(int sm_count, int n_seqs, int n_rows, int n_kv_heads, int group, bool f32, int max_q, int max_ctx,
                   size_t workspace_bytes, int head_dim) {
  AttnPlan        p    = {};
  const long long cols = (long long) max_q * group;
  p.splits = p.groups = p.col_tiles = p.col_groups = 1;
  long long jobs;  // CTAs of one pass over the contexts
  if (cols > 32 && group <= 128) {
    p.tile              = true;
    const int per_tile  = 128 / group;
    p.two_row_tiles     = !f32 && max_q > per_tile;
    const int per_cta   = p.two_row_tiles ? 2 * per_tile : per_tile;
    p.row_slots         = n_rows / per_cta + (long long) n_seqs;
    jobs                = ((long long) n_rows + per_cta - 1) / per_cta * n_kv_heads;
  } else {
    p.col_tiles  = cols > 8 ? 2 : 1;
    p.col_groups = (int) ((cols + 8 * p.col_tiles - 1) / (8 * p.col_tiles));
    jobs         = (long long) n_seqs * n_kv_heads * p.col_groups;
    const long long slots = (long long) sm_count * (p.col_tiles == 1 ? 3 : 2);  // CTAs resident at once
    const long long most  = ((long long) max_ctx + kStep * kWarps - 1) / (kStep * kWarps);  // a step per warp
    // Few short contexts: a cluster over each, joined in shared memory - one launch (700 tokens of one sequence
    // and 8 heads: 7.3 us in clusters of 8, 9.7 us through the workspace, 12.5 us unsplit).
    if (jobs * 8 <= slots && max_ctx <= 8192) {
      while (p.splits < 8 && p.splits < most) {
        p.splits *= 2;
      }
      return p;
    }
    // Else independent CTAs joined by a second launch, which leave no SM waiting for a cluster's worth of room:
    // one wave of equal shares when there are fewer jobs than CTAs fit (2 x 8 jobs of 131072 tokens: 112 us in 27
    // shares, 138 in 32, 154 in clusters of 8), about four waves, for lengths that differ, otherwise (64 x 8
    // jobs of 1 .. 8192 tokens: 101 us in 4 shares, 119 unsplit, 113 in 8, 110 in clusters of 2).
    long long want_groups = jobs >= slots / 2 ? (4 * slots + jobs - 1) / jobs : slots / jobs;
    want_groups = want_groups < max_ctx / 1024 ? want_groups : max_ctx / 1024;
    p.groups    = want_groups < 1 ? 1 : (want_groups > 64 ? 64 : (int) want_groups);
    if (attn_part_bytes(n_seqs, max_q, n_kv_heads * group, head_dim, p.groups) > workspace_bytes) {
      // no room to join them: clusters, and as many shares as the room allows
      p.groups = 1;
      while (p.splits < 8 && jobs * p.splits < slots && p.splits < most) {
        p.splits *= 2;
      }
      while (p.groups < 16 && jobs * p.splits * p.groups * 2 <= slots && max_ctx / (2 * p.groups) >= 4096 &&
             attn_part_bytes(n_seqs, max_q, n_kv_heads * group, head_dim, 2 * p.groups) <= workspace_bytes) {
        p.groups *= 2;
      }
    }
    return p;
  }
  // several CTAs over one context whose results a second launch joins: when each still has enough keys
  while (p.groups < 16 && jobs * p.groups < sm_count && max_ctx / (2 * p.groups) >= 1024) {
    p.groups *= 2;
  }
  while (p.groups > 1 && attn_part_bytes(n_seqs, max_q, n_kv_heads * group, head_dim, p.groups) > workspace_bytes) {
    p.groups /= 2;
  }
  return p;
}

cudaError_t attn_decode_launch(const AttnArgs &a, const AttnPlan &p, int head_dim, int kv_type, bool a16, bool pdl,
                               cudaStream_t st) {
  if (head_dim == 64) {
    if (kv_type == kKvI8) {
      return a16 ? launch_tiles<kKvI8, 64, false>(a, p, pdl, st) : launch_tiles<kKvI8, 64, true>(a, p, pdl, st);
    }
    return a16 ? launch_tiles<kKvE4m3, 64, false>(a, p, pdl, st) : launch_tiles<kKvE4m3, 64, true>(a, p, pdl, st);
  }
  if (kv_type == kKvI8) {
    return a16 ? launch_tiles<kKvI8, 128, false>(a, p, pdl, st) : launch_tiles<kKvI8, 128, true>(a, p, pdl, st);
  }
  return a16 ? launch_tiles<kKvE4m3, 128, false>(a, p, pdl, st) : launch_tiles<kKvE4m3, 128, true>(a, p, pdl, st);
}

}  // namespace htp
