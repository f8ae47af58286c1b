// Attention over the paged 8-bit cache for many rows per sequence (formula: include/htp_ops_b200.h,
// htp_b200_attn_paged), on the 5th-generation tensor cores.
//
// A tile is 128 rows = query rows x heads of one key/value head, against 128 keys at a time:
//   S = Q . K^T (128 x 128 fp32, tensor memory)      A = Q, B = K in shared memory
//   O += P . V  (128 x head_dim fp32, tensor memory) A = P in tensor memory, over S; B = V in shared memory
// Two streams of such tiles run in one CTA, each with its own S, O and four softmax warps, so that one
// stream's softmax runs under the other's matrix products:
//   ROWS  two row tiles walk the same keys: the keys' conversion is shared by 256 rows;
//   KEYS  one row tile, the streams take the key tiles in turn and join their results at the end: fp32
//         queries, whose two fp16 terms fill the room of the second row tile, and short prompts.
//
// Codes become fp16 exactly in four converter warps (global memory -> registers -> 128-byte swizzled shared
// memory, the next tile's loads in flight meanwhile); scales are applied as in attn_decode.cu: a weight is
// 2^(s * k_scale * scale * log2 e + log2 v_scale - M), the denominator divides v_scale out again.  fp32 weights are
// two fp16 terms each.  M follows the row's maximum only when it lags by more than kSlack, so O is rarely rescaled.
//
// Bound: per 128 x 128 scores 1024 cycles of tensor core at head_dim 128 and as many of the exponential unit
// (16 per cycle and SM); fp32 doubles the tensor-core part.  Measured: a prompt of 8192 rows, 32 + 8 heads of 128, fp16:
// 643 us = 855 TF/s, 0.52 of the measured cuBLAS rate; per tile of two streams 4983 clocks, of which a stream's
// softmax takes 2858, its wait for the next scores 1737 (the other stream's products, commits, the way through the
// barriers), the MMA thread 2430.  6.5 k rows with a window of 1024, fp32: 376 us.
//
// Roles: warps 0-3 and 4-7 softmax of stream 0 and 1 (thread = row = TMEM lane), 8-11 converters, 12 MMA
// issuer and tensor-memory owner, 13 scales.  All waits are bounded; one that runs out records error 311, raises the abort
// flag, and every role leaves.
#include <cuda_fp16.h>

#include "attn_common.cuh"
#include "ptx.cuh"
#include "tcgen05.cuh"
#include "unpack.cuh"

namespace htp {

namespace {

constexpr int kSoftWarps = 8;
constexpr int kConvWarp0 = 8;
constexpr int kMmaWarp   = 12;
constexpr int kScaleWarp = 13;
constexpr int kThreads   = 14 * 32;
constexpr int kKeys      = 128;  // keys of a tile
constexpr int kScaleRing = 4;    // key tiles whose scales are kept: one more than a softmax warp may lag behind

// The accumulator cuts off what lies below its last bit: sums come out short, on the average by about 1e-8 for each
// instruction that a growing sum has gone through, 16 a tile with two terms (measured per tile: 1.6e-7 over 5 to 7 tiles,
// 1.3e-7 over 28).  fp32 results get that back (prompts of 3300 keys: 1.6e-6 off without, 9.7e-7 with it; three quarters of it where the
// second terms have sums of their own); what fp16
// results round away is a thousand times more.
constexpr float kCut = 1.4e-7f;

struct Bars {
  uint64_t q_full, k_full[2], v_full[2], k_empty[2], v_empty[2], s_full[2], p_ready[2], o_done[2], drained;
  uint32_t tmem;
  int      abort_flag;
  float    by[kScaleRing][8], up[kScaleRing][8], inv[kScaleRing][8];  // of the tile's 16-key blocks
  float    unit[128];     // fp32 queries: the power of two that a row was divided by
  float    ml[2][2][128];  // KEYS: maximum and denominator of each stream's rows
  // element offsets of the tiles' rows in the queries and in the output, -1 for rows that are nobody's
  long long q_at[256], out_at[256];
};

template <int D>
struct Sizes {
  static constexpr int kTile = 128 * D * 2;  // 128 rows of fp16
  // two query parts, two key and two value tiles; at least half of an SM's, so that two CTAs never wait
  // for each other's tensor memory
  static constexpr int kSmem = (6 * kTile > 120 * 1024 ? 6 * kTile : 120 * 1024) + 1024 + (int) sizeof(Bars);
  static_assert(kSmem <= 232448, "shared memory");
};

struct Waiter {
  volatile int *abort_flag;
  int          *err;
  // the whole warp waits; true when the barrier's phase has completed
  __device__ __forceinline__ bool operator()(uint64_t *bar, uint32_t parity) const {
    bool ok = false;
    for (uint32_t i = 0; i < kWaitCap && !ok; ++i) {
      ok = mbar_try_wait(bar, parity);
      if (!ok && i >= 4096) {
        if (*abort_flag) {
          break;
        }
        __nanosleep(128);
      }
    }
    ok = __all_sync(0xffffffffu, ok);
    if (!ok && *abort_flag == 0) {
      record_error(err, kErrWait);
      *abort_flag = 1;
    }
    return ok;
  }
};

// byte offset of the 16-byte chunk `c` (8 halves) of row `r` in a 128-row operand tile: 64 halves of all rows
// after each other, 128-byte swizzle
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return (uint32_t) ((c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

template <int KVT, int D, bool F32, bool ROWS>
__global__ void __launch_bounds__(kThreads, 1) attn_prompt_kernel(const __grid_constant__ AttnArgs a) {
  static_assert(!(F32 && ROWS), "fp32 queries take the room of both row tiles");
  constexpr int TILE  = Sizes<D>::kTile;
  constexpr int TERMS = F32 ? 2 : 1;
  // fp32 at head_dim 64: tensor memory has room to sum the second terms apart, in the columns behind O
  constexpr int O2 = F32 && D == 64 ? 64 : 0;
  extern __shared__ uint8_t smem_raw[];
  // (an offset, not a rounded address: the compiler keeps seeing shared memory)
  uint8_t *smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
  uint8_t *sQ = smem, *sK = smem + 2 * TILE, *sV = smem + 4 * TILE;
  Bars    *bar = reinterpret_cast<Bars *>(smem + 6 * TILE);
  pdl_launch_dependents();
  pdl_wait_prior_grids();

  const KvView &kv   = a.kv;
  const int     warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // ---- which rows: sequence b has the row blocks from q_start[b] / per_cta + b on, at least as many as it
  // needs; late blocks first, they see the most keys
  const int per_tile = 128 / a.group;  // query rows of a tile
  const int per_cta  = ROWS ? 2 * per_tile : per_tile;
  unsigned  id       = blockIdx.x;
  const int grp      = id % a.groups;
  id /= a.groups;
  const int head = id % kv.n_kv_heads;
  id /= kv.n_kv_heads;
  const long long slot = (long long) (a.row_slots - 1) - id;
  auto            at   = [&](int i) { return (long long) (kv.q_start[i] / per_cta) + i; };
  const int       b    = interval_of(kv.n_seqs, slot, at);
  if (b >= kv.n_seqs) {
    return;
  }
  int q0, q_len, ctx;
  if (!sequence_of(kv, b, a.max_q, a.max_ctx, q0, q_len, ctx)) {
    if (threadIdx.x == 0) {
      record_error(a.err, kErrSequence);
    }
    return;
  }
  const long long block = slot - at(b);
  if (block < 0 || block * per_cta >= q_len) {
    return;
  }
  const int i0 = (int) block * per_cta, i1 = i0 + per_cta < q_len ? i0 + per_cta : q_len;
  const int past = ctx - q_len;
  int       lo = 0, hi = past + i1;
  hi = hi < 0 ? 0 : hi;
  if (a.window > 0 && past + i0 - a.window + 1 > 0) {
    lo = past + i0 - a.window + 1;
  }
  int       first_tile = lo / kKeys, n = hi > lo ? (hi + kKeys - 1) / kKeys - first_tile : 0;
  const int share0 = (int) ((long long) n * grp / a.groups), share1 = (int) ((long long) n * (grp + 1) / a.groups);
  first_tile += share0;
  n = share1 - share0;  // key tiles of this CTA
  // tile j of stream x is key tile j (ROWS) or 2 j + x (KEYS)
  const int n_of[2] = { ROWS ? n : (n + 1) / 2, ROWS ? n : n / 2 };

  if (threadIdx.x == 0) {
    mbar_init(&bar->q_full, kSoftWarps);
    mbar_init(&bar->drained, 1);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->k_full[i], 5), mbar_init(&bar->v_full[i], 4);  // (the converters; keys: and the scales)
      mbar_init(&bar->k_empty[i], 1), mbar_init(&bar->v_empty[i], 1);
      mbar_init(&bar->s_full[i], 2), mbar_init(&bar->p_ready[i], 4), mbar_init(&bar->o_done[i], 1);
    }
    bar->abort_flag = 0;
    mbar_fence_init();
  }
  if (threadIdx.x < (ROWS ? 256 : 128)) {
    const int       r = threadIdx.x & 127, q = i0 + (int) (threadIdx.x >> 7) * per_tile + r / a.group;
    const bool      in = r < per_tile * a.group && q < i1;
    const long long h  = (long long) (head * a.group + r % a.group) * D;
    bar->q_at[threadIdx.x]   = in ? (q0 + (long long) q) * a.q_stride + h : -1;
    bar->out_at[threadIdx.x] = in ? (q0 + (long long) q) * a.out_stride + h : -1;
  }
  if (warp == kMmaWarp) {
    tmem_alloc<false>(&bar->tmem, 512);
    tmem_relinquish<false>();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&bar->tmem);
  const Waiter   wait{ &bar->abort_flag, a.err };
  const int     *table = kv.page_table + (long long) b * kv.table_stride;
  auto           seen  = [&](int key) { return key < hi && key + 16 > lo; };  // some row sees some of these 16 keys
  // Slot t & 1 is free for tile t when the scores made of tile t - 2's keys, or the results made of its values,
  // are complete.  KEYS: tile t / 2 - 1 of the slot's own stream, whose barriers say so.  ROWS: of both
  // streams; the barriers of one could be two phases on by now, so the slots have their own.
  auto slot_free = [&](int t, uint64_t *empty, uint64_t *own) {
    return t < 2 || wait(ROWS ? empty + (t & 1) : own + (t & 1), ((t >> 1) & 1) ^ 1);
  };
  auto           s_at = [&](int x) { return tmem + (uint32_t) x * 128; };
  auto           o_at = [&](int x) { return tmem + 256 + (uint32_t) x * 128; };

  if (warp < kSoftWarps) {
    // ---------------- softmax
    const int x = warp >> 2, row = (warp & 3) * 32 + lane;
    // queries -> shared memory: 128 rows of one or two parts, a batch of loads in flight
    constexpr int CH    = D / 8;  // 16-byte chunks of a row
    constexpr int ITEMS = (ROWS ? 2 : 1) * 128 * CH / (kSoftWarps * 32), BATCH = F32 ? 4 : 16;
    static_assert(ITEMS % 4 == 0, "whole batches");
#pragma unroll
    for (int i0_ = 0; i0_ < ITEMS; i0_ += BATCH < ITEMS ? BATCH : ITEMS) {
      constexpr int NB = BATCH < ITEMS ? BATCH : ITEMS;
      uint4         v[NB][F32 ? 2 : 1];
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int       it = threadIdx.x + (i0_ + i) * kSoftWarps * 32, c = it % CH;
        const long long at = bar->q_at[it / CH];
        const bool      in = at >= 0;
        const uint4    *from = reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(a.q) + (at + c * 8) * (F32 ? 4 : 2));
#pragma unroll
        for (int u = 0; u < (F32 ? 2 : 1); ++u) {
          v[i][u] = make_uint4(0, 0, 0, 0);
          if (in) {
            v[i][u] = from[u];
          }
        }
      }
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int it = threadIdx.x + (i0_ + i) * kSoftWarps * 32, part = it / (128 * CH), r = it / CH % 128, c = it % CH;
        uint8_t  *to = sQ + part * TILE + chunk_at(r, c);
        if constexpr (F32) {
          float f[8] = { __uint_as_float(v[i][0].x), __uint_as_float(v[i][0].y), __uint_as_float(v[i][0].z), __uint_as_float(v[i][0].w),
                         __uint_as_float(v[i][1].x), __uint_as_float(v[i][1].y), __uint_as_float(v[i][1].z), __uint_as_float(v[i][1].w) };
          float m    = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            m = fmaxf(m, fabsf(f[e]));
          }
#pragma unroll
          for (int o = CH / 2; o > 0; o >>= 1) {  // (CH lanes hold a row)
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
          }
          float unit, by;
          query_unit(m, unit, by);
          if (c == 0) {
            bar->unit[r] = unit;
          }
          uint32_t h[4], l[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            split_h2(f[2 * e] * by, f[2 * e + 1] * by, h[e], l[e]);
          }
          *reinterpret_cast<uint4 *>(to)        = make_uint4(h[0], h[1], h[2], h[3]);
          *reinterpret_cast<uint4 *>(to + TILE) = make_uint4(l[0], l[1], l[2], l[3]);
        } else {
          *reinterpret_cast<uint4 *>(to) = v[i][0];
        }
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      mbar_arrive(&bar->q_full);
    }
    bool ok = wait(&bar->q_full, 0);  // (the rows' units)
    const float unit = F32 ? bar->unit[row] : 1.f;

    const int  my_q   = i0 + (ROWS ? x * per_tile : 0) + row / a.group;
    const bool mine   = row < per_tile * a.group && my_q < i1;
    // rows that are nobody's see everything: they cost no mask, and are not stored
    const int last  = mine ? past + my_q : 0x7fffffff;
    const int first = mine && a.window > 0 ? past + my_q - a.window + 1 : (int) 0x80000000;
    const uint32_t lanes = (uint32_t) ((warp & 3) * 32) << 16;
    const uint32_t s_addr = s_at(x) + lanes, o_addr = o_at(x) + lanes;
    float          mx = kFloor, l = 0.f;
    bool           huge = false;
    // multiplies what a row has by f: the weights of this tile's first c chunks of 32 keys and, from the second
    // tile on, O
    auto rescale = [&](int j, int c, float f) {
      uint32_t w[16];
      if (c > 0) {
        tmem_st_wait();
#pragma unroll 1
        for (int d = 0; d < 2 * c; d += F32 ? 1 : 2) {
          tmem_ld16_issue(s_addr + 16 * d, w);
          tmem_ld_wait(w);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 u = __half22float2(u32_as_h2(w[e]));
            w[e]           = pack_h2(u.x * f, u.y * f);
          }
          tmem_st16(s_addr + 16 * d, w);
        }
      }
      if (j > 0) {
        if (!wait(&bar->o_done[x], (j - 1) & 1)) {
          return false;
        }
        tc_fence_after();
#pragma unroll 1
        for (int d = 0; d < (D + O2) / 16; ++d) {
          tmem_ld16_issue(o_addr + 16 * d, w);
          tmem_ld_wait(w);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            w[e] = __float_as_uint(__uint_as_float(w[e]) * f);
          }
          tmem_st16(o_addr + 16 * d, w);
        }
      }
      return true;
    };
    for (int j = 0; j < n_of[x] && ok; ++j) {
      const int    t    = ROWS ? j : 2 * j + x;
      const int    key0 = (first_tile + t) * kKeys;
      const float *by_ = bar->by[t % kScaleRing], *up_ = bar->up[t % kScaleRing], *inv_ = bar->inv[t % kScaleRing];
      if (!(ok = wait(&bar->s_full[x], j & 1))) {
        break;
      }
      tc_fence_after();
      const bool full = __all_sync(0xffffffffu, key0 >= first && key0 + kKeys - 1 <= last);
      // 64 keys at a time; the registers of 32 are filled with later scores as soon as their weights are made
      uint32_t s[2][32];
      tmem_ld32_issue(s_addr, s[0]);
      tmem_ld32_issue(s_addr + 32, s[1]);
#pragma unroll 1
      for (int c = 0; c < 4 && ok; c += 2) {
        tmem_ld_wait32(s[0]);
        tmem_ld_wait32(s[1]);
        if (!full) {
#pragma unroll
          for (int e = 0; e < 64; ++e) {
            const int key     = key0 + 32 * c + e;
            s[e >> 5][e & 31] = key <= last && key >= first ? s[e >> 5][e & 31] : 0xff800000u;
          }
        }
        float by[4], up[4], off[4], most[4], top = -INFINITY;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const uint32_t *v = s[h >> 1] + 16 * (h & 1);
          float m0 = __uint_as_float(v[0]), m1 = __uint_as_float(v[1]);
#pragma unroll
          for (int e = 2; e < 14; e += 4) {
            m0 = max3(m0, __uint_as_float(v[e]), __uint_as_float(v[e + 1]));
            m1 = max3(m1, __uint_as_float(v[e + 2]), __uint_as_float(v[e + 3]));
          }
          m0      = max3(m0, __uint_as_float(v[14]), __uint_as_float(v[15]));
          most[h] = fmaxf(m0, m1);
          by[h]   = by_[2 * c + h] * unit;
          up[h]   = up_[2 * c + h];
          off[h]  = up[h] - mx + kLift;
          top     = fmaxf(top, huge ? fmaf(most[h], by[h], up[h]) - mx + kLift : fmaf(most[h], by[h], off[h]));
        }
        if (__any_sync(0xffffffffu, top > kLift + kSlack)) {
          // ---- a row's maximum has moved away: M follows by a power of two (exact for what is there already;
          // straight to the maximum when nothing is)
          float x0 = fmaf(most[0], by[0], up[0]);
#pragma unroll
          for (int h = 1; h < 4; ++h) {
            x0 = fmaxf(x0, fmaf(most[h], by[h], up[h]));
          }
          // (first on a grid of 1 / 256, so that adding whole numbers is exact; never below the score, where a step is so
          // large that it rounds)
          const float m = mx == kFloor ? fmaxf(ceilf(x0 * 256.f) * 0.00390625f, kFloor) : fmaxf(mx + fmaxf(ceilf(x0 - mx), 0.f), x0);
          const int   k = __float2int_rn(fminf(m - mx, 127.f));
          const float f = __int_as_float((127 - k) << 23);  // (2^-127 and less: 0)
          mx = m;
          l *= f;
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            off[h] = up[h] - mx + kLift;
          }
          huge = __any_sync(0xffffffffu, fabsf(mx) > kHuge && mx != kFloor);
          ok   = rescale(j, c, f);
          if (!ok) {
            break;
          }
        }
        if (huge) {  // (see kHuge)
#pragma unroll
          for (int e = 0; e < 64; ++e) {
            uint32_t &v = s[e >> 5][e & 31];
            v = __float_as_uint(fmaf(__uint_as_float(v), by[e >> 4], up[e >> 4]) - mx + kLift);
          }
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            by[h] = 1.f, off[h] = 0.f;
          }
        }
        // ---- weights, over the scores: 32 keys in the first 16 of their 32 columns, second terms in the others
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          uint32_t p[16], p2[16];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 b2 = make_float2(by[2 * d + h], by[2 * d + h]), o2 = make_float2(off[2 * d + h], off[2 * d + h]);
            float2       sum[2];
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              float2 w = fma2(make_float2(__uint_as_float(s[d][16 * h + e]), __uint_as_float(s[d][16 * h + e + 1])), b2, o2);
              w.x = exp2_approx(w.x), w.y = exp2_approx(w.y);
              sum[(e >> 1) & 1] = e < 4 ? w : add2(sum[(e >> 1) & 1], w);
              if constexpr (F32) {
                split_h2(w.x, w.y, p[8 * h + e / 2], p2[8 * h + e / 2]);
              } else {
                p[8 * h + e / 2] = pack_h2(w.x, w.y);
              }
            }
            const float2 both = add2(sum[0], sum[1]);
            l                 = fmaf(both.x + both.y, inv_[2 * (c + d) + h], l);
          }
          if (c == 0) {
            tmem_ld32_issue(s_addr + 32 * (2 + d), s[d]);
          }
          tmem_st16(s_addr + 32 * (c + d), p);
          if constexpr (F32) {
            tmem_st16(s_addr + 32 * (c + d) + 16, p2);
          }
        }
      }
      if (!ok) {
        break;
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bar->p_ready[x]);
      }
    }
    // ---- results
    if (ok && n_of[x] > 0) {
      ok = wait(&bar->o_done[x], (n_of[x] - 1) & 1);
    }
    float f0 = 1.f, f1 = 0.f;
    if constexpr (!ROWS) {
      if (ok && n_of[x ^ 1] > 0) {
        ok = wait(&bar->o_done[x ^ 1], (n_of[x ^ 1] - 1) & 1);
      }
      bar->ml[x][0][row] = mx, bar->ml[x][1][row] = l;
      named_bar_sync(1, kSoftWarps * 32);
      const float m = fmaxf(bar->ml[0][0][row], bar->ml[1][0][row]);
      f0 = exp2_approx(bar->ml[0][0][row] - m), f1 = exp2_approx(bar->ml[1][0][row] - m);
      l  = fmaf(f1, bar->ml[1][1][row], f0 * bar->ml[0][1][row]);
      mx = m;
    }
    tc_fence_after();
    if (ok) {
      const int  h  = head * a.group + row % a.group;
      const bool part = a.groups > 1;
      const float scale = part ? 1.f : (l > 0.f ? 1.f / l : 0.f);
      float      *to = part ? a.part + ((((long long) grp * kv.n_seqs + b) * a.max_q + my_q) * a.n_heads + h) * (D + 4) : nullptr;
      // bytes of a row that this warp stages: all of it, or its stream's half of the columns
      constexpr int ROWB  = (ROWS ? D : D / 2) * (F32 ? 4 : 2);
      uint8_t      *stage = sQ + (warp * 32) * ROWB;
      constexpr int SWZ = ROWB / 16 < 8 ? ROWB / 16 - 1 : 7;
      static_assert(kSoftWarps * 32 * ROWB <= 2 * TILE, "the query parts hold the results");
      if (part && mine && (ROWS || x == 0)) {
        *reinterpret_cast<float2 *>(to + D) = make_float2(mx, l);
      }
      __syncwarp();
      // ROWS: every thread stores its row; KEYS: the streams' warps store one half of the columns each
      constexpr int C0 = ROWS ? D / 32 : D / 64;
#pragma unroll
      for (int k = 0; k < C0; ++k) {
        const int c = ROWS ? k : x * C0 + k;
        float     v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          v[e] = 0.f;
        }
#pragma unroll
        for (int y = 0; y < (ROWS ? 1 : 2); ++y) {
          const int   z = ROWS ? x : y;
          const float f = (y ? f1 : f0) * scale * (F32 ? fmaf((float) n_of[z], O2 ? 0.75f * kCut : kCut, 1.f) : 1.f);
          if (n_of[z] > 0) {
            uint32_t o[32];
            tmem_ld32_issue(o_at(z) + lanes + 32 * c, o);
            tmem_ld_wait32(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              v[e] = fmaf(__uint_as_float(o[e]), f, v[e]);
            }
            if constexpr (O2 > 0) {
              tmem_ld32_issue(o_at(z) + O2 + lanes + 32 * c, o);
              tmem_ld_wait32(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                v[e] = fmaf(__uint_as_float(o[e]), f, v[e]);
              }
            }
          }
        }
        if (part) {
          if (mine) {
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              *reinterpret_cast<float4 *>(to + 32 * c + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
            }
          }
        } else {
          // to the warp's rows of the (no longer needed) query parts, 16-byte chunks swizzled by the row
          uint8_t *srow = stage + lane * ROWB;
          constexpr int PER = F32 ? 4 : 8;
#pragma unroll
          for (int e = 0; e < 32; e += PER) {
            uint4 u;
            if constexpr (F32) {
              u = make_uint4(__float_as_uint(v[e]), __float_as_uint(v[e + 1]), __float_as_uint(v[e + 2]), __float_as_uint(v[e + 3]));
            } else {
              u = make_uint4(pack_h2(v[e], v[e + 1]), pack_h2(v[e + 2], v[e + 3]), pack_h2(v[e + 4], v[e + 5]), pack_h2(v[e + 6], v[e + 7]));
            }
            const int chunk = (32 * k + e) / PER;
            *reinterpret_cast<uint4 *>(srow + ((chunk ^ (lane & SWZ)) << 4)) = u;
          }
        }
        __syncwarp();  // (the next tensor-memory load is the whole warp's)
      }
      if (!part) {  // rows leave as contiguous runs
        constexpr int CPR = ROWB / 16;  // chunks of a row
#pragma unroll
        for (int k = 0; k < CPR; ++k) {
          const int       i = k * 32 + lane, r = i / CPR, chunk = i % CPR;
          const long long at_o = bar->out_at[(ROWS ? warp : warp & 3) * 32 + r];
          if (at_o >= 0) {
            const uint4 u = *reinterpret_cast<const uint4 *>(stage + r * ROWB + ((chunk ^ (r & SWZ)) << 4));
            *reinterpret_cast<uint4 *>(static_cast<uint8_t *>(a.out) + at_o * (F32 ? 4 : 2) + (ROWS ? 0 : x * ROWB) + chunk * 16) = u;
          }
        }
      }
    }
    tc_fence_before();
  } else if (warp < kMmaWarp) {
    // ---------------- converters: a warp takes 32 keys (two 16-key blocks) of every tile
    constexpr int PIECES = D / 16;            // 16-byte pieces of a key's codes
    constexpr int RPL    = 32 / PIECES;       // keys of one warp-wide load
    constexpr int LOADS  = 32 / RPL;          // loads of a lane per tile
    const int cw = warp - kConvWarp0, piece = lane % PIECES, sub = lane / PIECES;
    // page numbers of the warp's two blocks in tile t, as they stand in the table; checked when they are used
    auto ask = [&](int t, int (&raw)[2]) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = (first_tile + t) * kKeys + cw * 32 + 16 * h;
        raw[h]        = t < n && seen(key) ? table[key >> kv.page_shift] : -1;
      }
    };
    auto checked = [&](const int (&raw)[2], int (&pg)[2]) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        pg[h] = raw[h] < kv.n_pages ? raw[h] : -1;  // (negative: nothing is read)
      }
    };
    constexpr int HALF = LOADS / 2;  // loads of a block
    const int     lane_at = sub * D + piece * 16;
    auto load = [&](const uint8_t *codes, int t, const int (&pg)[2], uint4 (&r)[LOADS]) {
      const int key0 = (first_tile + t) * kKeys + cw * 32;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int      key  = key0 + 16 * h;
        const uint8_t *from = codes + ((((long long) pg[h] * kv.n_kv_heads + head) << kv.page_shift) + (key & (kv.page_size - 1))) * D + lane_at;
        if (pg[h] >= 0 && key >= lo && key + 16 <= hi) {
#pragma unroll
          for (int i = 0; i < HALF; ++i) {
            r[h * HALF + i] = ld_stream16(from + i * RPL * D);
          }
        } else {  // zeros outside what any row sees: what lies there may be no numbers
#pragma unroll
          for (int i = 0; i < HALF; ++i) {
            const int k = key + i * RPL + sub;
            r[h * HALF + i] = make_uint4(0, 0, 0, 0);
            if (pg[h] >= 0 && k >= lo && k < hi) {
              r[h * HALF + i] = ld_stream16(from + i * RPL * D);
            }
          }
        }
      }
    };
    // where the lane's two chunks of its keys go (the swizzle takes the row modulo 8: with 4 keys a load, two
    // cases); the upper half of a 128-element key's pieces stores its chunks in the other order: no two lanes
    // of a row on one bank
    const int swap = D == 128 ? piece >> 2 : 0;
    uint32_t  put[2][2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int k = cw * 32 + e * RPL + sub;
      put[e][0]   = chunk_at(k, 2 * piece + swap) - e * RPL * 128;
      put[e][1]   = chunk_at(k, 2 * piece + 1 - swap) - e * RPL * 128;
    }
    auto convert = [&](uint8_t *tile, const uint4 (&r)[LOADS]) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const uint32_t w[4] = { r[i].x, r[i].y, r[i].z, r[i].w };
        uint32_t       h[4][2];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          codes_to_h2<KVT>(swap ? w[e ^ 2] : w[e], h[e]);
        }
        *reinterpret_cast<uint4 *>(tile + put[i & 1][0] + i * RPL * 128) = make_uint4(h[0][0], h[0][1], h[1][0], h[1][1]);
        *reinterpret_cast<uint4 *>(tile + put[i & 1][1] + i * RPL * 128) = make_uint4(h[2][0], h[2][1], h[3][0], h[3][1]);
      }
    };
    auto publish = [&](uint64_t *full) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(full);
      }
    };
    // Keys go one tile ahead of values: the next scores are wanted before this tile's results.  Loads are in
    // flight for a tile's time: a tile's keys and values are asked for when the registers of the tile
    // before have been converted, its page numbers a tile earlier.
    uint4 rk[LOADS], rv[LOADS];
    int   raw[2], pk[2], pv[2];
    ask(0, raw);
    checked(raw, pk);
    load(kv.k_codes, 0, pk, rk);
    load(kv.v_codes, 0, pk, rv);
    ask(1, raw);
    bool ok = true;
    auto keys = [&](int t) {
      const int i = t & 1;
      if (!(ok = slot_free(t, bar->k_empty, bar->s_full))) {
        return;
      }
      convert(sK + i * TILE, rk);
      publish(&bar->k_full[i]);
      checked(raw, pk);
      load(kv.k_codes, t + 1, pk, rk);
      ask(t + 2, raw);
    };
    if (n > 0) {
      keys(0);
    }
#pragma unroll 1
    for (int t = 0; t < n && ok; ++t) {
      pv[0] = pk[0], pv[1] = pk[1];  // (of tile t + 1)
      if (t + 1 < n) {
        keys(t + 1);
      }
      if (!ok || !(ok = slot_free(t, bar->v_empty, bar->o_done))) {
        break;
      }
      convert(sV + (t & 1) * TILE, rv);
      publish(&bar->v_full[t & 1]);
      load(kv.v_codes, t + 1, pv, rv);
    }
  } else if (warp == kScaleWarp) {
    // ---------------- scales of the tiles' 16-key blocks, a lane each; what is no block gets the weight 0
#pragma unroll 1
    for (int t = 0; t < n; ++t) {
      const int key = (first_tile + t) * kKeys + 16 * (lane & 7);
      float     by = a.scale_log2, up = -INFINITY, inv = 0.f;
      if (seen(key)) {
        const int p = table[key >> kv.page_shift];
        if (p < 0 || p >= kv.n_pages) {
          record_error(a.err, kErrPage);
        } else {
          const long long at_p = (long long) p * kv.n_kv_heads + head;
          block_scales(kv.k_scale[at_p], kv.v_scale[at_p], a.scale_log2, by, up, inv);
        }
      }
      __syncwarp();
      if (!slot_free(t, bar->k_empty, bar->s_full)) {
        break;
      }
      if (lane < 8) {
        bar->by[t % kScaleRing][lane] = by, bar->up[t % kScaleRing][lane] = up, bar->inv[t % kScaleRing][lane] = inv;
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bar->k_full[t & 1]);
      }
    }
  } else {
    // ---------------- MMA issuer: the whole warp walks the loop, one elected lane issues
    constexpr uint32_t IDESC_S = instr_desc_f16(128, kKeys), IDESC_O = instr_desc_f16(128, D) | kInstrBMajorMn;
    bool ok = n == 0 || wait(&bar->q_full, 0);
    auto scores = [&](int x, int j) {
      const int t = ROWS ? j : 2 * j + x, i = t & 1;
      if (!ROWS || x == 0) {
        ok = ok && wait(&bar->k_full[i], (t >> 1) & 1);
      }
      if (!ok) {
        return;
      }
      tc_fence_after();
      if (elect_one()) {
        const uint64_t kd = smem_desc_sw128(sK + i * TILE);
#pragma unroll
        for (int i_ = 0; i_ < TERMS; ++i_) {  // (the small second term first: its sums lose nothing to the accumulator's steps)
          const int      term = TERMS - 1 - i_;
          const uint64_t qd   = smem_desc_sw128(sQ + (ROWS ? x : term) * TILE);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = (k >> 2) * (16384 >> 4) + (k & 3) * 2;
            umma_f16_ss(s_at(x), qd + off, kd + off, IDESC_S, (i_ | k) ? 1u : 0u);
          }
        }
        umma_commit<false>(&bar->s_full[x]);
        mbar_arrive(&bar->s_full[x]);  // (carries the converters' scales on to the softmax warps)
        if (ROWS && x == 1) {
          umma_commit<false>(&bar->k_empty[i]);
        }
      }
      __syncwarp();
    };
    for (int x = 0; x < 2 && ok; ++x) {
      if (n_of[x] > 0) {
        scores(x, 0);
      }
    }
    for (int j = 0; j < n_of[0] && ok; ++j) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (j >= n_of[x] || !ok) {
          continue;
        }
        const int t = ROWS ? j : 2 * j + x, i = t & 1;
        if (!ROWS || x == 0) {
          ok = wait(&bar->v_full[i], (t >> 1) & 1);
        }
        ok = ok && wait(&bar->p_ready[x], j & 1);
        if (!ok) {
          continue;
        }
        tc_fence_after();
        if (elect_one()) {
          const uint64_t vd = smem_desc_sw128_mn(sV + i * TILE, 16384);
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k) {
#pragma unroll
            for (int term = 0; term < TERMS; ++term) {
              umma_f16_ts<false>(o_at(x) + O2 * term, s_at(x) + 32 * (k >> 1) + 8 * (k & 1) + 16 * term, vd + k * (2048 >> 4), IDESC_O,
                                 (j | k | (O2 ? 0 : term)) ? 1u : 0u);
            }
          }
          umma_commit<false>(&bar->o_done[x]);
          if (ROWS && x == 1) {
            umma_commit<false>(&bar->v_empty[i]);
          }
        }
        __syncwarp();
        if (j + 1 < n_of[x]) {
          scores(x, j + 1);
        }
      }
    }
    if (!ok) {  // what has been issued still reads shared memory: let it end
      if (elect_one()) {
        umma_commit<false>(&bar->drained);
      }
      __syncwarp();
      for (uint32_t i = 0; i < kWaitCap && !mbar_try_wait(&bar->drained, 0); ++i) {
        __nanosleep(64);
      }
    }
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc<false>(tmem, 512);
  }
}

template <int KVT, int D, bool F32, bool ROWS>
cudaError_t launch(const AttnArgs &a, bool pdl, cudaStream_t st) {
  const long long grid = a.row_slots * a.kv.n_kv_heads * a.groups;
  if (grid > 0x7fffffffll) {
    return cudaErrorInvalidConfiguration;
  }
  constexpr int     smem = Sizes<D>::kSmem;
  const cudaError_t e    = allow_smem(reinterpret_cast<const void *>(attn_prompt_kernel<KVT, D, F32, ROWS>), smem);
  return e != cudaSuccess ? e : launch_decoder_kernel(attn_prompt_kernel<KVT, D, F32, ROWS>, a, (unsigned) grid, kThreads, smem, pdl, 1, st);
}

template <int KVT, int D>
cudaError_t launch_type(const AttnArgs &a, const AttnPlan &p, bool a16, bool pdl, cudaStream_t st) {
  if (!a16) {
    return launch<KVT, D, true, false>(a, pdl, st);
  }
  return p.two_row_tiles ? launch<KVT, D, false, true>(a, pdl, st) : launch<KVT, D, false, false>(a, pdl, st);
}

}  // namespace

cudaError_t attn_prompt_launch(const AttnArgs &a, const AttnPlan &p, int head_dim, int kv_type, bool a16, bool pdl,
                               cudaStream_t st) {
  cudaError_t e;
  if (head_dim == 64) {
    e = kv_type == kKvI8 ? launch_type<kKvI8, 64>(a, p, a16, pdl, st) : launch_type<kKvE4m3, 64>(a, p, a16, pdl, st);
  } else {
    e = kv_type == kKvI8 ? launch_type<kKvI8, 128>(a, p, a16, pdl, st) : launch_type<kKvE4m3, 128>(a, p, a16, pdl, st);
  }
  return e != cudaSuccess || p.groups == 1 ? e : attn_join_launch(a, head_dim, a16, pdl, st);
}

}  // namespace htp
