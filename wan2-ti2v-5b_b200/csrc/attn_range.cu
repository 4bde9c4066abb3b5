// Attention over one key range per query row:
//   s_ij = scale q_i . k_j,  s' = cap tanh(s / cap)  (cap > 0),  t = s' + b_h(j - pos_i),
//   o_i = sum_{lo_i <= j < hi_i} e^(t_ij) v_j / sum e^(t_ij);  an empty range gives o_i = 0.
// Document, causal, frame-causal, prefix, window and padding masks all are one range per row.
//
// The query heads of one key head are packed into the rows of a query tile (row = token * group +
// head in group), so grouped heads read K and V once.  Two forms:
//   * up to 16 packed rows (single tokens, a few draft tokens): range_decode_kernel, bound by reading
//     K and V once from HBM;
//   * more: range_attn_kernel, tcgen05 tiles of 128 rows x 128 keys over the key tiles that a row of
//     the tile sees, bound by the exponentials and the tensor pipe.
//
// Hidden keys must not reach a row even where they hold NaN or infinities.  Scores are selected away,
// but a weight of 0 still turns a NaN in V into a NaN of the sum.  So wherever a block of keys is
// not seen by every row, non-finite entries of V are replaced by zeros before the product, and
// added one by one to the rows that do see them (never with finite values).
#include <atomic>

#include <cooperative_groups.h>

#include "common.cuh"
#include "internal.h"

namespace wanb200 {

namespace cg = cooperative_groups;

constexpr float RA_LOG2E = 1.4426950408889634f;
constexpr float RA_RESCALE = 8.f;  // log2 units by which a maximum must grow before sums are rescaled

enum RangeBias : int { kBiasNone = 0, kBiasSlopes = 1, kBiasTable = 2 };

struct RangeArgs {
  const __nv_bfloat16 *q, *k, *v;
  __nv_bfloat16* o;
  int64_t q_tok, q_batch, k_tok, k_batch, v_tok, v_batch, o_tok, o_batch;
  int batch, kv_heads, group, q_len, kv_len;
  // log2 units: no cap: t = s * sl2; cap: t = cap2 - 2 cap2 / (1 + 2^(s * sl2)), which is
  // cap tanh(s scale / cap) log2(e) with sl2 = 2 log2(e) scale / cap, cap2 = cap log2(e)
  float sl2, cap2;
  const int32_t *lo, *hi, *pos;
  int64_t range_batch;  // elements between the batches of lo / hi / pos, 0 when they are shared
  const float* slopes;  // [heads]
  const float* table;   // [heads, 2 * reach + 1]
  int reach;
};

__device__ __forceinline__ void row_range(const RangeArgs& a, int b, int i, int& lo, int& hi) {
  const int64_t r = b * a.range_batch + i;
  lo = max(__ldg(a.lo + r), 0);
  hi = min(__ldg(a.hi + r), a.kv_len);
}

__device__ __forceinline__ int row_pos(const RangeArgs& a, int b, int i) {
  return a.pos ? min(max(__ldg(a.pos + b * a.range_batch + i), -(1 << 30)), 1 << 30) : i;
}

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// min(x, 30) that keeps a NaN (30: 2^30 + 1 rounds tanh to 1, and four such factors stay below 2^127).
__device__ __forceinline__ float min30(float x) {
  float y;
  asm("min.NaN.f32 %0, %1, 0f41F00000;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ bool nonfinite_bf16(__nv_bfloat16 x) { return !isfinite(__bfloat162float(x)); }

// 2^t-units score of one (row, key) from its raw product, for the forms that take keys one by one.
template <bool CAP, int BIAS>
__device__ __forceinline__ float score_log2(const RangeArgs& a, float s, int h, int dist) {
  float t = s * a.sl2;
  if constexpr (CAP) t = a.cap2 - 2.f * a.cap2 * rcp_approx(1.f + ex2_approx(t));
  if constexpr (BIAS == kBiasSlopes) t = fmaf(-RA_LOG2E * __ldg(a.slopes + h), fabsf((float)dist), t);
  if constexpr (BIAS == kBiasTable)
    t = fmaf(RA_LOG2E, __ldg(a.table + (int64_t)h * (2 * a.reach + 1) + min(max(dist, -a.reach), a.reach) + a.reach), t);
  return t;
}

// ================================================================== few rows: one pass over K and V
// One cluster of blocks per (key head, batch element); the warps of a cluster take blocks of 16 keys in
// turn and keep their own running maximum, sum and output, merged at the end over the block's
// shared memory and then over the cluster's.  K and V pass through a ring of asynchronous copies,
// each lane's own 16-byte pieces, to the operand registers of mma.sync m16n8k16 (16 rows x 16
// keys): a dot product does not care about the order of its channels, so a lane's piece is taken as
// the operand of two K steps, q permuted alike, and the output channels come out permuted the same
// way.  The tensor work is far below the bandwidth bound, so the warp-level MMA is enough here.
constexpr int RD_WARPS = 4, RD_KEYS = 16, RD_STAGES = 2, RD_BLOCKS = 3;

template <int D>
struct RangeDecodeCfg {
  static constexpr int KC = D / 32, VC = D / 64;     // 16-byte pieces per K row, per V row
  static constexpr int PIECES = 2 * KC + 4 * VC;     // of a lane in one stage: 2 K rows, 4 V rows
  static constexpr int RING = RD_WARPS * RD_STAGES * PIECES * 512;
};

template <int D, bool TWO, bool CAP, int BIAS>  // TWO: 9 to 16 rows (the second half of the MMA's rows is used)
__global__ void __launch_bounds__(RD_WARPS * 32, RD_BLOCKS) range_decode_kernel(const RangeArgs a) {
  constexpr int KC = RangeDecodeCfg<D>::KC, VC = RangeDecodeCfg<D>::VC, PIECES = RangeDecodeCfg<D>::PIECES;
  constexpr int HR = TWO ? 2 : 1;          // rows held by a lane: lane / 4 and, with TWO, lane / 4 + 8
  constexpr int ROWS = TWO ? 16 : 8;
  // the ring [warp][stage][piece][lane], and after it the warps' outputs
  extern __shared__ uint4 ring[];
  float(*o_sh)[ROWS][D + 4] = reinterpret_cast<float(*)[ROWS][D + 4]>(ring);
  static_assert(RD_WARPS * ROWS * (D + 4) * 4 <= RangeDecodeCfg<D>::RING, "the outputs reuse the ring");
  __shared__ float2 ml_sh[RD_WARPS][ROWS];
  __shared__ float o_cta[ROWS][D];
  __shared__ float2 ml_cta[ROWS];
  cg::cluster_group cluster = cg::this_cluster();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g4 = lane >> 2, q4 = lane & 3;
  const int b = blockIdx.z, kh = blockIdx.y, csize = gridDim.x, crank = blockIdx.x;
  const int rows = a.q_len * a.group;

  // the rows' ranges: each lane's own, and over all rows what any and what all of them see
  int lo[HR], hi[HR], pos[HR], head[HR];
  int all_lo = 0, all_hi = INT32_MAX, any_lo = INT32_MAX, any_hi = 0;
#pragma unroll
  for (int x = 0; x < HR; ++x) {
    const int r = g4 + 8 * x;
    lo[x] = hi[x] = pos[x] = head[x] = 0;
    if (r < rows) {
      const int tok = r / a.group;
      row_range(a, b, tok, lo[x], hi[x]);
      pos[x] = row_pos(a, b, tok);
      head[x] = kh * a.group + r % a.group;
      if (lo[x] < hi[x]) {
        any_lo = min(any_lo, lo[x]);
        any_hi = max(any_hi, hi[x]);
      }
      all_lo = max(all_lo, lo[x]);
      all_hi = min(all_hi, hi[x]);
    }
  }
  all_lo = __reduce_max_sync(0xffffffffu, all_lo);
  all_hi = __reduce_min_sync(0xffffffffu, all_hi);
  any_lo = __reduce_min_sync(0xffffffffu, any_lo);
  any_hi = __reduce_max_sync(0xffffffffu, any_hi);

  uint32_t qa[HR][2 * KC][2];  // A operand: [row half][K step][the two k pairs]
#pragma unroll
  for (int x = 0; x < HR; ++x) {
    const int r = g4 + 8 * x;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      uint4 u = make_uint4(0u, 0u, 0u, 0u);
      if (r < rows)
        u = __ldg(reinterpret_cast<const uint4*>(a.q + b * a.q_batch + (int64_t)(r / a.group) * a.q_tok +
                                                 (int64_t)(kh * a.group + r % a.group) * D + 32 * c + 8 * q4));
      qa[x][2 * c][0] = u.x;
      qa[x][2 * c][1] = u.y;
      qa[x][2 * c + 1][0] = u.z;
      qa[x][2 * c + 1][1] = u.w;
    }
  }

  const int step = csize * RD_WARPS * RD_KEYS;
  const bool some = any_lo < any_hi;
  int key0 = (some ? any_lo : 0) + (crank * RD_WARPS + warp) * RD_KEYS, fkey = key0, stage = 0;
  // this lane's rows of the block of keys to be asked for next: K rows g4, g4 + 8; V rows 2 q4 + {0, 1}, + 8
  const __nv_bfloat16* kp = a.k + b * a.k_batch + (int64_t)kh * D + 8 * q4 + (key0 + g4) * a.k_tok;
  const __nv_bfloat16* vp = a.v + b * a.v_batch + (int64_t)kh * D + 8 * g4 + (key0 + 2 * q4) * a.v_tok;
  const int64_t k8 = 8 * a.k_tok, v8 = 8 * a.v_tok, kstep = step * a.k_tok, vstep = step * a.v_tok;
  const __nv_bfloat16 *k_any = a.k, *v_any = a.v;  // a valid address for the copies that write zeros
  const uint32_t base = smem_u32(ring + warp * (RD_STAGES * PIECES * 32) + lane);
  auto fetch = [&](int stg) {  // keys behind the last seen one are not read
    const uint32_t dst = base + stg * PIECES * 512;
    if (fkey < any_hi) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const bool in = fkey + 8 * t + g4 < any_hi;
        const __nv_bfloat16* src = in ? kp + t * k8 : k_any;
#pragma unroll
        for (int c = 0; c < KC; ++c) cp_async16(dst + (t * KC + c) * 512, src + 32 * c, in);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const bool in = fkey + (t >> 1) * 8 + 2 * q4 + (t & 1) < any_hi;
        const __nv_bfloat16* src = in ? vp + (t >> 1) * v8 + (t & 1) * a.v_tok : v_any;
#pragma unroll
        for (int c = 0; c < VC; ++c) cp_async16(dst + (2 * KC + t * VC + c) * 512, src + 64 * c, in);
      }
    }
    cp_async_commit();
    fkey += step;
    kp += kstep;
    vp += vstep;
  };

  float o[VC * 8][2 * HR];  // n tile 8 c + i: channels 64 c + 8 (2 q4 + {0, 1}) + i of the lane's rows
#pragma unroll
  for (int n = 0; n < VC * 8; ++n)
#pragma unroll
    for (int e = 0; e < 2 * HR; ++e) o[n][e] = 0.f;
  float m[HR], l[HR];
#pragma unroll
  for (int x = 0; x < HR; ++x) m[x] = -INFINITY, l[x] = 0.f;

#pragma unroll
  for (int i = 0; i < RD_STAGES - 1; ++i) fetch(i);
  for (; some && key0 < any_hi; key0 += step) {
    fetch(stage == 0 ? RD_STAGES - 1 : stage - 1);  // the stage used last
    cp_async_wait<RD_STAGES - 1>();
    const uint32_t src = base + stage * PIECES * 512;
    if (++stage == RD_STAGES) stage = 0;
    float s[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float odd[4] = {0.f, 0.f, 0.f, 0.f};  // two chains of products, half as long
      s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const uint4 k = ld_shared16(src + (t * KC + c) * 512);
        mma_16816(s[t], qa[0][2 * c][0], TWO ? qa[HR - 1][2 * c][0] : 0u, qa[0][2 * c][1], TWO ? qa[HR - 1][2 * c][1] : 0u, k.x,
                  k.y);
        mma_16816(odd, qa[0][2 * c + 1][0], TWO ? qa[HR - 1][2 * c + 1][0] : 0u, qa[0][2 * c + 1][1],
                  TWO ? qa[HR - 1][2 * c + 1][1] : 0u, k.z, k.w);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) s[t][e] += odd[e];
    }

    // the lane's scores: rows g4 (+ 8), keys key0 + 8 t + 2 q4 + e
    float p[HR][4];
    bool raise = false;
    float mx[HR];
#pragma unroll
    for (int x = 0; x < HR; ++x) {
      mx[x] = -INFINITY;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = key0 + 8 * t + 2 * q4 + e;
          const float v = score_log2<CAP, BIAS>(a, s[t][2 * x + e], head[x], j - pos[x]);
          p[x][2 * t + e] = j >= lo[x] && j < hi[x] ? v : -INFINITY;
          mx[x] = fmaxf(mx[x], p[x][2 * t + e]);
        }
      mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 1));
      mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 2));
      raise |= mx[x] > m[x] + RA_RESCALE;
    }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int x = 0; x < HR; ++x) {
        const float mn = mx[x] > m[x] + RA_RESCALE ? mx[x] : m[x];
        const float alpha = mn == m[x] ? 1.f : ex2_approx(m[x] - mn);
        m[x] = mn;
        l[x] *= alpha;
#pragma unroll
        for (int n = 0; n < VC * 8; ++n) {
          o[n][2 * x] *= alpha;
          o[n][2 * x + 1] *= alpha;
        }
      }
    }
    uint32_t pa[HR][2];
#pragma unroll
    for (int x = 0; x < HR; ++x) {
      const float neg = m[x] == -INFINITY ? 0.f : -m[x];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[x][e] = ex2_approx(p[x][e] + neg);
        l[x] += p[x][e];
      }
      pa[x][0] = pack_bf16x2(p[x][0], p[x][1]);  // weights in bf16, the MMA's operand type; the sum keeps fp32
      pa[x][1] = pack_bf16x2(p[x][2], p[x][3]);
    }
    uint4 vr[4][VC];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int c = 0; c < VC; ++c) vr[t][c] = ld_shared16(src + (2 * KC + t * VC + c) * 512);
    if (key0 < all_lo || key0 + RD_KEYS > all_hi) {  // some row does not see some key of this block
      uint32_t bad = 0;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int c = 0; c < VC; ++c) bad |= nonfinite_bits(vr[t][c]);
      if (__any_sync(0xffffffffu, bad)) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int c = 0; c < VC; ++c)
            vr[t][c] = make_uint4(zero_nonfinite(vr[t][c].x), zero_nonfinite(vr[t][c].y), zero_nonfinite(vr[t][c].z),
                                  zero_nonfinite(vr[t][c].w));
#pragma unroll 1
        for (int kk = 0; kk < RD_KEYS; ++kk) {
          const int j = key0 + kk, src = (lane & ~3) | ((kk & 7) >> 1), e = (kk >> 3) * 2 + (kk & 1);
#pragma unroll
          for (int x = 0; x < HR; ++x) {
            const float p0 = __shfl_sync(0xffffffffu, p[x][0], src), p1 = __shfl_sync(0xffffffffu, p[x][1], src);
            const float p2 = __shfl_sync(0xffffffffu, p[x][2], src), p3 = __shfl_sync(0xffffffffu, p[x][3], src);
            const float pj = e == 0 ? p0 : e == 1 ? p1 : e == 2 ? p2 : p3;
            if (j >= lo[x] && j < hi[x]) {
              const __nv_bfloat16* vp = a.v + b * a.v_batch + j * a.v_tok + (int64_t)kh * D;
#pragma unroll
              for (int n = 0; n < VC * 8; ++n)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                  const __nv_bfloat16 vv = vp[64 * (n >> 3) + 8 * (2 * q4 + y) + (n & 7)];
                  if (nonfinite_bf16(vv)) o[n][2 * x + y] += pj * __bfloat162float(vv);
                }
            }
          }
        }
      }
    }
#pragma unroll
    for (int c = 0; c < VC; ++c) {
      const uint32_t w0[4] = {vr[0][c].x, vr[0][c].y, vr[0][c].z, vr[0][c].w};
      const uint32_t w1[4] = {vr[1][c].x, vr[1][c].y, vr[1][c].z, vr[1][c].w};
      const uint32_t w2[4] = {vr[2][c].x, vr[2][c].y, vr[2][c].z, vr[2][c].w};
      const uint32_t w3[4] = {vr[3][c].x, vr[3][c].y, vr[3][c].z, vr[3][c].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t sel = i & 1 ? 0x7632u : 0x5410u;
        float acc[4] = {o[8 * c + i][0], o[8 * c + i][1], TWO ? o[8 * c + i][2 * HR - 2] : 0.f,
                        TWO ? o[8 * c + i][2 * HR - 1] : 0.f};
        mma_16816(acc, pa[0][0], TWO ? pa[HR - 1][0] : 0u, pa[0][1], TWO ? pa[HR - 1][1] : 0u,
                  __byte_perm(w0[i >> 1], w1[i >> 1], sel), __byte_perm(w2[i >> 1], w3[i >> 1], sel));
        o[8 * c + i][0] = acc[0];
        o[8 * c + i][1] = acc[1];
        if constexpr (TWO) {
          o[8 * c + i][2] = acc[2];
          o[8 * c + i][3] = acc[3];
        }
      }
    }
  }
  cp_async_wait<0>();
  __syncthreads();  // the ring becomes the merge buffer

  // merge: warps of the block, then blocks of the cluster (row r of the result by rank r % csize)
#pragma unroll
  for (int x = 0; x < HR; ++x) {
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
    const int r = g4 + 8 * x;
    if (q4 == 0) ml_sh[warp][r] = make_float2(m[x], l[x]);
#pragma unroll
    for (int n = 0; n < VC * 8; ++n)
#pragma unroll
      for (int y = 0; y < 2; ++y) o_sh[warp][r][64 * (n >> 3) + 8 * (2 * q4 + y) + (n & 7)] = o[n][2 * x + y];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * D; i += RD_WARPS * 32) {
    const int r = i / D, d = i % D;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < RD_WARPS; ++w) mm = fmaxf(mm, ml_sh[w][r].x);
    float ll = 0.f, oo = 0.f;
#pragma unroll
    for (int w = 0; w < RD_WARPS; ++w) {
      const float2 ml = ml_sh[w][r];
      // a warp that saw nothing, or only scores of minus infinity: its sums are 0, or NaN to be kept
      const float f = ml.x == -INFINITY ? 1.f : ex2_approx(ml.x - mm);
      ll = fmaf(f, ml.y, ll);
      oo = fmaf(f, o_sh[w][r][d], oo);
    }
    o_cta[r][d] = oo;
    if (d == 0) ml_cta[r] = make_float2(mm, ll);
  }
  cluster.sync();
  for (int r = crank; r < rows; r += csize) {
    const int tok = r / a.group;
    int rlo, rhi;
    row_range(a, b, tok, rlo, rhi);
    float mm = -INFINITY;
    for (int c = 0; c < csize; ++c) mm = fmaxf(mm, cluster.map_shared_rank(ml_cta, c)[r].x);
    for (int d = threadIdx.x; d < D; d += RD_WARPS * 32) {
      float ll = 0.f, oo = 0.f;
      for (int c = 0; c < csize; ++c) {
        const float2 ml = cluster.map_shared_rank(ml_cta, c)[r];
        const float f = ml.x == -INFINITY ? 1.f : ex2_approx(ml.x - mm);
        ll = fmaf(f, ml.y, ll);
        oo = fmaf(f, cluster.map_shared_rank(&o_cta[0][0], c)[r * D + d], oo);
      }
      a.o[b * a.o_batch + (int64_t)tok * a.o_tok + (int64_t)(kh * a.group + r % a.group) * D + d] =
          __float2bfloat16(rlo < rhi ? oo / ll : 0.f);
    }
  }
  cluster.sync();  // a block's shared memory stays until all have read it
}

// ================================================================== many rows: tcgen05 tiles
// One work unit = (pair of 128-row query tiles t = 0, 1; key head; batch element; key split).  A tile
// holds tpt = 128 / group tokens x group heads.  Per 128-key tile j that some row of tile t sees:
//   S_t = Q_t K_j^T (TMEM columns 128 t ..), P_t = 2^(score - m) in bf16 over the first 64 columns
//   of S_t, O_t += P_t V_j (TMEM columns 256 + D t ..).
// The MMAs of one tile run while the other tile's warps exponentiate; the running maximum moves
// only when a tile exceeds it by 2^8, and only then is O rescaled in TMEM.  Key tiles that no row
// of a tile sees are neither loaded nor multiplied; tiles that every row sees skip the mask.
//
// Warps: 0-3 / 4-7 softmax and output of tile 0 / 1 (thread = row = TMEM lane), 8 unit queue + TMA,
// 9 TMEM + MMA issue, 10-11 look through the V tiles that are not seen by every row.
//
// The costs of units differ by the mask, so units are taken from a counter (zeroed by the plan
// kernel in front), longest first; which block runs a unit does not change its result.
constexpr int RT_M = 128, RT_N = 128;
constexpr int RT_THREADS = 384;
constexpr int RT_BLK = 16384;  // 128 rows of one 128-byte swizzle row
constexpr int RT_P_SPLIT = 96;
constexpr int RT_QUEUE = 2;
constexpr int RT_SORT_MAX = 2048;  // pairs that the plan kernel sorts

template <int D>
struct RangeTileCfg {
  static constexpr int TILE = RT_M * D * 2;
  static constexpr int RING = D == 128 ? 5 : 8;
  static constexpr int OFF_R = 2 * TILE, META = (2 + RING) * TILE;
  static constexpr int SMEM = META + 640 + 1024;
};

// What the rows of one tile pair see: [t] key range of any row, key range of every row.
struct RangePair {
  int any_lo[2], any_hi[2], all_lo[2], all_hi[2];
};

struct RangeTileArgs {
  RangeArgs a;
  int tpt, nqp;          // tokens per tile, tile pairs per sequence
  int entries;           // planned pairs: nqp, times the batch where the ranges differ by batch
  int streams;           // (key head, batch) combinations of an entry
  int stream_group;      // streams that run next to each other (their K and V fit L2)
  int splits, units;
  const RangePair* pairs;
  const int* order;
  int* counter;
  float* o_part;   // [splits][batch * kv_heads * q_len * group][D]
  float2* ml_part;
  int64_t part_rows;
  int* err;
};

struct PlanArgs {
  RangeArgs a;
  int tpt, nqp, entries;
  RangePair* pairs;
  int* order;
  int* counter;
};

// The key ranges of every tile pair (one warp each), and the pairs from the most key tiles to the
// fewest (bitonic sort, up to RT_SORT_MAX pairs; more are taken from the last to the first).
__global__ void __launch_bounds__(1024) range_plan_kernel(const PlanArgs p) {
  __shared__ uint32_t key[RT_SORT_MAX];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int n2 = 1;
  while (n2 < p.entries) n2 *= 2;
  const bool sort = n2 <= RT_SORT_MAX;
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.counter = 0;
  if (sort)
    for (int i = threadIdx.x; i < n2; i += 1024) key[i] = 0u;
  __syncthreads();
  const int warps = sort ? 32 : gridDim.x * 32;
  for (int e = (sort ? 0 : blockIdx.x * 32) + warp; e < p.entries; e += warps) {
    const int b = e / p.nqp, tok0 = e % p.nqp * 2 * p.tpt;
    RangePair r;
    int tiles = 0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      int any_lo = INT32_MAX, any_hi = 0, all_lo = 0, all_hi = INT32_MAX;
      for (int i = tok0 + t * p.tpt + lane; i < min(tok0 + (t + 1) * p.tpt, p.a.q_len); i += 32) {
        int lo, hi;
        row_range(p.a, b, i, lo, hi);
        if (lo < hi) any_lo = min(any_lo, lo), any_hi = max(any_hi, hi);
        all_lo = max(all_lo, lo);
        all_hi = min(all_hi, hi);
      }
      r.any_lo[t] = __reduce_min_sync(0xffffffffu, any_lo);
      r.any_hi[t] = __reduce_max_sync(0xffffffffu, any_hi);
      r.all_lo[t] = __reduce_max_sync(0xffffffffu, all_lo);
      r.all_hi[t] = __reduce_min_sync(0xffffffffu, all_hi);
      if (r.any_lo[t] >= r.any_hi[t]) r.any_lo[t] = r.any_hi[t] = 0;
      tiles += (r.any_hi[t] + RT_N - 1) / RT_N - r.any_lo[t] / RT_N;
    }
    if (lane == 0) {
      p.pairs[e] = r;
      if (sort)
        key[e] = (uint32_t)min(tiles, (1 << 20) - 1) << 11 | (uint32_t)e;
      else
        p.order[e] = p.entries - 1 - e;
    }
  }
  if (!sort) return;
  __syncthreads();
  for (int k = 2; k <= n2; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = threadIdx.x; i < n2; i += 1024) {
        const int x = i ^ j;
        if (x > i) {
          const uint32_t u = key[i], v = key[x];
          if (((i & k) == 0) ? u < v : u > v) key[i] = v, key[x] = u;  // descending
        }
      }
      __syncthreads();
    }
  // the padding keys are 0, and so is that of entry 0 without any keys: it may end up among them
  for (int i = threadIdx.x; i < p.entries; i += 1024) p.order[i] = (int)(key[i] & (RT_SORT_MAX - 1));
}

struct RangeUnit {
  int tok0, b, mb, kh, split, k0, k1;  // key tiles [k0, k1) of this split
  int a[2], z[2];                      // tile t: key tiles [a, z)
  int full_lo[2], full_hi[2];          // keys that every row of the tile sees
};

__device__ __forceinline__ RangeUnit range_unit(const RangeTileArgs& g, int u) {
  RangeUnit r;
  const int per_group = g.stream_group * g.entries * g.splits;
  const int grp = u / per_group, first = grp * g.stream_group, size = min(g.stream_group, g.streams - first);
  int x = u - grp * per_group;
  r.split = x % g.splits;
  x /= g.splits;
  const int stream = first + x % size, e = __ldg(g.order + x / size);
  r.kh = stream % g.a.kv_heads;
  r.mb = e / g.nqp;
  r.b = g.a.range_batch ? r.mb : stream / g.a.kv_heads;
  r.tok0 = e % g.nqp * 2 * g.tpt;
  const int4* pp = reinterpret_cast<const int4*>(g.pairs + e);
  const int4 any = __ldg(pp), all = __ldg(pp + 1);
  r.a[0] = any.x / RT_N, r.a[1] = any.y / RT_N;
  r.z[0] = (any.z + RT_N - 1) / RT_N, r.z[1] = (any.w + RT_N - 1) / RT_N;
  r.full_lo[0] = all.x, r.full_lo[1] = all.y, r.full_hi[0] = all.z, r.full_hi[1] = all.w;
  // [k0, k1) is the hull of the tiles' ranges: when not empty, its first and last key tiles are loaded
  auto hull = [&]() {
    const bool e0 = r.a[0] >= r.z[0], e1 = r.a[1] >= r.z[1];
    r.k0 = e0 ? r.a[1] : e1 ? r.a[0] : min(r.a[0], r.a[1]);
    r.k1 = e0 && e1 ? r.k0 : e0 ? r.z[1] : e1 ? r.z[0] : max(r.z[0], r.z[1]);
  };
  hull();
  if (g.splits > 1) {
    const int per = (r.k1 - r.k0 + g.splits - 1) / g.splits;
    const int from = min(r.k1, r.k0 + r.split * per), to = min(r.k1, from + per);
#pragma unroll
    for (int t = 0; t < 2; ++t) r.a[t] = max(r.a[t], from), r.z[t] = min(r.z[t], to);
    hull();
  }
  return r;
}

__device__ __forceinline__ bool unit_has(const RangeUnit& u, int t, int j) { return j >= u.a[t] && j < u.z[t]; }
__device__ __forceinline__ bool unit_full(const RangeUnit& u, int t, int j) {
  return j * RT_N >= u.full_lo[t] && (j + 1) * RT_N <= u.full_hi[t];
}
// Whether key tile j is loaded, and whether some row of an active tile does not see all of it.
__device__ __forceinline__ bool unit_loads(const RangeUnit& u, int j) { return unit_has(u, 0, j) || unit_has(u, 1, j); }
__device__ __forceinline__ bool unit_partial(const RangeUnit& u, int j) {
  return (unit_has(u, 0, j) && !unit_full(u, 0, j)) || (unit_has(u, 1, j) && !unit_full(u, 1, j));
}

// The non-finite values of V in the flagged keys of tile j (zeroed in shared memory), added to the
// rows that see them: o += p v.  Runs in a whole warp; the scores are formed anew.
template <int D, bool CAP, int BIAS>
__device__ __noinline__ void range_poison(const RangeArgs* ap, const uint32_t* bad, int b, int kh, int j0, int tok, int head,
                                          int lo, int hi, int pos, float neg, uint32_t t_o) {
  const RangeArgs& a = *ap;
#pragma unroll 1
  for (int c = 0; c < D / 32; ++c) {
    float o[32];
    tmem_ld32(t_o + c * 32, o);
#pragma unroll 1
    for (int k = 0; k < RT_N; ++k) {
      if (!((bad[k >> 5] >> (k & 31)) & 1u)) continue;  // warp-uniform
      const int j = j0 + k;
      if (j < lo || j >= hi) continue;
      const __nv_bfloat16* qp = a.q + b * a.q_batch + tok * a.q_tok + (int64_t)head * D;
      const __nv_bfloat16* kp = a.k + b * a.k_batch + j * a.k_tok + (int64_t)kh * D;
      const __nv_bfloat16* vp = a.v + b * a.v_batch + j * a.v_tok + (int64_t)kh * D + c * 32;
      float s = 0.f;
      for (int d = 0; d < D; ++d) s = fmaf(__bfloat162float(qp[d]), __bfloat162float(kp[d]), s);
      const float p = ex2_approx(score_log2<CAP, BIAS>(a, s, head, j - pos) + neg);
#pragma unroll
      for (int d = 0; d < 32; ++d)
        if (nonfinite_bf16(vp[d])) o[d] += p * __bfloat162float(vp[d]);
    }
    __syncwarp();
    tmem_st32(t_o + c * 32, o);
  }
}

template <int D, bool CAP, int BIAS>
__global__ void __maxnreg__(160)
    range_attn_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const __grid_constant__ RangeTileArgs g) {
  using C = RangeTileCfg<D>;
  constexpr int TILE = C::TILE, RING = C::RING, HALVES = D / 64;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
  const uint32_t sbase = smem_u32(smem);
  uint8_t* meta = smem + C::META;
  const uint32_t m0 = smem_u32(meta);
  const uint32_t kv_full = m0, kv_empty = m0 + 64, v_ok = m0 + 128;  // RING (<= 8) each
  const uint32_t q_full = m0 + 192, q_empty = m0 + 200;
  const uint32_t s_full = m0 + 208, p_part = m0 + 224, p_full = m0 + 240, o_done = m0 + 256;  // 2 each
  const uint32_t u_full = m0 + 272, u_empty = m0 + 288;  // RT_QUEUE each
  const uint32_t done_bar = m0 + 304;
  volatile int* queue = reinterpret_cast<volatile int*>(meta + 312);  // RT_QUEUE
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(meta + 320);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(meta + 324);
  uint32_t* bad = reinterpret_cast<uint32_t*>(meta + 336);  // [RING][4]: keys of the V tile with non-finite values
  const uint32_t v_req = m0 + 464;  // RING
  int* err = g.err;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < RING; ++s) {
      mbar_init(v_req + 8 * s, 1);
      mbar_init(kv_full + 8 * s, 1);
      mbar_init(kv_empty + 8 * s, 1);
      mbar_init(v_ok + 8 * s, 2);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(s_full + 8 * t, 1);
      mbar_init(p_part + 8 * t, 4);
      mbar_init(p_full + 8 * t, 4);
      mbar_init(o_done + 8 * t, 1);
    }
    for (int s = 0; s < RT_QUEUE; ++s) {
      mbar_init(u_full + 8 * s, 1);
      mbar_init(u_empty + 8 * s, 11);  // MMA, 8 softmax warps, 2 checking warps
    }
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // The next unit for a consuming warp (or its one lane): -1 = no more, -2 = aborted.
  int un = 0;
  auto next_unit = [&](int code) -> int {
    const int s = un % RT_QUEUE;
    if (!mbar_wait(u_full + 8 * s, (un / RT_QUEUE) & 1, abort_flag, err, code)) return -2;
    const int u = queue[s];
    ++un;
    return u;
  };
  auto release_unit = [&]() { mbar_arrive(u_empty + 8 * ((un - 1) % RT_QUEUE)); };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;\n" ::: "memory");
    if (warp == 8) {
      // ---------------------------------------------------------- unit queue and TMA
      {  // the whole warp walks the issue loops: see elect_one
        uint32_t issued = 0, last_ph = 0, q_ph = 0;
        int gk = 0, qi = 0;
        bool ok = true, q_pending = false;
        for (int i = 0; ok; ++i) {
          const int s = i % RT_QUEUE;
          if (!mbar_wait_warp(u_empty + 8 * s, ((i / RT_QUEUE) & 1) ^ 1, abort_flag, err, kErrTimeoutAttnProducer)) {
            ok = false;
            break;
          }
          int u = 0;
          if (lane == 0) {
            u = atomicAdd(g.counter, 1);
            if (u >= g.units) u = -1;
            queue[s] = u;
            mbar_arrive(u_full + 8 * s);
          }
          u = __shfl_sync(0xffffffffu, u, 0);
          if (u < 0) break;
          const RangeUnit w = range_unit(g, u);
          if (w.k0 >= w.k1) continue;
          if (!mbar_wait_warp(q_empty, (qi & 1) ^ 1, abort_flag, err, kErrTimeoutAttnProducer)) {
            ok = false;
            break;
          }
          if (elect_one()) {
            mbar_expect_tx(q_full, 2 * HALVES * g.tpt * g.a.group * 128);
            for (int t = 0; t < 2; ++t)
              for (int h = 0; h < HALVES; ++h)
                tma_load_4d(sbase + t * TILE + h * RT_BLK, &tmQ, q_full, 64 * h, w.kh * g.a.group, w.tok0 + t * g.tpt, w.b);
          }
          __syncwarp();
          q_pending = true;
          q_ph = qi & 1;
          ++qi;
          for (int j = w.k0; ok && j < w.k1; ++j) {
            if (!unit_loads(w, j)) continue;
            for (int x = 0; x < 2; ++x, ++gk) {
              const int slot = gk % RING;
              const uint32_t ph = (gk / RING) & 1;
              if (!mbar_wait_warp(kv_empty + 8 * slot, ph ^ 1, abort_flag, err, kErrTimeoutAttnProducer)) {
                ok = false;
                break;
              }
              const void* map = x ? static_cast<const void*>(&tmV) : static_cast<const void*>(&tmK);
              const uint32_t dst = sbase + C::OFF_R + slot * TILE;
              if (elect_one()) {
                mbar_expect_tx(kv_full + 8 * slot, TILE);
                for (int h = 0; h < HALVES; ++h)
                  tma_load_4d(dst + h * RT_BLK, map, kv_full + 8 * slot, 64 * h, w.kh, j * RT_N, w.b);
                if (x && unit_partial(w, j)) mbar_arrive(v_req + 8 * slot);
              }
              __syncwarp();
              issued |= 1u << slot;
              last_ph = (last_ph & ~(1u << slot)) | (ph << slot);
            }
          }
        }
        if (!ok) {  // let every load in flight land before the block's shared memory goes away
          if (q_pending) mbar_drain(q_full, q_ph, err);
          for (int s = 0; s < RING; ++s)
            if ((issued >> s) & 1) mbar_drain(kv_full + 8 * s, (last_ph >> s) & 1, err);
        }
      }
    } else if (warp == 9) {
      // ---------------------------------------------------------- MMA issue
      {
        constexpr uint32_t idesc_s = idesc_bf16_f32(RT_M, RT_N, false, false);
        constexpr uint32_t idesc_o = idesc_bf16_f32(RT_M, D, false, true);
        constexpr uint32_t hi = sw128_hi(1024);
        const uint32_t q_lo = sw128_lo(sbase, 16), k_lo = sw128_lo(sbase + C::OFF_R, 16), v_lo = sw128_lo(sbase + C::OFF_R, RT_BLK);
        auto commit = [](bool yes, uint32_t bar) {
          if (yes && elect_one()) umma_commit(bar);
          __syncwarp();
        };
        int gk = 0, qi = 0, np[2] = {0, 0};
        uint32_t ok_ph = 0;  // phase of v_ok per ring slot
        bool ok = true;
        while (ok) {
          const int u = next_unit(kErrTimeoutAttnMma);
          if (!__all_sync(0xffffffffu, u != -2) || u < 0) break;
          const RangeUnit w = range_unit(g, u);
          __syncwarp();
          if (lane == 0) release_unit();
          if (w.k0 >= w.k1) continue;
          auto kv_wait = [&](int r) -> bool {
            return mbar_wait_warp(kv_full + 8 * (r % RING), (r / RING) & 1, abort_flag, err, kErrTimeoutAttnMma);
          };
          auto qk = [&](int t, int slot) {
            tc_fence_after();
            const uint32_t d = tmem_base + t * RT_N, qb = q_lo + t * (TILE >> 4), kb = k_lo + slot * (TILE >> 4);
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk) {
                const uint32_t off = ((kk >> 2) * RT_BLK + (kk & 3) * 32) >> 4;
                umma_bf16_w(d, qb + off, kb + off, hi, idesc_s, kk != 0);
              }
              umma_commit(s_full + 8 * t);
            }
            __syncwarp();
          };
          auto pv = [&](int t, int slot, bool last) -> bool {
            // P_t comes in two parts: the MMA over its first keys runs while the warps exponentiate the rest
            const uint32_t ph = np[t]++ & 1;
            if (!mbar_wait_warp(p_part + 8 * t, ph, abort_flag, err, kErrTimeoutAttnMma)) return false;
            tc_fence_after();
            const uint32_t d = tmem_base + 2 * RT_N + t * D, pa = tmem_base + t * RT_N, vb = v_lo + slot * (TILE >> 4);
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < RT_P_SPLIT / 16; ++kk)
                umma_bf16_tmem_a_w(d, pa + kk * 8, vb + kk * (2048 >> 4), hi, idesc_o);
            }
            __syncwarp();
            if (!mbar_wait_warp(p_full + 8 * t, ph, abort_flag, err, kErrTimeoutAttnMma)) return false;
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int kk = RT_P_SPLIT / 16; kk < RT_N / 16; ++kk)
                umma_bf16_tmem_a_w(d, pa + kk * 8, vb + kk * (2048 >> 4), hi, idesc_o);
              if (last) umma_commit(o_done + 8 * t);
            }
            __syncwarp();
            return true;
          };
          int j = w.k0;
          ok = mbar_wait_warp(q_full, qi & 1, abort_flag, err, kErrTimeoutAttnMma) && kv_wait(gk);
          ++qi;
          if (!ok) break;
          int jn = j + 1;
          while (jn < w.k1 && !unit_loads(w, jn)) ++jn;
          for (int t = 0; t < 2; ++t)
            if (unit_has(w, t, j)) qk(t, gk % RING);
          commit(true, kv_empty + 8 * (gk % RING));
          commit(jn >= w.k1, q_empty);
          while (true) {
            const int vslot = (gk + 1) % RING, kslot = (gk + 2) % RING;
            const bool more = jn < w.k1;
            if (!kv_wait(gk + 1)) { ok = false; break; }
            if (unit_partial(w, j)) {
              if (!mbar_wait_warp(v_ok + 8 * vslot, (ok_ph >> vslot) & 1, abort_flag, err, kErrTimeoutAttnMma)) { ok = false; break; }
              ok_ph ^= 1u << vslot;
            }
            if (unit_has(w, 0, j) && !pv(0, vslot, j == w.z[0] - 1)) { ok = false; break; }
            if (more) {
              if (!kv_wait(gk + 2)) { ok = false; break; }
              if (unit_has(w, 0, jn)) qk(0, kslot);
            }
            if (unit_has(w, 1, j) && !pv(1, vslot, j == w.z[1] - 1)) { ok = false; break; }
            commit(true, kv_empty + 8 * vslot);
            gk += 2;
            if (!more) break;
            if (unit_has(w, 1, jn)) qk(1, kslot);
            commit(true, kv_empty + 8 * kslot);
            j = jn++;
            while (jn < w.k1 && !unit_loads(w, jn)) ++jn;
            commit(jn >= w.k1, q_empty);  // the unit's last QK is issued: Q may be overwritten after it
          }
        }
        commit(true, done_bar);
        mbar_drain(done_bar, 0, err);
      }
    } else {
      // ---------------------------------------------------------- non-finite values in partly seen V tiles
      // The producer announces such a tile (v_req), so these warps pass over the others without a
      // wait: the phases of v_req move only with the tiles they handle, and neither they nor
      // kv_full can get a phase ahead before v_ok is given.
      int gk = 0;
      uint32_t req_ph = 0;  // phase of v_req per ring slot
      bool ok = true;
      while (ok) {
        const int u = next_unit(kErrTimeoutAttnProducer);
        if (!__all_sync(0xffffffffu, u != -2) || u < 0) break;
        const RangeUnit w = range_unit(g, u);
        __syncwarp();
        if (lane == 0) release_unit();
        for (int j = w.k0; ok && j < w.k1; ++j) {
          if (!unit_loads(w, j)) continue;
          const int slot = (gk + 1) % RING;
          if (unit_partial(w, j)) {
            ok = mbar_wait_warp(v_req + 8 * slot, (req_ph >> slot) & 1, abort_flag, err, kErrTimeoutAttnProducer) &&
                 mbar_wait_warp(kv_full + 8 * slot, ((gk + 1) / RING) & 1, abort_flag, err, kErrTimeoutAttnProducer);
            if (!ok) break;
            req_ph ^= 1u << slot;
            bool wrote = false;
#pragma unroll 1
            for (int x = 0; x < 2; ++x) {
              const int word = 2 * x + (warp - 10);
              uint8_t* row = smem + C::OFF_R + slot * TILE + (word * 32 + lane) * 128;
              bool hit = false;
#pragma unroll
              for (int h = 0; h < HALVES; ++h) hit |= clean_row128(row + h * RT_BLK, lane);
              const uint32_t bits = __ballot_sync(0xffffffffu, hit);
              if (lane == 0) bad[slot * 4 + word] = bits;
              wrote |= bits != 0;
            }
            if (wrote) fence_proxy_async_smem();  // uniform over the warp: each lane for its own stores
            __syncwarp();
            if (lane == 0) mbar_arrive(v_ok + 8 * slot);
          }
          gk += 2;
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;\n" ::: "memory");
    // ------------------------------------------------------------ softmax + output (warps 0..7)
    const int t = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lane_off = uint32_t((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem_base + lane_off + t * RT_N;
    const uint32_t t_o = tmem_base + lane_off + 2 * RT_N + t * D;
    const RangeArgs& a = g.a;
    const int rtok = r / a.group, rhead = r - rtok * a.group;
    auto zero_o = [&]() {
      const float z[32] = {};
#pragma unroll
      for (int c = 0; c < D / 32; ++c) tmem_st32(t_o + c * 32, z);
    };
    zero_o();  // every P V accumulates; the first is issued after this thread's first p_part arrival
    int gk = 0, ns = 0, no = 0;
    uint32_t ok_ph = 0;
    bool ok = true;
    while (ok) {
      const int u = next_unit(kErrTimeoutAttnSoftmax);
      if (!__all_sync(0xffffffffu, u != -2) || u < 0) break;
      const RangeUnit w = range_unit(g, u);
      __syncwarp();
      if (lane == 0) release_unit();
      const int tok = w.tok0 + t * g.tpt + rtok;
      const bool live = rtok < g.tpt && tok < a.q_len;
      const int head = w.kh * a.group + rhead;
      int lo = 0, hi = 0, pos = 0;
      if (live) {
        row_range(a, w.b, tok, lo, hi);
        if constexpr (BIAS != kBiasNone) pos = row_pos(a, w.b, tok);
      }
      float slope2 = 0.f;
      const float* trow = nullptr;
      if constexpr (BIAS == kBiasSlopes) slope2 = live ? RA_LOG2E * __ldg(a.slopes + head) : 0.f;
      if constexpr (BIAS == kBiasTable) trow = a.table + (live ? (int64_t)head * (2 * a.reach + 1) : 0) + a.reach;
      float m_used = -INFINITY, l_run = 0.f;
      bool any_tile = false;
      for (int j = w.k0; j < w.k1; ++j) {
        if (!unit_loads(w, j)) continue;
        const int slot = (gk + 1) % RING;
        const bool partial = unit_partial(w, j);
        gk += 2;
        if (!unit_has(w, t, j)) {
          if (partial) ok_ph ^= 1u << slot;
          continue;
        }
        if (!mbar_wait_warp(s_full + 8 * t, ns & 1, abort_flag, err, kErrTimeoutAttnSoftmax)) {
          ok = false;
          break;
        }
        ++ns;
        tc_fence_after();
        uint32_t sr[RT_N];
#pragma unroll
        for (int c = 0; c < RT_N / 32; ++c) tmem_ld32_nowait(t_s + c * 32, sr + c * 32);
        tmem_wait_ld();
        float* s = reinterpret_cast<float*>(sr);
        const int kbase = j * RT_N;
        const bool masked = !unit_full(w, t, j);
        uint32_t mask[4];
        if (masked) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {  // bit k: key kbase + 32 x + k is seen
            const int l0 = lo - kbase - 32 * x, h0 = hi - kbase - 32 * x;
            const uint32_t below = h0 >= 32 ? 0xffffffffu : h0 <= 0 ? 0u : (1u << h0) - 1u;
            mask[x] = below & (l0 <= 0 ? 0xffffffffu : l0 >= 32 ? 0u : 0xffffffffu << l0);
          }
          if constexpr (CAP) {  // a hidden NaN must not reach the four that share a reciprocal
#pragma unroll
            for (int k = 0; k < RT_N; ++k)
              if (!((mask[k >> 5] >> (k & 31)) & 1u)) s[k] = 0.f;
          }
        }
        if constexpr (CAP) {
          // cap2 tanh = cap2 - 2 cap2 / (1 + 2^x); four reciprocals from one (MUFU is what bounds this form)
          const float n2c = -2.f * a.cap2;
#pragma unroll
          for (int k = 0; k < RT_N; k += 4) {
            const float d0 = 1.f + ex2_approx(min30(s[k] * a.sl2)), d1 = 1.f + ex2_approx(min30(s[k + 1] * a.sl2));
            const float d2 = 1.f + ex2_approx(min30(s[k + 2] * a.sl2)), d3 = 1.f + ex2_approx(min30(s[k + 3] * a.sl2));
            const float p01 = d0 * d1, p23 = d2 * d3;
            const float rc = n2c * rcp_approx(p01 * p23);
            const float r01 = rc * p23, r23 = rc * p01;
            s[k] = fmaf(r01, d1, a.cap2);
            s[k + 1] = fmaf(r01, d0, a.cap2);
            s[k + 2] = fmaf(r23, d3, a.cap2);
            s[k + 3] = fmaf(r23, d2, a.cap2);
          }
        }
        const float sl2 = CAP ? 1.f : a.sl2;
        if constexpr (BIAS == kBiasSlopes) {
          const float d0 = (float)(kbase - pos);
#pragma unroll
          for (int k = 0; k < RT_N; ++k) s[k] = fmaf(-slope2, fabsf(d0 + (float)k), CAP ? s[k] : s[k] * sl2);
        }
        if constexpr (BIAS == kBiasTable) {
          const int d0 = kbase - pos;
          if (__all_sync(0xffffffffu, d0 >= a.reach || d0 + RT_N - 1 <= -a.reach)) {
            const float far = RA_LOG2E * __ldg(trow + (d0 >= a.reach ? a.reach : -a.reach));
#pragma unroll
            for (int k = 0; k < RT_N; ++k) s[k] = CAP ? s[k] + far : fmaf(s[k], sl2, far);
          } else {
#pragma unroll
            for (int k = 0; k < RT_N; ++k)
              s[k] = fmaf(RA_LOG2E, __ldg(trow + min(max(d0 + k, -a.reach), a.reach)), CAP ? s[k] : s[k] * sl2);
          }
        }
        const float mul = BIAS == kBiasNone && !CAP ? a.sl2 : 1.f;  // what is left to apply in the exponent
        if (masked) {
#pragma unroll
          for (int k = 0; k < RT_N; ++k)
            if (!((mask[k >> 5] >> (k & 31)) & 1u)) s[k] = -INFINITY;
        }
        float m8[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) m8[c] = fmaxf(s[2 * c], s[2 * c + 1]);
#pragma unroll
        for (int q = 1; q < RT_N / 16; ++q)
#pragma unroll
          for (int c = 0; c < 8; ++c) m8[c] = fmax3(m8[c], s[16 * q + 2 * c], s[16 * q + 2 * c + 1]);
        const float mx = fmax3(fmax3(m8[0], m8[1], m8[2]), fmax3(m8[3], m8[4], m8[5]), fmaxf(m8[6], m8[7]));
        const float m_cand = mx * mul;
        const bool need = m_cand > m_used + RA_RESCALE;
        const bool any_need = __any_sync(0xffffffffu, need);
        float alpha = 1.f;
        if (any_need) {
          const float m_new = need ? m_cand : m_used;
          if (need) alpha = ex2_approx(m_used - m_new);
          l_run *= alpha;
          m_used = m_new;
        }
        // O_t may be changed here: S_t(j) was issued after the previous P V of this tile, and this
        // tile's waits for the p_part arrival below
        if (any_need && any_tile) {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            float o[32];
            tmem_ld32(t_o + c * 32, o);
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] *= alpha;
            tmem_st32(t_o + c * 32, o);
          }
        }
        any_tile = true;
        const float neg = m_used == -INFINITY ? 0.f : -m_used;
        if (partial) {
          if (!mbar_wait_warp(v_ok + 8 * slot, (ok_ph >> slot) & 1, abort_flag, err, kErrTimeoutAttnSoftmax)) {
            ok = false;
            break;
          }
          ok_ph ^= 1u << slot;
          const uint32_t* bw = bad + slot * 4;
          if (bw[0] | bw[1] | bw[2] | bw[3])
            range_poison<D, CAP, BIAS>(&g.a, bw, w.b, w.kh, kbase, tok, head, lo, hi, pos, neg, t_o);
        }
        const float2 mulv = make_float2(mul, mul), negv = make_float2(neg, neg);
        float2 acc2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int c = 0; c < RT_N / 32; ++c) {
          if (c == RT_P_SPLIT / 32) {  // the first part of P_t is in TMEM: hand it over
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_part + 8 * t);
          }
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            const float2 x = __ffma2_rn(make_float2(s[c * 32 + k], s[c * 32 + k + 1]), mulv, negv);
            const float p0 = ex2_approx(x.x), p1 = ex2_approx(x.y);
            acc2[(k >> 1) & 1] = __fadd2_rn(acc2[(k >> 1) & 1], make_float2(p0, p1));
            pk[k >> 1] = pack_bf16x2(p0, p1);  // weights in bf16, the MMA's operand type; the row sum keeps fp32
          }
          tmem_st16_nowait(t_s + c * 16, pk);
        }
        tmem_wait_st();
        l_run += (acc2[0].x + acc2[0].y) + (acc2[1].x + acc2[1].y);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + 8 * t);
      }
      if (!ok) break;
      if (any_tile) {
        if (!mbar_wait_warp(o_done + 8 * t, no & 1, abort_flag, err, kErrTimeoutAttnSoftmax)) {
          ok = false;
          break;
        }
        ++no;
        tc_fence_after();
      }
      if (g.splits > 1) {
        const int64_t prow = (int64_t)w.split * g.part_rows +
                             (((int64_t)w.b * a.kv_heads + w.kh) * a.q_len + tok) * a.group + rhead;
        float4* dst = reinterpret_cast<float4*>(g.o_part + prow * D);
        if (any_tile) {  // otherwise the sum and maximum say that this split saw nothing
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            float o[32];
            tmem_ld32(t_o + c * 32, o);
            if (live) {
#pragma unroll
              for (int q = 0; q < 8; ++q) dst[c * 8 + q] = make_float4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
            }
          }
        }
        if (live) g.ml_part[prow] = make_float2(any_tile ? m_used : -INFINITY, any_tile ? l_run : -1.f);
      } else {
        const float inv_l = lo < hi ? 1.f / l_run : 0.f;
        uint4* dst = reinterpret_cast<uint4*>(a.o + (int64_t)w.b * a.o_batch + (int64_t)tok * a.o_tok + (int64_t)head * D);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          tmem_ld32(t_o + c * 32, o);
          if (live) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint4 x;
              x.x = pack_bf16x2(o[q * 8 + 0] * inv_l, o[q * 8 + 1] * inv_l);
              x.y = pack_bf16x2(o[q * 8 + 2] * inv_l, o[q * 8 + 3] * inv_l);
              x.z = pack_bf16x2(o[q * 8 + 4] * inv_l, o[q * 8 + 5] * inv_l);
              x.w = pack_bf16x2(o[q * 8 + 6] * inv_l, o[q * 8 + 7] * inv_l);
              dst[c * 4 + q] = x;
            }
          }
        }
      }
      if (any_tile) zero_o();
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem_base, 512);
}

// Merge of the key splits: one warp per packed row.  A split that saw no key tile left l = -1 and no O.
template <int D>
__global__ void __launch_bounds__(256) range_combine_kernel(const RangeTileArgs g) {
  constexpr int E = D / 32;
  const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (w >= g.part_rows) return;
  const RangeArgs& a = g.a;
  const int hg = (int)(w % a.group);
  int64_t x = w / a.group;
  const int tok = (int)(x % a.q_len);
  x /= a.q_len;
  const int kh = (int)(x % a.kv_heads), b = (int)(x / a.kv_heads);
  int lo, hi;
  row_range(a, b, tok, lo, hi);
  float m = -INFINITY;
  for (int s = 0; s < g.splits; ++s) m = fmaxf(m, g.ml_part[s * g.part_rows + w].x);
  float l = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int s = 0; s < g.splits; ++s) {
    const float2 ml = g.ml_part[s * g.part_rows + w];
    if (ml.y == -1.f) continue;
    const float f = ml.x == -INFINITY ? 1.f : ex2_approx(ml.x - m);
    l = fmaf(f, ml.y, l);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(f, g.o_part[(s * g.part_rows + w) * D + lane * E + e], o[e]);
  }
  __nv_bfloat16* op = a.o + b * a.o_batch + (int64_t)tok * a.o_tok + (int64_t)(kh * a.group + hg) * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) op[e] = __float2bfloat16(lo < hi ? o[e] / l : 0.f);
}

// ------------------------------------------------------------------ host launcher
// Packed rows up to which the few-rows kernel runs (the 16 rows of its MMA).
constexpr int RD_ROWS = 16;

struct RangeLayout {
  int tpt, nqp, entries, streams, splits;
  int64_t units, part_rows, order_off, counter_off, part_off, ml_off, bytes;
};

static RangeLayout range_layout(const wanb200_range_attn_params* p) {
  RangeLayout l = {};
  const int group = (int)(p->heads / p->kv_heads);
  if (p->q_len * group <= RD_ROWS) return l;
  const bool per_batch = p->range_batch_stride > 0;
  l.tpt = RT_M / group;
  l.nqp = (int)((p->q_len + 2 * l.tpt - 1) / (2 * l.tpt));
  const int64_t entries = per_batch ? p->batch * l.nqp : l.nqp, streams = per_batch ? p->kv_heads : p->kv_heads * p->batch;
  if (entries > INT32_MAX / 64 || streams > INT32_MAX / 64) return l;
  l.entries = (int)entries;
  l.streams = (int)streams;
  // split the keys when the units leave SMs idle: at least two key tiles a split
  const int64_t units = entries * streams, tiles = (p->kv_len + RT_N - 1) / RT_N;
  l.splits = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(num_sms() / units, tiles / 2), 32));
  l.units = units * l.splits;
  l.part_rows = p->batch * p->heads * p->q_len;
  auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
  l.order_off = up(entries * (int64_t)sizeof(RangePair));
  l.counter_off = l.order_off + up(entries * 4);
  l.part_off = l.counter_off + 256;
  l.ml_off = l.part_off + (l.splits > 1 ? up(l.splits * l.part_rows * p->head_dim * 4) : 0);
  l.bytes = l.ml_off + (l.splits > 1 ? up(l.splits * l.part_rows * 8) : 0);
  return l;
}

static int range_validate(const wanb200_range_attn_params* p) {
  if (!p) return set_error(WANB200_EINVAL, "range_attn: null params");
  if (!p->q || !p->k || !p->v || !p->o || !p->lo || !p->hi)
    return set_error(WANB200_EINVAL, "range_attn: null q/k/v/o/lo/hi");
  if (p->head_dim != 64 && p->head_dim != 128) return set_error(WANB200_EINVAL, "range_attn: head_dim must be 64 or 128");
  if (p->batch <= 0 || p->heads <= 0 || p->kv_heads <= 0 || p->q_len <= 0 || p->kv_len <= 0)
    return set_error(WANB200_EINVAL, "range_attn: batch, heads, kv_heads, q_len, kv_len must be positive");
  if (p->heads % p->kv_heads || p->heads / p->kv_heads > 128)
    return set_error(WANB200_EINVAL, "range_attn: heads must be a multiple of kv_heads, at most 128 heads each");
  if (p->batch > 65535 || p->heads > 65535 || p->q_len > INT32_MAX / 2 || p->kv_len > INT32_MAX / 2)
    return set_error(WANB200_EINVAL, "range_attn: batch/heads/lengths too large");
  const int64_t strides[8] = {p->q_tok_stride, p->q_batch_stride, p->k_tok_stride, p->k_batch_stride,
                              p->v_tok_stride, p->v_batch_stride, p->o_tok_stride, p->o_batch_stride};
  for (int i = 0; i < 8; ++i)
    if (strides[i] <= 0 || strides[i] % 8)
      return set_error(WANB200_EINVAL, "range_attn: strides must be positive multiples of 8");
  if (p->q_tok_stride < p->heads * p->head_dim || p->o_tok_stride < p->heads * p->head_dim ||
      p->k_tok_stride < p->kv_heads * p->head_dim || p->v_tok_stride < p->kv_heads * p->head_dim)
    return set_error(WANB200_EINVAL, "range_attn: token stride smaller than heads * head_dim");
  if (!aligned16(p->q) || !aligned16(p->k) || !aligned16(p->v) || !aligned16(p->o))
    return set_error(WANB200_EINVAL, "range_attn: q/k/v/o must be 16-byte aligned");
  if (!(p->softmax_scale > 0.f) || !(p->softmax_scale < INFINITY))
    return set_error(WANB200_EINVAL, "range_attn: softmax_scale must be positive");
  if (!(p->softcap >= 0.f) || !(p->softcap < INFINITY))
    return set_error(WANB200_EINVAL, "range_attn: softcap must be >= 0 (0 = none)");
  if (p->slopes && p->dist_bias) return set_error(WANB200_EINVAL, "range_attn: slopes or dist_bias, not both");
  if (p->dist_bias && (p->reach < 0 || p->reach > (1 << 24)))
    return set_error(WANB200_EINVAL, "range_attn: dist_bias needs 0 <= reach <= 2^24");
  if (p->range_batch_stride < 0) return set_error(WANB200_EINVAL, "range_attn: negative range_batch_stride");
  return WANB200_OK;
}

int64_t range_attn_workspace_bytes(const wanb200_range_attn_params* p) {
  if (!p || p->batch <= 0 || p->heads <= 0 || p->kv_heads <= 0 || p->heads % p->kv_heads || p->heads / p->kv_heads > RT_M ||
      p->q_len <= 0 || p->kv_len <= 0 || p->q_len > INT32_MAX / 2 || p->batch > 65535 || p->heads > 65535 ||
      (p->head_dim != 64 && p->head_dim != 128))
    return 0;
  return range_layout(p).bytes;
}

template <int D, bool TWO, bool CAP, int BIAS>
static cudaError_t launch_range_decode(const RangeArgs& a, const cudaLaunchConfig_t& cfg, int dev) {
  static std::atomic<bool> attr_set[kMaxDevices] = {};
  if (!attr_set[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(range_decode_kernel<D, TWO, CAP, BIAS>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, RangeDecodeCfg<D>::RING);
    if (e != cudaSuccess) return e;
    attr_set[dev].store(true, std::memory_order_release);
  }
  return cudaLaunchKernelEx(&cfg, range_decode_kernel<D, TWO, CAP, BIAS>, a);
}

template <int D, bool CAP, int BIAS>
static int launch_range_decode(const RangeArgs& a, int rows, cudaStream_t st) {
  // Blocks of a cluster share one (key head, batch element).  The cluster size is the one with the
  // smallest waves x (keys of a block + 160): the block's fixed costs (start, merges) weigh about as much
  // as 160 keys.
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= kMaxDevices) return set_error(WANB200_EINVAL, "device index out of range");
  const int64_t units = (int64_t)a.batch * a.kv_heads, slots = (int64_t)num_sms() * RD_BLOCKS;
  int best = 1;
  double best_t = 1e300;
  for (int c = 1; c <= 8; c *= 2) {
    const double t = (double)((units * c + slots - 1) / slots) * ((double)a.kv_len / c + 160.0);
    if (t < best_t - 1e-9) best_t = t, best = c;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)best, (unsigned)a.kv_heads, (unsigned)a.batch);
  cfg.blockDim = dim3(RD_WARPS * 32);
  cfg.dynamicSmemBytes = RangeDecodeCfg<D>::RING;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)best;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = rows > 8 ? launch_range_decode<D, true, CAP, BIAS>(a, cfg, dev)
                                 : launch_range_decode<D, false, CAP, BIAS>(a, cfg, dev);
  if (e != cudaSuccess) return set_cuda_error("range_decode_kernel launch", e);
  return WANB200_OK;
}

template <int D, bool CAP, int BIAS>
static int launch_range_tiles(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const RangeTileArgs& g,
                              cudaStream_t st) {
  static std::atomic<bool> attr_set[kMaxDevices] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= kMaxDevices) return set_error(WANB200_EINVAL, "device index out of range");
  if (!attr_set[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(range_attn_kernel<D, CAP, BIAS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               RangeTileCfg<D>::SMEM);
    if (e != cudaSuccess) return set_cuda_error("cudaFuncSetAttribute(range_attn)", e);
    attr_set[dev].store(true, std::memory_order_release);
  }
  PlanArgs pl;
  pl.a = g.a;
  pl.tpt = g.tpt;
  pl.nqp = g.nqp;
  pl.entries = g.entries;
  pl.pairs = const_cast<RangePair*>(g.pairs);
  pl.order = const_cast<int*>(g.order);
  pl.counter = g.counter;
  const int plan_blocks = g.entries <= RT_SORT_MAX ? 1 : std::min((g.entries + 31) / 32, num_sms());
  range_plan_kernel<<<plan_blocks, 1024, 0, st>>>(pl);
  const unsigned grid = (unsigned)std::min<int64_t>(g.units, num_sms());
  range_attn_kernel<D, CAP, BIAS><<<grid, RT_THREADS, RangeTileCfg<D>::SMEM, st>>>(tq, tk, tv, g);
  if (g.splits > 1) range_combine_kernel<D><<<(unsigned)((g.part_rows + 7) / 8), 256, 0, st>>>(g);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error("range attention launch", e);
  return WANB200_OK;
}

template <int D>
static int range_dispatch(const RangeArgs& a, const RangeTileArgs* g, const CUtensorMap* maps, int rows, cudaStream_t st) {
  const int bias = a.slopes ? kBiasSlopes : a.table ? kBiasTable : kBiasNone;
#define WANB200_RANGE_CASE(cap, bs) \
  return g ? launch_range_tiles<D, cap, bs>(maps[0], maps[1], maps[2], *g, st) : launch_range_decode<D, cap, bs>(a, rows, st)
  if (a.cap2 > 0.f) {
    if (bias == kBiasSlopes) WANB200_RANGE_CASE(true, kBiasSlopes);
    if (bias == kBiasTable) WANB200_RANGE_CASE(true, kBiasTable);
    WANB200_RANGE_CASE(true, kBiasNone);
  }
  if (bias == kBiasSlopes) WANB200_RANGE_CASE(false, kBiasSlopes);
  if (bias == kBiasTable) WANB200_RANGE_CASE(false, kBiasTable);
  WANB200_RANGE_CASE(false, kBiasNone);
#undef WANB200_RANGE_CASE
}

int range_attn_fwd(const wanb200_range_attn_params* p, cudaStream_t st) {
  int rc = range_validate(p);
  if (rc) return rc;
  RangeArgs a;
  a.q = reinterpret_cast<const __nv_bfloat16*>(p->q);
  a.k = reinterpret_cast<const __nv_bfloat16*>(p->k);
  a.v = reinterpret_cast<const __nv_bfloat16*>(p->v);
  a.o = reinterpret_cast<__nv_bfloat16*>(p->o);
  a.q_tok = p->q_tok_stride; a.q_batch = p->q_batch_stride;
  a.k_tok = p->k_tok_stride; a.k_batch = p->k_batch_stride;
  a.v_tok = p->v_tok_stride; a.v_batch = p->v_batch_stride;
  a.o_tok = p->o_tok_stride; a.o_batch = p->o_batch_stride;
  a.batch = (int)p->batch;
  a.kv_heads = (int)p->kv_heads;
  a.group = (int)(p->heads / p->kv_heads);
  a.q_len = (int)p->q_len;
  a.kv_len = (int)p->kv_len;
  a.sl2 = p->softcap > 0.f ? 2.f * RA_LOG2E * p->softmax_scale / p->softcap : RA_LOG2E * p->softmax_scale;
  a.cap2 = p->softcap * RA_LOG2E;
  a.lo = p->lo;
  a.hi = p->hi;
  a.pos = p->pos;
  a.range_batch = p->range_batch_stride;
  a.slopes = p->slopes;
  a.table = p->dist_bias;
  a.reach = p->reach;
  const int64_t rows = p->q_len * a.group;
  if (rows <= RD_ROWS) {
    return p->head_dim == 64 ? range_dispatch<64>(a, nullptr, nullptr, (int)rows, st)
                             : range_dispatch<128>(a, nullptr, nullptr, (int)rows, st);
  }
  const RangeLayout l = range_layout(p);
  if (l.units <= 0 || l.units > INT32_MAX / 2 || (l.part_rows + 7) / 8 > INT32_MAX)
    return set_error(WANB200_EINVAL, "range_attn: too many rows");
  if (!p->workspace || (reinterpret_cast<uintptr_t>(p->workspace) & 255u) || p->workspace_bytes < l.bytes)
    return set_error(WANB200_EINVAL, "range_attn: need a 256-byte aligned workspace of wanb200_range_attn_workspace_bytes()");
  int* err = device_error_word();
  if (!err) return WANB200_ECUDA;
  CUtensorMap maps[3];
  const int D = (int)p->head_dim;
  const int64_t dq[4] = {D, p->heads, p->q_len, p->batch}, sq[4] = {1, D, p->q_tok_stride, p->q_batch_stride};
  const int boxq[4] = {64, a.group, l.tpt, 1}, boxk[4] = {64, 1, RT_N, 1};
  rc = make_tmap_4d(&maps[0], p->q, dq, sq, boxq);
  if (rc) return rc;
  const int64_t dk[4] = {D, p->kv_heads, p->kv_len, p->batch}, sk[4] = {1, D, p->k_tok_stride, p->k_batch_stride};
  rc = make_tmap_4d(&maps[1], p->k, dk, sk, boxk);
  if (rc) return rc;
  const int64_t sv[4] = {1, D, p->v_tok_stride, p->v_batch_stride};
  rc = make_tmap_4d(&maps[2], p->v, dk, sv, boxk);
  if (rc) return rc;
  uint8_t* ws = static_cast<uint8_t*>(p->workspace);
  RangeTileArgs g;
  g.a = a;
  g.tpt = l.tpt;
  g.nqp = l.nqp;
  g.entries = l.entries;
  g.streams = l.streams;
  // streams side by side: as many as keep their K and V in about 64 MB of the L2
  g.stream_group = (int)std::min<int64_t>(l.streams, std::max<int64_t>(1, (64 << 20) / (p->kv_len * D * 4)));
  g.splits = l.splits;
  g.units = (int)l.units;
  g.pairs = reinterpret_cast<const RangePair*>(ws);
  g.order = reinterpret_cast<const int*>(ws + l.order_off);
  g.counter = reinterpret_cast<int*>(ws + l.counter_off);
  g.o_part = reinterpret_cast<float*>(ws + l.part_off);
  g.ml_part = reinterpret_cast<float2*>(ws + l.ml_off);
  g.part_rows = l.part_rows;
  g.err = err;
  return D == 64 ? range_dispatch<64>(a, &g, maps, 0, st) : range_dispatch<128>(a, &g, maps, 0, st);
}

}  // namespace wanb200
