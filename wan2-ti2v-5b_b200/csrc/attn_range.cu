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

#include "common.cuh"
#include "internal.h"

namespace wanb200 {

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

// Unnormalised results of the key splits: slot i holds one split's [slot_rows][D] outputs and [slot_rows]
// (maximum in log2 units, sum).  Of the few-rows kernel: the splits of row group x (slot_rows rows of one
// batch element and key head) are the slots first[x].x + k * first[x].z for k < first[x].y, merged by
// range_combine_kernel.  Of the tiles: slots x, x + groups, ... of `splits`, merged by range_join_kernel;
// a split that saw no key tile has sum -1 and no output.
struct RangeParts {
  float* o;
  float2* ml;
  int4* first;  // few-rows kernel only
  int slot_rows, groups, splits;
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

// A table's bias, such that a finite one stays finite in log2 units: times log2(e) the type's lowest value
// would become -inf, and a row whose keys all have it 0 / 0 instead of equal weights.  Infinities and NaN
// stay as they are.  2.3e38 log2(e) = 3.32e38 < 2^128.
__device__ __forceinline__ float table_bias(float b) {
  return fabsf(b) < INFINITY ? fminf(fmaxf(b, -2.3e38f), 2.3e38f) : b;
}

// The cap's two forms.  cap2 - 2 cap2 / (1 + 2^x) is off by up to 3e-7 of the cap whatever the score: 1e-4
// log2 units at a cap of 256, a twentieth of a bf16 weight's half step, but 0.2 at 1e6, where it is all of
// a small score.  The other: where |x| = |score| / cap <= 0.6, tanh x = x P(x^2), P fitted to 5.9e-7 (least
// maximum error of an odd polynomial of degree 7 on [0, 0.6]), within 9e-6 of the score itself.
// Caps above 256 take the form that fits each score (kCapLarge).  For the others one form a tile is enough
// and faster: picking costs 20% where scores pass 0.6 of the cap (4900 rows, 16 heads on 4, 82 -> 98 us)
// and, by its registers, 3% where none does (70 -> 72), so the two are kernels of their own.
enum RangeCap : int { kCapNone = 0, kCapSmall = 1, kCapLarge = 2 };
constexpr float RA_CAP_SMALL = 256.f;
constexpr float RA_TANH_MAX = 0.6f;
constexpr float RA_TANH0 = 0.999991018f, RA_TANH1 = -0.332989737f, RA_TANH2 = 0.129745518f, RA_TANH3 = -0.0396112428f;

template <int CAP>
__device__ __forceinline__ float capped_log2(const RangeArgs& a, float s) {
  const float t = s * a.sl2, y = a.cap2 - 2.f * a.cap2 * rcp_approx(1.f + ex2_approx(t));
  if constexpr (CAP == kCapSmall) return y;
  const float x = t * (0.5f / RA_LOG2E), x2 = x * x;
  const float near0 = a.cap2 * (x * fmaf(x2, fmaf(x2, fmaf(x2, RA_TANH3, RA_TANH2), RA_TANH1), RA_TANH0));
  return fabsf(x) <= RA_TANH_MAX ? near0 : y;
}

// 2^t-units score of one (row, key) from its raw product, for the forms that take keys one by one.
template <int CAP, int BIAS>
__device__ __forceinline__ float score_log2(const RangeArgs& a, float s, int h, int dist) {
  float t;
  if constexpr (CAP != kCapNone)
    t = capped_log2<CAP>(a, s);
  else
    t = s * a.sl2;
  if constexpr (BIAS == kBiasSlopes) t = fmaf(-RA_LOG2E * __ldg(a.slopes + h), fabsf((float)dist), t);
  if constexpr (BIAS == kBiasTable)
    t = fmaf(RA_LOG2E, table_bias(__ldg(a.table + (int64_t)h * (2 * a.reach + 1) + min(max(dist, -a.reach), a.reach) + a.reach)), t);
  return t;
}

// ================================================================== few rows: one pass over K and V
// Several blocks per (key head, batch element) take tiles of 64 keys in turn: one warp feeds a ring of
// K and V tiles by TMA, four warps take 16 keys of each tile and keep their own running maximum, sum
// and output, merged at the end over the block's shared memory, and over the blocks by
// range_combine_kernel.  The batch elements' key counts differ, so every block reads them all and
// the blocks are dealt out in equal shares of keys.  (With cp.async or plain loads by the warps
// themselves the reads stopped at 4.1 TB/s whatever the depth of the ring.)  The operands of mma.sync
// m16n8k16 are transposed: S^T (16 keys x 8 rows) = K Q^T and O^T (16 channels x 8 rows) += V^T P^T, so
// that up to 8 rows cost one MMA column tile and nothing of it is wasted.  A dot product does not
// care about the order of its channels: a lane's 16 bytes of K are taken as the operand of two K
// steps, q permuted alike, and the output channels come out permuted as the pieces of V lie.  The
// tensor work is far below the bandwidth bound, so the warp-level MMA is enough; what counts is few
// instructions for each 16 keys (about 200; with rows as the MMA's 16-row side it was 565).
constexpr int RD_WARPS = 4, RD_KEYS = 16, RD_TILE = RD_WARPS * RD_KEYS;
constexpr int RD_THREADS = (RD_WARPS + 1) * 32;
constexpr int RD_SHARE = 2;   // key tiles of a block at least
constexpr int RD_BLOCKS = 3, RD_BLOCKS_TWO = 2;  // blocks an SM holds: by shared memory; with 9 to 16 rows by registers

template <int D>
struct RangeDecodeCfg {
  static constexpr int HALF = RD_TILE * 128;               // 64 channels of a tile: 128-byte swizzled rows
  static constexpr int STAGE = 2 * (D / 64) * HALF;        // K, then V
  static constexpr int STAGES = D == 128 ? 2 : 4;
  static constexpr int RING = STAGES * STAGE;              // 64 KB
  static constexpr int SMEM = RING + 1024;
};

__device__ __forceinline__ int decode_key_tiles(const RangeArgs& a, int b) {
  int from = INT32_MAX, to = 0;
  for (int t = 0; t < a.q_len; ++t) {
    int lo, hi;
    row_range(a, b, t, lo, hi);
    if (lo < hi) from = min(from, lo), to = max(to, hi);
  }
  return from < to ? (to - from + RD_TILE - 1) / RD_TILE : 0;
}

template <int D, bool TWO, int CAP, int BIAS>  // TWO: 9 to 16 rows, two column tiles
__global__ void __launch_bounds__(RD_THREADS, TWO ? RD_BLOCKS_TWO : RD_BLOCKS)
    range_decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                        const __grid_constant__ RangeArgs a, const __grid_constant__ RangeParts out, const int slots, int* err) {
  using C = RangeDecodeCfg<D>;
  constexpr int KC = D / 32, VC = D / 64;         // 16-byte pieces per K row, per V row of a lane
  constexpr int NR = TWO ? 2 : 1, ROWS = 8 * NR;  // a lane holds rows 8 x + 2 q4 + y (x < NR, y < 2)
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);  // the ring, after it the warps' outputs
  const uint32_t sbase = smem_u32(smem);
  float(*o_sh)[ROWS][D + 4] = reinterpret_cast<float(*)[ROWS][D + 4]>(smem);
  static_assert(RD_WARPS * ROWS * (D + 4) * 4 <= C::RING, "the outputs reuse the ring");
  __shared__ float2 ml_sh[RD_WARPS][ROWS];
  __shared__ uint64_t bars[2 * C::STAGES];
  __shared__ int abort_word;
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * C::STAGES;
  volatile int* abort_flag = &abort_word;
  pdl_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g4 = lane >> 2, q4 = lane & 3;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(full0 + 8 * i, 1);
      mbar_init(empty0 + 8 * i, RD_WARPS);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  const int rows = a.q_len * a.group;
  int b = (int)blockIdx.x / a.kv_heads, kh = (int)blockIdx.x % a.kv_heads, csize = 1, crank = 0;
  if (slots > 0) {  // else one block for each (key head, batch element)
    __shared__ int deal[4];  // batch element, its first block, its blocks of each head; -1 = none left
    if (threadIdx.x < 32) {
      // tiles of every batch element (all heads alike), then the share of one block
      const int mine = lane < a.batch ? decode_key_tiles(a, lane) : 0;
      int total = mine;
      for (int i = lane + 32; i < a.batch; i += 32) total += decode_key_tiles(a, i);
      total = __reduce_add_sync(0xffffffffu, total);
      const int64_t all = (int64_t)total * a.kv_heads;
      const int each = (int)max((all + slots - 1) / slots, (int64_t)RD_SHARE);
      int before = 0;
      if (lane == 0) deal[0] = -1;
      __syncwarp();
      for (int i0 = 0; i0 < a.batch; i0 += 32) {
        const int i = i0 + lane;
        const int n = i < a.batch ? max(1, ((i0 ? decode_key_tiles(a, i) : mine) + each - 1) / each) : 0;
        int sum = n;
#pragma unroll
        for (int w = 1; w < 32; w *= 2) {
          const int v = __shfl_up_sync(0xffffffffu, sum, w);
          if (lane >= w) sum += v;
        }
        const int first = (before + sum - n) * a.kv_heads;
        if (n > 0 && (int)blockIdx.x >= first && (int)blockIdx.x < first + n * a.kv_heads)
          deal[0] = i, deal[1] = first, deal[2] = n;
        before += __shfl_sync(0xffffffffu, sum, 31);
      }
    }
    __syncthreads();
    b = deal[0];
    if (b < 0) return;  // more blocks were launched than there are shares
    csize = deal[2];
    const int x = (int)blockIdx.x - deal[1];
    kh = x % a.kv_heads;
    crank = x / a.kv_heads;
    if (crank == 0 && threadIdx.x == 0) out.first[b * a.kv_heads + kh] = make_int4((int)blockIdx.x, csize, a.kv_heads, 0);
  } else {
    __syncthreads();  // the barriers are set up
  }

  // the rows' ranges: each lane's own, and over all rows what any and what all of them see
  int lo[NR][2], hi[NR][2], pos[NR][2], head[NR][2];
  int all_lo = 0, all_hi = INT32_MAX, any_lo = INT32_MAX, any_hi = 0;
#pragma unroll
  for (int x = 0; x < NR; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int r = 8 * x + 2 * q4 + y;
      lo[x][y] = hi[x][y] = pos[x][y] = head[x][y] = 0;
      if (r < rows) {
        const int tok = r / a.group;
        row_range(a, b, tok, lo[x][y], hi[x][y]);
        pos[x][y] = BIAS == kBiasNone ? 0 : row_pos(a, b, tok);
        head[x][y] = kh * a.group + r % a.group;
        if (lo[x][y] < hi[x][y]) {
          any_lo = min(any_lo, lo[x][y]);
          any_hi = max(any_hi, hi[x][y]);
        }
        all_lo = max(all_lo, lo[x][y]);
        all_hi = min(all_hi, hi[x][y]);
      }
    }
  all_lo = __reduce_max_sync(0xffffffffu, all_lo);
  all_hi = __reduce_min_sync(0xffffffffu, all_hi);
  any_lo = __reduce_min_sync(0xffffffffu, any_lo);
  any_hi = __reduce_max_sync(0xffffffffu, any_hi);

  const int tiles = any_lo < any_hi ? (any_hi - any_lo + RD_TILE - 1) / RD_TILE : 0;
  if (warp == RD_WARPS) {  // the whole warp walks the loop: see elect_one
    int n = 0;
    bool ok = true;
    for (int t = crank; t < tiles; t += csize, ++n) {
      const int stage = n % C::STAGES, key0 = any_lo + t * RD_TILE;
      ok = mbar_wait_warp(empty0 + 8 * stage, ((n / C::STAGES) & 1) ^ 1, abort_flag, err, kErrTimeoutAttnProducer);
      if (!ok) break;
      if (elect_one()) {
        const uint32_t dst = sbase + stage * C::STAGE;
        mbar_expect_tx(full0 + 8 * stage, C::STAGE);
        for (int h = 0; h < VC; ++h) {
          tma_load_4d(dst + h * C::HALF, &tmK, full0 + 8 * stage, 64 * h, kh, key0, b);
          tma_load_4d(dst + (VC + h) * C::HALF, &tmV, full0 + 8 * stage, 64 * h, kh, key0, b);
        }
      }
      __syncwarp();
    }
    if (!ok)  // let every load in flight land before the block's shared memory goes away
      for (int i = max(0, n - C::STAGES); i < n; ++i) mbar_drain(full0 + 8 * (i % C::STAGES), (i / C::STAGES) & 1, err);
    __syncthreads();
    __syncthreads();
    return;
  }

  uint32_t qb[NR][2 * KC][2];  // B operand of S^T: row 8 x + g4, [K step][the two k pairs]
#pragma unroll
  for (int x = 0; x < NR; ++x) {
    const int r = 8 * x + g4;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      uint4 u = make_uint4(0u, 0u, 0u, 0u);
      if (r < rows)
        u = __ldg(reinterpret_cast<const uint4*>(a.q + b * a.q_batch + (int64_t)(r / a.group) * a.q_tok +
                                                 (int64_t)(kh * a.group + r % a.group) * D + 32 * c + 8 * q4));
      qb[x][2 * c][0] = u.x;
      qb[x][2 * c][1] = u.y;
      qb[x][2 * c + 1][0] = u.z;
      qb[x][2 * c + 1][1] = u.w;
    }
  }
  // o[x][4 c + p][2 e + y]: channel 64 c + 8 g4 + 2 p + e of row 8 x + 2 q4 + y
  float o[NR][4 * VC][4], m[NR][2], l[NR][2];
#pragma unroll
  for (int x = 0; x < NR; ++x) {
#pragma unroll
    for (int n = 0; n < 4 * VC; ++n) o[x][n][0] = o[x][n][1] = o[x][n][2] = o[x][n][3] = 0.f;
    m[x][0] = m[x][1] = -INFINITY;
    l[x][0] = l[x][1] = 0.f;
  }

  // 16 bytes of this lane: K row g4 (+ 8), channels 32 c + 8 q4; V row 2 q4 + t % 2 (+ 8), channels 64 c + 8 g4
  const uint32_t krow = sbase + (warp * RD_KEYS + g4) * 128, vrow = sbase + VC * C::HALF + (warp * RD_KEYS + 2 * q4) * 128;
  auto k_piece = [&](int stage, int t, int c) {
    return ld_shared16(krow + stage * C::STAGE + (c >> 1) * C::HALF + t * 1024 + ((((c & 1) * 4 + q4) ^ g4) << 4));
  };
  auto v_piece = [&](int stage, int t, int c) {
    return ld_shared16(vrow + stage * C::STAGE + c * C::HALF + (t >> 1) * 1024 + (t & 1) * 128 + ((g4 ^ (2 * q4 + (t & 1))) << 4));
  };
  int n = 0;
  for (int tile = crank; tile < tiles; tile += csize, ++n) {
    const int stage = n % C::STAGES, key0 = any_lo + tile * RD_TILE + warp * RD_KEYS;
    if (!mbar_wait_warp(full0 + 8 * stage, (n / C::STAGES) & 1, abort_flag, err, kErrTimeoutAttnSoftmax)) break;
    float s[NR][2][4];  // two chains of products, half as long; keys g4 + 8 (e / 2), rows 2 q4 + e % 2
#pragma unroll
    for (int x = 0; x < NR; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[x][0][e] = s[x][1][e] = 0.f;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const uint4 k0 = k_piece(stage, 0, c), k1 = k_piece(stage, 1, c);
#pragma unroll
      for (int x = 0; x < NR; ++x) {
        mma_16816(s[x][0], k0.x, k1.x, k0.y, k1.y, qb[x][2 * c][0], qb[x][2 * c][1]);
        mma_16816(s[x][1], k0.z, k1.z, k0.w, k1.w, qb[x][2 * c + 1][0], qb[x][2 * c + 1][1]);
      }
    }
    const bool full = key0 >= all_lo && key0 + RD_KEYS <= all_hi;  // every row sees every key of this block
    float p[NR][4];
    bool raise = false;
#pragma unroll
    for (int x = 0; x < NR; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = key0 + g4 + 8 * (e >> 1), y = e & 1;
        const float v = score_log2<CAP, BIAS>(a, s[x][0][e] + s[x][1][e], head[x][y], j - pos[x][y]);
        p[x][e] = full || (j >= lo[x][y] && j < hi[x][y]) ? v : -INFINITY;
        raise |= p[x][e] > m[x][y] + RA_RESCALE;
      }
    // the running maximum moves only when a score passes it by 2^8 (exact all the same)
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int x = 0; x < NR; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          float mx = fmaxf(p[x][y], p[x][2 + y]);
#pragma unroll
          for (int w = 4; w < 32; w *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
          const float mn = mx > m[x][y] + RA_RESCALE ? mx : m[x][y];
          const float alpha = mn == m[x][y] ? 1.f : ex2_approx(m[x][y] - mn);
          m[x][y] = mn;
          l[x][y] *= alpha;
#pragma unroll
          for (int n = 0; n < 4 * VC; ++n) o[x][n][y] *= alpha, o[x][n][2 + y] *= alpha;
        }
    }
    uint32_t pb[NR][2];
#pragma unroll
    for (int x = 0; x < NR; ++x) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float mm = m[x][e & 1];
        p[x][e] = ex2_approx(p[x][e] - (mm == -INFINITY ? 0.f : mm));
        l[x][e & 1] += p[x][e];
      }
      // weights in bf16, the MMA's operand type; the sum keeps fp32
      pb[x][0] = transpose_8x8(pack_bf16x2(p[x][0], p[x][1]));
      pb[x][1] = transpose_8x8(pack_bf16x2(p[x][2], p[x][3]));
    }
    uint4 vr[4][VC];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int c = 0; c < VC; ++c) vr[t][c] = v_piece(stage, t, c);
    __syncwarp();
    if (lane == 0) mbar_arrive(empty0 + 8 * stage);  // K and V of this stage are in registers
    if (!full) {
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
          const int j = key0 + kk, from = (kk & 7) * 4 + q4;
#pragma unroll
          for (int x = 0; x < NR; ++x)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const float pa = __shfl_sync(0xffffffffu, p[x][y], from), pc = __shfl_sync(0xffffffffu, p[x][2 + y], from);
              if (j >= lo[x][y] && j < hi[x][y]) {
                const __nv_bfloat16* row = a.v + b * a.v_batch + j * a.v_tok + (int64_t)kh * D + 8 * g4;
#pragma unroll
                for (int n = 0; n < 4 * VC; ++n)
#pragma unroll
                  for (int e = 0; e < 2; ++e) {
                    const __nv_bfloat16 vv = row[64 * (n >> 2) + 2 * (n & 3) + e];
                    if (nonfinite_bf16(vv)) o[x][n][2 * e + y] += (kk < 8 ? pa : pc) * __bfloat162float(vv);
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
      for (int i = 0; i < 4; ++i) {
        const uint32_t a0 = __byte_perm(w0[i], w1[i], 0x5410u), a1 = __byte_perm(w0[i], w1[i], 0x7632u);
        const uint32_t a2 = __byte_perm(w2[i], w3[i], 0x5410u), a3 = __byte_perm(w2[i], w3[i], 0x7632u);
#pragma unroll
        for (int x = 0; x < NR; ++x) mma_16816(o[x][4 * c + i], a0, a1, a2, a3, pb[x][0], pb[x][1]);
      }
    }
  }
  __syncthreads();  // the ring becomes the merge buffer
#pragma unroll
  for (int x = 0; x < NR; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int r = 8 * x + 2 * q4 + y;
#pragma unroll
      for (int w = 4; w < 32; w *= 2) l[x][y] += __shfl_xor_sync(0xffffffffu, l[x][y], w);
      if (g4 == 0) ml_sh[warp][r] = make_float2(m[x][y], l[x][y]);
#pragma unroll
      for (int n = 0; n < 4 * VC; ++n)
        *reinterpret_cast<float2*>(&o_sh[warp][r][64 * (n >> 2) + 8 * g4 + 2 * (n & 3)]) = make_float2(o[x][n][y], o[x][n][2 + y]);
    }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * (D / 4); i += RD_WARPS * 32) {  // four channels a thread
    const int r = i / (D / 4), d = i % (D / 4) * 4, tok = r / a.group;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < RD_WARPS; ++w) mm = fmaxf(mm, ml_sh[w][r].x);
    float ll = 0.f;
    float4 oo = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < RD_WARPS; ++w) {
      const float2 ml = ml_sh[w][r];
      const float4 x = *reinterpret_cast<const float4*>(&o_sh[w][r][d]);
      // a warp that saw nothing, or only scores of minus infinity: its sums are 0, or NaN to be kept
      const float f = ml.x == -INFINITY ? 1.f : ex2_approx(ml.x - mm);
      ll = fmaf(f, ml.y, ll);
      oo.x = fmaf(f, x.x, oo.x), oo.y = fmaf(f, x.y, oo.y), oo.z = fmaf(f, x.z, oo.z), oo.w = fmaf(f, x.w, oo.w);
    }
    if (csize > 1) {
      const int64_t prow = (int64_t)blockIdx.x * rows + r;
      *reinterpret_cast<float4*>(out.o + prow * D + d) = oo;
      if (d == 0) out.ml[prow] = make_float2(mm, ll);
    } else {
      int rlo, rhi;
      row_range(a, b, tok, rlo, rhi);
      const float inv = 1.f / ll;
      *reinterpret_cast<uint2*>(a.o + b * a.o_batch + (int64_t)tok * a.o_tok + (int64_t)(kh * a.group + r % a.group) * D + d) =
          rlo < rhi ? make_uint2(pack_bf16x2(oo.x * inv, oo.y * inv), pack_bf16x2(oo.z * inv, oo.w * inv)) : make_uint2(0u, 0u);
    }
  }
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
constexpr int RT_SORT_MAX = 1024;  // pairs that the plan kernel sorts
constexpr int RT_SPLITS = 32;  // of a tile pair's keys at most: a lane each in range_join_kernel
constexpr int RT_REACH_MAX = 8192;  // of a bias table (it is copied with padded ends at every call)

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
  RangeParts parts;
  const float* padded;  // the bias table in log2 units, its ends repeated RT_N times
  float cap_scale;      // softmax_scale / softcap
  int* err;
};

// Entry RT_N + reach + d of a padded row is table[clamp(d, -reach, reach)] log2(e), -reach - RT_N <= d < reach + RT_N.
__host__ __device__ constexpr int range_padded(int reach) { return 2 * (reach + RT_N); }

struct PlanArgs {
  RangeArgs a;
  int tpt, nqp, entries;
  RangePair* pairs;
  int* order;
  int* counter;
  float* padded;
};

// Block 0: the key ranges of every tile pair (one warp each) and the pairs from the most key tiles to
// the fewest (each counts those in front of it, up to RT_SORT_MAX pairs; more are spread over the
// blocks and taken from the last to the first).  The other blocks: the padded bias table.
__global__ void __launch_bounds__(1024) range_plan_kernel(const PlanArgs p) {
  __shared__ __align__(16) int tiles_of[RT_SORT_MAX];
  pdl_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool sort = p.entries <= RT_SORT_MAX;
  if (p.padded) {
    const int row = range_padded(p.a.reach), n = p.a.kv_heads * p.a.group * row;
    for (int i = blockIdx.x * 1024 + threadIdx.x; i < n; i += gridDim.x * 1024) {
      const int h = i / row, d = min(max(i - h * row - RT_N - p.a.reach, -p.a.reach), p.a.reach);
      p.padded[i] = RA_LOG2E * table_bias(__ldg(p.a.table + (int64_t)h * (2 * p.a.reach + 1) + d + p.a.reach));
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.counter = 0;
  if (sort && blockIdx.x != 0) return;
  const int warps = sort ? 32 : gridDim.x * 32;
  for (int e = (sort ? 0 : blockIdx.x * 32) + warp; e < p.entries; e += warps) {
    const int b = e / p.nqp, tok0 = e % p.nqp * 2 * p.tpt;
    // a tile's rows four a lane, all loads first; lanes behind the last row repeat it
    int lo[2][4], hi[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = min(p.tpt, p.a.q_len - (tok0 + t * p.tpt));
        lo[t][q] = hi[t][q] = 0;
        if (n > 0) row_range(p.a, b, tok0 + t * p.tpt + min(lane + 32 * q, n - 1), lo[t][q], hi[t][q]);
      }
    int any_lo[2], any_hi[2], all_lo[2], all_hi[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      any_lo[t] = INT32_MAX, any_hi[t] = 0, all_lo[t] = 0, all_hi[t] = INT32_MAX;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const bool some = lo[t][q] < hi[t][q];
        any_lo[t] = some ? min(any_lo[t], lo[t][q]) : any_lo[t];
        any_hi[t] = some ? max(any_hi[t], hi[t][q]) : any_hi[t];
        all_lo[t] = max(all_lo[t], lo[t][q]);
        all_hi[t] = min(all_hi[t], hi[t][q]);
      }
    }
    RangePair r;
    int tiles = 0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      r.any_lo[t] = __reduce_min_sync(0xffffffffu, any_lo[t]);
      r.any_hi[t] = __reduce_max_sync(0xffffffffu, any_hi[t]);
      r.all_lo[t] = __reduce_max_sync(0xffffffffu, all_lo[t]);
      r.all_hi[t] = __reduce_min_sync(0xffffffffu, all_hi[t]);
      if (r.any_lo[t] >= r.any_hi[t]) r.any_lo[t] = r.any_hi[t] = 0;
      tiles += (r.any_hi[t] + RT_N - 1) / RT_N - r.any_lo[t] / RT_N;
    }
    if (lane == 0) {
      p.pairs[e] = r;
      if (sort)
        tiles_of[e] = tiles;
      else
        p.order[e] = p.entries - 1 - e;
    }
  }
  if (!sort) return;
  if (threadIdx.x < 4 && p.entries + threadIdx.x < RT_SORT_MAX) tiles_of[p.entries + threadIdx.x] = -1;  // behind the last
  __syncthreads();
  const int e = threadIdx.x;  // entries <= 1024: one each
  if (e < p.entries) {
    const int mine = tiles_of[e];
    int place = 0;
#pragma unroll 4
    for (int i = 0; i < p.entries; i += 4) {
      const int4 v = *reinterpret_cast<const int4*>(tiles_of + i);
      place += (v.x > mine || (v.x == mine && i < e)) + (v.y > mine || (v.y == mine && i + 1 < e)) +
               (v.z > mine || (v.z == mine && i + 2 < e)) + (v.w > mine || (v.w == mine && i + 3 < e));
    }
    p.order[place] = e;
  }
}

struct RangeUnit {
  int tok0, b, mb, kh, split, k0, k1;  // key tiles [k0, k1) of this split
  int a[2], z[2];                      // tile t: key tiles [a, z)
  int full_lo[2], full_hi[2];          // keys that every row of the tile sees
};

// The plan (order, pairs, padded) is written while this kernel already runs, so it is read with plain loads:
// the read-only path is for memory that stays as it is over the whole kernel, and its loads may be moved up
// past the wait for the plan.
__device__ __forceinline__ RangeUnit range_unit(const RangeTileArgs& g, int u) {
  RangeUnit r;
  const int per_group = g.stream_group * g.entries * g.splits;
  const int grp = u / per_group, first = grp * g.stream_group, size = min(g.stream_group, g.streams - first);
  int x = u - grp * per_group;
  r.split = x % g.splits;
  x /= g.splits;
  const int stream = first + x % size, e = g.order[x / size];
  r.kh = stream % g.a.kv_heads;
  r.mb = e / g.nqp;
  r.b = g.a.range_batch ? r.mb : stream / g.a.kv_heads;
  r.tok0 = e % g.nqp * 2 * g.tpt;
  const int4* pp = reinterpret_cast<const int4*>(g.pairs + e);
  const int4 any = pp[0], all = pp[1];
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
template <int D, int CAP, int BIAS>
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

template <int D, int CAP, int BIAS>
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
  pdl_wait();  // the plan; its launch ran beside the set-up above

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
      // this tile's bounds as scalars (indexing the unit by t would put it into local memory)
      const int a_t = t ? w.a[1] : w.a[0], z_t = t ? w.z[1] : w.z[0];
      const int flo_t = t ? w.full_lo[1] : w.full_lo[0], fhi_t = t ? w.full_hi[1] : w.full_hi[0];
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
      if constexpr (BIAS == kBiasTable) trow = g.padded + (live ? (int64_t)head * range_padded(a.reach) : 0) + a.reach + RT_N;
      float m_used = -INFINITY, l_run = 0.f;
      bool any_tile = false;
      for (int j = w.k0; j < w.k1; ++j) {
        if (!unit_loads(w, j)) continue;
        const int slot = (gk + 1) % RING;
        const bool partial = unit_partial(w, j);
        gk += 2;
        if (j < a_t || j >= z_t) {
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
        const bool masked = kbase < flo_t || kbase + RT_N > fhi_t;
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
        float mx = -INFINITY;
        if constexpr (CAP) {
          float hi8[4], lo8[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) hi8[c] = fmaxf(s[2 * c], s[2 * c + 1]), lo8[c] = fminf(s[2 * c], s[2 * c + 1]);
#pragma unroll
          for (int q = 1; q < RT_N / 8; ++q)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              hi8[c] = fmax3(hi8[c], s[8 * q + 2 * c], s[8 * q + 2 * c + 1]);
              lo8[c] = fmin3(lo8[c], s[8 * q + 2 * c], s[8 * q + 2 * c + 1]);
            }
          const float top_hi = fmax3(hi8[0], hi8[1], fmaxf(hi8[2], hi8[3]));
          // rows that are not stored do not hold the others back from the short form
          const float top = live ? fmaxf(top_hi, -fmin3(lo8[0], lo8[1], fminf(lo8[2], lo8[3]))) : 0.f;
          if (__all_sync(0xffffffffu, top * g.cap_scale <= RA_TANH_MAX)) {
            // the polynomial alone: no MUFU, which bounds the general form
            const float2 kx = make_float2(g.cap_scale, g.cap_scale);
            const float c0 = RA_TANH0 * a.cap2, c1 = RA_TANH1 * a.cap2, c2 = RA_TANH2 * a.cap2, c3 = RA_TANH3 * a.cap2;
            const float2 p0 = make_float2(c0, c0), p1 = make_float2(c1, c1), p2 = make_float2(c2, c2), p3 = make_float2(c3, c3);
#pragma unroll
            for (int k = 0; k < RT_N; k += 2) {
              const float2 x = __fmul2_rn(make_float2(s[k], s[k + 1]), kx);
              const float2 x2 = __fmul2_rn(x, x);
              const float2 y = __fmul2_rn(x, __ffma2_rn(x2, __ffma2_rn(x2, __ffma2_rn(x2, p3, p2), p1), p0));
              s[k] = y.x;
              s[k + 1] = y.y;
            }
            const float x = top_hi * g.cap_scale, x2 = x * x;
            mx = x * fmaf(x2, fmaf(x2, fmaf(x2, c3, c2), c1), c0);
          } else if constexpr (CAP == kCapLarge) {
#pragma unroll
            for (int k = 0; k < RT_N; ++k) s[k] = capped_log2<CAP>(a, s[k]);
            mx = capped_log2<CAP>(a, top_hi);
          } else {
            // cap2 tanh = cap2 - 2 cap2 / (1 + 2^x); four reciprocals from one (MUFU bounds this form)
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
            mx = fmaf(n2c, rcp_approx(1.f + ex2_approx(min30(top_hi * a.sl2))), a.cap2);
          }
        }
        const float sl2 = CAP ? 1.f : a.sl2;
        if constexpr (BIAS == kBiasSlopes) {
          const float d0 = (float)(kbase - pos);
#pragma unroll
          for (int k = 0; k < RT_N; ++k) s[k] = fmaf(-slope2, fabsf(d0 + (float)k), CAP ? s[k] : s[k] * sl2);
        }
        if constexpr (BIAS == kBiasTable) {  // the padded table: one clamp a row, fixed offsets for its keys
          const float* tp = trow + min(max(kbase - pos, -a.reach - RT_N), a.reach);
#pragma unroll
          for (int k = 0; k < RT_N; ++k) s[k] = CAP ? s[k] + tp[k] : fmaf(s[k], sl2, tp[k]);
        }
        const float mul = BIAS == kBiasNone && !CAP ? a.sl2 : 1.f;  // what is left to apply in the exponent
        if (masked) {
#pragma unroll
          for (int k = 0; k < RT_N; ++k)
            if (!((mask[k >> 5] >> (k & 31)) & 1u)) s[k] = -INFINITY;
        }
        // the capped maximum of a fully seen tile follows from that of the raw scores (tanh grows with
        // its argument); m only has to be near the true maximum, so the two need not agree to the bit
        if (!CAP || BIAS != kBiasNone || masked) {
          float m8[8];
#pragma unroll
          for (int c = 0; c < 8; ++c) m8[c] = fmaxf(s[2 * c], s[2 * c + 1]);
#pragma unroll
          for (int q = 1; q < RT_N / 16; ++q)
#pragma unroll
            for (int c = 0; c < 8; ++c) m8[c] = fmax3(m8[c], s[16 * q + 2 * c], s[16 * q + 2 * c + 1]);
          mx = fmax3(fmax3(m8[0], m8[1], m8[2]), fmax3(m8[3], m8[4], m8[5]), fmaxf(m8[6], m8[7]));
        }
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
        const int64_t prow = ((int64_t)w.split * g.parts.groups + (int64_t)w.b * a.kv_heads + w.kh) * g.parts.slot_rows +
                             (int64_t)tok * a.group + rhead;
        float4* dst = reinterpret_cast<float4*>(g.parts.o + prow * D);
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
        if (live) g.parts.ml[prow] = make_float2(any_tile ? m_used : -INFINITY, any_tile ? l_run : -1.f);
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

// Merge of the few-rows kernel's splits: one block per packed row, its warps taking the splits in turn
// (few rows with up to hundreds of splits).
constexpr int RC_WARPS = 4;

template <int D>
__global__ void __launch_bounds__(RC_WARPS * 32) range_combine_kernel(const RangeArgs a, const RangeParts in) {
  constexpr int E = D / 32;
  __shared__ float l_sh[RC_WARPS], o_sh[RC_WARPS][D];
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int x = (int)(blockIdx.x / in.slot_rows), r = (int)(blockIdx.x - (int64_t)x * in.slot_rows);
  const int hg = r % a.group, tok = r / a.group, kh = x % a.kv_heads, b = x / a.kv_heads;
  const int4 f4 = in.first[x];
  if (f4.y == 1) return;  // its one block wrote the output
  int lo, hi;
  row_range(a, b, tok, lo, hi);
  const int64_t row0 = (int64_t)f4.x * in.slot_rows + r, next = (int64_t)f4.z * in.slot_rows;
  float m = -INFINITY;
  for (int s = lane; s < f4.y; s += 32) m = fmaxf(m, in.ml[row0 + s * next].x);
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float l = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll 4
  for (int s = warp; s < f4.y; s += RC_WARPS) {
    const float2 ml = in.ml[row0 + s * next];
    const float f = ml.x == -INFINITY ? 1.f : ex2_approx(ml.x - m);
    l = fmaf(f, ml.y, l);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(f, in.o[(row0 + s * next) * D + lane * E + e], o[e]);
  }
  if (lane == 0) l_sh[warp] = l;
#pragma unroll
  for (int e = 0; e < E; ++e) o_sh[warp][lane * E + e] = o[e];
  __syncthreads();
  if (threadIdx.x < D) {
    float ll = 0.f, oo = 0.f;
#pragma unroll
    for (int w = 0; w < RC_WARPS; ++w) ll += l_sh[w], oo += o_sh[w][threadIdx.x];
    a.o[b * a.o_batch + (int64_t)tok * a.o_tok + (int64_t)(kh * a.group + hg) * D + threadIdx.x] =
        __float2bfloat16(lo < hi ? oo / ll : 0.f);
  }
}

// Merge of the tiles' splits (at most RT_SPLITS): many rows with few splits, so one warp a row, eight
// rows a block, the loads of four splits in flight.  With one block a row 15,000 rows of 2 splits took
// 12 us longer (the whole call 36 against 24).
constexpr int RJ_WARPS = 8;

template <int D>
__global__ void __launch_bounds__(RJ_WARPS * 32) range_join_kernel(const RangeArgs a, const RangeParts in) {
  constexpr int E = D / 32;
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t rows = (int64_t)in.groups * in.slot_rows, row = (int64_t)blockIdx.x * RJ_WARPS + (threadIdx.x >> 5);
  if (row >= rows) return;  // warp-uniform
  const int x = (int)(row / in.slot_rows), r = (int)(row - (int64_t)x * in.slot_rows);
  const int hg = r % a.group, tok = r / a.group, kh = x % a.kv_heads, b = x / a.kv_heads;
  int lo, hi;
  row_range(a, b, tok, lo, hi);
  const float2 ml = lane < in.splits ? in.ml[row + lane * rows] : make_float2(-INFINITY, -1.f);
  const bool some = ml.y != -1.f;  // this lane's split saw a key tile of the row
  float m = ml.x;
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float f = !some ? 0.f : ml.x == -INFINITY ? 1.f : ex2_approx(ml.x - m);
  float l = some ? f * ml.y : 0.f, o[E];
#pragma unroll
  for (int w = 16; w; w >>= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
  const uint32_t has = __ballot_sync(0xffffffffu, some);
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll 4
  for (int s = 0; s < in.splits; ++s) {
    const float fs = __shfl_sync(0xffffffffu, f, s);
    const float* src = in.o + (row + s * rows) * D + lane * E;
    if ((has >> s) & 1u) {  // else nothing was written there
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 v = *reinterpret_cast<const float2*>(src + e);
        o[e] = fmaf(fs, v.x, o[e]);
        o[e + 1] = fmaf(fs, v.y, o[e + 1]);
      }
    }
  }
  const float inv = lo < hi ? 1.f / l : 0.f;
  uint32_t* dst = reinterpret_cast<uint32_t*>(a.o + b * a.o_batch + (int64_t)tok * a.o_tok + (int64_t)(kh * a.group + hg) * D) +
                  lane * (E / 2);
#pragma unroll
  for (int e = 0; e < E; e += 2) dst[e / 2] = lo < hi ? pack_bf16x2(o[e] * inv, o[e + 1] * inv) : 0u;
}

// ------------------------------------------------------------------ host launcher
// Packed rows up to which the few-rows kernel runs: two column tiles of 8 rows of its MMA.  Measured at
// 16 rows, few-rows kernel / tiles (us; batch x 8 key heads of 128, all keys seen): 1 x 1024 keys
// 11.7 / 13.4, 1 x 16384 26 / 29, 16 x 4096 55 / 64, 16 x 16384 165 / 217, and with lengths between a
// quarter of that and all of it 124 / 206.  Only many short caches go the other way (16 x 256: 18 / 14).
constexpr int RD_ROWS = 16;

struct RangeLayout {
  int tpt, nqp, entries, streams, splits;
  int64_t units, part_rows, order_off, counter_off, pad_off, part_off, ml_off, bytes;
};

static int64_t range_up(int64_t x) { return (x + 255) / 256 * 256; }

// The few-rows kernel's blocks: as many as the SMs hold at once, less half a block for each (key head,
// batch element), whose last share is half full on average.  More elements than blocks: one block each.
static int range_decode_slots(const wanb200_range_attn_params* p) {
  const bool two = p->q_len * (p->heads / p->kv_heads) > 8;
  const int64_t units = p->batch * p->kv_heads, slots = (int64_t)num_sms() * (two ? RD_BLOCKS_TWO : RD_BLOCKS);
  return units >= slots || p->kv_len <= RD_TILE * RD_SHARE ? 0 : (int)std::max(slots - units / 2, slots / 4);
}

static int64_t range_decode_blocks(const wanb200_range_attn_params* p) {  // an upper bound: the lengths are on the device
  const int64_t units = p->batch * p->kv_heads, slots = range_decode_slots(p);
  const int64_t most = (p->kv_len + RD_TILE * RD_SHARE - 1) / (RD_TILE * RD_SHARE);
  return slots ? std::min(slots + units, units * most) : units;
}

static RangeLayout range_layout(const wanb200_range_attn_params* p) {
  RangeLayout l = {};
  const int group = (int)(p->heads / p->kv_heads);
  l.part_rows = p->batch * p->heads * p->q_len;
  auto parts = [&](int64_t at, int64_t rows) {  // rows of all slots
    l.part_off = at;
    l.ml_off = at + range_up(rows * p->head_dim * 4);
    l.bytes = l.ml_off + range_up(rows * 8);
  };
  if (p->q_len * group <= RD_ROWS) {
    l.splits = 1;
    if (range_decode_slots(p)) {
      l.splits = 2;  // some element may have several blocks
      parts(range_up(p->batch * p->kv_heads * 16), range_decode_blocks(p) * p->q_len * group);
    }
    return l;
  }
  const bool per_batch = p->range_batch_stride > 0;
  l.tpt = RT_M / group;
  l.nqp = (int)((p->q_len + 2 * l.tpt - 1) / (2 * l.tpt));
  const int64_t entries = per_batch ? p->batch * l.nqp : l.nqp, streams = per_batch ? p->kv_heads : p->kv_heads * p->batch;
  if (entries > INT32_MAX / 64 || streams > INT32_MAX / 64) return l;
  l.entries = (int)entries;
  l.streams = (int)streams;
  // Split the keys when the units leave SMs idle: at least two key tiles a split.  Measured, causal order (us,
  // 1 split / as chosen): 24 units of up to 47 tiles 93 / 36, 40 of 20 45 / 28, 40 rows against 4 caches of up to
  // 8000 keys 108 / 40; with 5 tiles 21 / 22.5.  More splits than that, in two rounds of units: 96 units 28.6 as
  // chosen, 40 with 2 splits; 128 units of up to 32 tiles 70 and 67.
  const int64_t units = entries * streams, tiles = (p->kv_len + RT_N - 1) / RT_N;
  l.splits = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(num_sms() / units, tiles / 2), RT_SPLITS));
  l.units = units * l.splits;
  l.order_off = range_up(entries * (int64_t)sizeof(RangePair));
  l.counter_off = l.order_off + range_up(entries * 4);
  l.pad_off = l.counter_off + 256;
  parts(l.pad_off + (p->dist_bias ? range_up(p->heads * (int64_t)range_padded(p->reach) * 4) : 0),
        l.splits > 1 ? l.splits * l.part_rows : 0);
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
  if (!(p->softmax_scale >= 1e-12f && p->softmax_scale <= 1e12f))
    return set_error(WANB200_EINVAL, "range_attn: softmax_scale must lie in 1e-12 .. 1e12");
  if (p->softcap != 0.f && !(p->softcap >= 1e-6f && p->softcap <= 1e6f))
    return set_error(WANB200_EINVAL, "range_attn: softcap must be 0 (none) or in 1e-6 .. 1e6");
  if (p->slopes && p->dist_bias) return set_error(WANB200_EINVAL, "range_attn: slopes or dist_bias, not both");
  if (p->dist_bias && (p->reach < 0 || p->reach > RT_REACH_MAX))
    return set_error(WANB200_EINVAL, "range_attn: dist_bias needs 0 <= reach <= 8192");
  if (p->range_batch_stride < 0) return set_error(WANB200_EINVAL, "range_attn: negative range_batch_stride");
  return WANB200_OK;
}

int64_t range_attn_workspace_bytes(const wanb200_range_attn_params* p) {
  if (!p || p->batch <= 0 || p->heads <= 0 || p->kv_heads <= 0 || p->heads % p->kv_heads || p->heads / p->kv_heads > RT_M ||
      p->q_len <= 0 || p->kv_len <= 0 || p->q_len > INT32_MAX / 2 || p->batch > 65535 || p->heads > 65535 ||
      (p->head_dim != 64 && p->head_dim != 128) || p->reach < 0 || p->reach > RT_REACH_MAX)
    return 0;
  return range_layout(p).bytes;
}

template <int D>
static int launch_range_combine(const RangeArgs& a, const RangeParts& parts, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(parts.groups * parts.slot_rows));
  cfg.blockDim = dim3(RC_WARPS * 32);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, range_combine_kernel<D>, a, parts);
  if (e != cudaSuccess) return set_cuda_error("range_combine_kernel launch", e);
  return WANB200_OK;
}

struct DecodeLaunch {
  RangeParts parts;
  CUtensorMap k, v;
  int rows, blocks, slots;
  int* err;
};

template <int D, bool TWO, int CAP, int BIAS>
static cudaError_t launch_range_decode(const RangeArgs& a, const DecodeLaunch& d, int dev, cudaStream_t st) {
  static std::atomic<bool> attr_set[kMaxDevices] = {};
  if (!attr_set[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(range_decode_kernel<D, TWO, CAP, BIAS>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, RangeDecodeCfg<D>::SMEM);
    if (e != cudaSuccess) return e;
    attr_set[dev].store(true, std::memory_order_release);
  }
  range_decode_kernel<D, TWO, CAP, BIAS><<<(unsigned)d.blocks, RD_THREADS, RangeDecodeCfg<D>::SMEM, st>>>(d.k, d.v, a, d.parts,
                                                                                                          d.slots, d.err);
  return cudaGetLastError();
}

template <int D, int CAP, int BIAS>
static int launch_range_decode(const RangeArgs& a, const DecodeLaunch& d, cudaStream_t st) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= kMaxDevices) return set_error(WANB200_EINVAL, "device index out of range");
  const cudaError_t e = d.rows > 8 ? launch_range_decode<D, true, CAP, BIAS>(a, d, dev, st)
                                   : launch_range_decode<D, false, CAP, BIAS>(a, d, dev, st);
  if (e != cudaSuccess) return set_cuda_error("range_decode_kernel launch", e);
  return d.parts.splits > 1 ? launch_range_combine<D>(a, d.parts, st) : WANB200_OK;
}

template <int D, int CAP, int BIAS>
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
  pl.padded = const_cast<float*>(g.padded);
  int plan_blocks = g.entries <= RT_SORT_MAX ? 1 : std::min((g.entries + 31) / 32, num_sms());
  if (BIAS == kBiasTable)
    plan_blocks = std::max(plan_blocks, std::min(1 + g.a.kv_heads * g.a.group * range_padded(g.a.reach) / 4096, num_sms()));
  range_plan_kernel<<<plan_blocks, 1024, 0, st>>>(pl);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min<int64_t>(g.units, num_sms()));
  cfg.blockDim = dim3(RT_THREADS);
  cfg.dynamicSmemBytes = RangeTileCfg<D>::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, range_attn_kernel<D, CAP, BIAS>, tq, tk, tv, g);
  if (e != cudaSuccess) return set_cuda_error("range_attn_kernel launch", e);
  if (g.splits == 1) return WANB200_OK;
  const int64_t join_rows = (int64_t)g.parts.groups * g.parts.slot_rows;
  cfg.gridDim = dim3((unsigned)((join_rows + RJ_WARPS - 1) / RJ_WARPS));
  cfg.blockDim = dim3(RJ_WARPS * 32);
  cfg.dynamicSmemBytes = 0;
  e = cudaLaunchKernelEx(&cfg, range_join_kernel<D>, g.a, g.parts);
  if (e != cudaSuccess) return set_cuda_error("range_join_kernel launch", e);
  return WANB200_OK;
}

// The few-rows kernel (d) or the tiles (g with the maps of q, k and v).
template <int D>
static int range_dispatch(const RangeArgs& a, const DecodeLaunch* d, const RangeTileArgs* g, const CUtensorMap* maps,
                          cudaStream_t st) {
  const int bias = a.slopes ? kBiasSlopes : a.table ? kBiasTable : kBiasNone;
#define WANB200_RANGE_CASE(cap, bs) \
  return g ? launch_range_tiles<D, cap, bs>(maps[0], maps[1], maps[2], *g, st) : launch_range_decode<D, cap, bs>(a, *d, st)
#define WANB200_RANGE_CAP(cap)                                        \
  do {                                                                \
    if (bias == kBiasSlopes) WANB200_RANGE_CASE(cap, kBiasSlopes);    \
    if (bias == kBiasTable) WANB200_RANGE_CASE(cap, kBiasTable);      \
    WANB200_RANGE_CASE(cap, kBiasNone);                               \
  } while (0)
  if (a.cap2 <= 0.f) WANB200_RANGE_CAP(kCapNone);
  if (a.cap2 <= RA_CAP_SMALL * RA_LOG2E) WANB200_RANGE_CAP(kCapSmall);
  WANB200_RANGE_CAP(kCapLarge);
#undef WANB200_RANGE_CAP
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
  const bool few = rows <= RD_ROWS;
  const RangeLayout l = range_layout(p);
  if ((!few && l.units <= 0) || l.units > INT32_MAX / 2 || l.part_rows > INT32_MAX)
    return set_error(WANB200_EINVAL, "range_attn: too many rows");
  if (l.bytes > 0 &&
      (!p->workspace || (reinterpret_cast<uintptr_t>(p->workspace) & 255u) || p->workspace_bytes < l.bytes))
    return set_error(WANB200_EINVAL, "range_attn: need a 256-byte aligned workspace of wanb200_range_attn_workspace_bytes()");
  uint8_t* ws = static_cast<uint8_t*>(p->workspace);
  RangeParts parts;
  parts.o = reinterpret_cast<float*>(ws + l.part_off);
  parts.ml = reinterpret_cast<float2*>(ws + l.ml_off);
  parts.first = few ? reinterpret_cast<int4*>(ws) : nullptr;
  parts.slot_rows = (int)rows;
  parts.groups = (int)(p->batch * p->kv_heads);
  parts.splits = l.splits;
  int* err = device_error_word();
  if (!err) return WANB200_ECUDA;
  CUtensorMap maps[3];
  const int D = (int)p->head_dim;
  const int boxk[4] = {64, 1, few ? RD_TILE : RT_N, 1};
  const int64_t dk[4] = {D, p->kv_heads, p->kv_len, p->batch}, sk[4] = {1, D, p->k_tok_stride, p->k_batch_stride};
  rc = make_tmap_4d(&maps[1], p->k, dk, sk, boxk);
  if (rc) return rc;
  const int64_t sv[4] = {1, D, p->v_tok_stride, p->v_batch_stride};
  rc = make_tmap_4d(&maps[2], p->v, dk, sv, boxk);
  if (rc) return rc;
  if (few) {
    const int64_t blocks = range_decode_blocks(p);
    if (blocks > INT32_MAX) return set_error(WANB200_EINVAL, "range_attn: too many rows");
    DecodeLaunch d;
    d.parts = parts;
    d.k = maps[1];
    d.v = maps[2];
    d.rows = (int)rows;
    d.blocks = (int)blocks;
    d.slots = range_decode_slots(p);
    d.err = err;
    return D == 64 ? range_dispatch<64>(a, &d, nullptr, nullptr, st) : range_dispatch<128>(a, &d, nullptr, nullptr, st);
  }
  if (rows > INT32_MAX || p->batch * p->kv_heads > INT32_MAX) return set_error(WANB200_EINVAL, "range_attn: too many rows");
  const int64_t dq[4] = {D, p->heads, p->q_len, p->batch}, sq[4] = {1, D, p->q_tok_stride, p->q_batch_stride};
  const int boxq[4] = {64, a.group, l.tpt, 1};
  rc = make_tmap_4d(&maps[0], p->q, dq, sq, boxq);
  if (rc) return rc;
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
  g.parts = parts;
  g.padded = p->dist_bias ? reinterpret_cast<const float*>(ws + l.pad_off) : nullptr;
  g.cap_scale = p->softcap > 0.f ? p->softmax_scale / p->softcap : 0.f;
  g.err = err;
  return D == 64 ? range_dispatch<64>(a, nullptr, &g, maps, st) : range_dispatch<128>(a, nullptr, &g, maps, st);
}

}  // namespace wanb200
