// Low-rank adapters of many requests beside one projection:
//   y = epilogue(x W^T + bias + s_id (x A_id^T) B_id^T),  id = ids[row], none where id < 0.
// More than 16 rows: lora_down_kernel forms h = s_id x A_id^T for every row into the columns of its
// adapter, zero in the other columns that the row's 128-row tile uses, and the GEMM (gemm.cu) runs
// those columns as further K steps: acc += h . B^T with B as stored [N, adapters * rank].  A
// tile multiplies only the 16-column steps that one of its rows uses, so sorted requests cost one
// adapter's rank per tile and interleaved ones the ranks that really occur in it.
// Up to 16 rows: reading W once bounds the call, and two small kernels stream it.
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "lora.h"

namespace wanb200 {

constexpr int LD_THREADS = 192;  // TMA, MMA, 4 epilogue warps
constexpr int LD_BM = 128, LD_BK = 64, LD_GROUP = 4, LD_GROUP_F32 = 2;  // chunks of one pass
constexpr int LD_STAGES = 4;
constexpr int LD_STAGE_BYTES = LD_BM * LD_BK * 2 + LD_GROUP * LORA_CHUNK * LD_BK * 2;  // 48 KB
constexpr int LD_RED_LD = LD_GROUP * LORA_CHUNK + 4;  // fp32 row of the partial sums, padded against bank conflicts
constexpr int LD_SMEM = LD_STAGES * LD_STAGE_BYTES + 1024;
static_assert(LD_BM * LD_RED_LD * 4 <= LD_STAGES * LD_STAGE_BYTES, "the partial sums reuse the ring");

struct LoraDownArgs {
  int M, K;
  const float* scales;
  const int32_t* ids;
  int adapters, rank, cols, planes, kblocks_per_rank;
  int64_t rows_pad;
  uint32_t* step_mask;
  int* mixed;
  __nv_bfloat16* h;
  int* err;
};

__device__ __forceinline__ uint2 bf16x4(const float4& v) { return make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w)); }

// Four adjacent columns of a row of h: the row's adapter's columns scaled, zeros elsewhere (selected,
// so a NaN of another adapter's product goes no further), rounded to bf16 -- the operand type of the
// MMA that takes them.  For an fp32 output two more planes hold what the rounding left: 3 x 8 significant
// bits are those of fp32, and both remainders are exact.  (With the planes as a loop to a run-time bound the
// down-projection of 15708 rows took 53 us, unrolled 34.)
template <int PLANES>
__device__ __forceinline__ void lora_store_h(const LoraDownArgs& a, int row, int col, float4 v, int first, int last, float scale) {
  v.x = col >= first && col < last ? v.x * scale : 0.f;
  v.y = col + 1 >= first && col + 1 < last ? v.y * scale : 0.f;
  v.z = col + 2 >= first && col + 2 < last ? v.z * scale : 0.f;
  v.w = col + 3 >= first && col + 3 < last ? v.w * scale : 0.f;
  __nv_bfloat16* hp = a.h + (int64_t)row * a.cols + col;
#pragma unroll
  for (int pl = 0; pl < PLANES; ++pl) {
    const uint2 hi = bf16x4(v);
    *reinterpret_cast<uint2*>(hp) = hi;
    if (pl + 1 == PLANES) break;
    v.x -= __uint_as_float(hi.x << 16);
    v.y -= __uint_as_float(hi.x & 0xffff0000u);
    v.z -= __uint_as_float(hi.y << 16);
    v.w -= __uint_as_float(hi.y & 0xffff0000u);
    // an infinite h has no remainder
    v.x = isfinite(v.x) ? v.x : 0.f, v.y = isfinite(v.y) ? v.y : 0.f;
    v.z = isfinite(v.z) ? v.z : 0.f, v.w = isfinite(v.w) ? v.w : 0.f;
    hp += a.rows_pad * a.cols;
  }
}

// One cluster per 128-row tile, its blocks sharing K (one block where there are row tiles enough to
// fill the SMs): x tile x the tile's used chunks of A, up to four (N = 256) in one pass over x.  The
// read of x bounds it; with few row tiles the split of K brings enough SMs to the read.  The
// partial sums meet in the cluster's shared memory, each block adding its share of the rows.
// F32 (fp32 outputs): two chunks a pass, their sums over runs of LORA_RUN K blocks in two accumulators
// in turn, added up in fp32 registers, since the tensor core cuts sums off (as in gemm.cu).
template <bool F32>
__global__ void __launch_bounds__(LD_THREADS, 1)
    lora_down_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmD,
                     const __grid_constant__ LoraDownArgs a) {
  constexpr int GROUP = F32 ? LD_GROUP_F32 : LD_GROUP, ACCS = F32 ? 2 : 1, ACC_COLS = GROUP * LORA_CHUNK;
  constexpr int RUN = F32 ? LORA_RUN : 1 << 30;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bars[2 * LD_STAGES + 2 * ACCS + 1];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  __shared__ uint32_t bits[LORA_MASK_WORDS];
  __shared__ int ids[LD_BM];
  __shared__ int chunks[LORA_MAX_COLS / LORA_CHUNK];
  __shared__ int num_chunks;
  pdl_launch();  // the GEMM behind starts its own K loop; it waits for this kernel before it reads h
  const int krank = blockIdx.x, ksize = gridDim.x, m0 = blockIdx.y * LD_BM;
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sbase = smem_u32(smem);
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * LD_STAGES, tfull0 = empty0 + 8 * LD_STAGES;
  const uint32_t tempty0 = tfull0 + 8 * ACCS, done_bar = tempty0 + 8 * ACCS;
  volatile int* abort_flag = &abort_word;
  int* err = a.err;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x < LORA_MASK_WORDS) bits[threadIdx.x] = 0u;
  if (threadIdx.x == 0) {
    for (int s = 0; s < LD_STAGES; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int b = 0; b < ACCS; ++b) {
      mbar_init(tfull0 + 8 * b, 1);
      mbar_init(tempty0 + 8 * b, 128);
    }
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmD);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_slot), ACCS * ACC_COLS);
    tmem_relinquish();
  }
  __syncthreads();
  if (threadIdx.x < LD_BM) {
    const int row = m0 + threadIdx.x;
    int id = row < a.M ? __ldg(a.ids + row) : -1;
    if (id >= a.adapters) {
      atomicCAS(a.err, 0, kErrBadAdapter);
      id = -1;
    }
    ids[threadIdx.x] = id;
    if (id >= 0)
      for (int s = id * a.rank / LORA_STEP; s * LORA_STEP < (id + 1) * a.rank; ++s) atomicOr(bits + (s >> 5), 1u << (s & 31));
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (threadIdx.x < LORA_MASK_WORDS && krank == 0)
    a.step_mask[blockIdx.y * LORA_MASK_WORDS + threadIdx.x] = bits[threadIdx.x];
  // a row is mixed with an adapter that it does not use where the tile's rows differ, or where a step at
  // either end of its own adapter's columns holds some of the next one's (ranks that are no multiple of 16);
  // and several planes of h must not meet an infinite weight one by one: its product with a plane that is
  // zero, or of the other sign, makes a NaN of what is an infinity
  int mixed = a.planes > 1;
  if (threadIdx.x < LD_BM && m0 + (int)threadIdx.x < a.M) {
    const int id = ids[threadIdx.x], first = id * a.rank, last = first + a.rank;
    mixed |= id != ids[0] || (id >= 0 && (first % LORA_STEP || (last % LORA_STEP && id + 1 < a.adapters)));
  }
  mixed = __syncthreads_or(mixed);
  if (threadIdx.x == 0 && krank == 0) a.mixed[blockIdx.y] = mixed != 0;
  if (threadIdx.x == 0) {
    int n = 0;
    for (int c = 0; c < a.cols / LORA_CHUNK; ++c)
      if ((bits[c >> 3] >> ((c & 7) * 4)) & 0xfu) chunks[n++] = c;
    num_chunks = n;
  }
  __syncthreads();
  const uint32_t tmem_base = tmem_slot;
  const int kb0 = krank * a.kblocks_per_rank, kblocks = min(a.K / LD_BK - kb0, a.kblocks_per_rank);  // >= 1 (host)
  const int passes = (num_chunks + GROUP - 1) / GROUP;
  uint32_t ph = 0, issued = 0, last_ph = 0;  // ring phases, per role
  int stage = 0, run = 0;                    // run: of all passes, counted by the MMA warp and the epilogue

  for (int pass = 0; pass < passes; ++pass) {
    const int c0 = pass * GROUP, nc = min(GROUP, num_chunks - c0);
    // (the whole warp walks the issue loops: see elect_one)
    if (warp == 0) {
      for (int kb = 0; kb < kblocks; ++kb) {
        if (!mbar_wait_warp(empty0 + 8 * stage, ph ^ 1, abort_flag, err, kErrTimeoutGemmProducer)) break;
        const uint32_t dst = sbase + stage * LD_STAGE_BYTES;
        if (elect_one()) {
          mbar_expect_tx(full0 + 8 * stage, LD_BM * LD_BK * 2 + nc * LORA_CHUNK * LD_BK * 2);
          tma_load_2d(dst, &tmX, full0 + 8 * stage, (kb0 + kb) * LD_BK, m0);
          for (int c = 0; c < nc; ++c)
            tma_load_2d(dst + LD_BM * LD_BK * 2 + c * LORA_CHUNK * LD_BK * 2, &tmD, full0 + 8 * stage, (kb0 + kb) * LD_BK,
                        chunks[c0 + c] * LORA_CHUNK);
        }
        __syncwarp();
        issued |= 1u << stage;
        last_ph = (last_ph & ~(1u << stage)) | (ph << stage);
        if (++stage == LD_STAGES) stage = 0, ph ^= 1;
      }
    } else if (warp == 1) {
      const uint32_t idesc = idesc_bf16_f32(LD_BM, nc * LORA_CHUNK, false, false);
      bool ok = true;
      for (int r0 = 0; ok && r0 < kblocks; r0 += RUN, ++run) {
        const int acc = run % ACCS;
        const uint32_t d_tmem = tmem_base + acc * ACC_COLS;
        ok = mbar_wait_warp(tempty0 + 8 * acc, ((run / ACCS) & 1) ^ 1, abort_flag, err, kErrTimeoutGemmMma);
        tc_fence_after();
        for (int kb = r0; ok && kb < min(kblocks, r0 + RUN); ++kb) {
          ok = mbar_wait_warp(full0 + 8 * stage, ph, abort_flag, err, kErrTimeoutGemmMma);
          if (!ok) break;
          tc_fence_after();
          const uint32_t x_lo = sw128_lo(sbase, 16) + stage * (LD_STAGE_BYTES >> 4), d_lo = x_lo + (LD_BM * LD_BK * 2 >> 4);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < LD_BK / 16; ++kk)
              umma_bf16_w(d_tmem, x_lo + kk * 2, d_lo + kk * 2, sw128_hi(1024), idesc, ((kb - r0) | kk) != 0);
            umma_commit(empty0 + 8 * stage);
          }
          __syncwarp();
          if (++stage == LD_STAGES) stage = 0, ph ^= 1;
        }
        if (ok && elect_one()) umma_commit(tfull0 + 8 * acc);
        __syncwarp();
      }
    } else {
      const int quad = warp & 3, r = quad * 32 + lane, row = m0 + r;
      const int id = ids[r];
      const int first = id < 0 ? 0 : id * a.rank, last = id < 0 ? 0 : first + a.rank;
      const float scale = id >= 0 && a.scales ? __ldg(a.scales + id) : 1.f;
      // 32 columns from c * 32 on: h, or this block's part of it
      auto put = [&](int c, const float (&v)[32]) {
        if (ksize == 1) {
          if (row < a.M) {
            const int col = chunks[c0 + (c >> 1)] * LORA_CHUNK + (c & 1) * 32;
#pragma unroll
            for (int q = 0; q < 8; ++q)
              lora_store_h<F32 ? LORA_F32_PLANES : 1>(a, row, col + 4 * q, make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]), first, last,
                           scale);
          }
        } else {  // the ring is free: every MMA of the pass has completed
          float4* red = reinterpret_cast<float4*>(smem + (r * LD_RED_LD + c * 32) * 4);
#pragma unroll
          for (int q = 0; q < 8; ++q) red[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
        }
      };
      const uint32_t t_row = tmem_base + (uint32_t(quad * 32) << 16);
      if constexpr (F32) {
        float sum[2 * GROUP][32];
#pragma unroll
        for (int c = 0; c < 2 * GROUP; ++c)
#pragma unroll
          for (int j = 0; j < 32; ++j) sum[c][j] = 0.f;
        bool ok = true;
        for (int r0 = 0; ok && r0 < kblocks; r0 += RUN, ++run) {
          const int acc = run % ACCS;
          ok = mbar_wait_warp(tfull0 + 8 * acc, (run / ACCS) & 1, abort_flag, err, kErrTimeoutGemmEpilogue);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < 2 * GROUP; ++c)
            if (c < 2 * nc) {
              float v[32];
              tmem_ld32(t_row + acc * ACC_COLS + c * 32, v);
#pragma unroll
              for (int j = 0; j < 32; ++j) sum[c][j] += v[j];
            }
          tc_fence_before();
          mbar_arrive(tempty0 + 8 * acc);
        }
        if (ok) {
#pragma unroll
          for (int c = 0; c < 2 * GROUP; ++c)
            if (c < 2 * nc) put(c, sum[c]);
        }
      } else {
        const bool ok = mbar_wait_warp(tfull0, run++ & 1, abort_flag, err, kErrTimeoutGemmEpilogue);
        if (ok) {
          tc_fence_after();
          for (int c = 0; c < nc * 2; ++c) {
            float v[32];
            tmem_ld32(t_row + c * 32, v);
            put(c, v);
          }
        }
        tc_fence_before();
        mbar_arrive(tempty0);
      }
    }
    if (ksize > 1) {
      cluster_sync_all();
      // Each block takes its share of the rows.  Reads from the other SMs are slow (12 bytes a clock were
      // measured), so of a row only its own adapter's columns are read; the others are zero.
      const int per = LD_BM / ksize, own = a.rank / 4;
      for (int i = threadIdx.x; i < per * own; i += LD_THREADS) {
        const int r = krank * per + i / own, row = m0 + r, id = ids[r];
        if (row >= a.M || id < 0) continue;
        const int first = id * a.rank, col = first + i % own * 4;
        int g = -1;
        for (int c = 0; c < nc; ++c)
          if (chunks[c0 + c] == col / LORA_CHUNK) g = c;
        if (g < 0) continue;  // another pass has these columns
        const uint32_t at = sbase + (r * LD_RED_LD + g * LORA_CHUNK + col % LORA_CHUNK) * 4;
        float4 x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < ksize) x[k] = ld_cluster16(at, k);
        float4 sum = x[0];
#pragma unroll
        for (int k = 1; k < 8; ++k)  // in order, so that the sum is the same in every run
          if (k < ksize) sum.x += x[k].x, sum.y += x[k].y, sum.z += x[k].z, sum.w += x[k].w;
        lora_store_h<F32 ? LORA_F32_PLANES : 1>(a, row, col, sum, first, first + a.rank, a.scales ? __ldg(a.scales + id) : 1.f);
      }
      const int groups = nc * LORA_CHUNK / 8;
      for (int i = threadIdx.x; i < per * groups; i += LD_THREADS) {
        const int r = krank * per + i / groups, g = i % groups, row = m0 + r, id = ids[r];
        const int col = chunks[c0 + g / 8] * LORA_CHUNK + g % 8 * 8;
        if (row >= a.M || (id >= 0 && col >= id * a.rank && col < (id + 1) * a.rank)) continue;
        for (int pl = 0; pl < a.planes; ++pl)
          *reinterpret_cast<uint4*>(a.h + (pl * a.rows_pad + row) * a.cols + col) = make_uint4(0u, 0u, 0u, 0u);
      }
      fence_proxy_async_smem();  // the next pass's loads overwrite what was read and written here
      cluster_sync_all();
    }
  }
  if (warp == 0 && lane == 0 && *abort_flag) {  // let every load in flight land
    for (int s = 0; s < LD_STAGES; ++s)
      if ((issued >> s) & 1) mbar_drain(full0 + 8 * s, (last_ph >> s) & 1, err);
  }
  if (warp == 1) {
    if (elect_one()) umma_commit(done_bar);
    __syncwarp();
    mbar_drain(done_bar, 0, err);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, ACCS * ACC_COLS);
}

// ================================================================== up to 16 rows: W is read once
// Measured, these kernels / the tiles (us; K = N = 4096, 8 adapters of rank 16): 1 row 9.5 / 20.4, 4 rows
// 9.8 / 20.7, 16 rows 13.4 / 22.1; K = 8192, N = 2048, 16 rows 18.9 / 19.9, where the gain ends.
constexpr int LF_ROWS = 16, LF_WARPS = 8;

struct LoraFewArgs {
  const __nv_bfloat16* x;
  int64_t ldx;
  const __nv_bfloat16* w;
  int64_t ldw;
  void* d;
  int64_t ldd;
  int M, N, K, out_f32, res_f32;
  const __nv_bfloat16* bias;
  const void* residual;
  int64_t ldr;
  const __nv_bfloat16* gate_mod;
  const float* gate_e0;
  int64_t gate_frame_stride, seq_len, tokens_per_frame, row_offset, rows_per_seq;
  const __nv_bfloat16 *down, *up;
  const float* scales;
  const int32_t* ids;
  int adapters, rank;
  float* h;  // [M][rank]
  int* err;
};

__device__ __forceinline__ int few_id(const LoraFewArgs& a, int row) {
  const int id = __ldg(a.ids + row);
  return id >= 0 && id < a.adapters ? id : -1;
}

// h[row][i] = scale * x[row] . down[id][i] in fp32.  A block has one row and LF_RANKS values i; its 256
// threads share K, so that (up to K = 4096) every load is in flight at once: the GEMM behind waits for
// this latency.
constexpr int LF_RANKS = 4;

__global__ void __launch_bounds__(256) lora_few_down_kernel(const LoraFewArgs a) {
  __shared__ float part[8][LF_RANKS];
  pdl_launch();
  const int per = a.rank / LF_RANKS, row = blockIdx.x / per, i0 = (blockIdx.x - row * per) * LF_RANKS;
  const int id = few_id(a, row);
  if (id < 0) {
    if (threadIdx.x == 0 && i0 == 0 && __ldg(a.ids + row) >= a.adapters) atomicCAS(a.err, 0, kErrBadAdapter);
    return;
  }
  const uint4* xp = reinterpret_cast<const uint4*>(a.x + row * a.ldx);
  const uint4* dp = reinterpret_cast<const uint4*>(a.down + ((int64_t)id * a.rank + i0) * a.K);
  const int n = a.K / 8;
  float v[LF_RANKS] = {};
  for (int k0 = threadIdx.x; k0 < n; k0 += 512) {
    const bool second = k0 + 256 < n;
    uint4 x[2], d[2][LF_RANKS];
    x[0] = __ldg(xp + k0);
    x[1] = second ? __ldg(xp + k0 + 256) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int r = 0; r < LF_RANKS; ++r) {
      d[0][r] = __ldg(dp + r * n + k0);
      d[1][r] = second ? __ldg(dp + r * n + k0 + 256) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      float f[8];
      unpack_bf16x8(x[y], f);
#pragma unroll
      for (int r = 0; r < LF_RANKS; ++r) {
        float g[8];
        unpack_bf16x8(d[y][r], g);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[r] = fmaf(f[e], g[e], v[r]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < LF_RANKS; ++r) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v[r] += __shfl_xor_sync(0xffffffffu, v[r], o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5][r] = v[r];
  }
  __syncthreads();
  if (threadIdx.x < LF_RANKS) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) t += part[w][threadIdx.x];
    a.h[row * a.rank + i0 + threadIdx.x] = t * (a.scales ? __ldg(a.scales + id) : 1.f);
  }
}

// 8 columns of the output a block (16 or 32 were slower up to N = 14336: fewer blocks to hide a block's
// merge behind); its warps take blocks of 64 K values in turn.  W goes from
// memory straight to the operand registers of mma.sync (16 rows x 8 columns): a dot product does
// not care about the order of K, so a lane's 16 bytes serve two K steps with x permuted alike.  Bound by
// the read of W, far below even the warp-level MMA's rate.  The partial sums of the warps meet in
// shared memory; the adapter's part is added there in fp32, its h formed by the launch before while
// W streams.
template <int EPI, bool TWO>
__global__ void __launch_bounds__(LF_WARPS * 32) lora_few_kernel(const LoraFewArgs a) {
  constexpr int COLS = 8, ROWS = TWO ? 16 : 8, UNROLL = 4;
  __shared__ float red[LF_WARPS][ROWS][COLS + 1];
  __shared__ float delta[ROWS][COLS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g4 = lane >> 2, q4 = lane & 3;
  const int n0 = blockIdx.x * COLS;
  const __nv_bfloat16* wp = a.w + (int64_t)(n0 + g4) * a.ldw + 8 * q4;
  // rows behind the last repeat it: their sums are not stored
  const __nv_bfloat16* x0 = a.x + min(g4, a.M - 1) * a.ldx + 8 * q4;
  const __nv_bfloat16* x1 = a.x + min(g4 + 8, a.M - 1) * a.ldx + 8 * q4;
  // the adapters' part of this block's outputs is read at the end: brought to the L2 meanwhile
  for (int i = threadIdx.x; i < a.M * COLS; i += LF_WARPS * 32) {
    const int id = few_id(a, i / COLS);
    if (id >= 0) {
      const __nv_bfloat16* up = a.up + ((int64_t)(n0 + i % COLS) * a.adapters + id) * a.rank;
      for (int k = 0; k < a.rank; k += 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(up + k));
    }
  }
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  // a warp's turn: UNROLL blocks of 64 K values (one 128-byte line of each W row), all loads first
  auto turn = [&](int c0, auto unroll) {
    constexpr int U = decltype(unroll)::value;
    uint4 wv[U][2], xv[U][2][TWO ? 2 : 1];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int k = 64 * (c0 + u * LF_WARPS) + 32 * y;
        wv[u][y] = ld_stream(wp + k);
        xv[u][y][0] = __ldg(reinterpret_cast<const uint4*>(x0 + k));
        if constexpr (TWO) xv[u][y][1] = __ldg(reinterpret_cast<const uint4*>(x1 + k));
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const uint4 lo = xv[u][y][0], hi = TWO ? xv[u][y][TWO ? 1 : 0] : make_uint4(0u, 0u, 0u, 0u);
        mma_16816(acc, lo.x, hi.x, lo.y, hi.y, wv[u][y].x, wv[u][y].y);
        mma_16816(acc, lo.z, hi.z, lo.w, hi.w, wv[u][y].z, wv[u][y].w);
      }
  };
  const int blocks = a.K / 64;
  int c0 = warp;
  for (; c0 + (UNROLL - 1) * LF_WARPS < blocks; c0 += LF_WARPS * UNROLL) turn(c0, std::integral_constant<int, UNROLL>());
  for (; c0 < blocks; c0 += LF_WARPS) turn(c0, std::integral_constant<int, 1>());
#pragma unroll
  for (int e = 0; e < (TWO ? 4 : 2); ++e) red[warp][g4 + 8 * (e >> 1)][2 * q4 + (e & 1)] = acc[e];
  pdl_wait();
  // h . up[n][id], eight lanes an output so that its rank values are read as whole lines
  const int l8 = lane & 7;
#pragma unroll 2
  for (int i = threadIdx.x >> 3; i < a.M * COLS; i += LF_WARPS * 4) {
    const int row = i / COLS, id = few_id(a, row);
    float s0 = 0.f, s1 = 0.f;
    if (id >= 0) {
      const uint4* up = reinterpret_cast<const uint4*>(a.up + ((int64_t)(n0 + i % COLS) * a.adapters + id) * a.rank);
      const float4* h = reinterpret_cast<const float4*>(a.h + row * a.rank);
      for (int k = l8; k < a.rank / 8; k += 8) {
        float u[8];
        unpack_bf16x8(__ldg(up + k), u);
        const float4 h0 = h[2 * k], h1 = h[2 * k + 1];
        s0 = fmaf(h0.x, u[0], s0), s1 = fmaf(h0.y, u[1], s1), s0 = fmaf(h0.z, u[2], s0), s1 = fmaf(h0.w, u[3], s1);
        s0 = fmaf(h1.x, u[4], s0), s1 = fmaf(h1.y, u[5], s1), s0 = fmaf(h1.z, u[6], s0), s1 = fmaf(h1.w, u[7], s1);
      }
    }
    s0 += s1;
#pragma unroll
    for (int o = 4; o; o >>= 1) s0 += __shfl_xor_sync(0xffu << (lane & 24), s0, o);
    if (l8 == 0) delta[row][i % COLS] = s0;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.M * COLS; i += LF_WARPS * 32) {
    const int row = i / COLS, col = i % COLS, n = n0 + col;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < LF_WARPS; ++w) v += red[w][row][col];
    v += delta[row][col];
    if constexpr (EPI != WANB200_EPI_NONE) v += __bfloat162float(a.bias[n]);
    if constexpr (EPI == WANB200_EPI_BIAS_GELU) v = gelu_tanh(v);
    if constexpr (EPI == WANB200_EPI_BIAS_SILU) v = silu(v);
    if constexpr (EPI == WANB200_EPI_BIAS_GATE_RES || EPI == WANB200_EPI_BIAS_RES) {
      const int64_t at = row * a.ldr + n;
      const float r = a.res_f32 ? static_cast<const float*>(a.residual)[at]
                                : __bfloat162float(static_cast<const __nv_bfloat16*>(a.residual)[at]);
      if constexpr (EPI == WANB200_EPI_BIAS_GATE_RES) {
        const int64_t f = frame_of_row(row, a.rows_per_seq, a.row_offset, a.seq_len, a.tokens_per_frame);
        v = r + v * (__bfloat162float(a.gate_mod[n]) + a.gate_e0[f * a.gate_frame_stride + n]);
      } else {
        v += r;
      }
    }
    if (a.out_f32)
      static_cast<float*>(a.d)[row * a.ldd + n] = v;
    else
      static_cast<__nv_bfloat16*>(a.d)[row * a.ldd + n] = __float2bfloat16(v);
  }
}

template <int EPI>
static cudaError_t launch_lora_few(const LoraFewArgs& a, const cudaLaunchConfig_t& cfg) {
  return a.M > 8 ? cudaLaunchKernelEx(&cfg, lora_few_kernel<EPI, true>, a) : cudaLaunchKernelEx(&cfg, lora_few_kernel<EPI, false>, a);
}

static int lora_few(const wanb200_lora_params* p, float* h, int* err, cudaStream_t st) {
  const wanb200_gemm_params* g = &p->gemm;
  LoraFewArgs a;
  a.x = reinterpret_cast<const __nv_bfloat16*>(g->a);
  a.ldx = g->lda;
  a.w = reinterpret_cast<const __nv_bfloat16*>(g->w);
  a.ldw = g->ldw;
  a.d = g->d;
  a.ldd = g->ldd;
  a.M = (int)g->M;
  a.N = (int)g->N;
  a.K = (int)g->K;
  a.out_f32 = g->out_f32 != 0;
  a.res_f32 = g->residual_f32 != 0;
  a.bias = reinterpret_cast<const __nv_bfloat16*>(g->bias);
  a.residual = g->residual;
  a.ldr = g->ldr;
  a.gate_mod = reinterpret_cast<const __nv_bfloat16*>(g->gate_mod);
  a.gate_e0 = g->gate_e0;
  a.gate_frame_stride = g->gate_frame_stride;
  a.seq_len = g->seq_len > 0 ? g->seq_len : 1;
  a.tokens_per_frame = g->tokens_per_frame > 0 ? g->tokens_per_frame : 1;
  a.row_offset = g->row_offset;
  a.rows_per_seq = g->rows_per_seq;
  a.down = reinterpret_cast<const __nv_bfloat16*>(p->down);
  a.up = reinterpret_cast<const __nv_bfloat16*>(p->up);
  a.scales = p->scales;
  a.ids = p->ids;
  a.adapters = p->adapters;
  a.rank = p->rank;
  a.h = h;
  a.err = err;
  lora_few_down_kernel<<<(unsigned)(a.M * (a.rank / LF_RANKS)), 256, 0, st>>>(a);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.N / 8));
  cfg.blockDim = dim3(LF_WARPS * 32);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e;
  switch (g->epilogue) {
    case WANB200_EPI_NONE: e = launch_lora_few<WANB200_EPI_NONE>(a, cfg); break;
    case WANB200_EPI_BIAS: e = launch_lora_few<WANB200_EPI_BIAS>(a, cfg); break;
    case WANB200_EPI_BIAS_GELU: e = launch_lora_few<WANB200_EPI_BIAS_GELU>(a, cfg); break;
    case WANB200_EPI_BIAS_SILU: e = launch_lora_few<WANB200_EPI_BIAS_SILU>(a, cfg); break;
    case WANB200_EPI_BIAS_GATE_RES: e = launch_lora_few<WANB200_EPI_BIAS_GATE_RES>(a, cfg); break;
    default: e = launch_lora_few<WANB200_EPI_BIAS_RES>(a, cfg); break;
  }
  if (e != cudaSuccess) return set_cuda_error("lora_few_kernel launch", e);
  return WANB200_OK;
}

// ------------------------------------------------------------------ host launcher
struct LoraLayout {
  int64_t rows_pad, num_m, mixed_off, h_off, bytes;
  int cols, planes;
};

static LoraLayout lora_layout(int64_t M, int adapters, int rank, int out_f32) {
  LoraLayout l = {};
  if (M <= LF_ROWS) {  // h in fp32
    l.num_m = 1;
    l.bytes = M * rank * 4;
    return l;
  }
  l.num_m = (M + LD_BM - 1) / LD_BM;
  l.rows_pad = l.num_m * LD_BM;
  l.cols = (adapters * rank + LORA_CHUNK - 1) / LORA_CHUNK * LORA_CHUNK;
  l.planes = out_f32 ? LORA_F32_PLANES : 1;
  l.mixed_off = l.num_m * LORA_MASK_WORDS * 4;
  l.h_off = (l.mixed_off + l.num_m * 4 + 255) / 256 * 256;
  l.bytes = l.h_off + l.planes * l.rows_pad * l.cols * 2;
  return l;
}

static bool lora_sizes_ok(int64_t M, int adapters, int rank) {
  return M > 0 && M <= INT32_MAX / 2 && adapters > 0 && rank > 0 && rank % 8 == 0 &&
         (int64_t)adapters * rank <= LORA_MAX_COLS;
}

int64_t lora_workspace_bytes(int64_t M, int adapters, int rank, int out_f32) {
  return lora_sizes_ok(M, adapters, rank) ? lora_layout(M, adapters, rank, out_f32).bytes : 0;
}

// Blocks per row tile of the down-projection, and the GEMM's tile width, K split and grid, by a cost
// model in which a K block of 64 costs max(200, width) of a tile (the loads into an SM bound narrow
// tiles, the tensor pipe 256-wide ones: about 215 and 280 ns) and 300 in the down-projection, whose
// fixed part weighs 3000.
// The two kernels run side by side where the SMs beside the down-projection's suffice for the GEMM
// (it waits for h only at the end of its first K loop), else one after the other.  Few tiles
// share K over a cluster; its join reads (ks - 1) / ks of a tile from other SMs.
// Measured (us): 509 x 2048 x 4096, 16 adapters of rank 16: 25 as chosen, 46 without a split of the
// down-projection, 34 without one of the GEMM; 128 x 4096 x 4096, 4 of rank 64: 23, 45 and 35; 1964 x
// 8192 x 2048, 3 of rank 32, has tiles enough: 67 whatever is allowed.
struct LoraLaunch {
  int down_ksize, bn, ksplit, grid;
};

static LoraLaunch lora_plan_launch(int64_t M, int64_t N, int kblocks, int tile_n, int sms) {
  const int64_t num_m = (M + LD_BM - 1) / LD_BM;
  LoraLaunch best = {};
  double best_t = 1e300;
  auto shares = [&](int k) { return (kblocks + k - 1) / k; };
  for (int ds = 1; ds <= 8; ds *= 2) {
    if (ds > 1 && ((int64_t)(ds - 1) * shares(ds) >= kblocks || shares(ds) < 4 || num_m * ds > sms)) break;
    const int64_t down_blocks = num_m * ds;
    const double down = (double)((down_blocks + sms - 1) / sms) * (shares(ds) * 300.0 + 3000.0);
    for (int bn = tile_n ? tile_n : 256; bn >= (tile_n ? tile_n : 128); bn -= 32) {
      const int64_t tiles = num_m * ((N + bn - 1) / bn);
      const double kb = std::max(200, bn);
      for (int ks = 1; ks <= 4; ks *= 2) {
        if (ks > 1 && ((int64_t)(ks - 1) * shares(ks) >= kblocks || shares(ks) < 4 || tiles * ks > sms)) break;
        const double tile = shares(ks) * kb + (ks > 1 ? 40.0 * bn * (ks - 1) / ks : 0.0) + 64.0 * shares(ks);
        for (int beside = 0; beside < 2; ++beside) {
          const int64_t room = beside ? sms - down_blocks : sms;
          if (room < ks || (ks > 1 && tiles * ks > room)) continue;
          const double t = beside ? std::max((double)((tiles + room - 1) / room) * tile, down + 1600.0)
                                  : down + (double)((tiles + sms - 1) / sms) * tile;
          if (t < best_t - 1e-9) {
            best_t = t;
            best = {ds, bn, ks, (int)(ks > 1 ? tiles * ks : std::min<int64_t>(tiles, room))};
          }
        }
      }
    }
  }
  return best;
}

template <bool F32>
static int launch_lora_down(const CUtensorMap& tx, const CUtensorMap& td, const LoraDownArgs& a, int ksize, int64_t num_m,
                            cudaStream_t st) {
  static std::atomic<bool> attr_set[kMaxDevices] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= kMaxDevices) return set_error(WANB200_EINVAL, "device index out of range");
  cudaError_t e;
  if (!attr_set[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(lora_down_kernel<F32>, cudaFuncAttributeMaxDynamicSharedMemorySize, LD_SMEM);
    if (e != cudaSuccess) return set_cuda_error("cudaFuncSetAttribute(lora_down)", e);
    attr_set[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ksize, (unsigned)num_m);
  cfg.blockDim = dim3(LD_THREADS);
  cfg.dynamicSmemBytes = LD_SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ksize;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, lora_down_kernel<F32>, tx, td, a);
  if (e != cudaSuccess) return set_cuda_error("lora_down_kernel launch", e);
  return WANB200_OK;
}

int gemm_lora(const wanb200_lora_params* p, cudaStream_t st) {
  if (!p) return set_error(WANB200_EINVAL, "gemm_lora: null params");
  const wanb200_gemm_params* g = &p->gemm;
  if (g->epilogue == WANB200_EPI_SCATTER || g->epilogue == WANB200_EPI_BIAS_SUMSQ)
    return set_error(WANB200_EINVAL, "gemm_lora: the SCATTER and SUMSQ epilogues take no adapters");
  int rc = gemm_validate(g);
  if (rc) return rc;
  if (!lora_sizes_ok(g->M, p->adapters, p->rank))
    return set_error(WANB200_EINVAL, "gemm_lora: need adapters > 0, rank a positive multiple of 8, adapters * rank <= 4096");
  if (!p->down || !p->up || !p->ids || !aligned16(p->down) || !aligned16(p->up))
    return set_error(WANB200_EINVAL, "gemm_lora: need ids and 16-byte aligned down and up");
  const LoraLayout l = lora_layout(g->M, p->adapters, p->rank, g->out_f32 != 0);
  if (!p->lora_workspace || (reinterpret_cast<uintptr_t>(p->lora_workspace) & 255u) || p->lora_workspace_bytes < l.bytes)
    return set_error(WANB200_EINVAL, "gemm_lora: need a 256-byte aligned workspace of wanb200_lora_workspace_bytes()");
  if (l.num_m > 65535) return set_error(WANB200_EINVAL, "gemm_lora: too many rows");
  int* err = device_error_word();
  if (!err) return WANB200_ECUDA;
  if (g->M <= LF_ROWS) return lora_few(p, static_cast<float*>(p->lora_workspace), err, st);
  uint8_t* ws = static_cast<uint8_t*>(p->lora_workspace);
  CUtensorMap tx, td;
  rc = make_tmap_2d(&tx, g->a, g->K, g->M, g->lda, LD_BK, LD_BM);
  if (rc) return rc;
  rc = make_tmap_2d(&td, p->down, g->K, (int64_t)p->adapters * p->rank, g->K, LD_BK, LORA_CHUNK);
  if (rc) return rc;
  LoraDownArgs a;
  a.M = (int)g->M;
  a.K = (int)g->K;
  a.scales = p->scales;
  a.ids = p->ids;
  a.adapters = p->adapters;
  a.rank = p->rank;
  a.cols = l.cols;
  a.planes = l.planes;
  a.rows_pad = l.rows_pad;
  a.step_mask = reinterpret_cast<uint32_t*>(ws);
  a.mixed = reinterpret_cast<int*>(ws + l.mixed_off);
  a.h = reinterpret_cast<__nv_bfloat16*>(ws + l.h_off);
  a.err = err;
  const LoraLaunch pl = lora_plan_launch(g->M, g->N, a.K / LD_BK, g->tile_n, num_sms());
  const int ksize = pl.down_ksize;
  a.kblocks_per_rank = (a.K / LD_BK + ksize - 1) / ksize;
  rc = g->out_f32 ? launch_lora_down<true>(tx, td, a, ksize, l.num_m, st) : launch_lora_down<false>(tx, td, a, ksize, l.num_m, st);
  if (rc) return rc;
  LoraPlan plan;
  plan.step_mask = a.step_mask;
  plan.mixed = a.mixed;
  plan.h = a.h;
  plan.up = reinterpret_cast<const __nv_bfloat16*>(p->up);
  plan.ids = a.ids;
  plan.adapters = a.adapters;
  plan.rank = a.rank;
  plan.cols = a.cols;
  plan.planes = a.planes;
  plan.rows_pad = a.rows_pad;
  plan.bn = pl.bn;
  plan.ksplit = pl.ksplit;
  plan.grid = pl.grid;
  return gemm_launch(g, &plan, err, st);
}

}  // namespace wanb200
