// Low-rank adapters of many requests beside one projection:
//   y = epilogue(x W^T + bias + s_id (x A_id^T) B_id^T),  id = ids[row], none where id < 0.
// Two launches: this file's kernel forms h = s_id x A_id^T for every row into the columns of its
// adapter, zero in the other columns that the row's 128-row tile uses, and the GEMM (gemm.cu) runs
// those columns as further K steps: acc += h . B^T with B as stored [N, adapters * rank].  A
// tile multiplies only the 16-column steps that one of its rows uses, so sorted requests cost one
// adapter's rank per tile and interleaved ones the ranks that really occur in it.
#include "common.cuh"
#include "lora.h"

namespace wanb200 {

struct LoraDownArgs {
  const __nv_bfloat16* x;
  int64_t ldx;
  int M, N, K;
  const __nv_bfloat16* down;  // [adapters * rank, K]
  const __nv_bfloat16* up;    // [N, adapters * rank]
  const float* scales;
  const int32_t* ids;
  int adapters, rank, cols, steps, planes;
  int64_t rows_pad;
  uint32_t* step_mask;
  int* bad;
  __nv_bfloat16* h;
  int num_m;
  int* err;
};

__device__ __forceinline__ int lora_id(const LoraDownArgs& a, int row) {
  const int id = __ldg(a.ids + row);
  if (id >= a.adapters) atomicCAS(a.err, 0, kErrBadAdapter);
  return id >= 0 && id < a.adapters ? id : -1;
}

// Blocks 0 .. num_m - 1: the step bits of a row tile.  The others: one (step, slice of N) each, a
// scan of the step's `up` columns for values that are not finite.  h = 0 keeps a row clear of
// another adapter's finite values, but 0 * NaN does not, so the GEMM leaves such steps out and its
// epilogue adds them to the rows that use them one by one.
__global__ void __launch_bounds__(128) lora_plan_kernel(const LoraDownArgs a) {
  if ((int)blockIdx.x < a.num_m) {
    __shared__ uint32_t bits[LORA_MASK_WORDS];
    if (threadIdx.x < LORA_MASK_WORDS) bits[threadIdx.x] = 0u;
    __syncthreads();
    const int row = blockIdx.x * 128 + threadIdx.x;
    const int id = row < a.M ? lora_id(a, row) : -1;
    if (id >= 0)
      for (int s = id * a.rank / LORA_STEP; s * LORA_STEP < (id + 1) * a.rank; ++s) atomicOr(bits + (s >> 5), 1u << (s & 31));
    __syncthreads();
    if (threadIdx.x < LORA_MASK_WORDS) a.step_mask[blockIdx.x * LORA_MASK_WORDS + threadIdx.x] = bits[threadIdx.x];
    return;
  }
  const int unit = blockIdx.x - a.num_m, step = unit / LORA_SCAN, slice = unit % LORA_SCAN;
  const int c0 = step * LORA_STEP, c1 = min(c0 + LORA_STEP, a.adapters * a.rank);
  int used = 0, bad = 0;
  for (int row = threadIdx.x; row < a.M && !used; row += 128) {
    const int id = __ldg(a.ids + row);
    used = id >= 0 && id < a.adapters && id * a.rank < c1 && (id + 1) * a.rank > c0;
  }
  if (__syncthreads_or(used)) {
    const int n1 = min(a.N, (slice + 1) * ((a.N + LORA_SCAN - 1) / LORA_SCAN));
    for (int n = slice * ((a.N + LORA_SCAN - 1) / LORA_SCAN) + threadIdx.x; n < n1; n += 128) {
      const uint4* p = reinterpret_cast<const uint4*>(a.up + (int64_t)n * a.adapters * a.rank + c0);
      for (int q = 0; q < (c1 - c0) / 8; ++q) {
        const uint4 u = __ldg(p + q);
        bad |= nonfinite_bf16x2(u.x) | nonfinite_bf16x2(u.y) | nonfinite_bf16x2(u.z) | nonfinite_bf16x2(u.w);
      }
    }
  }
  bad = __syncthreads_or(bad);
  if (threadIdx.x == 0) a.bad[unit] = bad;
}

// One block per row, one warp per column of the tile's used steps.
__global__ void __launch_bounds__(256) lora_down_rows_kernel(const LoraDownArgs a) {
  const int row = blockIdx.x, lane = threadIdx.x & 31;
  const int id = lora_id(a, row);
  const float scale = id >= 0 && a.scales ? __ldg(a.scales + id) : 1.f;
  const uint32_t* mask = a.step_mask + (row >> 7) * LORA_MASK_WORDS;
  for (int c = threadIdx.x >> 5; c < a.cols; c += 8) {
    if (!((__ldg(mask + (c >> 9)) >> ((c >> 4) & 31)) & 1u)) continue;
    float v = 0.f;
    if (id >= 0 && c >= id * a.rank && c < (id + 1) * a.rank) {
      const uint4* xp = reinterpret_cast<const uint4*>(a.x + row * a.ldx);
      const uint4* dp = reinterpret_cast<const uint4*>(a.down + (int64_t)c * a.K);
      for (int k = lane; k < a.K / 8; k += 32) {
        float f[8], g[8];
        unpack_bf16x8(__ldg(xp + k), f);
        unpack_bf16x8(__ldg(dp + k), g);
#pragma unroll
        for (int i = 0; i < 8; ++i) v = fmaf(f[i], g[i], v);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      v *= scale;
    }
    if (lane == 0) {
      __nv_bfloat16* hp = a.h + (int64_t)row * a.cols + c;
      const __nv_bfloat16 hi = __float2bfloat16(v);
      hp[0] = hi;
      // the second plane keeps h's rounding out of an fp32 output
      if (a.planes > 1) hp[a.rows_pad * a.cols] = __float2bfloat16(isfinite(v) ? v - __bfloat162float(hi) : 0.f);
    }
  }
}

struct LoraLayout {
  int64_t rows_pad, num_m, bad_off, h_off, bytes;
  int cols, steps, planes;
};

static LoraLayout lora_layout(int64_t M, int adapters, int rank, int out_f32) {
  LoraLayout l;
  l.num_m = (M + 127) / 128;
  l.rows_pad = l.num_m * 128;
  l.cols = (adapters * rank + LORA_CHUNK - 1) / LORA_CHUNK * LORA_CHUNK;
  l.steps = (adapters * rank + LORA_STEP - 1) / LORA_STEP;
  l.planes = out_f32 ? 2 : 1;
  l.bad_off = (l.num_m * LORA_MASK_WORDS * 4 + 255) / 256 * 256;
  l.h_off = l.bad_off + (l.steps * LORA_SCAN * 4 + 255) / 256 * 256;
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

int gemm_lora(const wanb200_lora_params* p, cudaStream_t st) {
  if (!p) return set_error(WANB200_EINVAL, "gemm_lora: null params");
  const wanb200_gemm_params* g = &p->gemm;
  if (g->epilogue == WANB200_EPI_SCATTER || g->epilogue == WANB200_EPI_BIAS_SUMSQ)
    return set_error(WANB200_EINVAL, "gemm_lora: the SCATTER and SUMSQ epilogues take no adapters");
  const int rc = gemm_validate(g);
  if (rc) return rc;
  if (!lora_sizes_ok(g->M, p->adapters, p->rank))
    return set_error(WANB200_EINVAL, "gemm_lora: need adapters > 0, rank a positive multiple of 8, adapters * rank <= 4096");
  if (!p->down || !p->up || !p->ids || !aligned16(p->down) || !aligned16(p->up))
    return set_error(WANB200_EINVAL, "gemm_lora: need ids and 16-byte aligned down and up");
  const LoraLayout l = lora_layout(g->M, p->adapters, p->rank, g->out_f32 != 0);
  if (!p->lora_workspace || (reinterpret_cast<uintptr_t>(p->lora_workspace) & 255u) || p->lora_workspace_bytes < l.bytes)
    return set_error(WANB200_EINVAL, "gemm_lora: need a 256-byte aligned workspace of wanb200_lora_workspace_bytes()");
  int* err = device_error_word();
  if (!err) return WANB200_ECUDA;
  uint8_t* ws = static_cast<uint8_t*>(p->lora_workspace);
  LoraDownArgs a;
  a.x = reinterpret_cast<const __nv_bfloat16*>(g->a);
  a.ldx = g->lda;
  a.M = (int)g->M;
  a.N = (int)g->N;
  a.K = (int)g->K;
  a.down = reinterpret_cast<const __nv_bfloat16*>(p->down);
  a.up = reinterpret_cast<const __nv_bfloat16*>(p->up);
  a.scales = p->scales;
  a.ids = p->ids;
  a.adapters = p->adapters;
  a.rank = p->rank;
  a.cols = l.cols;
  a.steps = l.steps;
  a.planes = l.planes;
  a.rows_pad = l.rows_pad;
  a.step_mask = reinterpret_cast<uint32_t*>(ws);
  a.bad = reinterpret_cast<int*>(ws + l.bad_off);
  a.h = reinterpret_cast<__nv_bfloat16*>(ws + l.h_off);
  a.num_m = (int)l.num_m;
  a.err = err;
  lora_plan_kernel<<<(unsigned)(l.num_m + l.steps * LORA_SCAN), 128, 0, st>>>(a);
  lora_down_rows_kernel<<<(unsigned)g->M, 256, 0, st>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error("lora down-projection launch", e);
  LoraPlan plan;
  plan.step_mask = a.step_mask;
  plan.bad = a.bad;
  plan.h = a.h;
  plan.up = a.up;
  plan.ids = a.ids;
  plan.adapters = a.adapters;
  plan.rank = a.rank;
  plan.cols = a.cols;
  plan.steps = a.steps;
  plan.planes = a.planes;
  plan.rows_pad = a.rows_pad;
  return gemm_launch(g, &plan, err, st);
}

}  // namespace wanb200
