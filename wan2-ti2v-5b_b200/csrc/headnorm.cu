// RMS norm of every head of the query and key sections with the position rotation in the same
// pass.  Per head x[0..D): y = x * rsqrt(mean(x^2) + eps) * gamma, then the pairs (a, b) of the
// first `rot` channels become (a c - b s, a s + b c) with the angle of the row's position.  One
// read and one write of 2 bytes per value: HBM-bound, and latency-bound at a few rows.
#include "common.cuh"
#include "internal.h"

namespace wanb200 {

struct HeadNormArgs {
  const __nv_bfloat16* x;
  __nv_bfloat16* out;
  int64_t ldx, ldo, rows;
  int64_t col0[2];
  int heads0, heads1;
  const __nv_bfloat16* gamma[2];
  float eps;
  int rot;
  const float* cos;
  const float* sin;
  const int32_t* positions;
  int64_t table_rows;
  int groups0, groups;  // warps per row: of section 0, of both
  int* err;
};

// A head is LPH = D / 8 lanes of 16 bytes, so a warp holds 32 / LPH heads at once and takes NV such
// passes over heads of one section of one row, all loads in flight before the first use.  Sums and the
// norm are fp32 over the head's lanes (a butterfly inside the lane group).  Gains and angles are the
// same for all heads of the warp, so their products are formed once: a pair becomes
//   a' = r (a (g_a c) - b (g_b s)),  b' = r (a (g_a s) + b (g_b c)),  r = rsqrt(mean + eps).
// Interleaved pairs live inside a lane; half-split pairs (i, i + rot/2) are exchanged with the partner
// lane by shuffles.  One rounding, to bf16, at the store.  x and the output go past the L1 (streaming
// hints), which keeps the angles that a row's warps share.
//
// With gains and angles applied head by head the kernel issued 21 instructions a value and stood at
// 78 us for 15708 rows of 48 heads of 128 (390 MB) with its issue slots 68% busy; with the products
// formed once it is 70 us, 5.56 TB/s, 0.86 of the copy rate, issue 59%.
template <int LPH, int NV, bool INTER>
__global__ void __launch_bounds__(256, 4) head_norm_rope_kernel(const HeadNormArgs a) {
  constexpr int HP = 32 / LPH, D = LPH * 8;
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int64_t row = w / a.groups;
  if (row >= a.rows) return;  // warp-uniform
  int grp = (int)(w - row * a.groups);
  const int sec = grp >= a.groups0;  // warp-uniform
  grp -= sec ? a.groups0 : 0;
  const int heads = sec ? a.heads1 : a.heads0;
  const int h0 = grp * (HP * NV) + lane / LPH;
  const int c = lane % LPH;  // this lane's 8 channels: 8c .. 8c + 7
  const int64_t col = (sec ? a.col0[1] : a.col0[0]) + 8 * c;
  const __nv_bfloat16* xr = a.x + row * a.ldx + col;
  uint4 raw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int h = h0 + i * HP;
    raw[i] = h < heads ? __ldcs(reinterpret_cast<const uint4*>(xr + h * D)) : make_uint4(0u, 0u, 0u, 0u);
  }
  const int half = a.rot >> 4;  // lanes of one half of the rotated channels (half-split pairs)
  const bool turned = a.cos && 8 * c < a.rot;
  const int partner = (lane + (c < half ? half : -half)) & 31;
  const __nv_bfloat16* gamma = sec ? a.gamma[1] : a.gamma[0];
  // own[k], other[k]: factors of the value itself and of its pair's other value
  float own[8], other[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) own[k] = 1.f, other[k] = 0.f;
  if (gamma) unpack_bf16x8(__ldg(reinterpret_cast<const uint4*>(gamma) + c), own);
  if (a.cos) {
    const int64_t pos = a.positions ? (int64_t)__ldg(a.positions + row) : row % a.table_rows;
    if (pos < 0 || pos >= a.table_rows) {  // warp-uniform: the row is left as it was
      if (lane == 0) atomicCAS(a.err, 0, kErrBadPosition);
      return;
    }
    float g2[8];  // the gains of the pairs' other values
#pragma unroll
    for (int k = 0; k < 8; ++k) g2[k] = INTER ? own[k ^ 1] : __shfl_sync(0xffffffffu, own[k], partner);
    if (turned) {
      const int p0 = INTER ? 4 * c : 8 * (c < half ? c : c - half);
      const float4* cp = reinterpret_cast<const float4*>(a.cos + pos * (a.rot >> 1) + p0);
      const float4* sp = reinterpret_cast<const float4*>(a.sin + pos * (a.rot >> 1) + p0);
      float cs[8], sn[8];
#pragma unroll
      for (int q = 0; q < (INTER ? 1 : 2); ++q) {
        const float4 cv = __ldg(cp + q), sv = __ldg(sp + q);
        cs[4 * q] = cv.x; cs[4 * q + 1] = cv.y; cs[4 * q + 2] = cv.z; cs[4 * q + 3] = cv.w;
        sn[4 * q] = sv.x; sn[4 * q + 1] = sv.y; sn[4 * q + 2] = sv.z; sn[4 * q + 3] = sv.w;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const bool first = INTER ? (k & 1) == 0 : c < half;
        const int p = INTER ? k >> 1 : k;
        own[k] *= cs[p];
        other[k] = first ? -g2[k] * sn[p] : g2[k] * sn[p];
      }
    }
  }
  __nv_bfloat16* outr = a.out + row * a.ldo + col;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int h = h0 + i * HP;
    float x[8];
    unpack_bf16x8(raw[i], x);
    float r = 1.f;
    if (gamma) {
      float q = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) q = fmaf(x[k], x[k], q);
#pragma unroll
      for (int o = LPH / 2; o; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
      r = rsqrtf(q * (1.f / D) + a.eps);
    }
    float y[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = x[k] * own[k];
    if (a.cos) {
      if constexpr (INTER) {
        if (turned) {
#pragma unroll
          for (int k = 0; k < 8; ++k) y[k] = fmaf(x[k ^ 1], other[k], y[k]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float o = __shfl_sync(0xffffffffu, x[k], partner);
          if (turned) y[k] = fmaf(o, other[k], y[k]);
        }
      }
    }
    if (h < heads) {
      uint4 u;
      u.x = pack_bf16x2(y[0] * r, y[1] * r);
      u.y = pack_bf16x2(y[2] * r, y[3] * r);
      u.z = pack_bf16x2(y[4] * r, y[5] * r);
      u.w = pack_bf16x2(y[6] * r, y[7] * r);
      __stcs(reinterpret_cast<uint4*>(outr + h * D), u);
    }
  }
}

template <int LPH, int NV>
static void launch_head_norm(const HeadNormArgs& a, bool inter, unsigned blocks, cudaStream_t st) {
  if (inter)
    head_norm_rope_kernel<LPH, NV, true><<<blocks, 256, 0, st>>>(a);
  else
    head_norm_rope_kernel<LPH, NV, false><<<blocks, 256, 0, st>>>(a);
}

template <int LPH>
static void launch_head_norm(const HeadNormArgs& a, int nv, bool inter, unsigned blocks, cudaStream_t st) {
  if (nv == 1)
    launch_head_norm<LPH, 1>(a, inter, blocks, st);
  else if (nv == 2)
    launch_head_norm<LPH, 2>(a, inter, blocks, st);
  else
    launch_head_norm<LPH, 6>(a, inter, blocks, st);
}

int head_norm_rope(const wanb200_headnorm_params* p, cudaStream_t st) {
  if (!p) return set_error(WANB200_EINVAL, "head_norm_rope: null params");
  if (!p->x || !p->out || p->rows <= 0) return set_error(WANB200_EINVAL, "head_norm_rope: need x, out, rows > 0");
  if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256)
    return set_error(WANB200_EINVAL, "head_norm_rope: head_dim must be 64, 128 or 256");
  if (p->nsections < 1 || p->nsections > 2)
    return set_error(WANB200_EINVAL, "head_norm_rope: nsections must be 1 or 2");
  if (p->ldx <= 0 || p->ldo <= 0 || p->ldx % 8 || p->ldo % 8 || !aligned16(p->x) || !aligned16(p->out))
    return set_error(WANB200_EINVAL, "head_norm_rope: x / out need 16-byte aligned pointers and row strides % 8 == 0");
  if (p->x == p->out && p->ldx != p->ldo)
    return set_error(WANB200_EINVAL, "head_norm_rope: in place needs equal row strides");
  for (int s = 0; s < p->nsections; ++s) {
    if (p->heads[s] <= 0 || p->heads[s] > 65535 || p->col0[s] < 0 || p->col0[s] % 8 ||
        p->col0[s] + (int64_t)p->heads[s] * p->head_dim > std::min(p->ldx, p->ldo) || !aligned16(p->gamma[s]))
      return set_error(WANB200_EINVAL, "head_norm_rope: bad section (col0 % 8 == 0, heads * head_dim inside the row, "
                                       "16-byte aligned gamma)");
  }
  if (p->nsections == 2) {  // a warp may hold heads of both, so they must not share channels
    const int64_t e0 = p->col0[0] + (int64_t)p->heads[0] * p->head_dim, e1 = p->col0[1] + (int64_t)p->heads[1] * p->head_dim;
    if (p->col0[0] < e1 && p->col0[1] < e0) return set_error(WANB200_EINVAL, "head_norm_rope: the sections overlap");
  }
  if ((!p->cos) != (!p->sin)) return set_error(WANB200_EINVAL, "head_norm_rope: cos and sin come together");
  if (p->cos) {
    if (p->rot <= 0 || p->rot % 16 || p->rot > p->head_dim)
      return set_error(WANB200_EINVAL, "head_norm_rope: rot must be a multiple of 16 in 16..head_dim");
    if (p->table_rows <= 0 || !aligned16(p->cos) || !aligned16(p->sin))
      return set_error(WANB200_EINVAL, "head_norm_rope: rotation needs 16-byte aligned tables and table_rows > 0");
  } else if (!p->gamma[0] && (p->nsections == 1 || !p->gamma[1])) {
    return set_error(WANB200_EINVAL, "head_norm_rope: neither a gamma nor a rotation");
  }
  int* err = device_error_word();
  if (!err) return WANB200_ECUDA;
  HeadNormArgs a;
  a.x = reinterpret_cast<const __nv_bfloat16*>(p->x);
  a.out = reinterpret_cast<__nv_bfloat16*>(p->out);
  a.ldx = p->ldx;
  a.ldo = p->ldo;
  a.rows = p->rows;
  a.col0[0] = p->col0[0];
  a.col0[1] = p->nsections > 1 ? p->col0[1] : 0;
  a.heads0 = p->heads[0];
  a.heads1 = p->nsections > 1 ? p->heads[1] : 0;
  a.gamma[0] = reinterpret_cast<const __nv_bfloat16*>(p->gamma[0]);
  a.gamma[1] = p->nsections > 1 ? reinterpret_cast<const __nv_bfloat16*>(p->gamma[1]) : nullptr;
  a.eps = p->eps;
  a.rot = p->cos ? p->rot : 0;
  a.cos = p->cos;
  a.sin = p->sin;
  a.positions = p->cos ? p->positions : nullptr;
  a.table_rows = p->cos ? p->table_rows : 1;
  a.err = err;
  const int lph = p->head_dim / 8, hp = 32 / lph;
  // The passes of a warp: six where that leaves every SM its 32 warps and at most half as many idle
  // passes again (a section's heads fill whole warps), two where that leaves 16, else one, for latency.
  // Measured (us, 1 / 2 / 6 passes): 1 row of 48 heads of 128 2.2 / 2.3 / 3.2; 640 rows 6.0 / 4.8 / 5.0;
  // 15708 rows 109 / 79 / 69, of 32 + 8 heads of 64 (8 + 2 passes in 18 places) 47 / 35 / 41, of 16 + 2
  // heads of 256 (18 in 24) 83 / 68 / 62.
  const int64_t p0 = (a.heads0 + hp - 1) / hp, p1 = (a.heads1 + hp - 1) / hp, fill = (int64_t)num_sms() * 32;
  const int64_t warps6 = (p0 + 5) / 6 + (p1 + 5) / 6, warps2 = (p0 + 1) / 2 + (p1 + 1) / 2;
  const int nv = p->rows * warps6 >= fill && 4 * warps6 <= p0 + p1 ? 6 : p->rows * warps2 >= fill / 2 ? 2 : 1;
  a.groups0 = (a.heads0 + hp * nv - 1) / (hp * nv);
  a.groups = a.groups0 + (a.heads1 + hp * nv - 1) / (hp * nv);
  const int64_t blocks = (p->rows * a.groups + 7) / 8;
  if (p->rows > INT32_MAX || blocks > INT32_MAX) return set_error(WANB200_EINVAL, "head_norm_rope: too many rows");
  if (lph == 8)
    launch_head_norm<8>(a, nv, p->interleaved != 0, (unsigned)blocks, st);
  else if (lph == 16)
    launch_head_norm<16>(a, nv, p->interleaved != 0, (unsigned)blocks, st);
  else
    launch_head_norm<32>(a, nv, p->interleaved != 0, (unsigned)blocks, st);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error("head_norm_rope_kernel launch", e);
  return WANB200_OK;
}

}  // namespace wanb200
