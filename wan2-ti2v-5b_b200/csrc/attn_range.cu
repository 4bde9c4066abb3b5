// Attention over one key range per query row:
//   s_ij = scale q_i . k_j,  s' = cap tanh(s / cap)  (cap > 0),  t = s' + b_h(j - pos_i),
//   o_i = sum_{lo_i <= j < hi_i} e^(t_ij) v_j / sum e^(t_ij);  an empty range gives o_i = 0.
// Document, causal, frame-causal, prefix, window and padding masks all are one range per row.
#include "common.cuh"
#include "internal.h"

namespace wanb200 {

constexpr float RA_LOG2E = 1.4426950408889634f;

struct RangeArgs {
  const __nv_bfloat16 *q, *k, *v;
  __nv_bfloat16* o;
  int64_t q_tok, q_batch, k_tok, k_batch, v_tok, v_batch, o_tok, o_batch;
  int batch, heads, group, q_len, kv_len;
  float scale, cap;
  const int32_t *lo, *hi, *pos;
  int64_t range_batch;  // elements between the batches of lo / hi / pos, 0 when they are shared
  const float* slopes;  // [heads]
  const float* table;   // [heads, 2 * reach + 1]
  int reach;
};

// One warp per (batch, row, head); lane l holds D / 32 channels.  The straightforward form: one
// key after the other with the running maximum and sum.
template <int D>
__global__ void __launch_bounds__(256) range_attn_rows_kernel(const RangeArgs a) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (w >= (int64_t)a.batch * a.q_len * a.heads) return;
  const int h = (int)(w % a.heads);
  const int64_t bi = w / a.heads;
  const int i = (int)(bi % a.q_len), b = (int)(bi / a.q_len);
  const int64_t r = b * a.range_batch + i;
  const int lo = max(__ldg(a.lo + r), 0), hi = min(__ldg(a.hi + r), a.kv_len);
  const int pos = a.pos ? __ldg(a.pos + r) : i;
  float q[E], o[E];
  const __nv_bfloat16* qp = a.q + b * a.q_batch + i * a.q_tok + (int64_t)h * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = __bfloat162float(qp[e]) * a.scale;
    o[e] = 0.f;
  }
  const int kh = h / a.group;
  float m = -INFINITY, l = 0.f;
  for (int j = lo; j < hi; ++j) {
    const __nv_bfloat16* kp = a.k + b * a.k_batch + j * a.k_tok + (int64_t)kh * D + lane * E;
    const __nv_bfloat16* vp = a.v + b * a.v_batch + j * a.v_tok + (int64_t)kh * D + lane * E;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(q[e], __bfloat162float(kp[e]), s);
#pragma unroll
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    if (a.cap > 0.f) s = a.cap * tanhf(s / a.cap);
    if (a.slopes) s -= __ldg(a.slopes + h) * fabsf((float)(j - pos));
    if (a.table) s += __ldg(a.table + (int64_t)h * (2 * a.reach + 1) + min(max(j - pos, -a.reach), a.reach) + a.reach);
    const float mn = fmaxf(m, s);
    const float corr = m == mn ? 1.f : ex2_approx((m - mn) * RA_LOG2E), p = ex2_approx((s - mn) * RA_LOG2E);
    m = mn;
    l = l * corr + p;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * corr + p * __bfloat162float(vp[e]);
  }
  __nv_bfloat16* op = a.o + b * a.o_batch + i * a.o_tok + (int64_t)h * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) op[e] = __float2bfloat16(lo < hi ? o[e] / l : 0.f);
}

int64_t range_attn_workspace_bytes(const wanb200_range_attn_params*) { return 0; }

int range_attn_fwd(const wanb200_range_attn_params* p, cudaStream_t st) {
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
  a.heads = (int)p->heads;
  a.group = (int)(p->heads / p->kv_heads);
  a.q_len = (int)p->q_len;
  a.kv_len = (int)p->kv_len;
  a.scale = p->softmax_scale;
  a.cap = p->softcap;
  a.lo = p->lo;
  a.hi = p->hi;
  a.pos = p->pos;
  a.range_batch = p->range_batch_stride;
  a.slopes = p->slopes;
  a.table = p->dist_bias;
  a.reach = p->reach;
  const int64_t blocks = (p->batch * p->q_len * p->heads + 7) / 8;
  if (blocks > INT32_MAX) return set_error(WANB200_EINVAL, "range_attn: too many rows");
  if (p->head_dim == 64)
    range_attn_rows_kernel<64><<<(unsigned)blocks, 256, 0, st>>>(a);
  else
    range_attn_rows_kernel<128><<<(unsigned)blocks, 256, 0, st>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error("range attention launch", e);
  return WANB200_OK;
}

}  // namespace wanb200
