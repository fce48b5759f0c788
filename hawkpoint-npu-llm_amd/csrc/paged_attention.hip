// Attention of a batch's new tokens over a paged KV cache (hk_paged_attention).
//
// Row (token t of an entry, head h) stands at position p = length - count + t
// and sees the slots j <= p (with a window, j > p - window) whose page exists:
//   s_j = scale (q . k_j),  m = max s_j,  l = sum exp(s_j - m)
//   out = sum exp(s_j - m) v_j / l,  lse = m + ln l
#include "hk_common.h"
#include "hk_internal.h"
#include "paged.h"

namespace hk {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// A pool element as a float.
template <bool E4M3>
__device__ __forceinline__ float pool_value(const char* p, int64_t i) {
  if constexpr (E4M3) return __builtin_amdgcn_cvt_f32_fp8(((const uint8_t*)p)[i], 0);
  return bf16_to_f32(((const uint16_t*)p)[i]);
}

// One wave per row: 64 slots at a time, a lane per slot for the scores, a lane
// per D / 64 dimensions for P @ V.
template <int D, bool E4M3>
__global__ __launch_bounds__(64) void paged_attention_row_kernel(PagedAttnArgs a) {
  constexpr int kPer = D / 64;
  __shared__ float qs[D], ps[64];
  __shared__ int64_t at[64];
  __shared__ int found;
  const int tok = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, g = h / a.group;
  if (lane == 0) found = -1;
  __syncthreads();
  for (int e = lane; e < a.b.n; e += 64) {
    const int2 r = entry_rows(a.b, e);
    if (tok >= r.x && tok < r.y) found = e;
  }
  __syncthreads();
  const int e = found;
  if (e < 0) return;
  const int2 r = entry_rows(a.b, e), s = entry_seq(a.c, a.b, e);
  const int p = s.y - r.y + tok;
  const int low = a.window > 0 ? max(0, p - a.window + 1) : 0;
  for (int d = lane; d < D; d += 64) qs[d] = bf16_to_f32(a.q[tok * a.q_stride + h * D + d]);
  const float ks = (E4M3 ? a.c.k_scale[g] : 1.0f) * a.scale * kLog2e, vs = E4M3 ? a.c.v_scale[g] : 1.0f;
  float m = -INFINITY, l = 0.0f, o[kPer] = {};
  for (int j0 = low & ~63; j0 <= p; j0 += 64) {
    const int j = j0 + lane;
    int page = -1;
    if (j >= low && j <= p) page = a.c.table[(int64_t)s.x * a.c.width + (j >> a.c.page_shift)];
    const bool on = (unsigned)page < (unsigned)a.c.pages;
    const int slot = j & ((1 << a.c.page_shift) - 1);
    const int64_t off = on ? page * a.c.page_bytes + (((int64_t)g << a.c.page_shift) + slot) * D * a.c.elt : 0;
    __syncthreads();
    float sc = -INFINITY;
    if (on) {
      float d = 0.0f;
      for (int i = 0; i < D; ++i) d = fmaf(qs[i], pool_value<E4M3>(a.c.k + off, i), d);
      sc = d * ks;
    }
    const float m_new = fmaxf(m, group_max<64>(sc)), m_use = m_new == -INFINITY ? 0.0f : m_new;
    const float e2 = on ? __builtin_amdgcn_exp2f(sc - m_use) : 0.0f, f = __builtin_amdgcn_exp2f(m - m_use);
    l = l * f + group_sum<64>(e2);
    m = m_new;
    ps[lane] = e2;
    at[lane] = on ? off : -1;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kPer; ++q) o[q] *= f;
    for (int i = 0; i < 64; ++i) {
      if (at[i] < 0) continue;
#pragma unroll
      for (int q = 0; q < kPer; ++q) o[q] = fmaf(ps[i], pool_value<E4M3>(a.c.v + at[i], lane + 64 * q), o[q]);
    }
  }
#pragma unroll
  for (int q = 0; q < kPer; ++q)
    a.out[tok * a.out_stride + h * D + lane + 64 * q] = (uint16_t)f32_to_bf16(l == 0.0f ? 0.0f : o[q] / l * vs);
  if (a.lse && lane == 0)
    a.lse[(int64_t)tok * a.q_heads + h] = l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

}  // namespace

int launch_paged_attention(const PagedAttnArgs& a, int head_dim, hipStream_t stream) {
  const dim3 grid(a.b.tokens, a.q_heads);
  if (head_dim == 64 && a.c.elt == 2)
    hipLaunchKernelGGL((paged_attention_row_kernel<64, false>), grid, dim3(64), 0, stream, a);
  else if (head_dim == 64)
    hipLaunchKernelGGL((paged_attention_row_kernel<64, true>), grid, dim3(64), 0, stream, a);
  else if (a.c.elt == 2)
    hipLaunchKernelGGL((paged_attention_row_kernel<128, false>), grid, dim3(64), 0, stream, a);
  else
    hipLaunchKernelGGL((paged_attention_row_kernel<128, true>), grid, dim3(64), 0, stream, a);
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? 0 : hip_fail(err, "paged attention launch");
}

}  // namespace hk
