// paged_u4.cu -- paged attention over a cache held in 4 bits (u4.cuh has the row format).
//
// Semantics are those of the other paged kernels: positions at or past min(ctx, max_pages * page_size),
// holes (page id < 0 or >= P) and, with the causal limit, keys after l + ctx - L are skipped; a row that
// sees nothing is zero, and a key that no row sees has no influence whatever it holds.
#include "nvm_internal.h"
#include "u4.cuh"

namespace nvm {
namespace {

constexpr int kWarps = 4;

// One warp a query row: lane j scores key j of 32, then every lane adds its elements of V.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32) paged_u4_rows_kernel(const PagedArgs a) {
  __shared__ float qs[kWarps][128];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = (int)a.D, groups = D / kU4Group;
  const int64_t row = (int64_t)blockIdx.x * kWarps + warp;
  if (row >= a.B * a.Hq * a.L) return;
  const int64_t n = row / a.L, l = row % a.L, b = n / a.Hq, kvh = n % a.Hq / (a.Hq / a.Hkv);
  const int64_t ctx = a.context_lens[b], cap = a.max_pages * a.page_size;
  int64_t keys = ctx < cap ? ctx : cap;
  if (a.is_causal && l + ctx - a.L + 1 < keys) keys = l + ctx - a.L + 1;
  for (int d = lane; d < D; d += 32) qs[warp][d] = load_dyn(a.q, row * D + d, a.q_dtype);
  __syncwarp();
  const uint8_t *kp = static_cast<const uint8_t*>(a.k_pages), *vp = static_cast<const uint8_t*>(a.v_pages);
  const uint32_t *ks = static_cast<const uint32_t*>(a.k_scales), *vs = static_cast<const uint32_t*>(a.v_scales);
  float m = -INFINITY, sum = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int64_t j0 = 0; j0 < keys; j0 += 32) {
    const int64_t key = j0 + lane;
    int64_t at = -1;
    if (key < keys) {
      const int64_t pid = a.block_table[b * a.max_pages + key / a.page_size];
      if (pid >= 0 && pid < a.P) at = (pid * a.Hkv + kvh) * a.page_size + key % a.page_size;
    }
    float s = -INFINITY;
    if (at >= 0) {
      s = 0.0f;
      for (int g = 0; g < groups; ++g) {
        const float2 sz = u4_pair<T>(ks[at * groups + g]);
        for (int d = 0; d < kU4Group; d += 2) {
          const int byte = kp[at * (D / 2) + (g * kU4Group + d) / 2];
          s += qs[warp][g * kU4Group + d] * fmaf(sz.x, (float)(byte & 15), sz.y);
          s += qs[warp][g * kU4Group + d + 1] * fmaf(sz.x, (float)(byte >> 4), sz.y);
        }
      }
      s *= a.scale;
    }
    const float m_new = fmaxf(m, warp_max(s));
    if (m_new == -INFINITY) continue;
    const float fade = expf(m - m_new), p = at >= 0 ? expf(s - m_new) : 0.0f;
    sum = sum * fade + warp_sum(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= fade;
    for (int j = 0; j < 32; ++j) {
      const int64_t atj = __shfl_sync(0xffffffffu, at, j);
      const float pj = __shfl_sync(0xffffffffu, p, j);
      if (atj < 0) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = lane + 32 * i;
        if (d >= D) continue;
        const float2 sz = u4_pair<T>(vs[atj * groups + d / kU4Group]);
        acc[i] += pj * fmaf(sz.x, (float)(vp[atj * (D / 2) + d / 2] >> (d % 2 * 4) & 15), sz.y);
      }
    }
    m = m_new;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i < D) store_dyn(a.out, row * D + lane + 32 * i, a.out_dtype, sum == 0.0f ? 0.0f : acc[i] / sum);
}

}  // namespace

int launch_paged_u4(const PagedArgs& a, cudaStream_t s) {
  const unsigned grid = (unsigned)((a.B * a.Hq * a.L + kWarps - 1) / kWarps);
  if (a.scale_dtype == NVM_BF16)
    paged_u4_rows_kernel<__nv_bfloat16><<<grid, kWarps * 32, 0, s>>>(a);
  else
    paged_u4_rows_kernel<__half><<<grid, kWarps * 32, 0, s>>>(a);
  return check_cuda(cudaGetLastError(), "paged_attention: 4-bit kernel launch");
}

}  // namespace nvm
