// key_mass.cu -- accumulated attention weight of every cached key.
//
// For kv head h of sequence b, with rows (q head i of h's group, query token l) at
// positions pos = l + ctx - L:
//   mass[b, h, s] = (s < ctx - L ? mass[b, h, s] : 0) + sum_rows 2^(z[row, s] - lse[row])
// where z is the scaled score in base 2 and lse[row] = log2 sum_s 2^z[row, s] comes from
// the attention kernel that ran before on the same stream (+inf for a row without a key,
// which then gives every key weight 0).  Keys of unmapped pages gain nothing.  No atomics:
// one warp owns a key, so results do not depend on the order of anything.
#include "nvm_common.cuh"
#include "nvm_internal.h"

namespace nvm {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct MassParams {
  const void* q;
  const void* k;
  const void* ks;
  const int32_t* block_table;
  const int32_t* context_lens;
  const float* lse;
  float* mass;
  int64_t stride_b, stride_h, len;
  int q_dtype, kv_dtype, scale_dtype;
  int64_t B, Hq, Hkv, L, D, P, ps, mp, g;
  float scale_log2;
  int causal;
  int64_t window, sinks;
};

// Any head dim <= 256, page size and dtype: a warp per key, lanes along the query rows.
constexpr int kGenWarps = 4;
__global__ void __launch_bounds__(kGenWarps * 32) key_mass_generic_kernel(MassParams p) {
  __shared__ float krow[kGenWarps][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t b = blockIdx.y / p.Hkv, h = blockIdx.y % p.Hkv;
  const int64_t ctx = p.context_lens[b];
  const int64_t cap = p.mp * p.ps;
  int64_t end = ctx < cap ? ctx : cap;
  if (p.len < end) end = p.len;
  for (int64_t s = (int64_t)blockIdx.x * kGenWarps + warp; s < end; s += (int64_t)gridDim.x * kGenWarps) {
    const int64_t page = s / p.ps, off = s - page * p.ps;
    const int64_t pid = p.block_table[b * p.mp + page];
    float sum = 0.f;
    if (pid >= 0 && pid < p.P) {
      const int64_t base = (pid * p.Hkv + h) * p.ps + off;
      const float ksc = p.kv_dtype == NVM_I8 ? load_dyn(p.ks, base, p.scale_dtype) : 1.f;
      for (int64_t d = lane; d < p.D; d += 32) krow[warp][d] = load_dyn(p.k, base * p.D + d, p.kv_dtype);
      __syncwarp();
      for (int64_t r = lane; r < p.g * p.L; r += 32) {
        const int64_t l = r % p.L, pos = l + ctx - p.L;
        const bool seen = (!p.causal || s <= pos) && (p.window == 0 || s < p.sinks || s > pos - p.window);
        if (!seen) continue;
        const int64_t row = (b * p.Hq + h * p.g) * p.L + r;
        float dot = 0.f;
        for (int64_t d = 0; d < p.D; ++d) dot += load_dyn(p.q, row * p.D + d, p.q_dtype) * krow[warp][d];
        if (p.kv_dtype == NVM_I8) dot *= ksc;
        sum += exp2f(dot * p.scale_log2 - p.lse[row]);
      }
      __syncwarp();
      sum = warp_sum(sum);
    }
    if (lane == 0) {
      float* m = p.mass + b * p.stride_b + h * p.stride_h + s;
      *m = (s < ctx - p.L ? *m : 0.f) + sum;
    }
  }
}

}  // namespace

int launch_key_mass(const PagedArgs& a, const KeyMassArgs& m, cudaStream_t s) {
  MassParams p{};
  p.q = a.q; p.k = a.k_pages; p.ks = a.k_scales; p.block_table = a.block_table; p.context_lens = a.context_lens;
  p.lse = a.lse; p.mass = m.mass; p.stride_b = m.stride_b; p.stride_h = m.stride_h; p.len = m.len;
  p.q_dtype = a.q_dtype; p.kv_dtype = a.kv_dtype; p.scale_dtype = a.scale_dtype;
  p.B = a.B; p.Hq = a.Hq; p.Hkv = a.Hkv; p.L = a.L; p.D = a.D; p.P = a.P; p.ps = a.page_size; p.mp = a.max_pages;
  p.g = a.Hq / a.Hkv;
  p.scale_log2 = a.scale * kLog2e;
  p.causal = a.is_causal; p.window = a.window; p.sinks = a.sinks;
  int64_t keys = a.max_pages * a.page_size;
  if (m.len < keys) keys = m.len;
  if (keys <= 0 || a.B * a.Hkv == 0) return NVM_OK;
  int64_t bx = (keys + kGenWarps - 1) / kGenWarps;
  if (bx > 65536) bx = 65536;
  const dim3 grid((unsigned)bx, (unsigned)(a.B * a.Hkv));
  key_mass_generic_kernel<<<grid, kGenWarps * 32, 0, s>>>(p);
  return check_cuda(cudaGetLastError(), "paged_attention: key mass kernel launch");
}

}  // namespace nvm
