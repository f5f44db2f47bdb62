// paged_mma_window.cu -- instances of the tensor-core paged attention kernel (paged_mma.cuh)
// with a sliding window, sinks and row log-sum-exps, one per default variant of the plan.
// Measured on a B200: 64 requests of 4K-16K keys under a window of 4096 with 4 sinks, 32/8 heads,
// bf16: 170-177 us, 6.1-6.3 TB/s of the keys seen (0.93-0.96 of a copy's rate); 48 requests under 2048, 64/8
// heads, int8 pages: 59 us, 3.5 TB/s, bound by latency: two chunks a unit make 768 CTAs of 1184 slots,
// 9.5 warps an SM, which the int8 tile's conversions keep waiting (0.45 instructions a cycle).
#include "paged_mma.cuh"

namespace nvm {
namespace {

template <typename KvT, typename ScaleT, int D>
int launch_window_d(const PagedArgs& a, const MmaPlan& plan, void* ws, cudaStream_t s) {
  switch (plan.nwm) {
    case 0:
      return plan.variant == 2 ? launch_cfg<KvT, ScaleT, D, 0, 2, 2, true>(a, plan, ws, s)
                               : launch_cfg<KvT, ScaleT, D, 0, 2, 4, true>(a, plan, ws, s);
    case 1: return launch_cfg<KvT, ScaleT, D, 1, 2, 6, true>(a, plan, ws, s);
    case 2: return launch_cfg<KvT, ScaleT, D, 2, 2, 0, true>(a, plan, ws, s);
    case 3: return launch_cfg<KvT, ScaleT, D, 3, 1, 4, true>(a, plan, ws, s);
    default: return launch_cfg<KvT, ScaleT, D, 4, 1, 0, true>(a, plan, ws, s);
  }
}

}  // namespace

int launch_paged_mma_window(const PagedArgs& a, const MmaPlan& plan, void* ws, cudaStream_t s) {
  if (a.kv_dtype == NVM_F16) {
    return a.D == 64 ? launch_window_d<__half, __half, 64>(a, plan, ws, s)
                     : launch_window_d<__half, __half, 128>(a, plan, ws, s);
  }
  if (a.kv_dtype == NVM_BF16) {
    return a.D == 64 ? launch_window_d<__nv_bfloat16, __nv_bfloat16, 64>(a, plan, ws, s)
                     : launch_window_d<__nv_bfloat16, __nv_bfloat16, 128>(a, plan, ws, s);
  }
  if (a.scale_dtype == NVM_F16) return launch_window_d<int8_t, __half, 128>(a, plan, ws, s);
  return launch_window_d<int8_t, __nv_bfloat16, 128>(a, plan, ws, s);
}

}  // namespace nvm
