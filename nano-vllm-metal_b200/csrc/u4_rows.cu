// u4_rows.cu -- rows of the 4-bit cache: the scatter-write that quantises them, and the gather that
// reads slots of any page type back as values (u4.cuh has the format).
//
// Both move each byte once and compute a few operations an element.  One warp takes one (token, kv
// head) row of K and the same row of V.
#include "nvm_internal.h"
#include "u4.cuh"

namespace nvm {
namespace {

constexpr int kWarps = 8;

// Element offsets of a row: lane l holds elements 2l, 2l + 1 of group 0 (and of group 1, D = 128).
template <typename T>
__device__ __forceinline__ void write_row(const void* src, int64_t at, int dtype, uint8_t* codes, T* scales, int groups,
                                          int lane) {
  for (int g = 0; g < groups; ++g) {
    const float a = load_dyn(src, at + g * kU4Group + 2 * lane, dtype);
    const float b = load_dyn(src, at + g * kU4Group + 2 * lane + 1, dtype);
    float hi = max_nan(a, b), lo = max_nan(-a, -b);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      lo = max_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
    const float2 sz = u4_scale<T>(-lo, hi);
    const float r = u4_inverse(sz.x);
    bool amb_a, amb_b;
    int ca = u4_code_fast(a, sz.y, r, amb_a), cb = u4_code_fast(b, sz.y, r, amb_b);
    if (amb_a) ca = u4_code_div(a, sz.y, sz.x);
    if (amb_b) cb = u4_code_div(b, sz.y, sz.x);
    codes[g * (kU4Group / 2) + lane] = (uint8_t)(ca | cb << 4);
    if (lane == 0) reinterpret_cast<uint32_t*>(scales)[g] = u4_pack_pair<T>(sz);
  }
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
    u4_write_kernel(const void* k, const void* v, int dtype, int64_t st, int64_t sh, uint8_t* kp, uint8_t* vp, T* ks, T* vs,
                    const int64_t* slots, int64_t tokens, int64_t Hkv, int D, int64_t P, int64_t ps) {
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (w >= tokens * Hkv) return;
  const int64_t t = w / Hkv, h = w - t * Hkv, slot = slots[t];
  if (slot < 0 || slot / ps >= P) return;
  const int64_t row = (slot / ps * Hkv + h) * ps + slot % ps, at = t * st + h * sh;
  const int groups = D / kU4Group;
  write_row<T>(k, at, dtype, kp + row * (D / 2), ks + row * 2 * groups, groups, lane);
  write_row<T>(v, at, dtype, vp + row * (D / 2), vs + row * 2 * groups, groups, lane);
}

__device__ __forceinline__ float row_value(const void* pages, int kv_dtype, const void* scales, int scale_dtype, int64_t row,
                                           int64_t D, int64_t d) {
  if (kv_dtype == NVM_U4) {
    const int64_t g = row * (D / kU4Group) + d / kU4Group;
    const int code = static_cast<const uint8_t*>(pages)[row * (D / 2) + d / 2] >> (d % 2 * 4) & 15;
    return fmaf(load_dyn(scales, 2 * g, scale_dtype), (float)code, load_dyn(scales, 2 * g + 1, scale_dtype));
  }
  const float x = load_dyn(pages, row * D + d, kv_dtype);
  return kv_dtype == NVM_I8 ? __fmul_rn(x, load_dyn(scales, row, scale_dtype)) : x;
}

__global__ void __launch_bounds__(kWarps * 32)
    read_slots_kernel(const void* kp, const void* vp, int kv_dtype, const void* ks, const void* vs, int scale_dtype,
                      const int64_t* slots, void* k, void* v, int out_dtype, int64_t tokens, int64_t Hkv, int64_t D, int64_t P,
                      int64_t ps) {
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (w >= tokens * Hkv) return;
  const int64_t t = w / Hkv, h = w - t * Hkv, slot = slots[t];
  const bool there = slot >= 0 && slot / ps < P;
  const int64_t row = there ? (slot / ps * Hkv + h) * ps + slot % ps : 0;
  for (int64_t d = lane; d < D; d += 32) {
    store_dyn(k, w * D + d, out_dtype, there ? row_value(kp, kv_dtype, ks, scale_dtype, row, D, d) : 0.0f);
    store_dyn(v, w * D + d, out_dtype, there ? row_value(vp, kv_dtype, vs, scale_dtype, row, D, d) : 0.0f);
  }
}

}  // namespace

int launch_u4_write(const void* k, const void* v, int in_dtype, int64_t stride_t, int64_t stride_h, void* k_pages, void* v_pages,
                    void* k_scales, void* v_scales, int scale_dtype, const int64_t* slots, int64_t T, int64_t Hkv, int64_t D,
                    int64_t P, int64_t page_size, cudaStream_t s) {
  const unsigned grid = (unsigned)((T * Hkv + kWarps - 1) / kWarps);
  uint8_t *kp = static_cast<uint8_t*>(k_pages), *vp = static_cast<uint8_t*>(v_pages);
  if (scale_dtype == NVM_BF16)
    u4_write_kernel<<<grid, kWarps * 32, 0, s>>>(k, v, in_dtype, stride_t, stride_h, kp, vp,
                                                 static_cast<__nv_bfloat16*>(k_scales), static_cast<__nv_bfloat16*>(v_scales),
                                                 slots, T, Hkv, (int)D, P, page_size);
  else
    u4_write_kernel<<<grid, kWarps * 32, 0, s>>>(k, v, in_dtype, stride_t, stride_h, kp, vp, static_cast<__half*>(k_scales),
                                                 static_cast<__half*>(v_scales), slots, T, Hkv, (int)D, P, page_size);
  return check_cuda(cudaGetLastError(), "write_page_slice: kernel launch");
}

int launch_read_slots(const void* k_pages, const void* v_pages, int kv_dtype, const void* k_scales, const void* v_scales,
                      int scale_dtype, const int64_t* slots, void* k, void* v, int out_dtype, int64_t T, int64_t Hkv, int64_t D,
                      int64_t P, int64_t page_size, cudaStream_t s) {
  read_slots_kernel<<<(unsigned)((T * Hkv + kWarps - 1) / kWarps), kWarps * 32, 0, s>>>(
      k_pages, v_pages, kv_dtype, k_scales, v_scales, scale_dtype, slots, k, v, out_dtype, T, Hkv, D, P, page_size);
  return check_cuda(cudaGetLastError(), "read_slots: kernel launch");
}

}  // namespace nvm
