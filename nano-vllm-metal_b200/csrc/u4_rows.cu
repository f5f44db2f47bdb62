// u4_rows.cu -- rows of the 4-bit cache: the scatter-write that quantises them, and the gather that
// reads slots of any page type back as values (u4.cuh has the format).
//
// Both are bound by HBM and move each byte once: a thread owns eight elements of a K row and the same
// eight of the V row, 16 bytes on the 16-bit side and a word of codes on the other, so that both sides
// of a warp are whole lines; a group's 64 elements lie in eight neighbouring lanes, three shuffles
// from their extremes.  Four rows are in flight a thread when reading (two or eight 74 us for 72).
// 16 requests of 2K-8K tokens, 8 heads, bf16, are read in 72 us, 0.89 of a copy's rate; 8192 rows of 8 heads are
// written in 23 us, their slots in no order.
#include <algorithm>

#include "nvm_internal.h"
#include "u4.cuh"

namespace nvm {
namespace {

constexpr int kThreads = 128;  // 256: 79 us for 72
constexpr int kRead = 4;  // rows a thread reads at a time

struct RowsParams {
  const void* k;  // values, [tokens, Hkv, D] when reading
  const void* v;
  int64_t st, sh;  // elements between tokens and heads of the values when writing
  void* kp;
  void* vp;
  void* ks;
  void* vs;
  const int64_t* slots;
  int64_t P, ps;
  uint32_t items, Hkv, parts;  // items: threads with work, tokens * Hkv * parts; parts: D / 8
  FastDiv by_parts, by_heads, by_ps;
  int dtype, kv_dtype, scale_dtype, fast;  // fast: 16-byte vectors of the values, whole ones of the pages
};

// Where an item's row lies in the pool (false: it is skipped).
__device__ __forceinline__ bool find_row(const RowsParams& p, uint32_t item, uint32_t& t, uint32_t& h, uint32_t& part, int64_t& row) {
  const uint32_t w = p.by_parts(item);
  part = item - w * p.parts;
  t = p.by_heads(w);
  h = w - t * p.Hkv;
  const int64_t slot = __ldg(p.slots + t);
  if (slot < 0) return false;
  int64_t pid, off;
  if (slot <= 0x7fffffffLL) {  // a 64-bit division costs as much as the rest
    pid = p.by_ps((uint32_t)slot);
    off = (uint32_t)slot - (uint32_t)pid * (uint32_t)p.ps;
  } else {
    pid = slot / p.ps;
    off = slot - pid * p.ps;
  }
  row = (pid * p.Hkv + h) * p.ps + off;
  return pid < p.P;
}

__device__ __forceinline__ void unpack16(uint4 u, int dtype, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = dtype == NVM_BF16 ? u4_pair<__nv_bfloat16>(w[i]) : u4_pair<__half>(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

__device__ __forceinline__ void load8(const void* src, int64_t at, int dtype, bool fast, float (&x)[8]) {
  if (!fast) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = load_dyn(src, at + i, dtype);
  } else if (dtype == NVM_F32) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(src) + at));
    const float4 b = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(src) + at) + 1);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
    unpack16(__ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(src) + at)), dtype, x);
  }
}

// Eight lanes hold a group, eight elements each.
template <typename T>
__device__ __forceinline__ void write8(const float (&x)[8], uint8_t* codes, T* scales, int64_t row, uint32_t parts, uint32_t part,
                                       bool there) {
  float hi = x[0], lo = -x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    hi = max_nan(hi, x[i]);
    lo = max_nan(lo, -x[i]);
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    lo = max_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
  }
  const float2 sz = u4_scale<T>(-lo, hi);
  const float r = u4_inverse(sz.x);
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    bool amb;
    int c = u4_code_fast(x[i], sz.y, r, amb);
    if (amb) c = u4_code_div(x[i], sz.y, sz.x);
    word |= (uint32_t)c << (4 * i);
  }
  if (!there) return;
  reinterpret_cast<uint32_t*>(codes)[row * parts + part] = word;
  if (part % 8 == 0) reinterpret_cast<uint32_t*>(scales)[(row * parts + part) / 8] = u4_pack_pair<T>(sz);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) u4_write_kernel(const RowsParams p) {
  const uint32_t item = blockIdx.x * kThreads + threadIdx.x;
  uint32_t t = 0, h = 0, part = 0;
  int64_t row = 0;
  const bool there = item < p.items && find_row(p, item, t, h, part, row);
  float k[8] = {}, v[8] = {};
  if (there) {
    const int64_t at = t * p.st + h * p.sh + part * 8;
    load8(p.k, at, p.dtype, p.fast, k);
    load8(p.v, at, p.dtype, p.fast, v);
  }
  write8<T>(k, static_cast<uint8_t*>(p.kp), static_cast<T*>(p.ks), row, p.parts, part, there);
  write8<T>(v, static_cast<uint8_t*>(p.vp), static_cast<T*>(p.vs), row, p.parts, part, there);
}

// Eight elements of a pool row as they lie there.
template <int kKind>
struct Raw;
template <>
struct Raw<NVM_U4> {
  uint32_t codes, pair;
  __device__ __forceinline__ void load(const void* pages, const void* scales, int64_t row, uint32_t parts, uint32_t part) {
    codes = __ldg(static_cast<const uint32_t*>(pages) + row * parts + part);
    pair = __ldg(static_cast<const uint32_t*>(scales) + (row * parts + part) / 8);
  }
  __device__ __forceinline__ void values(int scale_dtype, float (&x)[8]) const {
    const float2 sz = scale_dtype == NVM_BF16 ? u4_pair<__nv_bfloat16>(pair) : u4_pair<__half>(pair);
    // the codes at 4 i and 4 i + 16 are the f16 subnormals code * 2^-24 once shifted: exact, two an operation;
    // the factor goes to the code, since bf16 scales go up to 2^124
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = codes >> (4 * i) & 0x000f000fu;
      const float2 c = __half22float2(*reinterpret_cast<const __half2*>(&w));
      x[i] = fmaf(sz.x, c.x * 0x1p24f, sz.y);
      x[i + 4] = fmaf(sz.x, c.y * 0x1p24f, sz.y);
    }
  }
};
template <>
struct Raw<NVM_I8> {
  uint2 q;
  float scale;
  __device__ __forceinline__ void load(const void* pages, const void* scales, int64_t row, uint32_t parts, uint32_t part, int dtype) {
    q = __ldg(static_cast<const uint2*>(pages) + row * parts + part);
    scale = load_dyn(scales, row, dtype);
  }
  __device__ __forceinline__ void values(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __fmul_rn((float)(int8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3))), scale);
  }
};

__device__ __forceinline__ void store8(void* dst, int64_t at, int dtype, const float (&x)[8]) {
  if (dtype == NVM_F32) {
    float4* d = reinterpret_cast<float4*>(static_cast<float*>(dst) + at);
    d[0] = make_float4(x[0], x[1], x[2], x[3]);
    d[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = dtype == NVM_BF16 ? pack2<__nv_bfloat16>(x[2 * i], x[2 * i + 1]) : pack2<__half>(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(dst) + at) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <int kKind>
__global__ void __launch_bounds__(kThreads) read_slots_kernel(const RowsParams p) {
  const uint32_t item0 = blockIdx.x * (kThreads * kRead) + threadIdx.x;
  if constexpr (kKind == NVM_U4) {
    Raw<NVM_U4> k[kRead] = {}, v[kRead] = {};
#pragma unroll
    for (int i = 0; i < kRead; ++i) {  // a slot that is not there keeps zeros: value 0 * 0 + 0
      const uint32_t item = item0 + i * kThreads;
      uint32_t t, h, part;
      int64_t row;
      if (item < p.items && find_row(p, item, t, h, part, row)) {
        k[i].load(p.kp, p.ks, row, p.parts, part);
        v[i].load(p.vp, p.vs, row, p.parts, part);
      }
    }
#pragma unroll
    for (int i = 0; i < kRead; ++i) {
      const uint32_t item = item0 + i * kThreads;
      if (item >= p.items) return;
      float x[8];
      k[i].values(p.scale_dtype, x);
      store8(const_cast<void*>(p.k), (int64_t)item * 8, p.dtype, x);
      v[i].values(p.scale_dtype, x);
      store8(const_cast<void*>(p.v), (int64_t)item * 8, p.dtype, x);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kRead; ++i) {
      const uint32_t item = item0 + i * kThreads;
      if (item >= p.items) return;
      uint32_t t, h, part;
      int64_t row;
      float x[8] = {}, y[8] = {};
      if (find_row(p, item, t, h, part, row)) {
        if constexpr (kKind == NVM_I8) {
          Raw<NVM_I8> k, v;
          k.load(p.kp, p.ks, row, p.parts, part, p.scale_dtype);
          v.load(p.vp, p.vs, row, p.parts, part, p.scale_dtype);
          k.values(x);
          v.values(y);
        } else {
          load8(p.kp, (row * p.parts + part) * 8, p.kv_dtype, true, x);
          load8(p.vp, (row * p.parts + part) * 8, p.kv_dtype, true, y);
        }
      }
      store8(const_cast<void*>(p.k), (int64_t)item * 8, p.dtype, x);
      store8(const_cast<void*>(p.v), (int64_t)item * 8, p.dtype, y);
    }
  }
}

// Rows that no vector fits (odd head dims, odd addresses): an element a thread, parts is D.  4-bit rows
// always fit.
__global__ void __launch_bounds__(kThreads) read_slots_odd_kernel(const RowsParams p) {
  const uint32_t item = blockIdx.x * kThreads + threadIdx.x;
  if (item >= p.items) return;
  uint32_t t, h, part;
  int64_t row;
  float x = 0.0f, y = 0.0f;
  if (find_row(p, item, t, h, part, row)) {
    x = load_dyn(p.kp, row * p.parts + part, p.kv_dtype);
    y = load_dyn(p.vp, row * p.parts + part, p.kv_dtype);
    if (p.kv_dtype == NVM_I8) {
      x = __fmul_rn(x, load_dyn(p.ks, row, p.scale_dtype));
      y = __fmul_rn(y, load_dyn(p.vs, row, p.scale_dtype));
    }
  }
  store_dyn(const_cast<void*>(p.k), item, p.dtype, x);
  store_dyn(const_cast<void*>(p.v), item, p.dtype, y);
}

bool aligned16(const void* a, const void* b) { return (((uintptr_t)a | (uintptr_t)b) & 15) == 0; }

}  // namespace

int launch_u4_write(const void* k, const void* v, int in_dtype, int64_t stride_t, int64_t stride_h, void* k_pages, void* v_pages,
                    void* k_scales, void* v_scales, int scale_dtype, const int64_t* slots, int64_t T, int64_t Hkv, int64_t D,
                    int64_t P, int64_t page_size, cudaStream_t s) {
  RowsParams p{};
  const int64_t e = (int64_t)dtype_size(in_dtype);
  p.st = stride_t; p.sh = stride_h; p.kp = k_pages; p.vp = v_pages; p.ks = k_scales; p.vs = v_scales;
  p.P = P; p.ps = page_size; p.Hkv = (uint32_t)Hkv; p.parts = (uint32_t)(D / 8);
  p.by_parts = FastDiv(p.parts);
  p.by_heads = FastDiv(Hkv);
  p.by_ps = FastDiv(page_size);
  p.dtype = in_dtype;
  p.fast = aligned16(k, v) && stride_t * e % 16 == 0 && stride_h * e % 16 == 0;
  const int64_t row_items = Hkv * (D / 8), most = INT32_MAX / row_items;  // tokens of a launch: items are counted in 32 bits
  for (int64_t t0 = 0; t0 < T; t0 += most) {
    const int64_t n = std::min(most, T - t0);
    p.k = static_cast<const uint8_t*>(k) + t0 * stride_t * e;
    p.v = static_cast<const uint8_t*>(v) + t0 * stride_t * e;
    p.slots = slots + t0;
    p.items = (uint32_t)(n * row_items);
    const unsigned grid = (unsigned)((p.items + kThreads - 1) / kThreads);
    if (scale_dtype == NVM_BF16)
      u4_write_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(p);
    else
      u4_write_kernel<__half><<<grid, kThreads, 0, s>>>(p);
    const int st = check_cuda(cudaGetLastError(), "write_page_slice: kernel launch");
    if (st != NVM_OK) return st;
  }
  return NVM_OK;
}

int launch_read_slots(const void* k_pages, const void* v_pages, int kv_dtype, const void* k_scales, const void* v_scales,
                      int scale_dtype, const int64_t* slots, void* k, void* v, int out_dtype, int64_t T, int64_t Hkv, int64_t D,
                      int64_t P, int64_t page_size, cudaStream_t s) {
  RowsParams p{};
  const int64_t e = (int64_t)dtype_size(out_dtype);
  p.kp = const_cast<void*>(k_pages); p.vp = const_cast<void*>(v_pages);
  p.ks = const_cast<void*>(k_scales); p.vs = const_cast<void*>(v_scales);
  p.P = P; p.ps = page_size; p.Hkv = (uint32_t)Hkv; p.dtype = out_dtype; p.kv_dtype = kv_dtype; p.scale_dtype = scale_dtype;
  const bool fast = D % 8 == 0 && aligned16(k, v) && aligned16(k_pages, v_pages);
  p.parts = (uint32_t)(fast ? D / 8 : D);
  p.by_parts = FastDiv(p.parts);
  p.by_heads = FastDiv(Hkv);
  p.by_ps = FastDiv(page_size);
  const int64_t row_items = Hkv * p.parts, most = INT32_MAX / row_items;
  if (most < 1) return fail(NVM_ERR_UNSUPPORTED, "read_slots: rows of more than 2^31 elements a token");
  for (int64_t t0 = 0; t0 < T; t0 += most) {
    const int64_t n = std::min(most, T - t0);
    p.k = static_cast<uint8_t*>(k) + t0 * Hkv * D * e;
    p.v = static_cast<uint8_t*>(v) + t0 * Hkv * D * e;
    p.slots = slots + t0;
    p.items = (uint32_t)(n * row_items);
    const unsigned grid = (unsigned)((p.items + kThreads * kRead - 1) / (kThreads * kRead));
    if (!fast)
      read_slots_odd_kernel<<<(unsigned)((p.items + kThreads - 1) / kThreads), kThreads, 0, s>>>(p);
    else if (kv_dtype == NVM_U4)
      read_slots_kernel<NVM_U4><<<grid, kThreads, 0, s>>>(p);
    else if (kv_dtype == NVM_I8)
      read_slots_kernel<NVM_I8><<<grid, kThreads, 0, s>>>(p);
    else
      read_slots_kernel<NVM_BF16><<<grid, kThreads, 0, s>>>(p);  // the page type is looked at in the kernel
    const int st = check_cuda(cudaGetLastError(), "read_slots: kernel launch");
    if (st != NVM_OK) return st;
  }
  return NVM_OK;
}

}  // namespace nvm
