// u4_prompt.cu -- many query rows over a 4-bit cache: the pages are unpacked once into f16 and the
// tcgen05 kernel (flash_sm100.cu) attends to those.
//
// A row block of paged_u4.cu unpacks the keys that it sees for itself, which costs it more than the
// matrix instructions do once a kv head has many blocks; here a key is unpacked once for all of them and
// the tensor cores run from TMA tiles: 4 x 512 tokens against 2K-8K keys, 32/8 heads, take 243 us, about 205
// of them the tcgen05 kernel's (pages of 24 tokens, in row blocks, 3.4 times as long).  Calls of fewer rows a kv head stay with the row blocks
// (kU4PromptRows has both sides).
// f16 rounds values and queries of bfloat16 range to 11 bits, eight times finer than bfloat16 would, as long
// as they lie in its range.  Fixed powers of two bring ordinary ones into its middle (Held; the queries' makes
// the softmax scale's power up), and are undone in the scores' scale and in the output.  They do not follow
// the data: a power of two from all keys of a request lets a key change rows that do not see it.  What f16
// cannot hold (larger, far smaller, NaN) is left out of the unpacked pages and noted: the rows that see such a
// key, or are themselves too large, are computed by the row blocks in a second step, which ends at once
// where there are none (3 us).  So which kernel computes a row, and from what, depends on what the row sees only.
// The unpacking is bound by HBM (144 bytes in, 512 out a key) and its result mostly stays in L2 for the
// attention.
#include <algorithm>
#include <cmath>

#include "nvm_internal.h"
#include "u4.cuh"

namespace nvm {
namespace {

constexpr int kD = 128;
constexpr int kThreads = 128;
constexpr int kUnroll = 4;                            // keys of a thread
constexpr int kKeys = kThreads / (kD / 8) * kUnroll;  // of a block
constexpr float kHalfMax = 65504.0f;
// Bytes that unpacked pages may take; larger batches are taken in parts.  They are sized by the table's width, since
// the lengths are on the device: one request may take kMostOfOne (2M keys of 8 heads), and is left to the row
// blocks, which need no copy, beyond that (a table a million pages wide asked for 4 TB).
constexpr int64_t kMostBytes = int64_t(1) << 30, kMostOfOne = int64_t(1) << 33;

// What K and V are multiplied by in f16, the most that they may be there, and the least size of a value group whose
// elements keep 12 bits of it there (below 2^-14 f16 has steps of 2^-24, here of 2^-30).  Numbers of float16
// pages are whole steps of f16 however small, and go as they are.
template <typename T>
struct Held;
template <>
struct Held<__nv_bfloat16> {
  static constexpr float kKeys = 0x1p4f, kMostKey = kHalfMax, kValues = 0x1p6f, kLeastValue = 0x1p-18f;
};
template <>
struct Held<__half> {
  static constexpr float kKeys = 1.0f, kMostKey = kHalfMax / 16, kValues = 1.0f, kLeastValue = 0.0f;
};
// Queries are multiplied by 2^8 and the softmax scale's power of two, and may be 2^15 then.  Scores (base 2) then stay
// below 128 * 2^7 * 4094 * 1.45 < 2^27, where the tcgen05 kernel's weights pass their reference by less than 2^12.
constexpr int kQueryShift = 8;
constexpr float kMostQuery = 0x1p15f;

struct PromptParams {
  const uint8_t* kp;
  const uint8_t* vp;
  const uint32_t* ks;
  const uint32_t* vs;
  const int32_t* block_table;
  const int32_t* context_lens;
  const void* q;
  __half* k16;        // [B * groups][Hkv][16][D]
  __half* v16;
  __half* q16;        // [B * Hq * L][D], or NULL: q goes as it is, and is only looked at
  int32_t* table;     // [B][groups]
  uint32_t* first;    // U4Some, zero to begin with but for the rows
  int* some;
  uint8_t* far_rows;
  FastDiv by_ps, by_heads, by_blocks;
  int B, Hq, Hkv, P, ps, mp, groups, blocks;  // blocks: of a (request, kv head)
  int64_t q_vectors, vectors_of_head;         // of eight elements, all of q's and those of a q head
  int q_dtype, q_fast, q_blocks;              // q_fast: 16-bit vectors
  float q_scale, q_size;                      // of the copy, and of what may be kMostQuery
};

__device__ __forceinline__ int64_t pool_row(const PromptParams& p, int b, int h, int key) {
  const int page = (int)p.by_ps((uint32_t)key), pid = __ldg(p.block_table + (int64_t)b * p.mp + page);
  return pid < 0 || pid >= p.P ? -1 : ((int64_t)pid * p.Hkv + h) * p.ps + (key - page * p.ps);
}

// Whether a group's values, which lie between z and z + 15 s, are in range.
template <typename T>
__device__ __forceinline__ bool fits(uint32_t pair, float factor, float most, float least) {
  const float2 sz = u4_pair<T>(pair);
  const float size = max_nan(fabsf(sz.y), fabsf(fmaf(15.0f, sz.x, sz.y)));
  return size * factor <= most && (size >= least || size == 0.0f);  // false for NaN
}

template <typename T>
__device__ __forceinline__ uint4 unpack8(uint32_t codes, uint32_t pair, float factor) {
  const float2 sz = u4_pair<T>(pair);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = __fsub_rn(__uint_as_float(0x4B000000u | (codes >> (8 * i) & 15)), 8388608.0f);
    const float b = __fsub_rn(__uint_as_float(0x4B000000u | (codes >> (8 * i + 4) & 15)), 8388608.0f);
    w[i] = pack2<__half>(fmaf(sz.x, a, sz.y) * factor, fmaf(sz.x, b, sz.y) * factor);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float into_half(float x) {  // NaN stays
  return x > kHalfMax ? kHalfMax : x < -kHalfMax ? -kHalfMax : x;
}

// q in f16, times q_scale, and the rows that are too large for it: kUnroll vectors a thread, a row in half a warp.
__device__ __forceinline__ void take_queries(const PromptParams& p, int64_t block) {
  const int64_t first = block * (kThreads * kUnroll) + threadIdx.x;
  const uint32_t half = 0xffffu << (threadIdx.x & 16);
  uint4 raw[kUnroll];
  if (p.q_fast) {
#pragma unroll
    for (int e = 0; e < kUnroll; ++e)
      if (first + e * kThreads < p.q_vectors) raw[e] = __ldg(static_cast<const uint4*>(p.q) + first + e * kThreads);
  }
#pragma unroll
  for (int e = 0; e < kUnroll; ++e) {
    const int64_t i = first + e * kThreads;
    if (i >= p.q_vectors) return;  // (whole rows)
    float x[8];
    const uint32_t u[4] = {raw[e].x, raw[e].y, raw[e].z, raw[e].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (p.q_fast) {
        const float2 v = p.q_dtype == NVM_BF16 ? u4_pair<__nv_bfloat16>(u[k]) : u4_pair<__half>(u[k]);
        x[2 * k] = v.x;
        x[2 * k + 1] = v.y;
      } else {
        x[2 * k] = load_dyn(p.q, i * 8 + 2 * k, p.q_dtype);
        x[2 * k + 1] = load_dyn(p.q, i * 8 + 2 * k + 1, p.q_dtype);
      }
    }
    float top = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(x[k]));
    if (p.q16 != nullptr) {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = pack2<__half>(into_half(x[2 * k] * p.q_scale), into_half(x[2 * k + 1] * p.q_scale));
      reinterpret_cast<uint4*>(p.q16)[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    const bool far = __any_sync(half, top * p.q_size > kMostQuery);
    if ((threadIdx.x & 15) == 0) {
      p.far_rows[i / (kD / 8)] = far;
      if (far) p.some[i / (p.vectors_of_head * p.Hq)] = 1;
    }
  }
}

// Block (request, kv head, kKeys keys); rows from the context's end to that of its group of 16 are zero
// (a weight of zero times what lies there).  The blocks of kv head 0 write the table of the groups, the
// first q_blocks take the queries.
template <typename T>
__global__ void __launch_bounds__(kThreads) u4_unpack_kernel(const PromptParams p) {
  if ((int)blockIdx.x < p.q_blocks) {
    take_queries(p, blockIdx.x);
    return;
  }
  const int block = blockIdx.x - p.q_blocks, bh = (int)p.by_blocks((uint32_t)block), k0 = (block - bh * p.blocks) * kKeys;
  const int b = (int)p.by_heads((uint32_t)bh), h = bh - b * p.Hkv;
  const int keys = max(min(__ldg(p.context_lens + b), p.mp * p.ps), 0);
  if (h == 0 && threadIdx.x < kKeys / 16) {
    const int g = k0 / 16 + threadIdx.x;
    if (g < p.groups) p.table[(int64_t)b * p.groups + g] = 16 * g < keys && pool_row(p, b, 0, 16 * g) >= 0 ? b * p.groups + g : -1;
  }
  if (k0 >= keys) return;
  const int part = threadIdx.x % (kD / 8);
  uint32_t codes[2][kUnroll], pairs[2][kUnroll];
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    const int key = k0 + threadIdx.x / (kD / 8) + i * (kKeys / kUnroll);
    const int64_t row = key < keys ? pool_row(p, b, h, key) : -1;
    codes[0][i] = codes[1][i] = pairs[0][i] = pairs[1][i] = 0;
    if (row >= 0) {
      codes[0][i] = __ldg(reinterpret_cast<const uint32_t*>(p.kp) + row * (kD / 8) + part);
      codes[1][i] = __ldg(reinterpret_cast<const uint32_t*>(p.vp) + row * (kD / 8) + part);
      pairs[0][i] = __ldg(p.ks + row * 2 + part / 8);
      pairs[1][i] = __ldg(p.vs + row * 2 + part / 8);
    }
  }
  uint32_t first = 0;  // the thread's first key that f16 does not hold: zeros there, and the rows that see it come later
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    const int key = k0 + threadIdx.x / (kD / 8) + i * (kKeys / kUnroll);
    if (key >= (keys + 15) / 16 * 16) break;
    if (!fits<T>(pairs[0][i], Held<T>::kKeys, Held<T>::kMostKey, 0.0f) ||
        !fits<T>(pairs[1][i], Held<T>::kValues, kHalfMax, Held<T>::kLeastValue)) {
      codes[0][i] = codes[1][i] = pairs[0][i] = pairs[1][i] = 0;
      first = max(first, (uint32_t)(INT32_MAX - key));
    }
    const int64_t to = ((((int64_t)b * p.groups + key / 16) * p.Hkv + h) * 16 + key % 16) * (kD / 8) + part;
    reinterpret_cast<uint4*>(p.k16)[to] = unpack8<T>(codes[0][i], pairs[0][i], Held<T>::kKeys);
    reinterpret_cast<uint4*>(p.v16)[to] = unpack8<T>(codes[1][i], pairs[1][i], Held<T>::kValues);
  }
  first = __reduce_max_sync(0xffffffffu, first);
  if (first != 0 && threadIdx.x % 32 == 0) {
    atomicMax(p.first + bh, first);
    p.some[b] = 1;
  }
}

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

struct Layout {
  size_t k, v, q, table, first, some, far_rows, total;  // `first` and `some` are neighbours
  int64_t groups;
};
Layout layout_of(const PagedArgs& a, size_t attention) {
  Layout w{};
  w.groups = (a.max_pages * a.page_size + 15) / 16;
  const size_t rows = (size_t)(a.B * w.groups * a.Hkv * 16);
  w.k = align256(std::max(attention, kTicketRegionBytes));
  w.v = w.k + rows * kD * 2;
  w.q = w.v + rows * kD * 2;
  w.table = w.q + align256((size_t)(a.B * a.Hq * a.L) * kD * 2);
  // the row blocks' workspace lies over all of the above, which they need no more
  w.first = align256(std::max(w.table + (size_t)(a.B * w.groups) * 4, plan_paged_u4(a).ws_bytes));
  w.some = w.first + (size_t)(a.B * a.Hkv) * 4;
  w.far_rows = w.some + (size_t)a.B * 4;
  w.total = w.far_rows + align256((size_t)(a.B * a.Hq * a.L));
  return w;
}

// The attention over unpacked pages, as the tcgen05 kernel takes it; `ws` NULL: sizes only.
PagedArgs unpacked(const PagedArgs& a, const Layout& w, uint8_t* ws) {
  PagedArgs x = a;
  x.kv_dtype = x.q_dtype = NVM_F16;
  x.P = a.B * w.groups;
  x.page_size = 16;
  x.max_pages = w.groups;
  x.k_scales = x.v_scales = nullptr;
  if (ws != nullptr) {
    x.k_pages = ws + w.k;
    x.v_pages = ws + w.v;
    x.block_table = reinterpret_cast<int32_t*>(ws + w.table);
  }
  return x;
}

}  // namespace

U4PromptPlan plan_u4_prompt(const PagedArgs& a) {
  U4PromptPlan plan{};
  const int64_t rows = a.Hq / a.Hkv * a.L;
  if (a.B <= 0 || a.D != kD || a.page_size % 16 != 0 || rows < kU4PromptRows || !(a.scale > 0.0f) || !std::isfinite(a.scale) ||
      (uintptr_t)a.out % 16 != 0 || a.P <= 0 || a.max_pages <= 0 || a.max_pages * a.page_size > INT32_MAX - 4096 ||
      a.Hq * a.L > INT32_MAX / 16)
    return plan;
  const int64_t keys = a.max_pages * a.page_size, blocks = a.Hkv * ((keys + kKeys - 1) / kKeys);  // of a request
  const int64_t one = blocks * (kKeys * kD * 4);
  if (one > kMostOfOne) return plan;
  PagedArgs x = a;
  x.B = std::min(a.B, std::max<int64_t>(kMostBytes / one, 1));
  while (x.B > 1 && (x.B * blocks > INT32_MAX / 2 || x.B * x.Hq * x.L > INT32_MAX / 2)) x.B = (x.B + 1) / 2;
  const int64_t parts = (a.B + x.B - 1) / x.B;
  x.B = (a.B + parts - 1) / parts;  // parts of one size
  const Layout none = layout_of(x, 0);
  const PagedArgs inner = unpacked(x, none, nullptr);
  const Sm100Plan attention = plan_sm100(inner, true);
  if (!attention.eligible) return plan;
  plan.attention_bytes = attention.ws_bytes;
  if (a.B % x.B != 0) {  // the last part's plan may cut the keys finer
    PagedArgs last = x;
    last.B = a.B % x.B;
    plan.attention_bytes = std::max(plan.attention_bytes, plan_sm100(unpacked(last, layout_of(last, 0), nullptr), true).ws_bytes);
  }
  plan.eligible = true;
  plan.batch = x.B;
  plan.ws_bytes = layout_of(x, plan.attention_bytes).total;
  return plan;
}

int launch_u4_prompt(const PagedArgs& a, const U4PromptPlan& plan, void* workspace, cudaStream_t s) {
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  int e = 0;
  const float mantissa = std::frexp(a.scale, &e);  // scale = mantissa * 2^e: the power goes into the queries
  const int shift = std::min(std::max(e + kQueryShift, -126), 127);
  for (int64_t b0 = 0; b0 < a.B; b0 += plan.batch) {
    PagedArgs x = a;
    x.B = std::min(plan.batch, a.B - b0);
    const int64_t first = b0 * a.Hq * a.L * a.D;
    x.q = static_cast<const uint8_t*>(a.q) + first * (int64_t)dtype_size(a.q_dtype);
    x.out = static_cast<uint8_t*>(a.out) + first * (int64_t)dtype_size(a.out_dtype);
    x.block_table = a.block_table + b0 * a.max_pages;
    x.context_lens = a.context_lens + b0;
    const Layout w = layout_of(x, plan.attention_bytes);
    PagedArgs y = unpacked(x, w, ws);
    const bool bf = a.scale_dtype == NVM_BF16;
    const bool scaled = bf || a.q_dtype != NVM_F16;  // queries
    const bool copied = scaled || (uintptr_t)x.q % 16 != 0;
    PromptParams p{};
    p.kp = static_cast<const uint8_t*>(a.k_pages);
    p.vp = static_cast<const uint8_t*>(a.v_pages);
    p.ks = static_cast<const uint32_t*>(a.k_scales);
    p.vs = static_cast<const uint32_t*>(a.v_scales);
    p.block_table = x.block_table;
    p.context_lens = x.context_lens;
    p.q = x.q;
    p.k16 = reinterpret_cast<__half*>(ws + w.k);
    p.v16 = reinterpret_cast<__half*>(ws + w.v);
    p.q16 = copied ? reinterpret_cast<__half*>(ws + w.q) : nullptr;
    p.table = reinterpret_cast<int32_t*>(ws + w.table);
    p.first = reinterpret_cast<uint32_t*>(ws + w.first);
    p.some = reinterpret_cast<int*>(ws + w.some);
    p.far_rows = ws + w.far_rows;
    p.by_ps = FastDiv(a.page_size);
    p.by_heads = FastDiv(a.Hkv);
    p.B = (int)x.B; p.Hq = (int)a.Hq; p.Hkv = (int)a.Hkv; p.P = (int)a.P; p.ps = (int)a.page_size; p.mp = (int)a.max_pages;
    p.groups = (int)w.groups;
    p.vectors_of_head = a.L * (kD / 8);
    p.q_vectors = x.B * a.Hq * p.vectors_of_head;
    p.q_dtype = a.q_dtype;
    p.q_size = std::ldexp(1.0f, shift);
    p.q_scale = scaled ? p.q_size : 1.0f;
    const int64_t keys = a.max_pages * a.page_size;
    int st = check_cuda(cudaMemsetAsync(p.first, 0, (size_t)(x.B * (a.Hkv + 1)) * 4, s), "paged_attention: cudaMemsetAsync");
    if (st != NVM_OK) return st;
    p.blocks = (int)((keys + kKeys - 1) / kKeys);
    p.by_blocks = FastDiv(p.blocks);
    p.q_fast = a.q_dtype != NVM_F32 && (uintptr_t)x.q % 16 == 0;
    p.q_blocks = (int)((p.q_vectors + kThreads * kUnroll - 1) / (kThreads * kUnroll));
    if (copied) y.q = p.q16;
    if (scaled) y.scale = std::ldexp(mantissa, e - shift);
    if (bf) {
      y.scale /= Held<__nv_bfloat16>::kKeys;
      y.out_scale = 1.0f / Held<__nv_bfloat16>::kValues;
    }
    const unsigned grid = (unsigned)(x.B * a.Hkv * p.blocks + p.q_blocks);
    bf ? u4_unpack_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(p) : u4_unpack_kernel<__half><<<grid, kThreads, 0, s>>>(p);
    st = check_cuda(cudaGetLastError(), "paged_attention: 4-bit unpack kernel launch");
    if (st != NVM_OK) return st;
    const Sm100Plan sp = plan_sm100(y, false);
    if (!sp.eligible || sp.ws_bytes > w.k) return fail(NVM_ERR_UNSUPPORTED, "paged_attention: 4-bit prompt plan");
    st = launch_sm100(y, sp, workspace, s);
    if (st != NVM_OK) return st;
    const U4Some rest{p.first, p.far_rows, p.some};
    st = launch_paged_u4(x, plan_paged_u4(x), workspace, s, &rest);
    if (st != NVM_OK) return st;
  }
  return NVM_OK;
}

}  // namespace nvm
