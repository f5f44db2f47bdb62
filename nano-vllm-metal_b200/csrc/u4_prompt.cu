// u4_prompt.cu -- many query rows over a 4-bit cache: the pages are unpacked once into f16 and the
// tcgen05 kernel (flash_sm100.cu) attends to those.
//
// A row block of paged_u4.cu unpacks the keys that it sees for itself, which costs it more than the
// matrix instructions do once a kv head has many blocks; here a key is unpacked once for all of them and
// the tensor cores run from TMA tiles: 4 x 512 tokens against 2K-8K keys, 32/8 heads, take 247 us, 200 of
// them the tcgen05 kernel's (885 us in row blocks).  Calls of fewer rows a kv head stay with the row blocks
// (kU4PromptRows has both sides).
// Values of bfloat16 range are brought into f16 by a power of two for every (request, kv head): K's goes
// into the queries together with the softmax scale's power of two, V's into the output; f16 then rounds
// them to 11 bits, eight times finer than bfloat16 would.  The unpacking is bound by HBM (144 bytes in,
// 512 out a key) and its result mostly stays in L2 for the attention.
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
constexpr int kSizeUnroll = 4;
constexpr int kSizeKeys = 256 * kSizeUnroll;          // keys of a block that looks at sizes
constexpr int kTarget = 4;  // values are brought below 2^(kTarget + 1)
// Bytes that unpacked pages may take; larger batches are taken in parts.
constexpr size_t kMostBytes = size_t(1) << 30;

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
  __half* q16;        // [B * Hq * L][D], or NULL: q goes as it is
  int32_t* table;     // [B][groups]
  uint32_t* sizes;    // bits of the largest |K| and |V|: [2][B * Hkv], or NULL: nothing is scaled
  float* out_scale;   // [B * Hkv]
  FastDiv by_ps, by_heads, by_blocks;
  int B, Hq, Hkv, P, ps, mp, groups, blocks;  // blocks: of a (request, kv head)
  int64_t q_vectors, vectors_of_head;         // of eight elements, all of q's and those of a q head
  int q_dtype, q_fast, q_blocks;              // q_fast: 16-bit vectors
  float q_scale;
};

// 2^e that brings numbers of this size below 2^(kTarget + 1), and back
__device__ __forceinline__ int exponent_of(uint32_t size) { return size == 0 ? kTarget : min(max((int)(size >> 23) - 127, -100), 127); }
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + min(max(e, -126), 127)) << 23); }

__device__ __forceinline__ int64_t pool_row(const PromptParams& p, int b, int h, int key) {
  const int page = (int)p.by_ps((uint32_t)key), pid = __ldg(p.block_table + (int64_t)b * p.mp + page);
  return pid < 0 || pid >= p.P ? -1 : ((int64_t)pid * p.Hkv + h) * p.ps + (key - page * p.ps);
}

template <typename T>
__device__ __forceinline__ float size_of(uint2 pairs) {
  const float2 a = u4_pair<T>(pairs.x), b = u4_pair<T>(pairs.y);
  const float m = fmaxf(fmaxf(fabsf(a.y), fabsf(fmaf(15.0f, a.x, a.y))), fmaxf(fabsf(b.y), fabsf(fmaf(15.0f, b.x, b.y))));
  return fminf(m, 3.0e38f);
}

template <typename T>
__global__ void __launch_bounds__(256) u4_sizes_kernel(const PromptParams p) {
  __shared__ float most[2][8];
  const int bh = (int)p.by_blocks(blockIdx.x), k0 = (blockIdx.x - bh * p.blocks) * kSizeKeys;
  const int b = (int)p.by_heads((uint32_t)bh), h = bh - b * p.Hkv;
  const int keys = min(min(__ldg(p.context_lens + b), p.mp * p.ps), k0 + kSizeKeys);
  float mk = 0.0f, mv = 0.0f;
  uint2 pk[kSizeUnroll], pv[kSizeUnroll];
#pragma unroll
  for (int i = 0; i < kSizeUnroll; ++i) {
    const int key = k0 + i * 256 + threadIdx.x;
    const int64_t row = key < keys ? pool_row(p, b, h, key) : -1;
    pk[i] = pv[i] = make_uint2(0, 0);
    if (row >= 0) {
      pk[i] = __ldg(reinterpret_cast<const uint2*>(p.ks) + row);
      pv[i] = __ldg(reinterpret_cast<const uint2*>(p.vs) + row);
    }
  }
#pragma unroll
  for (int i = 0; i < kSizeUnroll; ++i) {
    mk = fmaxf(mk, size_of<T>(pk[i]));
    mv = fmaxf(mv, size_of<T>(pv[i]));
  }
  mk = warp_max(mk);
  mv = warp_max(mv);
  if ((threadIdx.x & 31) == 0) {
    most[0][threadIdx.x >> 5] = mk;
    most[1][threadIdx.x >> 5] = mv;
  }
  __syncthreads();
  if (threadIdx.x < 2) {  // a maximum does not depend on the order of the blocks
    float m = 0.0f;
    for (int w = 0; w < 8; ++w) m = fmaxf(m, most[threadIdx.x][w]);
    if (m > 0.0f) atomicMax(p.sizes + threadIdx.x * (p.B * p.Hkv) + bh, __float_as_uint(m));
  }
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
  return x > 65504.0f ? 65504.0f : x < -65504.0f ? -65504.0f : x;
}

// q in f16, times the scale's power of two and what K was divided by: kUnroll vectors a thread
__device__ __forceinline__ void take_queries(const PromptParams& p, int64_t block) {
  const int64_t first = block * (kThreads * kUnroll) + threadIdx.x;
  if (p.sizes != nullptr)
    for (int64_t i = block * kThreads + threadIdx.x; i < (int64_t)p.B * p.Hkv; i += (int64_t)p.q_blocks * kThreads)
      p.out_scale[i] = power_of_two(exponent_of(__ldcg(p.sizes + (int64_t)p.B * p.Hkv + i)) - kTarget);
  uint4 raw[kUnroll];
  if (p.q_fast) {
#pragma unroll
    for (int e = 0; e < kUnroll; ++e)
      if (first + e * kThreads < p.q_vectors) raw[e] = __ldg(static_cast<const uint4*>(p.q) + first + e * kThreads);
  }
#pragma unroll
  for (int e = 0; e < kUnroll; ++e) {
    const int64_t i = first + e * kThreads;
    if (i >= p.q_vectors) return;
    float f = p.q_scale;
    if (p.sizes != nullptr) {
      const uint32_t head = (uint32_t)(i / p.vectors_of_head);  // b * Hq + q head: a kv head's are neighbours
      f = fminf(f * power_of_two(exponent_of(__ldcg(p.sizes + head / (uint32_t)(p.Hq / p.Hkv))) - kTarget), 3.0e38f);
    }
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
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = pack2<__half>(into_half(x[2 * k] * f), into_half(x[2 * k + 1] * f));
    reinterpret_cast<uint4*>(p.q16)[i] = make_uint4(w[0], w[1], w[2], w[3]);
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
  float fk = 1.0f, fv = 1.0f;
  if (p.sizes != nullptr) {
    fk = power_of_two(kTarget - exponent_of(__ldcg(p.sizes + bh)));
    fv = power_of_two(kTarget - exponent_of(__ldcg(p.sizes + p.B * p.Hkv + bh)));
  }
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
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    const int key = k0 + threadIdx.x / (kD / 8) + i * (kKeys / kUnroll);
    if (key >= (keys + 15) / 16 * 16) break;
    const int64_t to = ((((int64_t)b * p.groups + key / 16) * p.Hkv + h) * 16 + key % 16) * (kD / 8) + part;
    reinterpret_cast<uint4*>(p.k16)[to] = unpack8<T>(codes[0][i], pairs[0][i], fk);
    reinterpret_cast<uint4*>(p.v16)[to] = unpack8<T>(codes[1][i], pairs[1][i], fv);
  }
}

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

struct Layout {
  size_t k, v, q, table, sizes, out_scale, total;
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
  w.sizes = w.table + align256((size_t)(a.B * w.groups) * 4);
  w.out_scale = w.sizes + align256((size_t)(a.B * a.Hkv) * 8);
  w.total = w.out_scale + align256((size_t)(a.B * a.Hkv) * 4);
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
  PagedArgs x = a;
  const int64_t one = std::max<int64_t>(a.max_pages * a.page_size * a.Hkv * kD * 4, 1);
  const int64_t parts = (a.B * one + (int64_t)kMostBytes - 1) / (int64_t)kMostBytes;
  x.B = std::max<int64_t>((a.B + parts - 1) / parts, 1);
  for (; x.B > 1 && (x.B * x.Hkv * ((a.max_pages * a.page_size + kKeys - 1) / kKeys) > INT32_MAX / 2 || x.B * x.Hq * x.L > INT32_MAX / 2);)
    x.B = (x.B + 1) / 2;
  const Layout none = layout_of(x, 0);
  const PagedArgs inner = unpacked(x, none, nullptr);
  if (x.Hkv * ((a.max_pages * a.page_size + kKeys - 1) / kKeys) > INT32_MAX / 2) return plan;
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
    const bool sized = a.scale_dtype == NVM_BF16, copied = sized || a.q_dtype != NVM_F16 || (uintptr_t)x.q % 16 != 0;
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
    p.q16 = reinterpret_cast<__half*>(ws + w.q);
    p.table = reinterpret_cast<int32_t*>(ws + w.table);
    p.sizes = sized ? reinterpret_cast<uint32_t*>(ws + w.sizes) : nullptr;
    p.out_scale = reinterpret_cast<float*>(ws + w.out_scale);
    p.by_ps = FastDiv(a.page_size);
    p.by_heads = FastDiv(a.Hkv);
    p.B = (int)x.B; p.Hq = (int)a.Hq; p.Hkv = (int)a.Hkv; p.P = (int)a.P; p.ps = (int)a.page_size; p.mp = (int)a.max_pages;
    p.groups = (int)w.groups;
    p.vectors_of_head = a.L * (kD / 8);
    p.q_vectors = copied ? x.B * a.Hq * p.vectors_of_head : 0;
    p.q_dtype = a.q_dtype;
    p.q_scale = std::ldexp(1.0f, std::min(std::max(e, -126), 127));
    const int64_t keys = a.max_pages * a.page_size;
    const bool bf = a.scale_dtype == NVM_BF16;
    if (sized) {
      int st = check_cuda(cudaMemsetAsync(p.sizes, 0, (size_t)(x.B * a.Hkv) * 8, s), "paged_attention: cudaMemsetAsync");
      if (st != NVM_OK) return st;
      p.blocks = (int)((keys + kSizeKeys - 1) / kSizeKeys);
      p.by_blocks = FastDiv(p.blocks);
      u4_sizes_kernel<__nv_bfloat16><<<(unsigned)(x.B * a.Hkv * p.blocks), 256, 0, s>>>(p);
      st = check_cuda(cudaGetLastError(), "paged_attention: 4-bit sizes kernel launch");
      if (st != NVM_OK) return st;
    }
    p.blocks = (int)((keys + kKeys - 1) / kKeys);
    p.by_blocks = FastDiv(p.blocks);
    if (copied) {
      p.q_fast = a.q_dtype != NVM_F32 && (uintptr_t)x.q % 16 == 0;
      p.q_blocks = (int)((p.q_vectors + kThreads * kUnroll - 1) / (kThreads * kUnroll));
      y.q = p.q16;
      y.scale = mantissa;
      y.out_scale = sized ? p.out_scale : nullptr;
    }
    const unsigned grid = (unsigned)(x.B * a.Hkv * p.blocks + p.q_blocks);
    bf ? u4_unpack_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(p) : u4_unpack_kernel<__half><<<grid, kThreads, 0, s>>>(p);
    int st = check_cuda(cudaGetLastError(), "paged_attention: 4-bit unpack kernel launch");
    if (st != NVM_OK) return st;
    const Sm100Plan sp = plan_sm100(y, false);
    if (!sp.eligible || sp.ws_bytes > w.k) return fail(NVM_ERR_UNSUPPORTED, "paged_attention: 4-bit prompt plan");
    st = launch_sm100(y, sp, workspace, s);
    if (st != NVM_OK) return st;
  }
  return NVM_OK;
}

}  // namespace nvm
