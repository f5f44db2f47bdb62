// evict.cu -- eviction of cached tokens by accumulated attention weight.
//
// Request b of n = context_lens[b] tokens, per kv head, keeps `budget` of them: the first
// `sinks`, the last `recent` and, of the rest, the ones with the most accumulated weight
// (ties: the lowest position; NaN ranks below every number; -0 equals +0).  The kept rows
// of K, V, their scales and their weights move, in order, to the head's first `budget`
// slots of the request's own pages; weights behind them become zero.  n <= budget changes
// nothing.
//
// Two kernels.  evict_select: a CTA per (request, kv head) finds the k-th largest weight by
// radix selection on an order-preserving 32-bit image of the weight (four 8-bit digits),
// then walks the positions once in order, numbering the kept ones with ballots, and moves
// the weights.  evict_compact: a CTA per (request, kv head, column slice of K or V).  Slot i
// receives token keep[i] >= i, so a tile of slots read completely before it is written never
// overwrites a row that a later tile reads (later tiles read positions at or past their own
// first slot): in place, no second copy of the cache.  The column slices are independent,
// which is what spreads one (request, kv head) over several SMs.
#include "nvm_common.cuh"
#include "nvm_internal.h"

namespace nvm {
namespace {

constexpr int kSelThreads = 1024;

struct EvictParams {
  EvictArgs a;
  int64_t row_bytes;    // of one K (or V) row
  int slice_bytes;      // columns of one CTA
  int n_slices;
  int scale_bytes;      // 0: no scales
};

// Larger weight -> larger image; NaN -> 0, -0 -> the image of +0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictParams ep) {
  const EvictArgs& p = ep.a;
  __shared__ int hist[256];
  __shared__ int wsum[2][32];
  __shared__ int s_bad, s_digit, s_rank;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int64_t b = blockIdx.x / p.Hkv, h = blockIdx.x % p.Hkv;
  const int64_t n64 = p.context_lens[b];
  int32_t* keep = p.keep_index + (int64_t)blockIdx.x * p.budget;
  const float* mass = p.mass + b * p.stride_b + h * p.stride_h;
  float* mout = p.mass_out + b * p.out_stride_b + h * p.out_stride_h;

  // A request whose tokens would have to move is taken only if its row is sound: every page
  // that holds them mapped, and (with refcounts) owned by this request alone.
  if (t == 0) s_bad = 0;
  __syncthreads();
  if (n64 < 0 || n64 > p.len || n64 > p.max_pages * p.page_size) {
    if (t == 0) s_bad = 1;
  } else if (n64 > p.budget) {
    const int64_t first = p.sinks / p.page_size, last = (n64 - 1) / p.page_size;
    for (int64_t i = first + t; i <= last; i += kSelThreads) {
      const int64_t pid = p.block_table[b * p.max_pages + i];
      if (pid < 0 || pid >= p.P || (p.page_refcount != nullptr && p.page_refcount[pid] != 1)) s_bad = 1;
    }
  }
  __syncthreads();
  const bool bad = s_bad != 0;
  const int n = bad ? 0 : (int)n64;
  const bool evicts = n > p.budget;
  if (t == 0 && h == 0) {
    p.kept[b] = bad ? (int32_t)n64 : (evicts ? (int32_t)p.budget : n);
    p.dropped[b] = evicts ? n - (int32_t)p.budget : 0;
    if (bad) *p.status = NVM_ERR_INVALID_ARGUMENT;
  }
  if (!evicts) {  // everything stays (or the row is refused: no index, weights as they are)
    for (int64_t i = t; i < p.budget; i += kSelThreads) keep[i] = i < n ? (int32_t)i : -1;
    if (mout != mass)
      for (int64_t i = t; i < n; i += kSelThreads) mout[i] = mass[i];
    return;
  }

  // k-th largest of the middle [lo, hi): digits from the top, `rank` counted inside the prefix
  const int lo = (int)p.sinks, hi = n - (int)p.recent;
  int rank = (int)(p.budget - p.sinks - p.recent);
  uint32_t prefix = 0;
  int above = 0;  // weights larger than the threshold, so far
  if (rank > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (t < 256) hist[t] = 0;
      __syncthreads();
      for (int i = lo + t; i < hi; i += kSelThreads) {
        const uint32_t key = weight_key(mass[i]);
        if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255], 1);
      }
      __syncthreads();
      if (t == 0) {
        int left = rank, d = 255;
        while (d > 0 && hist[d] < left) left -= hist[d--];
        s_digit = d;
        s_rank = left;
      }
      __syncthreads();
      above += rank - s_rank;
      rank = s_rank;
      prefix |= (uint32_t)s_digit << shift;
      __syncthreads();
    }
  }
  // kept of the middle: every weight above the threshold, and the first `rank` equal ones
  const bool none = p.budget == p.sinks + p.recent;
  int out = 0, eq_seen = 0;  // kept / equal so far (all threads hold the same values)
  for (int base = 0; base < n; base += kSelThreads) {
    const int i = base + t;
    bool eq = false, take = false;
    float w = 0.f;
    if (i < n) {
      w = mass[i];
      if (i < lo || i >= hi) {
        take = true;
      } else if (!none) {
        const uint32_t key = weight_key(w);
        take = key > prefix;
        eq = key == prefix;
      }
    }
    const uint32_t beq = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) wsum[0][warp] = __popc(beq);
    __syncthreads();
    int before = 0, total_eq = 0;
    for (int w2 = 0; w2 < 32; ++w2) {
      if (w2 < warp) before += wsum[0][w2];
      total_eq += wsum[0][w2];
    }
    const int my_eq = eq_seen + before + __popc(beq & ((1u << lane) - 1u));
    if (eq && my_eq < rank) take = true;
    const uint32_t bt = __ballot_sync(0xffffffffu, take);
    if (lane == 0) wsum[1][warp] = __popc(bt);
    __syncthreads();  // every weight of this stretch has been read: they may be overwritten
    int slot = out, total = 0;
    for (int w2 = 0; w2 < 32; ++w2) {
      if (w2 < warp) slot += wsum[1][w2];
      total += wsum[1][w2];
    }
    slot += __popc(bt & ((1u << lane) - 1u));
    if (take) {
      keep[slot] = i;
      mout[slot] = w;
    }
    out += total;
    eq_seen += total_eq;
    __syncthreads();
  }
  for (int64_t i = p.budget + t; i < n; i += kSelThreads) mout[i] = 0.f;
}

template <typename V>
__device__ __forceinline__ void compact_rows(const EvictParams& ep, int64_t b, int64_t h, uint8_t* pool, int64_t row_bytes,
                                             int col0, int cols) {
  const EvictArgs& p = ep.a;
  constexpr int kU = 4;  // rows in flight per thread
  const int per_row = cols / (int)sizeof(V);
  const int rows_par = blockDim.x / per_row;  // rows one step of the CTA covers
  const int my_row = threadIdx.x / per_row, my_col = threadIdx.x % per_row;
  const int32_t* keep = p.keep_index + (b * p.Hkv + h) * p.budget;
  const int32_t* table = p.block_table + b * p.max_pages;
  const uint32_t ps = (uint32_t)p.page_size;
  auto at = [&](uint32_t tok) -> V* {
    const uint32_t page = tok / ps, off = tok - page * ps;
    return reinterpret_cast<V*>(pool + (((int64_t)table[page] * p.Hkv + h) * ps + off) * row_bytes + col0) + my_col;
  };
  for (int64_t base = p.sinks; base < p.budget; base += (int64_t)rows_par * kU) {
    V v[kU];
    bool mv[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int64_t i = base + u * rows_par + my_row;
      mv[u] = false;
      if (my_row < rows_par && i < p.budget) {
        const int src = keep[i];
        mv[u] = src != i;
        if (mv[u]) v[u] = *at((uint32_t)src);
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (mv[u]) *at((uint32_t)(base + u * rows_par + my_row)) = v[u];
  }
}

template <typename V>
__global__ void __launch_bounds__(256) evict_compact_kernel(const EvictParams ep) {
  const EvictArgs& p = ep.a;
  const int64_t b = blockIdx.x / p.Hkv, h = blockIdx.x % p.Hkv;
  if (p.dropped[b] == 0) return;
  const int y = blockIdx.y;
  if (y < 2 * ep.n_slices) {
    uint8_t* pool = static_cast<uint8_t*>(y < ep.n_slices ? p.k_pages : p.v_pages);
    const int sl = y % ep.n_slices, col0 = sl * ep.slice_bytes;
    const int left = (int)ep.row_bytes - col0;
    compact_rows<V>(ep, b, h, pool, ep.row_bytes, col0, left < ep.slice_bytes ? left : ep.slice_bytes);
  } else {
    uint8_t* pool = static_cast<uint8_t*>(y == 2 * ep.n_slices ? p.k_scales : p.v_scales);
    if (ep.scale_bytes == 4)
      compact_rows<uint32_t>(ep, b, h, pool, 4, 0, 4);
    else
      compact_rows<uint16_t>(ep, b, h, pool, 2, 0, 2);
  }
}

}  // namespace

int launch_evict(const EvictArgs& a, cudaStream_t s) {
  EvictParams ep{};
  ep.a = a;
  ep.row_bytes = a.D * (int64_t)dtype_size(a.kv_dtype);
  ep.scale_bytes = a.kv_dtype == NVM_I8 ? (int)dtype_size(a.scale_dtype) : 0;
  const dim3 sel((unsigned)(a.B * a.Hkv));
  evict_select_kernel<<<sel, kSelThreads, 0, s>>>(ep);
  int st = check_cuda(cudaGetLastError(), "evict: selection kernel launch");
  if (st != NVM_OK) return st;
  // the widest vector that rows and pools are aligned to
  const uint64_t al = (uint64_t)ep.row_bytes | reinterpret_cast<uintptr_t>(a.k_pages) | reinterpret_cast<uintptr_t>(a.v_pages);
  const int vec = (al & 15) == 0 ? 16 : (al & 3) == 0 ? 4 : (al & 1) == 0 ? 2 : 1;
  ep.slice_bytes = 32 * (vec >= 4 ? 4 : 1) * (vec >= 16 ? 4 : 1);
  if (ep.slice_bytes > ep.row_bytes) ep.slice_bytes = (int)ep.row_bytes;
  ep.n_slices = (int)((ep.row_bytes + ep.slice_bytes - 1) / ep.slice_bytes);
  const dim3 grid((unsigned)(a.B * a.Hkv), (unsigned)(2 * ep.n_slices + (ep.scale_bytes ? 2 : 0)));
  if (vec == 16) evict_compact_kernel<uint4><<<grid, 256, 0, s>>>(ep);
  else if (vec == 4) evict_compact_kernel<uint32_t><<<grid, 256, 0, s>>>(ep);
  else if (vec == 2) evict_compact_kernel<uint16_t><<<grid, 256, 0, s>>>(ep);
  else evict_compact_kernel<uint8_t><<<grid, 256, 0, s>>>(ep);
  return check_cuda(cudaGetLastError(), "evict: compaction kernel launch");
}

}  // namespace nvm
