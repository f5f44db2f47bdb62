// evict.cu -- eviction of cached tokens by accumulated attention weight.
//
// Request b of n = context_lens[b] tokens, per kv head, keeps `budget` of them: the first
// `sinks`, the last `recent` and, of the rest, the ones with the most accumulated weight
// (ties: the lowest position; NaN ranks below every number; -0 equals +0).  The kept rows
// of K, V, their scales and their weights move, in order, to the head's first `budget`
// slots of the request's own pages; weights behind them become zero.  n <= budget changes
// nothing.
//
// Two kernels.  evict_select: a CTA per (request, kv head) reads the weights once into
// registers (up to 32 a thread; longer rows re-read them from L2), finds the k-th largest by
// radix selection on an order-preserving 32-bit image (digits of 11, 11 and 10 bits,
// shared-memory histograms), numbers the kept positions with one scan over ballot
// counts in position order, and moves the weights.  evict_compact: a CTA per (request, kv
// head, column slice of K or V).  Slot i receives token keep[i] >= i, so a tile of slots that
// is read completely before it is written never overwrites a row that a later tile reads
// (those lie at or past their own first slot): in place, no second copy of the cache, and the
// next tile's rows can be on their way while this one is written.  The column slices are
// independent, which is what spreads one (request, kv head) over several SMs.
// Measured on a B200: 64 requests of 2.1K-8K tokens to 2048, 8 kv heads, bf16: selection 28 us,
// compaction 178 us for 1.07 GB read and written (6.0 TB/s); 32 requests to 4000, int8 pages:
// 20 and 95 us.
#include "nvm_common.cuh"
#include "nvm_internal.h"

namespace nvm {
namespace {

struct EvictParams {
  EvictArgs a;
  int64_t row_bytes;    // of one K (or V) row
  int slice_bytes;      // columns of one CTA
  int n_slices;
  int scale_bytes;      // 0: no scales
  int page_shift;       // log2 of page_size, -1 if it is no power of two
};

// Larger weight -> larger image; NaN -> 0, -0 -> the image of +0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Exclusive scan of one int per thread over the CTA (T threads); *total the sum.
template <int T>
__device__ __forceinline__ int cta_exclusive_scan(int v, int* wsum, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) wsum[warp] = x;
  __syncthreads();
  int w = lane < T / 32 ? wsum[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += y;
  }
  *total = __shfl_sync(0xffffffffu, w, 31);
  const int before = warp > 0 ? __shfl_sync(0xffffffffu, w, warp - 1) : 0;
  __syncthreads();  // wsum may be reused
  return before + x - v;
}

constexpr int kPer = 32;  // weights a thread holds in registers
// Digits of 11, 11 and 10 bits: the first one holds the exponent and two bits of the mantissa.
// With 8-bit digits a row's weights fall into a handful of first bins and their atomics
// serialise (512 rows of 5000: 42 us against 35 us).
constexpr int kBins = 2048;

template <int T>
struct SelSmem {
  int hist[kBins];
  int cnt[T];  // kept per (stretch, warp) of one sweep
  int wsum[32];
  int bad, digit, rank, count;
};
static_assert(kBins % 1024 == 0, "every thread clears and scans whole bins");

// Keeps, of positions [0, n): [0, lo), [hi, n) and the k of [lo, hi) with the largest weight;
// writes their positions and weights in order.  kHeld: the weights' images fit in registers,
// and so are made once (4700 instructions a warp were 2000 too many when every pass made them
// again); the weights themselves are read a second time when they move.
template <int T, bool kHeld>
__device__ __forceinline__ void select_row(SelSmem<T>& sm, const float* mass, float* mout, int32_t* keep, int n, int lo,
                                           int hi, int k) {
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int stretches = (n + T - 1) / T;
  uint32_t img[kPer];    // kHeld: the whole row's; else one sweep's
  uint32_t middle = 0;   // bit j: this thread's position of the sweep's stretch j is in [lo, hi)
  auto read_sweep = [&](int s0) {
    middle = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (s0 + j >= stretches) break;
      const int i = (s0 + j) * T + t;
      img[j] = i < n ? __float_as_uint(__ldcg(mass + i)) : 0u;
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (s0 + j >= stretches) break;
      const int i = (s0 + j) * T + t;
      img[j] = weight_key(__uint_as_float(img[j]));
      if (i >= lo && i < hi) middle |= 1u << j;
    }
  };
  if constexpr (kHeld) read_sweep(0);
  uint32_t prefix = 0;
  int rank = k;         // how many weights equal to the threshold are kept ..
  bool all_eq = true;   // .. all of them
  if (k > 0) {
    constexpr int kBinsPer = kBins / T;
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;  // 11, 11 and 10 bits
      const uint32_t digits = pass == 2 ? 1023u : 2047u;
#pragma unroll
      for (int x = 0; x < kBinsPer; ++x) sm.hist[t + x * T] = 0;
      __syncthreads();
      const int up = shift + (pass == 2 ? 10 : 11);
      for (int s0 = 0; s0 < stretches; s0 += kPer) {
        if constexpr (!kHeld) read_sweep(s0);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          if (s0 + j >= stretches) break;
          if (((middle >> j) & 1u) && (pass == 0 || (img[j] >> up) == (prefix >> up)))
            atomicAdd(&sm.hist[(img[j] >> shift) & digits], 1);
        }
      }
      __syncthreads();
      // thread t: digits kBins - 1 - kBinsPer t, downwards
      int c[kBinsPer], sum = 0, total;
#pragma unroll
      for (int x = 0; x < kBinsPer; ++x) sum += c[x] = sm.hist[kBins - 1 - kBinsPer * t - x];
      int above = cta_exclusive_scan<T>(sum, sm.wsum, &total);  // weights with a larger digit
      if (above < rank && rank <= above + sum) {
#pragma unroll
        for (int x = 0; x < kBinsPer; ++x) {
          if (above < rank && rank <= above + c[x]) {
            sm.digit = kBins - 1 - kBinsPer * t - x;
            sm.rank = rank - above;
            sm.count = c[x];
          }
          above += c[x];
        }
      }
      __syncthreads();
      rank = sm.rank;
      all_eq = rank == sm.count;
      prefix |= (uint32_t)sm.digit << shift;
    }
  }
  // Number the kept positions in sweeps of 32 stretches: first the weights equal to the
  // threshold (only the first `rank` stay), then all kept.
  int kept = 0, eq_seen = 0;
  for (int s0 = 0; s0 < stretches; s0 += kPer) {
    uint32_t eqs = 0, take = 0;  // bit j: this thread's position of stretch s0 + j
    if constexpr (!kHeld) read_sweep(s0);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (s0 + j >= stretches) break;
      if ((middle >> j) & 1u) {
        if (k > 0 && (img[j] > prefix || (all_eq && img[j] == prefix))) take |= 1u << j;
        if (img[j] == prefix) eqs |= 1u << j;
      } else if ((s0 + j) * T + t < n) {
        take |= 1u << j;
      }
    }
    const int in_sweep = stretches - s0 < kPer ? stretches - s0 : kPer;
    // position order within a sweep: stretch, warp, lane -> entry stretch * (T / 32) + warp
    auto number = [&](uint32_t bits, int* total, auto&& f) {
      sm.cnt[t] = 0;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if (j >= in_sweep) break;
        const uint32_t bal = __ballot_sync(0xffffffffu, (bits >> j) & 1u);
        if (lane == 0) sm.cnt[j * (T / 32) + warp] = __popc(bal);
      }
      __syncthreads();
      const int mine = cta_exclusive_scan<T>(sm.cnt[t], sm.wsum, total);
      sm.cnt[t] = mine;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if (j >= in_sweep) break;
        const uint32_t bal = __ballot_sync(0xffffffffu, (bits >> j) & 1u);
        if ((bits >> j) & 1u) f(j, sm.cnt[j * (T / 32) + warp] + __popc(bal & ((1u << lane) - 1u)));
      }
      __syncthreads();
    };
    if (!all_eq) {
      int total;
      number(eqs, &total, [&](int j, int at) {
        if (eq_seen + at < rank) take |= 1u << j;
      });
      eq_seen += total;
    }
    // The kept weights of this sweep, read before the barriers of the numbering: slots below
    // the sweep's end may be overwritten after it when the weights move in place.
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (s0 + j >= stretches) break;
      if ((take >> j) & 1u) img[j] = __float_as_uint(__ldcg(mass + (s0 + j) * T + t));
    }
    int total;
    number(take, &total, [&](int j, int at) {
      keep[kept + at] = (s0 + j) * T + t;
      mout[kept + at] = __uint_as_float(img[j]);
    });
    kept += total;
  }
  for (int i = kept + t; i < n; i += T) mout[i] = 0.f;
}

template <int T>
__global__ void __launch_bounds__(T, 1024 / T) evict_select_kernel(const EvictParams ep) {
  const EvictArgs& p = ep.a;
  __shared__ SelSmem<T> sm;
  const int t = threadIdx.x;
  const int64_t b = blockIdx.x / p.Hkv, h = blockIdx.x % p.Hkv;
  const int64_t n64 = p.context_lens[b];
  int32_t* keep = p.keep_index + (int64_t)blockIdx.x * p.budget;
  const float* mass = p.mass + b * p.stride_b + h * p.stride_h;
  float* mout = p.mass_out + b * p.out_stride_b + h * p.out_stride_h;

  // A request whose tokens would have to move is taken only if its row is sound: every page
  // that holds them mapped, and (with refcounts) owned by this request alone.
  if (t == 0) sm.bad = 0;
  __syncthreads();
  if (n64 < 0 || n64 > p.len || n64 > p.max_pages * p.page_size) {
    if (t == 0) sm.bad = 1;
  } else if (n64 > p.budget) {
    const int64_t first = p.sinks / p.page_size, last = (n64 - 1) / p.page_size;
    for (int64_t i = first + t; i <= last; i += T) {
      const int64_t pid = p.block_table[b * p.max_pages + i];
      if (pid < 0 || pid >= p.P || (p.page_refcount != nullptr && p.page_refcount[pid] != 1)) sm.bad = 1;
    }
  }
  __syncthreads();
  const bool bad = sm.bad != 0;
  const int n = bad ? 0 : (int)n64;
  const bool evicts = n > p.budget;
  if (t == 0 && h == 0) {
    p.kept[b] = bad ? (int32_t)n64 : (evicts ? (int32_t)p.budget : n);
    p.dropped[b] = evicts ? n - (int32_t)p.budget : 0;
    p.refused[b] = bad ? NVM_ERR_INVALID_ARGUMENT : NVM_OK;
    if (bad && p.status != nullptr) *p.status = NVM_ERR_INVALID_ARGUMENT;
  }
  if (!evicts) {  // everything stays (or the row is refused: no index, weights as they are)
    for (int64_t i = t; i < p.budget; i += T) keep[i] = i < n ? (int32_t)i : -1;
    if (mout != mass)
      for (int64_t i = t; i < n; i += T) mout[i] = mass[i];
    return;
  }
  const int lo = (int)p.sinks, hi = n - (int)p.recent, k = (int)(p.budget - p.sinks - p.recent);
  if (n <= kPer * T)
    select_row<T, true>(sm, mass, mout, keep, n, lo, hi, k);
  else
    select_row<T, false>(sm, mass, mout, keep, n, lo, hi, k);
}

// CTAs of 128 threads, seven to an SM (about 900 threads with 2 x 4 vectors each in flight):
// 512 (request, head) pairs x K and V are 6.9 CTAs an SM, one even wave.
// With no more than four CTAs an SM each has eight vectors a tile instead of four, and the
// registers for them (512 CTAs of int8 rows: 125 us with the selection against 139 us; 1024
// CTAs would take two waves, 257 us against 215 us).
constexpr int kCmpThreads = 128;

// Rows of one column slice: threads my_row = threadIdx / per_row of a step, kU steps a tile.
template <typename V, int kU>
__device__ __forceinline__ void compact_rows(const EvictParams& ep, int64_t b, int64_t h, uint8_t* pool, int64_t row_bytes,
                                             int col0, int cols) {
  const EvictArgs& p = ep.a;
  const int per_row = cols / (int)sizeof(V);
  const int rows_par = blockDim.x / per_row;  // rows one step of the CTA covers
  const int my_row = threadIdx.x / per_row, my_col = threadIdx.x % per_row;
  const bool active = my_row < rows_par;
  const int budget = (int)p.budget, tile = rows_par * kU;
  const int32_t* keep = p.keep_index + (b * p.Hkv + h) * p.budget;
  const int32_t* table = p.block_table + b * p.max_pages;
  const uint32_t ps = (uint32_t)p.page_size;
  const int shift = ep.page_shift;
  auto at = [&](uint32_t tok) -> V* {
    const uint32_t page = shift >= 0 ? tok >> shift : tok / ps, off = tok - page * ps;
    return reinterpret_cast<V*>(pool + (((int64_t)__ldg(table + page) * p.Hkv + h) * ps + off) * row_bytes + col0) + my_col;
  };
  // where this thread's rows of the tile at `base` come from (the slot itself: nothing moves)
  auto sources = [&](int base, int (&src)[kU]) {
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int i = base + u * rows_par + my_row;
      src[u] = active && i < budget ? __ldg(keep + i) : i;
    }
  };
  auto fetch = [&](int base, const int (&src)[kU], V (&v)[kU]) {
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (src[u] != base + u * rows_par + my_row) v[u] = __ldcs(at((uint32_t)src[u]));
  };
  int src[kU], src2[kU];
  V v[kU], v2[kU];
  sources((int)p.sinks, src);
  fetch((int)p.sinks, src, v);
  sources((int)p.sinks + tile, src2);
  for (int base = (int)p.sinks; base < budget; base += tile) {
    // the next tile's rows lie past this tile's slots: they can be read before it is written
    fetch(base + tile, src2, v2);
    int src3[kU];
    sources(base + 2 * tile, src3);
    __syncthreads();  // this tile's rows have been read by every thread
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int i = base + u * rows_par + my_row;
      if (src[u] != i) *at((uint32_t)i) = v[u];
      src[u] = src2[u];
      src2[u] = src3[u];
      v[u] = v2[u];
    }
  }
}

template <typename V, int kU>
__global__ void __launch_bounds__(kCmpThreads, kU > 4 ? 4 : 7) evict_compact_kernel(const EvictParams ep) {
  const EvictArgs& p = ep.a;
  const int64_t b = blockIdx.x / p.Hkv, h = blockIdx.x % p.Hkv;
  if (p.dropped[b] == 0) return;
  const int y = blockIdx.y;
  if (y < 2 * ep.n_slices) {
    uint8_t* pool = static_cast<uint8_t*>(y < ep.n_slices ? p.k_pages : p.v_pages);
    const int sl = y % ep.n_slices, col0 = sl * ep.slice_bytes;
    const int left = (int)ep.row_bytes - col0;
    compact_rows<V, kU>(ep, b, h, pool, ep.row_bytes, col0, left < ep.slice_bytes ? left : ep.slice_bytes);
  } else {
    uint8_t* pool = static_cast<uint8_t*>(y == 2 * ep.n_slices ? p.k_scales : p.v_scales);
    if (ep.scale_bytes == 4)
      compact_rows<uint32_t, kU>(ep, b, h, pool, 4, 0, 4);
    else
      compact_rows<uint16_t, kU>(ep, b, h, pool, 2, 0, 2);
  }
}

}  // namespace

int launch_evict(const EvictArgs& a, cudaStream_t s) {
  EvictParams ep{};
  ep.a = a;
  ep.row_bytes = a.D * (int64_t)dtype_size(a.kv_dtype);
  ep.scale_bytes = a.kv_dtype == NVM_I8 ? (int)dtype_size(a.scale_dtype) : 0;
  ep.page_shift = -1;
  for (int x = 0; x < 31; ++x)
    if (a.page_size == int64_t(1) << x) ep.page_shift = x;
  // Threads of a selection: enough to hold the longest row that the sizes allow, 32 weights a
  // thread; with no more rows than SMs, 8 a thread.  A CTA of 1024 fills an SM's registers:
  // 512 rows of 5000 took 72 us in CTAs of 1024 and 42 us in CTAs of 256 (8-bit digits).
  const dim3 sel((unsigned)(a.B * a.Hkv));
  const int64_t cap = a.len < a.max_pages * a.page_size ? a.len : a.max_pages * a.page_size;
  const int64_t per = a.B * a.Hkv <= 148 ? 8 : kPer;
  if (cap > 512 * per) evict_select_kernel<1024><<<sel, 1024, 0, s>>>(ep);
  else if (cap > 256 * per) evict_select_kernel<512><<<sel, 512, 0, s>>>(ep);
  else evict_select_kernel<256><<<sel, 256, 0, s>>>(ep);
  int st = check_cuda(cudaGetLastError(), "evict: selection kernel launch");
  if (st != NVM_OK) return st;
  // the widest vector that rows and pools are aligned to
  const uint64_t al = (uint64_t)ep.row_bytes | reinterpret_cast<uintptr_t>(a.k_pages) | reinterpret_cast<uintptr_t>(a.v_pages);
  const int vec = (al & 15) == 0 ? 16 : (al & 3) == 0 ? 4 : (al & 1) == 0 ? 2 : 1;
  // Columns of one CTA: up to 256 bytes (whole rows of 128 16-bit values), halved down to 32 while
  // the CTAs would be fewer than two per SM.  Narrow slices waste the memory's 64-byte accesses
  // (512 CTAs of whole 128-byte int8 rows 138 us with the selection, 1024 of half rows 147 us,
  // 2048 of quarter rows 236 us), but one request needs them (8 heads: 26 us against 43 us).
  int slice = vec >= 16 ? 256 : vec >= 4 ? 128 : 32;
  if (slice > ep.row_bytes) slice = (int)ep.row_bytes;
  while (slice > 32 && slice % 2 == 0 && (slice / 2) % vec == 0 &&
         a.B * a.Hkv * 2 * ((ep.row_bytes + slice - 1) / slice) < 2 * 148)
    slice /= 2;
  ep.slice_bytes = slice;
  ep.n_slices = (int)((ep.row_bytes + ep.slice_bytes - 1) / ep.slice_bytes);
  const dim3 grid((unsigned)(a.B * a.Hkv), (unsigned)(2 * ep.n_slices + (ep.scale_bytes ? 2 : 0)));
  if (vec == 16 && a.B * a.Hkv * 2 * ep.n_slices <= 4 * 148) evict_compact_kernel<uint4, 8><<<grid, kCmpThreads, 0, s>>>(ep);
  else if (vec == 16) evict_compact_kernel<uint4, 4><<<grid, kCmpThreads, 0, s>>>(ep);
  else if (vec == 4) evict_compact_kernel<uint32_t, 4><<<grid, kCmpThreads, 0, s>>>(ep);
  else if (vec == 2) evict_compact_kernel<uint16_t, 4><<<grid, kCmpThreads, 0, s>>>(ep);
  else evict_compact_kernel<uint8_t, 4><<<grid, kCmpThreads, 0, s>>>(ep);
  return check_cuda(cudaGetLastError(), "evict: compaction kernel launch");
}

}  // namespace nvm
