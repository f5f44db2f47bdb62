// u4_append.cu -- the step before attention over a 4-bit cache: q/k RMSNorm (optional), rotary position
// embedding of q and k, and K and V quantised into their slots (u4.cuh has the row format).
//
// The same operator as qk_prep.cu over another kind of pages, with its rounding points and, for the
// norm, its order of summation, so that q and the rows handed to the quantiser are bit for bit those
// that 16-bit pages would get.  A lane holds four neighbouring elements of each half of a row (8-byte
// vectors), so a warp works on 256 / D rows at once: a group's extremes are three or four shuffles away and
// a lane's codes of a half are 16 bits.  A warp walks rows of one kind of one token, all q, all k or all v,
// with the loads of the next kAhead steps in flight; few tokens are spread over more warps, down to one
// step each.  Bound by HBM (22 KB a token, 32/8 heads) as far as issue allows: 8192 tokens, bf16, 49 us
// without a norm (3.7 TB/s, issue slots 71 % busy) and 59 with one; one token 3.1 us.  In qk_prep.cu's
// layout (a row over 32 lanes, eight rows unrolled) the same took 1.4 and 1.5 times as long, one token twice.
#include <algorithm>

#include "nvm_internal.h"
#include "u4.cuh"

namespace nvm {
namespace {

constexpr int kWarps = 8;
constexpr int kBlocks = 4;  // of an SM (8192 f16 tokens appended and read back, 59.4 us: 3 67.0; 5, which spills, 62.8)
constexpr int kMost = 8;   // steps of a warp (the same: 4 59.5, 16 69.9)
constexpr int kAhead = 4;  // steps whose loads are in flight

struct AppendParams {
  const void* q;
  const void* k;
  const void* v;
  const void* wq;  // both NULL: rows are rotated as they are
  const void* wk;
  const float* cos_t;
  const float* sin_t;
  const int32_t* pos;
  const int64_t* slots;
  void* q_out;
  uint8_t* kp;
  uint8_t* vp;
  void* ks;
  void* vs;
  int* err;
  int64_t q_st, kv_st, table_rows, q_out_L, P, ps;
  FastDiv by_ps, by_warps;
  int T, Hq, Hkv, each, q_warps, kv_warps;  // each: steps of a warp; warps of a token
  float eps;
};

template <typename T>
__device__ __forceinline__ void unpack4(uint2 u, float* x) {
  const float2 a = u4_pair<T>(u.x), b = u4_pair<T>(u.y);
  x[0] = a.x;
  x[1] = a.y;
  x[2] = b.x;
  x[3] = b.y;
}
template <typename T>
__device__ __forceinline__ uint2 pack4(const float* x) {
  return make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
}

// Steps [0, n) of a warp's rows of one kind (a step is kRows heads, the lane's at `head` and up): rotated
// (kNorm: normalised first, with weights w), then stored at dst + step * dst_step or quantised into the rows at
// pool_row + step * pool_step of codes / scales.
template <typename T, int D, bool kTrad, bool kRope, bool kQuant, bool kNorm>
__device__ __forceinline__ void walk(const T* src, int head, int heads, int n, const uint2* w, float eps, const float (&c)[4],
                                     const float (&sn)[4], T* dst, int64_t dst_step, uint8_t* codes, uint32_t* scales,
                                     int64_t pool_row, int64_t pool_step, int j) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes, kHalf = D / 2;
  uint2 lo[kAhead], hi[kAhead];  // of the steps to come
  const uint2* at = reinterpret_cast<const uint2*>(src) + j;
  auto load = [&](int i, uint2& a, uint2& b) {
    a = b = make_uint2(0, 0);
    if (i < n && head + i * kRows < heads) {
      a = __ldg(at + i * (kRows * D / 4));
      b = __ldg(at + i * (kRows * D / 4) + kHalf / 4);
    }
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) load(i, lo[i], hi[i]);
  uint2 w_lo = make_uint2(0, 0), w_hi = w_lo;
  if (kNorm) {
    w_lo = __ldg(w + j);
    w_hi = __ldg(w + kHalf / 4 + j);
  }
#pragma unroll 1
  for (int i = 0; i < n; ++i) {
    float x[8];
    unpack4<T>(lo[0], x);
    unpack4<T>(hi[0], x + 4);
#pragma unroll
    for (int e = 0; e + 1 < kAhead; ++e) {
      lo[e] = lo[e + 1];
      hi[e] = hi[e + 1];
    }
    load(i + kAhead, lo[kAhead - 1], hi[kAhead - 1]);
    const bool mine = head + i * kRows < heads;
    if constexpr (kRope) {
      if constexpr (kNorm) {
        // the order of qk_prep.cu: its lane l holds elements l * D/64 and up of both halves, and sums over
        // lanes l ^ 16, 8, 4, 2, 1; two (D = 128) or four of its lanes are one here
        float part[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) part[e] = __fmul_rn(x[e], x[e]);
        if constexpr (D == 128) {
#pragma unroll
          for (int e = 0; e < 2; ++e)
            part[e] = __fadd_rn(__fadd_rn(__fadd_rn(part[2 * e], part[2 * e + 1]), __fmul_rn(x[4 + 2 * e], x[4 + 2 * e])),
                                __fmul_rn(x[5 + 2 * e], x[5 + 2 * e]));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) part[e] = __fadd_rn(part[e], __fmul_rn(x[4 + e], x[4 + e]));
        }
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1)
#pragma unroll
          for (int e = 0; e < (D == 128 ? 2 : 4); ++e) part[e] = __fadd_rn(part[e], __shfl_xor_sync(0xffffffffu, part[e], o));
        const float sum = D == 128 ? __fadd_rn(part[0], part[1])
                                   : __fadd_rn(__fadd_rn(part[0], part[2]), __fadd_rn(part[1], part[3]));
        const float inv = __frcp_rn(__fsqrt_rn(__fadd_rn(__fmul_rn(sum, 1.0f / (float)D), eps)));
        float wx[8];
        unpack4<T>(w_lo, wx);
        unpack4<T>(w_hi, wx + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __fmul_rn(__fmul_rn(x[e], inv), wx[e]);
        unpack4<T>(pack4<T>(x), x);
        unpack4<T>(pack4<T>(x + 4), x + 4);
      }
      float y[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int a = kTrad ? 2 * e : e, b = kTrad ? 2 * e + 1 : 4 + e;
        y[a] = __fsub_rn(__fmul_rn(x[a], c[e]), __fmul_rn(x[b], sn[e]));
        y[b] = __fadd_rn(__fmul_rn(x[a], sn[e]), __fmul_rn(x[b], c[e]));
      }
      const uint2 y_lo = pack4<T>(y), y_hi = pack4<T>(y + 4);
      if constexpr (kQuant) {
        unpack4<T>(y_lo, x);
        unpack4<T>(y_hi, x + 4);
      } else if (mine) {
        uint2* to = reinterpret_cast<uint2*>(dst + i * dst_step);
        to[j] = y_lo;
        to[kHalf / 4 + j] = y_hi;
      }
    }
    if constexpr (kQuant) {  // the groups are the halves (D = 128), or the row
      constexpr int G = D / kU4Group;
      float top[2], low[2];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const float* y = x + 4 * g;
        top[g] = max_nan(max_nan(y[0], y[1]), max_nan(y[2], y[3]));
        low[g] = max_nan(max_nan(-y[0], -y[1]), max_nan(-y[2], -y[3]));
      }
      if constexpr (G == 1) {
        top[0] = max_nan(top[0], top[1]);
        low[0] = max_nan(low[0], low[1]);
      }
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1)
#pragma unroll
        for (int g = 0; g < G; ++g) {
          top[g] = max_nan(top[g], __shfl_xor_sync(0xffffffffu, top[g], o));
          low[g] = max_nan(low[g], __shfl_xor_sync(0xffffffffu, low[g], o));
        }
      // half the lanes of a row work out one group's pair, half the other's
      const bool second = G == 2 && j >= kLanes / 2;
      const float2 own = u4_scale<T>(second ? -low[1] : -low[0], second ? top[1] : top[0]);
      float2 sz[2];
      sz[0] = sz[1] = own;
      if constexpr (G == 2) {
        const float2 other = make_float2(__shfl_xor_sync(0xffffffffu, own.x, kLanes / 2),
                                         __shfl_xor_sync(0xffffffffu, own.y, kLanes / 2));
        sz[0] = second ? other : own;
        sz[1] = second ? own : other;
      }
      int code[8];
      bool amb[8], any = false;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const float r = u4_inverse(sz[g].x);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          code[4 * g + e] = u4_code_fast(x[4 * g + e], sz[g].y, r, amb[4 * g + e]);
          any |= amb[4 * g + e];
        }
      }
      if (__any_sync(0xffffffffu, any)) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (amb[e]) code[e] = u4_code_div(x[e], sz[e / 4].y, sz[e / 4].x);
      }
      if (mine) {
        const int64_t row = pool_row + i * pool_step;
        uint16_t* to = reinterpret_cast<uint16_t*>(codes + row * kHalf);
#pragma unroll
        for (int g = 0; g < 2; ++g)
          to[g * kLanes + j] = (uint16_t)(code[4 * g] | code[4 * g + 1] << 4 | code[4 * g + 2] << 8 | code[4 * g + 3] << 12);
        if (j % (kLanes / 2) == 0 && j / (kLanes / 2) < G) scales[row * G + j / (kLanes / 2)] = u4_pack_pair<T>(own);
      }
    }
  }
}

template <typename T, int D, bool kTrad, bool kNorm>
__global__ void __launch_bounds__(kWarps * 32, kBlocks) u4_append_kernel(const AppendParams p) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes, kHalf = D / 2;  // lanes of a row, rows of a step
  const int lane = threadIdx.x & 31, j = lane % kLanes, sub = lane / kLanes;
  const int warp = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int t = (int)p.by_warps((uint32_t)warp);
  if (t >= p.T) return;
  // a token's warps: q_warps of q rows, then kv_warps of k, then of v, p.each steps each
  int part = warp - t * (p.q_warps + 2 * p.kv_warps);
  const int kind = (part >= p.q_warps) + (part >= p.q_warps + p.kv_warps);
  part -= (kind > 0 ? p.q_warps : 0) + (kind > 1 ? p.kv_warps : 0);
  const int heads = kind == 0 ? p.Hq : p.Hkv, steps = (heads + kRows - 1) / kRows;
  const int s0 = part * p.each, n = min(p.each, steps - s0), head = s0 * kRows + sub;

  int64_t pid = 0, off = 0;
  if (kind > 0) {
    const int64_t slot = __ldg(p.slots + t);
    if (slot < 0) return;
    if (slot <= 0x7fffffffLL) {
      pid = p.by_ps((uint32_t)slot);
      off = (uint32_t)slot - (uint32_t)pid * (uint32_t)p.ps;
    } else {
      pid = slot / p.ps;
      off = slot - pid * p.ps;
    }
    if (pid >= p.P) {
      if (lane == 0) record_error(p.err, kDevErrBadIndex);
      return;
    }
  }
  // cos / sin of the lane's elements: halves (element e and its partner share angle e), or pairs
  float c[4] = {}, sn[4] = {};
  if (kind < 2) {
    const int pos = __ldg(p.pos + t);
    if (pos < 0 || pos >= p.table_rows) {
      if (lane == 0) record_error(p.err, kDevErrBadIndex);
      return;
    }
    const float* ct = p.cos_t + (int64_t)pos * kHalf;
    const float* st = p.sin_t + (int64_t)pos * kHalf;
    if constexpr (kTrad) {
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const float2 a = __ldg(reinterpret_cast<const float2*>(ct + e * (kHalf / 4)) + j);
        const float2 b = __ldg(reinterpret_cast<const float2*>(st + e * (kHalf / 4)) + j);
        c[e] = a.x; c[e + 1] = a.y;
        sn[e] = b.x; sn[e + 1] = b.y;
      }
    } else {
      const float4 a = __ldg(reinterpret_cast<const float4*>(ct) + j), b = __ldg(reinterpret_cast<const float4*>(st) + j);
      c[0] = a.x; c[1] = a.y; c[2] = a.z; c[3] = a.w;
      sn[0] = b.x; sn[1] = b.y; sn[2] = b.z; sn[3] = b.w;
    }
  }
  const int64_t first = (int64_t)t * (kind == 0 ? p.q_st : p.kv_st) + (int64_t)head * D;
  if (kind == 0) {
    int64_t row = (int64_t)t * p.Hq + head, mul = 1;  // of q_out: [T, Hq, D], or [T / L, Hq, L, D]
    if (p.q_out_L > 0) {
      const int bb = t / (int)p.q_out_L;
      row = ((int64_t)bb * p.Hq + head) * p.q_out_L + (t - bb * (int)p.q_out_L);
      mul = p.q_out_L;
    }
    walk<T, D, kTrad, true, false, kNorm>(static_cast<const T*>(p.q) + first, head, heads, n, static_cast<const uint2*>(p.wq), p.eps, c, sn,
                                   static_cast<T*>(p.q_out) + row * D, mul * (kRows * D), nullptr, nullptr, 0, 0, j);
    return;
  }
  const int64_t row = (pid * p.Hkv + head) * p.ps + off, step = kRows * p.ps;
  if (kind == 1)
    walk<T, D, kTrad, true, true, kNorm>(static_cast<const T*>(p.k) + first, head, heads, n, static_cast<const uint2*>(p.wk), p.eps, c, sn,
                                  nullptr, 0, p.kp, static_cast<uint32_t*>(p.ks), row, step, j);
  else
    walk<T, D, kTrad, false, true, false>(static_cast<const T*>(p.v) + first, head, heads, n, nullptr, p.eps, c, sn, nullptr, 0, p.vp,
                                   static_cast<uint32_t*>(p.vs), row, step, j);
}

template <typename T, int D>
void launch(const AppendParams& p, bool traditional, unsigned grid, cudaStream_t s) {
  const bool norm = p.wq != nullptr;
  if (traditional)
    norm ? u4_append_kernel<T, D, true, true><<<grid, kWarps * 32, 0, s>>>(p) : u4_append_kernel<T, D, true, false><<<grid, kWarps * 32, 0, s>>>(p);
  else
    norm ? u4_append_kernel<T, D, false, true><<<grid, kWarps * 32, 0, s>>>(p) : u4_append_kernel<T, D, false, false><<<grid, kWarps * 32, 0, s>>>(p);
}

}  // namespace

int launch_u4_append(const U4AppendArgs& a, cudaStream_t s) {
  AppendParams p{};
  p.wq = a.wq; p.wk = a.wk; p.cos_t = a.cos_table; p.sin_t = a.sin_table;
  p.kp = static_cast<uint8_t*>(a.k_pages); p.vp = static_cast<uint8_t*>(a.v_pages); p.ks = a.k_scales; p.vs = a.v_scales;
  p.err = device_error_word();
  p.q_st = a.q_stride_t; p.kv_st = a.kv_stride_t; p.table_rows = a.table_rows; p.q_out_L = a.q_out_L; p.P = a.P; p.ps = a.page_size;
  p.Hq = (int)a.Hq; p.Hkv = (int)a.Hkv; p.eps = a.eps;
  const int rows = (int)(256 / a.D);  // of a step
  const int q_steps = (p.Hq + rows - 1) / rows, kv_steps = (p.Hkv + rows - 1) / rows;
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  // steps of a warp: few tokens are spread over as many warps as the SMs hold
  p.each = (int)std::min<int64_t>(kMost, std::max<int64_t>(1, a.T * (q_steps + 2 * kv_steps) / (kBlocks * kWarps * (int64_t)sms)));
  p.q_warps = (q_steps + p.each - 1) / p.each;
  p.kv_warps = (kv_steps + p.each - 1) / p.each;
  p.by_ps = FastDiv(a.page_size);
  p.by_warps = FastDiv(p.q_warps + 2 * p.kv_warps);
  const int64_t units = p.q_warps + 2 * p.kv_warps, L = a.q_out_L > 0 ? a.q_out_L : 1;
  // tokens of a launch: warps are counted in 32 bits, and q_out's batches are whole
  const int64_t most = std::max<int64_t>((INT32_MAX - kWarps) / units / L * L, L);
  if (most * units > INT32_MAX - kWarps) return fail(NVM_ERR_UNSUPPORTED, "qk_norm_rope_write: too many tokens a sequence");
  for (int64_t t0 = 0; t0 < a.T; t0 += most) {
    p.T = (int)std::min(most, a.T - t0);
    p.q = static_cast<const uint16_t*>(a.q) + t0 * a.q_stride_t;
    p.k = static_cast<const uint16_t*>(a.k) + t0 * a.kv_stride_t;
    p.v = static_cast<const uint16_t*>(a.v) + t0 * a.kv_stride_t;
    p.pos = a.positions + t0;
    p.slots = a.slots + t0;
    p.q_out = static_cast<uint16_t*>(a.q_out) + t0 * a.Hq * a.D;
    const unsigned grid = (unsigned)((p.T * units + kWarps - 1) / kWarps);
    if (a.dtype == NVM_BF16)
      a.D == 128 ? launch<__nv_bfloat16, 128>(p, a.traditional, grid, s) : launch<__nv_bfloat16, 64>(p, a.traditional, grid, s);
    else
      a.D == 128 ? launch<__half, 128>(p, a.traditional, grid, s) : launch<__half, 64>(p, a.traditional, grid, s);
    const int st = check_cuda(cudaGetLastError(), "qk_norm_rope_write: kernel launch");
    if (st != NVM_OK) return st;
  }
  return NVM_OK;
}

}  // namespace nvm
