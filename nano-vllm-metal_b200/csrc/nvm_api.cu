// nvm_api.cu -- the extern "C" entry points of libnvm_attn.so (include/nvm_attn.h):
// argument validation (messages keep the reference operators' prefixes, e.g.
// paged_attention.cpp:22-63 and flash_attention.cpp:20-56), kernel selection, the
// per-device error word and tensor-map encoding.
#include <cudaTypedefs.h>
#include <unistd.h>

#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <mutex>
#include <string>

#include "nvm_internal.h"

__device__ int g_nvm_error_word;

namespace nvm {

namespace {
thread_local std::string t_last_error;
std::mutex g_mu;
int* g_err_ptr[64] = {nullptr};
PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;

bool env_flag(const char* name) {
  const char* v = env_get(name);
  return v != nullptr && v[0] != '\0' && v[0] != '0';
}
}  // namespace

thread_local bool t_env_none = false;

const char* env_get(const char* name) { return t_env_none ? nullptr : std::getenv(name); }

EnvScope::EnvScope() {
  t_env_none = true;
  for (char** e = environ; e != nullptr && *e != nullptr; ++e)
    if (std::strncmp(*e, "NVM_", 4) == 0) t_env_none = false;
}

int fail(int status, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  t_last_error = buf;
  return status;
}

int check_cuda(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return NVM_OK;
  return fail(NVM_ERR_CUDA, "%s: CUDA error %d (%s)", what, (int)e, cudaGetErrorString(e));
}

int* device_error_word() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
  std::lock_guard<std::mutex> lock(g_mu);
  if (g_err_ptr[dev] == nullptr) {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_nvm_error_word) != cudaSuccess) return nullptr;
    g_err_ptr[dev] = static_cast<int*>(p);
  }
  return g_err_ptr[dev];
}

size_t dtype_size(int dtype) {
  switch (dtype) {
    case NVM_F32: case NVM_I32: return 4;
    case NVM_F16: case NVM_BF16: return 2;
    case NVM_I8: return 1;
    case NVM_I64: return 8;
    default: return 0;
  }
}

int encode_tmap(CUtensorMap* map, CUtensorMapDataType dt, int rank, const void* base, const uint64_t* dims,
                const uint64_t* strides_bytes, const uint32_t* box, CUtensorMapSwizzle swizzle) {
  {
    std::lock_guard<std::mutex> lock(g_mu);
    if (g_encode == nullptr) {
      void* fn = nullptr;
      cudaDriverEntryPointQueryResult q;
      cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
      if (e != cudaSuccess || fn == nullptr || q != cudaDriverEntryPointSuccess)
        return fail(NVM_ERR_CUDA, "nvm: cuTensorMapEncodeTiled entry point unavailable");
      g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    }
  }
  cuuint64_t gdim[5], gstride[4];
  cuuint32_t bdim[5], estride[5];
  for (int i = 0; i < rank; ++i) {
    gdim[i] = dims[i];
    bdim[i] = box[i];
    estride[i] = 1;
    if (i + 1 < rank) gstride[i] = strides_bytes[i];
  }
  auto encode = [&] {
    return g_encode(map, dt, (cuuint32_t)rank, const_cast<void*>(base), gdim, gstride, bdim, estride,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = encode();
  int dev = 0;
  // A driver call does not bind the device's context to a host thread that has called nothing
  // yet; the runtime does.
  if (r == CUDA_ERROR_INVALID_CONTEXT && cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) r = encode();
  if (r != CUDA_SUCCESS) return fail(NVM_ERR_CUDA, "nvm: cuTensorMapEncodeTiled failed (%d)", (int)r);
  return NVM_OK;
}

}  // namespace nvm

using namespace nvm;

namespace {

bool is_float_dtype(int d) { return d == NVM_F32 || d == NVM_F16 || d == NVM_BF16; }

// Shared validation of nvm_paged_attention / nvm_paged_attention_workspace_size.
int validate_paged(const PagedArgs& a, bool check_ptrs) {
  const char* op = a.kv_dtype == NVM_I8 ? "paged_attention_int8_decode" : "paged_attention";
  if (!is_float_dtype(a.q_dtype)) return fail(NVM_ERR_INVALID_ARGUMENT, "%s: q must be float32, float16 or bfloat16", op);
  if (!is_float_dtype(a.kv_dtype) && a.kv_dtype != NVM_I8)
    return fail(NVM_ERR_INVALID_ARGUMENT,
                "paged_attention: key_pages and value_pages must be float32, float16, bfloat16 or int8");
  if (!is_float_dtype(a.out_dtype)) return fail(NVM_ERR_INVALID_ARGUMENT, "%s: output dtype must be floating point", op);
  if (a.B < 0 || a.Hq <= 0 || a.Hkv <= 0 || a.L <= 0 || a.D <= 0 || a.P < 0 || a.page_size <= 0 ||
      a.max_pages < 0)
    return fail(NVM_ERR_INVALID_ARGUMENT, "%s: sizes must be positive (B=%lld Hq=%lld Hkv=%lld L=%lld D=%lld)", op,
                (long long)a.B, (long long)a.Hq, (long long)a.Hkv, (long long)a.L, (long long)a.D);
  if (a.Hq % a.Hkv != 0) return fail(NVM_ERR_INVALID_ARGUMENT, "%s: num_heads must be divisible by num_kv_heads", op);
  if (a.D > 256) return fail(NVM_ERR_UNSUPPORTED, "%s: head dimension must be <= 256 (got %lld)", op, (long long)a.D);
  if (a.kv_dtype == NVM_I8) {
    if (!is_float_dtype(a.scale_dtype))
      return fail(NVM_ERR_INVALID_ARGUMENT, "%s: key_scales and value_scales must be floating point", op);
    if (check_ptrs && (a.k_scales == nullptr || a.v_scales == nullptr))
      return fail(NVM_ERR_INVALID_ARGUMENT, "%s: int8 pages need key_scales and value_scales", op);
  }
  if (check_ptrs && a.B > 0) {
    if (a.q == nullptr || a.out == nullptr || a.context_lens == nullptr || a.block_table == nullptr)
      return fail(NVM_ERR_INVALID_ARGUMENT, "%s: null tensor pointer", op);
    if (a.max_pages > 0 && a.P > 0 && (a.k_pages == nullptr || a.v_pages == nullptr))
      return fail(NVM_ERR_INVALID_ARGUMENT, "%s: null page pointer", op);
  }
  if (a.B * a.Hq * a.L > (int64_t)INT32_MAX * 4)
    return fail(NVM_ERR_UNSUPPORTED, "%s: too many query rows", op);
  return NVM_OK;
}

// Bytes of the scores that the n8 decode tile keeps (key_mass.cu says why), 0 if it does not
// serve the plan.
size_t score_bytes(const PagedArgs& a, const MmaPlan& plan) {
  if (!plan.eligible || plan.nwm != 0) return 0;
  const int64_t rows = (a.Hq / a.Hkv * a.L + 1) & ~int64_t(1);
  return (size_t)(plan.n_units * plan.n_chunks * plan.chunk_tiles * 16 * rows) * sizeof(float);
}
// Scores of more than this are kept for a part of the batch at a time.  They are sized by the block
// tables' width, 4 bytes a query row and key, and stay with the stream's workspace (256 requests of
// 128K-token tables, 64/8 heads: 8.6 GB in one part).  Parts cost their last waves: 256 requests of
// 500-8000 tokens in such tables, 32/8 heads, 1041 us in one (4.3 GB) and 1144 us in two; of 100-1000
// tokens 463 and 470 us.
constexpr size_t kMaxScoreBytes = size_t(9) << 28;

// Sequences of each launch of the mma.sync kernel (but the last) and its plan: all of them, unless
// their units outnumber the merge tickets, or their kept scores (`scored`) the limit above.
int64_t plan_parts(const PagedArgs& a, bool scored, MmaPlan* plan) {
  PagedArgs x = a;
  for (;;) {
    *plan = plan_paged_mma(x);
    int64_t most = x.B;  // sequences of a part
    if (!plan->eligible && plan->max_batch > 0) most = plan->max_batch;
    const size_t bytes = scored ? score_bytes(x, *plan) : 0;
    if (bytes > kMaxScoreBytes) most = (int64_t)(kMaxScoreBytes / (bytes / (size_t)x.B));
    if (most < 1) most = 1;
    if (most >= x.B) return x.B;
    const int64_t parts = (a.B + most - 1) / most;
    x.B = (a.B + parts - 1) / parts;
  }
}
// Sequences b0 .. b0 + n - 1 of a call.
PagedArgs batch_part(const PagedArgs& a, int64_t b0, int64_t n) {
  PagedArgs x = a;
  const int64_t rows = b0 * a.Hq * a.L * a.D;
  x.B = n;
  x.q = static_cast<const uint8_t*>(a.q) + rows * (int64_t)dtype_size(a.q_dtype);
  x.out = static_cast<uint8_t*>(a.out) + rows * (int64_t)dtype_size(a.out_dtype);
  x.block_table = a.block_table + b0 * a.max_pages;
  x.context_lens = a.context_lens + b0;
  return x;
}
// The last part's plan differs in its batch: calls f(arguments, plan, first sequence) for every part
// until one fails.
template <typename F>
int each_part(const PagedArgs& a, int64_t n, const MmaPlan& plan, F&& f) {
  if (n >= a.B) return f(a, plan, (int64_t)0);
  for (int64_t b0 = 0; b0 < a.B; b0 += n) {
    const int64_t m = a.B - b0 < n ? a.B - b0 : n;
    const PagedArgs x = batch_part(a, b0, m);
    const int st = f(x, m == n ? plan : plan_paged_mma(x), b0);
    if (st != NVM_OK) return st;
  }
  return NVM_OK;
}
// Workspace of the mma.sync kernel's part of a call, over its parts.
size_t parts_ws(const PagedArgs& a, int64_t n, const MmaPlan& plan) {
  size_t need = plan.eligible ? plan.ws_bytes : 0;
  PagedArgs x = a;
  x.B = a.B % n;
  if (n < a.B && x.B != 0) {
    const MmaPlan last = plan_paged_mma(x);
    if (last.eligible && last.ws_bytes > need) need = last.ws_bytes;
  }
  return need;
}

// Stands for the log-sum-exp buffer while a call is planned, before its workspace is known.
float kLseLater;

// Scored decode through the workspace with fewer units than this leaves its merges to the kernel
// over the scores: the one CTA of 64 threads that ends a unit needs up to 40 us for 60 chunks
// while most SMs have run dry (4 kv-head units of 16K keys 59 -> 26 us, 32 of 1.3K-10.7K keys
// 51 -> 38 us).  With many units the merges hide behind the others' keys (512 units: 430 us,
// against 460 us deferred).
constexpr int64_t kDeferUnits = 148;

// Workspace of a windowed / scored call: the attention kernel's own part, then (with key
// mass) the log-sum-exp of every query row, behind the ticket region in any case: tickets of
// other calls that share the workspace must stay zero.
struct WindowWs {
  size_t lse, scores, total;
};
WindowWs window_ws(const PagedArgs& a, size_t attn_bytes, size_t score_bytes, bool with_mass) {
  auto al = [](size_t x) { return (x + 255) & ~size_t(255); };
  WindowWs w{};
  w.lse = al(attn_bytes > kTicketRegionBytes ? attn_bytes : kTicketRegionBytes);
  w.scores = w.lse + al((size_t)(a.B * a.Hq * a.L) * sizeof(float));
  w.total = with_mass ? w.scores + score_bytes : attn_bytes;
  return w;
}

// The same over the parts of a call whose batch the mma.sync kernel takes.
size_t parts_window_ws(const PagedArgs& a, int64_t n, const MmaPlan& plan, bool with_mass) {
  PagedArgs x = a;
  x.B = n;
  size_t need = window_ws(x, plan.eligible ? plan.ws_bytes : 0, score_bytes(x, plan), with_mass).total;
  x.B = a.B % n;
  if (n < a.B && x.B != 0) {
    const MmaPlan last = plan_paged_mma(x);
    const size_t t = window_ws(x, last.eligible ? last.ws_bytes : 0, score_bytes(x, last), with_mass).total;
    if (t > need) need = t;
  }
  return need;
}

int validate_window(int64_t window, int64_t sinks, const char* op) {
  if (window < 0) return fail(NVM_ERR_INVALID_ARGUMENT, "%s: window must be positive, or 0 for none", op);
  if (sinks < 0) return fail(NVM_ERR_INVALID_ARGUMENT, "%s: sinks must not be negative", op);
  if (window > INT32_MAX || sinks > INT32_MAX)
    return fail(NVM_ERR_UNSUPPORTED, "%s: window and sinks must be below 2^31", op);
  return NVM_OK;
}

}  // namespace

extern "C" {

const char* nvm_status_string(int status) {
  switch (status) {
    case NVM_OK: return "NVM_OK";
    case NVM_ERR_INVALID_ARGUMENT: return "NVM_ERR_INVALID_ARGUMENT";
    case NVM_ERR_UNSUPPORTED: return "NVM_ERR_UNSUPPORTED";
    case NVM_ERR_WORKSPACE: return "NVM_ERR_WORKSPACE";
    case NVM_ERR_CUDA: return "NVM_ERR_CUDA";
    case NVM_ERR_DEVICE_TIMEOUT: return "NVM_ERR_DEVICE_TIMEOUT";
    case NVM_ERR_OUT_OF_PAGES: return "NVM_ERR_OUT_OF_PAGES";
    default: return "NVM_ERR_UNKNOWN";
  }
}

const char* nvm_last_error(void) { return t_last_error.c_str(); }

const char* nvm_version(void) { return "nvm_attn 0.1 sm_100a"; }

int nvm_device_error(void* stream, int clear) {
  int* w = device_error_word();
  if (w == nullptr) return fail(NVM_ERR_CUDA, "nvm_device_error: no device error word");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int st = check_cuda(cudaStreamSynchronize(s), "nvm_device_error");
  if (st != NVM_OK) return st;
  int v = 0;
  st = check_cuda(cudaMemcpy(&v, w, sizeof(int), cudaMemcpyDeviceToHost), "nvm_device_error");
  if (st != NVM_OK) return st;
  if (clear && v != 0) {
    st = check_cuda(cudaMemset(w, 0, sizeof(int)), "nvm_device_error");
    if (st != NVM_OK) return st;
  }
  return v;
}

int nvm_stream_capture_id(void* stream, unsigned long long* id) {
  if (id == nullptr) return fail(NVM_ERR_INVALID_ARGUMENT, "nvm_stream_capture_id: null pointer");
  *id = 0;
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long which = 0;
  const int st = check_cuda(cudaStreamGetCaptureInfo(static_cast<cudaStream_t>(stream), &status, &which),
                            "nvm_stream_capture_id");
  if (st == NVM_OK && status == cudaStreamCaptureStatusActive) *id = which;
  return st;
}

size_t nvm_paged_attention_workspace_size(int64_t B, int64_t Hq, int64_t Hkv, int64_t L, int64_t D,
                                          int64_t page_size, int64_t max_pages, int kv_dtype) {
  PagedArgs a{};
  a.q_dtype = NVM_F32;
  a.kv_dtype = kv_dtype;
  a.scale_dtype = NVM_F16;
  a.out_dtype = NVM_F32;
  a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.L = L; a.D = D; a.P = 1; a.page_size = page_size; a.max_pages = max_pages;
  a.is_causal = 1;
  if (validate_paged(a, false) != NVM_OK) return 0;
  if (env_flag("NVM_ATTN_FORCE_GENERIC")) return 0;
  // q's dtype is not known here: cover the tcgen05 plan (taken when q matches the pages)
  // and the mma.sync plan (taken otherwise).
  MmaPlan plan{};
  const int64_t n = plan_parts(a, false, &plan);
  size_t need = n > 0 ? parts_ws(a, n, plan) : 0;
  if (!env_flag("NVM_ATTN_NO_SM100")) {
    const Sm100Plan sp = plan_sm100(a, true);
    if (sp.eligible && sp.ws_bytes > need) need = sp.ws_bytes;
  }
  return need;
}

int nvm_paged_attention(const void* q, int q_dtype, const void* k_pages, const void* v_pages, int kv_dtype,
                        const void* k_scales, const void* v_scales, int scale_dtype,
                        const int32_t* block_table, const int32_t* context_lens, void* out, int out_dtype,
                        int64_t B, int64_t Hq, int64_t Hkv, int64_t L, int64_t D, int64_t P, int64_t page_size,
                        int64_t max_pages, float scale, int is_causal, void* workspace, size_t workspace_bytes,
                        void* stream) {
  PagedArgs a{};
  a.q = q; a.q_dtype = q_dtype; a.k_pages = k_pages; a.v_pages = v_pages; a.kv_dtype = kv_dtype;
  a.k_scales = k_scales; a.v_scales = v_scales; a.scale_dtype = scale_dtype;
  a.block_table = block_table; a.context_lens = context_lens; a.out = out; a.out_dtype = out_dtype;
  a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.L = L; a.D = D; a.P = P; a.page_size = page_size; a.max_pages = max_pages;
  a.scale = scale; a.is_causal = is_causal ? 1 : 0; a.dense_ctx = 0;
  int st = validate_paged(a, true);
  if (st != NVM_OK) return st;
  if (B == 0) return NVM_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!env_flag("NVM_ATTN_FORCE_GENERIC")) {
    if (!env_flag("NVM_ATTN_NO_SM100") && flash2q_eligible(a)) return launch_flash2q(a, s);
    if (!env_flag("NVM_ATTN_NO_SM100")) {
      const Sm100Plan sp = plan_sm100(a, false);
      if (sp.eligible) {
        if (sp.ws_bytes > 0 && (workspace == nullptr || workspace_bytes < sp.ws_bytes))
          return fail(NVM_ERR_WORKSPACE, "paged_attention: workspace of %zu bytes required, %zu given", sp.ws_bytes,
                      workspace_bytes);
        return launch_sm100(a, sp, workspace, s);
      }
    }
    MmaPlan plan{};
    const int64_t n = plan_parts(a, false, &plan);
    if (plan.eligible) {
      const size_t need = parts_ws(a, n, plan);
      if (need > 0 && (workspace == nullptr || workspace_bytes < need))
        return fail(NVM_ERR_WORKSPACE, "paged_attention: workspace of %zu bytes required, %zu given", need,
                    workspace_bytes);
      return each_part(a, n, plan, [&](const PagedArgs& x, const MmaPlan& xp, int64_t) {
        return xp.eligible ? launch_paged_mma(x, xp, workspace, s) : launch_paged_generic(x, s);
      });
    }
  }
  return launch_paged_generic(a, s);
}

int nvm_flash_attention(const void* q, const void* k, const void* v, int dtype, const float* mask,
                        int64_t mask_stride_n, int64_t mask_stride_l, int64_t mask_stride_s, void* out,
                        int out_dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t L, int64_t S, int64_t D,
                        float scale, int is_causal, void* stream) {
  if (!is_float_dtype(dtype)) return fail(NVM_ERR_INVALID_ARGUMENT, "flash_attention: all input arrays must be float32, float16 or bfloat16");
  if (!is_float_dtype(out_dtype)) return fail(NVM_ERR_INVALID_ARGUMENT, "flash_attention: output dtype must be floating point");
  if (B < 0 || Hq <= 0 || Hkv <= 0 || L <= 0 || S <= 0 || D <= 0)
    return fail(NVM_ERR_INVALID_ARGUMENT, "flash_attention: sizes must be positive");
  if (Hq % Hkv != 0) return fail(NVM_ERR_INVALID_ARGUMENT, "flash_attention: num_heads must be divisible by num_kv_heads");
  if (D > 256) return fail(NVM_ERR_UNSUPPORTED, "flash_attention: E must be <= 256 (got %lld)", (long long)D);
  if (B == 0) return NVM_OK;
  if (q == nullptr || k == nullptr || v == nullptr || out == nullptr)
    return fail(NVM_ERR_INVALID_ARGUMENT, "flash_attention: null tensor pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (mask == nullptr && dtype != NVM_F32 && !env_flag("NVM_ATTN_FORCE_GENERIC")) {
    // Dense K/V [B*Hkv, S, D] viewed as a pool of B pages of size S (page id = b).
    PagedArgs a{};
    a.q = q; a.q_dtype = dtype; a.k_pages = k; a.v_pages = v; a.kv_dtype = dtype;
    a.block_table = nullptr; a.context_lens = nullptr; a.out = out; a.out_dtype = out_dtype;
    a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.L = L; a.D = D; a.P = B; a.page_size = S; a.max_pages = 1;
    a.scale = scale; a.is_causal = is_causal ? 1 : 0; a.dense = 1; a.dense_ctx = S;
    if (!env_flag("NVM_ATTN_NO_SM100")) {
      if (flash2q_eligible(a)) return launch_flash2q(a, s);
      const Sm100Plan sp = plan_sm100(a, false);
      if (sp.eligible && sp.ws_bytes == 0) return launch_sm100(a, sp, nullptr, s);
    }
    MmaPlan plan = plan_paged_mma(a);
    if (plan.eligible && plan.ws_bytes == 0) return launch_paged_mma(a, plan, nullptr, s);
  }
  FlashArgs f{};
  f.q = q; f.k = k; f.v = v; f.dtype = dtype; f.mask = mask;
  f.ms_n = mask_stride_n; f.ms_l = mask_stride_l; f.ms_s = mask_stride_s;
  f.out = out; f.out_dtype = out_dtype;
  f.B = B; f.Hq = Hq; f.Hkv = Hkv; f.L = L; f.S = S; f.D = D; f.scale = scale; f.is_causal = is_causal ? 1 : 0;
  return launch_flash_generic(f, s);
}

size_t nvm_paged_attention_window_workspace_size(int64_t B, int64_t Hq, int64_t Hkv, int64_t L, int64_t D,
                                                 int64_t page_size, int64_t max_pages, int kv_dtype, int64_t window,
                                                 int64_t sinks, int with_mass) {
  const EnvScope env;
  PagedArgs a{};
  a.q_dtype = NVM_F32;
  a.kv_dtype = kv_dtype;
  a.scale_dtype = NVM_F16;
  a.out_dtype = NVM_F32;
  a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.L = L; a.D = D; a.P = 1; a.page_size = page_size; a.max_pages = max_pages;
  a.window = window; a.sinks = sinks;
  if (validate_paged(a, false) != NVM_OK || validate_window(window, sinks, "paged_attention") != NVM_OK) return 0;
  if (with_mass) a.lse = &kLseLater;
  // q's dtype and the mask are not known here: cover both kernels' plans, and both masks (without
  // the causal limit the rows of a block see on to the last key, so windows take more chunks)
  size_t total = window_ws(a, 0, 0, with_mass != 0).total;
  for (int causal = 0; causal < 2 && !env_flag("NVM_ATTN_FORCE_GENERIC"); ++causal) {
    a.is_causal = causal;
    size_t t = 0;
    if (!env_flag("NVM_ATTN_NO_SM100")) {
      const Sm100Plan sp = plan_sm100(a, true);
      if (sp.eligible) t = window_ws(a, sp.ws_bytes, 0, with_mass != 0).total;
    }
    if (t > total) total = t;
    MmaPlan plan{};
    const int64_t n = plan_parts(a, with_mass != 0, &plan);
    if (n > 0) t = parts_window_ws(a, n, plan, with_mass != 0);
    if (t > total) total = t;
  }
  return total;
}

int nvm_paged_attention_window(const void* q, int q_dtype, const void* k_pages, const void* v_pages, int kv_dtype,
                               const void* k_scales, const void* v_scales, int scale_dtype,
                               const int32_t* block_table, const int32_t* context_lens, void* out, int out_dtype,
                               int64_t B, int64_t Hq, int64_t Hkv, int64_t L, int64_t D, int64_t P,
                               int64_t page_size, int64_t max_pages, float scale, int is_causal, int64_t window,
                               int64_t sinks, float* key_mass, int64_t mass_stride_b, int64_t mass_stride_h,
                               int64_t mass_len, void* workspace, size_t workspace_bytes, void* stream) {
  const EnvScope env;
  PagedArgs a{};
  a.q = q; a.q_dtype = q_dtype; a.k_pages = k_pages; a.v_pages = v_pages; a.kv_dtype = kv_dtype;
  a.k_scales = k_scales; a.v_scales = v_scales; a.scale_dtype = scale_dtype;
  a.block_table = block_table; a.context_lens = context_lens; a.out = out; a.out_dtype = out_dtype;
  a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.L = L; a.D = D; a.P = P; a.page_size = page_size; a.max_pages = max_pages;
  a.scale = scale; a.is_causal = is_causal ? 1 : 0; a.window = window; a.sinks = sinks;
  int st = validate_paged(a, true);
  if (st != NVM_OK) return st;
  st = validate_window(window, sinks, "paged_attention");
  if (st != NVM_OK) return st;
  if (key_mass != nullptr && (mass_len < 0 || mass_stride_b < 0 || mass_stride_h < 0))
    return fail(NVM_ERR_INVALID_ARGUMENT, "paged_attention: key_mass sizes must not be negative");
  if (B == 0) return NVM_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (key_mass != nullptr) a.lse = &kLseLater;
  Sm100Plan sp{};
  MmaPlan plan{};
  int64_t n = B;
  if (!env_flag("NVM_ATTN_FORCE_GENERIC")) {
    if (!env_flag("NVM_ATTN_NO_SM100")) sp = plan_sm100(a, false);
    if (!sp.eligible) n = plan_parts(a, key_mass != nullptr, &plan);
  }
  const size_t need = sp.eligible ? window_ws(a, sp.ws_bytes, 0, key_mass != nullptr).total
                                  : parts_window_ws(a, n, plan, key_mass != nullptr);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(NVM_ERR_WORKSPACE, "paged_attention: workspace of %zu bytes required, %zu given", need, workspace_bytes);
  return each_part(a, n, plan, [&](PagedArgs x, const MmaPlan& xp, int64_t b0) {
    KeyMassArgs m{key_mass, mass_stride_b, mass_stride_h, mass_len};
    if (key_mass != nullptr) {
      m.mass += b0 * mass_stride_b;
      const size_t kept = score_bytes(x, xp);
      const WindowWs ws = window_ws(x, sp.eligible ? sp.ws_bytes : xp.eligible ? xp.ws_bytes : 0, kept, true);
      x.lse = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + ws.lse);
      if (kept > 0) {
        x.scores = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + ws.scores);
        if (xp.ws_bytes == 0)
          x.mass = m.mass;  // the attention kernel weighs them too
        else
          x.defer = xp.n_units < kDeferUnits && mass_len > 0 ? 1 : 0;  // no entries: no kernel over the scores
        x.mass_sb = mass_stride_b; x.mass_sh = mass_stride_h; x.mass_len = mass_len;
      }
    }
    const int r = sp.eligible   ? launch_sm100(x, sp, workspace, s)
                  : xp.eligible ? launch_paged_mma(x, xp, workspace, s)
                                : launch_paged_generic(x, s);
    if (r != NVM_OK || key_mass == nullptr || x.mass != nullptr) return r;
    return launch_key_mass(x, m, &xp, workspace, sp.eligible || xp.eligible, s);
  });
}

int nvm_flash_attention_window(const void* q, const void* k, const void* v, int dtype, void* out, int out_dtype,
                               int64_t B, int64_t Hq, int64_t Hkv, int64_t L, int64_t S, int64_t D, float scale,
                               int is_causal, int64_t window, int64_t sinks, void* stream) {
  const EnvScope env;
  if (!is_float_dtype(dtype)) return fail(NVM_ERR_INVALID_ARGUMENT, "flash_attention: all input arrays must be float32, float16 or bfloat16");
  if (!is_float_dtype(out_dtype)) return fail(NVM_ERR_INVALID_ARGUMENT, "flash_attention: output dtype must be floating point");
  if (B < 0 || Hq <= 0 || Hkv <= 0 || L <= 0 || S <= 0 || D <= 0)
    return fail(NVM_ERR_INVALID_ARGUMENT, "flash_attention: sizes must be positive");
  if (Hq % Hkv != 0) return fail(NVM_ERR_INVALID_ARGUMENT, "flash_attention: num_heads must be divisible by num_kv_heads");
  if (D > 256) return fail(NVM_ERR_UNSUPPORTED, "flash_attention: E must be <= 256 (got %lld)", (long long)D);
  if (B * Hq * L > (int64_t)INT32_MAX * 4) return fail(NVM_ERR_UNSUPPORTED, "flash_attention: too many query rows");
  int st = validate_window(window, sinks, "flash_attention");
  if (st != NVM_OK) return st;
  if (B == 0) return NVM_OK;
  if (q == nullptr || k == nullptr || v == nullptr || out == nullptr)
    return fail(NVM_ERR_INVALID_ARGUMENT, "flash_attention: null tensor pointer");
  PagedArgs a{};  // dense K/V [B*Hkv, S, D] viewed as a pool of B pages of size S (page id = b)
  a.q = q; a.q_dtype = dtype; a.k_pages = k; a.v_pages = v; a.kv_dtype = dtype;
  a.out = out; a.out_dtype = out_dtype;
  a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.L = L; a.D = D; a.P = B; a.page_size = S; a.max_pages = 1;
  a.scale = scale; a.is_causal = is_causal ? 1 : 0; a.dense = 1; a.dense_ctx = S;
  a.window = window; a.sinks = sinks;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (window > 0 && dtype != NVM_F32 && !env_flag("NVM_ATTN_FORCE_GENERIC")) {
    if (!env_flag("NVM_ATTN_NO_SM100")) {
      const Sm100Plan sp = plan_sm100(a, false);
      if (sp.eligible && sp.ws_bytes == 0) return launch_sm100(a, sp, nullptr, s);
    }
    const MmaPlan plan = plan_paged_mma(a);
    if (plan.eligible && plan.ws_bytes == 0) return launch_paged_mma(a, plan, nullptr, s);
  }
  return launch_paged_generic(a, s);
}

int nvm_paged_evict(void* k_pages, void* v_pages, int kv_dtype, void* k_scales, void* v_scales, int scale_dtype,
                    const int32_t* block_table, const int32_t* context_lens, const int32_t* page_refcount,
                    const float* key_mass, int64_t mass_stride_b, int64_t mass_stride_h, int64_t mass_len,
                    float* mass_out, int64_t out_stride_b, int64_t out_stride_h, int64_t B, int64_t Hkv, int64_t D,
                    int64_t P, int64_t page_size, int64_t max_pages, int64_t budget, int64_t sinks, int64_t recent,
                    int32_t* keep_index, int32_t* kept, int32_t* dropped, int32_t* refused, int32_t* status,
                    void* stream) {
  if (!is_float_dtype(kv_dtype) && kv_dtype != NVM_I8)
    return fail(NVM_ERR_INVALID_ARGUMENT, "evict: pages must be float32, float16, bfloat16 or int8");
  if (kv_dtype == NVM_I8 && !is_float_dtype(scale_dtype))
    return fail(NVM_ERR_INVALID_ARGUMENT, "evict: int8 pages need floating-point key and value scales");
  if (B < 0 || Hkv <= 0 || D <= 0 || P < 0 || page_size <= 0 || max_pages < 0 || mass_len < 0)
    return fail(NVM_ERR_INVALID_ARGUMENT, "evict: sizes must be positive");
  if (mass_stride_b < 0 || mass_stride_h < 0 || out_stride_b < 0 || out_stride_h < 0)
    return fail(NVM_ERR_INVALID_ARGUMENT, "evict: strides must not be negative");
  if (budget < 1 || sinks < 0 || recent < 0 || sinks + recent > budget)
    return fail(NVM_ERR_INVALID_ARGUMENT, "evict: need budget >= 1, sinks >= 0, recent >= 0 and sinks + recent <= budget");
  if (D > 256) return fail(NVM_ERR_UNSUPPORTED, "evict: head dimension must be <= 256 (got %lld)", (long long)D);
  if (budget > INT32_MAX || page_size > INT32_MAX || B * Hkv > INT32_MAX)
    return fail(NVM_ERR_UNSUPPORTED, "evict: budget, page_size and B * Hkv must be below 2^31");
  // the kernels count a row's positions in 32 bits, up to a sweep of 32 x 1024 past its end
  if (mass_len > INT32_MAX - 65536 && max_pages > (INT32_MAX - 65536) / page_size)
    return fail(NVM_ERR_UNSUPPORTED, "evict: requests of more than 2^31 - 65537 tokens are not supported");
  if (B == 0) return NVM_OK;
  if (!k_pages || !v_pages || !block_table || !context_lens || !key_mass || !mass_out || !keep_index || !kept ||
      !dropped || !refused || (kv_dtype == NVM_I8 && (!k_scales || !v_scales)))
    return fail(NVM_ERR_INVALID_ARGUMENT, "evict: null tensor pointer");
  EvictArgs a{};
  a.k_pages = k_pages; a.v_pages = v_pages; a.kv_dtype = kv_dtype; a.k_scales = k_scales; a.v_scales = v_scales;
  a.scale_dtype = scale_dtype; a.block_table = block_table; a.context_lens = context_lens;
  a.page_refcount = page_refcount; a.mass = key_mass; a.mass_out = mass_out;
  a.stride_b = mass_stride_b; a.stride_h = mass_stride_h; a.len = mass_len;
  a.out_stride_b = out_stride_b; a.out_stride_h = out_stride_h;
  a.B = B; a.Hkv = Hkv; a.D = D; a.P = P; a.page_size = page_size; a.max_pages = max_pages;
  a.budget = budget; a.sinks = sinks; a.recent = recent;
  a.keep_index = keep_index; a.kept = kept; a.dropped = dropped; a.refused = refused; a.status = status;
  return launch_evict(a, static_cast<cudaStream_t>(stream));
}

int nvm_reshape_and_cache(const void* k, const void* v, int in_dtype, int64_t stride_t, int64_t stride_h,
                          void* k_pages, void* v_pages, int kv_dtype, void* k_scales, void* v_scales,
                          int scale_dtype, const int64_t* slot_mapping, int64_t T, int64_t Hkv, int64_t D,
                          int64_t P, int64_t page_size, void* stream) {
  if (!is_float_dtype(in_dtype)) return fail(NVM_ERR_INVALID_ARGUMENT, "write_page_slice: key/value must be floating point");
  if (kv_dtype != in_dtype && kv_dtype != NVM_I8)
    return fail(NVM_ERR_INVALID_ARGUMENT, "write_page_slice: page dtype must equal the input dtype or be int8");
  if (kv_dtype == NVM_I8 && (k_scales == nullptr || v_scales == nullptr || !is_float_dtype(scale_dtype)))
    return fail(NVM_ERR_INVALID_ARGUMENT, "write_page_slice: int8 pages need floating-point key/value scales");
  if (T < 0 || Hkv <= 0 || D <= 0 || P < 0 || page_size <= 0)
    return fail(NVM_ERR_INVALID_ARGUMENT, "write_page_slice: sizes must be positive");
  if (T == 0) return NVM_OK;
  if (k == nullptr || v == nullptr || k_pages == nullptr || v_pages == nullptr || slot_mapping == nullptr)
    return fail(NVM_ERR_INVALID_ARGUMENT, "write_page_slice: null tensor pointer");
  return launch_kv_write(k, v, in_dtype, stride_t, stride_h, k_pages, v_pages, kv_dtype, k_scales, v_scales,
                         scale_dtype, slot_mapping, T, Hkv, D, P, page_size, static_cast<cudaStream_t>(stream));
}

int nvm_paged_append(int32_t* block_table, int32_t* context_lens, const int32_t* new_tokens, int32_t* free_stack,
                     int32_t* free_top, int32_t* num_pages, int32_t* page_refcount, int64_t* slot_mapping,
                     int64_t slot_capacity, int32_t* status, int64_t B, int64_t max_pages, int64_t page_size,
                     int64_t capacity, void* stream) {
  if (B < 0 || B > 4096 || max_pages < 0 || page_size <= 0 || capacity < 0 || slot_capacity < 0)
    return fail(NVM_ERR_INVALID_ARGUMENT, "allocate_page: invalid sizes (B must be in [0, 4096])");
  if (B == 0) return NVM_OK;
  if (!block_table || !context_lens || !new_tokens || !free_stack || !free_top || !num_pages || !page_refcount ||
      !slot_mapping || !status)
    return fail(NVM_ERR_INVALID_ARGUMENT, "allocate_page: null tensor pointer");
  return launch_paged_append(block_table, context_lens, new_tokens, free_stack, free_top, num_pages, page_refcount,
                             slot_mapping, slot_capacity, status, B, max_pages, page_size, capacity,
                             static_cast<cudaStream_t>(stream));
}

int nvm_paged_rewind(int32_t* block_table, int32_t* context_lens, const int32_t* rewind, int32_t* free_stack,
                     int32_t* free_top, int32_t* page_refcount, int32_t* last_call, int32_t* status, int64_t B,
                     int64_t max_pages, int64_t page_size, int64_t capacity, void* stream) {
  if (B < 0 || B > 4096 || max_pages < 0 || page_size <= 0 || capacity < 0)
    return fail(NVM_ERR_INVALID_ARGUMENT, "rewind: invalid sizes (B must be in [0, 4096])");
  if (B == 0) return NVM_OK;
  if (!block_table || !context_lens || !rewind || !free_stack || !free_top || !page_refcount || !last_call || !status)
    return fail(NVM_ERR_INVALID_ARGUMENT, "rewind: null tensor pointer");
  return launch_paged_rewind(block_table, context_lens, rewind, free_stack, free_top, page_refcount, last_call, status,
                             B, max_pages, page_size, capacity, static_cast<cudaStream_t>(stream));
}

int nvm_paged_attach(int32_t* block_table, int32_t* context_lens, const int32_t* pages, const int32_t* count,
                     int32_t* page_refcount, int32_t* status, int64_t B, int64_t max_pages, int64_t page_size,
                     int64_t max_prefix, int64_t capacity, void* stream) {
  if (B < 0 || B > 4096 || max_pages < 0 || page_size <= 0 || max_prefix < 0 || capacity < 0)
    return fail(NVM_ERR_INVALID_ARGUMENT, "attach: invalid sizes (B must be in [0, 4096])");
  if (B == 0) return NVM_OK;
  if (!block_table || !context_lens || !count || !page_refcount || !status || (max_prefix > 0 && !pages))
    return fail(NVM_ERR_INVALID_ARGUMENT, "attach: null tensor pointer");
  return launch_paged_attach(block_table, context_lens, pages, count, page_refcount, status, B, max_pages, page_size,
                             max_prefix, capacity, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
