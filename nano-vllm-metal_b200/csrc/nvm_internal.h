// nvm_internal.h -- host-side declarations shared by the translation units of
// libnvm_attn.so (not part of the public ABI; see include/nvm_attn.h for that).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "nvm_attn.h"

namespace nvm {

// Records the message returned by nvm_last_error() for this thread; returns `status`.
int fail(int status, const char* fmt, ...);
// Maps a CUDA runtime error (after a launch or API call) to NVM_ERR_CUDA + message.
int check_cuda(cudaError_t e, const char* what);
// Device address of the calling device's error word (set up once per device).
int* device_error_word();

size_t dtype_size(int dtype);

// The tuning variables are read on every call, a dozen of them, and each getenv walks the whole
// environment (0.4 us among 130 variables).  While an EnvScope lives on this thread and one walk
// found no name that begins with NVM_, env_get answers without another.
extern thread_local bool t_env_none;
const char* env_get(const char* name);
struct EnvScope {
  EnvScope();
  ~EnvScope() { t_env_none = false; }
};

// Bytes at the start of every split-K workspace that hold the ticket counters: zero
// before a call, zero again after a successful one.  paged_mma.cu and flash_sm100.cu
// lay their counters out inside this region; noalloc.cu clears exactly this much.
constexpr size_t kTicketRegionBytes = size_t(1) << 20;

// Arguments of one paged-attention call after validation.  block_table == nullptr
// selects the dense identity layout used by flash attention: sequence b owns
// "page" b of size page_size == S, and context_lens == nullptr means every
// sequence holds `dense_ctx` tokens.
struct PagedArgs {
  const void* q;
  int q_dtype;
  const void* k_pages;
  const void* v_pages;
  int kv_dtype;
  const void* k_scales;
  const void* v_scales;
  int scale_dtype;
  const int32_t* block_table;
  const int32_t* context_lens;
  void* out;
  int out_dtype;
  int64_t B, Hq, Hkv, L, D, P, page_size, max_pages;
  float scale;
  int is_causal;
  int dense;          // 1: dense K/V viewed as one page per sequence (no block table)
  int64_t dense_ctx;  // tokens per sequence when dense
  // Windowed / scored calls (nvm_paged_attention_window, nvm_flash_attention_window); all
  // zero otherwise.  A row at position pos = l + ctx - L sees key s only if s < sinks or
  // s > pos - window (window == 0: no such limit).
  int64_t window, sinks;
  float* lse;         // [B*Hq*L] log2 of sum 2^(score * log2 e) of every row (+inf: no key), or NULL
  float* scores;      // n8 tile only: keep every base-2 score, [B*Hkv][virtual keys][rows, even], or NULL
  int defer;          // with scores: leave the merge through the workspace to the kernel over the scores
  float* mass;        // with scores, and no merge through the workspace: add the weights, or NULL
  int64_t mass_sb, mass_sh, mass_len;
  float out_scale = 1.0f;  // factor of the output, of the tcgen05 kernel only
};
inline bool paged_is_ext(const PagedArgs& a) { return a.window > 0 || a.lse != nullptr; }

// Generic CUDA-core kernel: any D <= 256, any page_size, F32/F16/BF16/I8 pages.
int launch_paged_generic(const PagedArgs& a, cudaStream_t s);

// Accumulated attention weight per cached key (key_mass.cu): for the calls' visible keys
// mass[b, h, s] = (s < ctx - L ? mass[b, h, s] : 0) + sum over the rows of kv head h of
// 2^(score_log2 - lse[row]); entries at or past min(ctx, mass_len) are left as they are.
struct KeyMassArgs {
  float* mass;
  int64_t stride_b, stride_h, len;
};
struct MmaPlan;
// plan, ws: the attention kernel's, when a.scores is set (with a.defer the launch merges its
// chunks too); tensor_cores: it was not the generic one.
int launch_key_mass(const PagedArgs& a, const KeyMassArgs& m, const MmaPlan* plan, const void* ws, bool tensor_cores,
                    cudaStream_t s);
// Where a plan's partial results lie in its workspace: (m, l) and O of [units][chunks][rows].
size_t mma_ws_ml();
size_t mma_ws_o(const MmaPlan& plan);

// Eviction by accumulated weight (evict.cu).
struct EvictArgs {
  void* k_pages;
  void* v_pages;
  int kv_dtype;
  void* k_scales;
  void* v_scales;
  int scale_dtype;
  const int32_t* block_table;
  const int32_t* context_lens;
  const int32_t* page_refcount;  // may be NULL
  const float* mass;
  float* mass_out;
  int64_t stride_b, stride_h, len;          // of mass
  int64_t out_stride_b, out_stride_h;       // of mass_out (same length)
  int64_t B, Hkv, D, P, page_size, max_pages, budget, sinks, recent;
  int32_t* keep_index;
  int32_t* kept;
  int32_t* dropped;
  int32_t* refused;
  int32_t* status;  // may be NULL
};
int launch_evict(const EvictArgs& a, cudaStream_t s);

// Generic dense flash attention with the reference's additive-mask semantics.
struct FlashArgs {
  const void* q;
  const void* k;
  const void* v;
  int dtype;
  const float* mask;
  int64_t ms_n, ms_l, ms_s;
  void* out;
  int out_dtype;
  int64_t B, Hq, Hkv, L, S, D;
  float scale;
  int is_causal;
};
int launch_flash_generic(const FlashArgs& a, cudaStream_t s);

// Tensor-core (mma.sync m16n8k16) paged kernel fed by TMA tiles.
struct MmaPlan {
  bool eligible;   // shapes/dtypes/alignment served by the tensor-core kernel
  int nwm;         // 16-row m-tiles per CTA (warps along rows)
  int nwk;         // warps splitting the key tiles of one CTA
  int variant;     // decode kernel variant (consumer warps x stage depth)
  int rows_per_block;
  int64_t n_row_blocks;
  int64_t rows_real;      // rows of one (seq, kv head) unit actually stored per block
  int64_t chunk_tiles;    // 16-token tiles per CTA (split-K granularity)
  int64_t n_chunks;       // max chunks per unit
  int64_t n_units;
  size_t ws_bytes;        // workspace for the split-K combine (0 if n_chunks == 1 or cluster)
  int64_t max_batch;      // not eligible for more tickets than the workspace has: the largest batch that is, or 0
  int64_t head_blocks;    // windowed calls: row blocks per q head (no block spans two), 0: over all rows
  int cluster;            // 1: a unit's n_chunks CTAs form one thread-block cluster and merge
                          // their partial results over distributed shared memory (no workspace)
};
MmaPlan plan_paged_mma(const PagedArgs& a);
int launch_paged_mma(const PagedArgs& a, const MmaPlan& plan, void* workspace, cudaStream_t s);
int launch_paged_mma_window(const PagedArgs& a, const MmaPlan& plan, void* workspace, cudaStream_t s);

// tcgen05 / TMEM causal prefill (dense or paged) for 16-bit Q/K/V, D == 128.
// tcgen05/TMEM kernel (flash_sm100.cu): prefill (>= 64 query rows per head) and grouped
// few-token calls (a kv head's g*L query rows as one tile, split-K over keys when paged).
struct Sm100Plan {
  bool eligible;
  int grouped;
  int64_t M_rows, n_outer, n_row_tiles, n_units, rows_real, ct, n_chunks;
  size_t ws_bytes;
  int cluster;         // the chunks of a unit merge inside a thread-block cluster
  int64_t tiles_full;  // 64-key tiles of the longest context without a window
};
// sizing_only: plan from shapes alone (q dtype, pointers and scale unknown), for
// nvm_paged_attention_workspace_size.
Sm100Plan plan_sm100(const PagedArgs& a, bool sizing_only);
int launch_sm100(const PagedArgs& a, const Sm100Plan& plan, void* ws, cudaStream_t s);

// tcgen05 kernel with two 128-row query tiles per CTA (flash_2q.cu): prefill with at least
// 256 query rows per head, 16-bit, D == 128; no workspace.
bool flash2q_eligible(const PagedArgs& a);
int launch_flash2q(const PagedArgs& a, cudaStream_t s);

int launch_kv_write(const void* k, const void* v, int in_dtype, int64_t stride_t, int64_t stride_h,
                    void* k_pages, void* v_pages, int kv_dtype, void* k_scales, void* v_scales,
                    int scale_dtype, const int64_t* slot_mapping, int64_t T, int64_t Hkv, int64_t D,
                    int64_t P, int64_t page_size, cudaStream_t s);

// 4-bit cache (u4.cuh): scatter-write, reading slots back (any page type), attention.
int launch_u4_write(const void* k, const void* v, int in_dtype, int64_t stride_t, int64_t stride_h, void* k_pages, void* v_pages,
                    void* k_scales, void* v_scales, int scale_dtype, const int64_t* slots, int64_t T, int64_t Hkv, int64_t D,
                    int64_t P, int64_t page_size, cudaStream_t s);
int launch_read_slots(const void* k_pages, const void* v_pages, int kv_dtype, const void* k_scales, const void* v_scales,
                      int scale_dtype, const int64_t* slots, void* k, void* v, int out_dtype, int64_t T, int64_t Hkv, int64_t D,
                      int64_t P, int64_t page_size, cudaStream_t s);
struct U4AppendArgs {
  const void* q;
  const void* k;
  const void* v;
  int dtype;
  int64_t q_stride_t, kv_stride_t;
  const void* wq;
  const void* wk;
  float eps;
  const float* cos_table;
  const float* sin_table;
  int64_t table_rows;
  bool traditional;
  const int32_t* positions;
  void* q_out;
  int64_t q_out_L;
  void* k_pages;
  void* v_pages;
  void* k_scales;
  void* v_scales;
  const int64_t* slots;
  int64_t T, Hq, Hkv, D, P, page_size;
};
int launch_u4_append(const U4AppendArgs& a, cudaStream_t s);
// Many query rows: pages unpacked into the workspace for the tcgen05 kernel (u4_prompt.cu), from so many a
// kv head.  Row blocks / unpacked, us: 32 requests of 4850 keys, 4 heads, 128 rows 246 / 320, 192 362 / 346, 256
// 473 / 373; 8 of 4000, 8 heads, 192 rows 164 / 225, 256 213 / 236, 320 262 / 225; 2 of 2000, 256 rows 45 / 57, 384
// 61 / 77: between what many requests and few would have.
constexpr int64_t kU4PromptRows = 256;
struct U4PromptPlan {
  bool eligible;
  int64_t batch;  // requests taken at a time
  size_t ws_bytes, attention_bytes;
};
U4PromptPlan plan_u4_prompt(const PagedArgs& a);
int launch_u4_prompt(const PagedArgs& a, const U4PromptPlan& plan, void* ws, cudaStream_t s);
struct U4Plan {
  int tiles;                   // of 8 query rows a unit
  int64_t row_blocks, blocks;  // row blocks of one (request, kv head), thread blocks
  size_t ws_bytes;
};
U4Plan plan_paged_u4(const PagedArgs& a);
// The query rows that a call over unpacked pages could not hold: those that see a key from `first` on (of each
// (request, kv head): 2^31 - 1 less the key, 0 for none) and those marked in `rows`; a request
// without any has a zero in `some`.
struct U4Some {
  const uint32_t* first;
  const uint8_t* rows;
  const int* some;
};
int launch_paged_u4(const PagedArgs& a, const U4Plan& plan, void* ws, cudaStream_t s, const U4Some* some = nullptr);

int launch_paged_append(int32_t* block_table, int32_t* context_lens, const int32_t* new_tokens,
                        int32_t* free_stack, int32_t* free_top, int32_t* num_pages,
                        int32_t* page_refcount, int64_t* slot_mapping, int64_t slot_capacity, int32_t* status, int64_t B,
                        int64_t max_pages, int64_t page_size, int64_t capacity, cudaStream_t s);
int launch_paged_rewind(int32_t* block_table, int32_t* context_lens, const int32_t* rewind, int32_t* free_stack,
                        int32_t* free_top, int32_t* page_refcount, int32_t* last_call, int32_t* status, int64_t B,
                        int64_t max_pages, int64_t page_size, int64_t capacity, cudaStream_t s);
int launch_paged_attach(int32_t* block_table, int32_t* context_lens, const int32_t* pages, const int32_t* count,
                        int32_t* page_refcount, int32_t* status, int64_t B, int64_t max_pages, int64_t page_size,
                        int64_t max_prefix, int64_t capacity, cudaStream_t s);

// cuTensorMapEncodeTiled through the runtime's driver entry point (no -lcuda).
int encode_tmap(CUtensorMap* map, CUtensorMapDataType dt, int rank, const void* base,
                const uint64_t* dims, const uint64_t* strides_bytes, const uint32_t* box,
                CUtensorMapSwizzle swizzle);

}  // namespace nvm
