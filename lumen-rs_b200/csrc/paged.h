// The uncompressed paged cache (lc_paged_*) and beam selection (lc_beam_*):
// kernel argument blocks and launchers shared by paged.cpp and the kernels.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "common.h"
#include "status.h"

namespace lc {

// Raises a kernel's dynamic shared memory limit once per device.
struct SmemOptIn {
  std::atomic<uint64_t> done{0};
  template <typename K>
  void operator()(K kernel, size_t bytes, int device) {
    const uint64_t bit = 1ull << (device & 63);
    if (done.load(std::memory_order_relaxed) & bit) return;
    LC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    done.fetch_or(bit);
  }
};

// The caller's pool and one call's tables. Row (page p, head h, slot t) of
// layer l starts at element l * layer + p * page + h * head + t * token of k
// and of v.
struct PagedView {
  void* k;
  void* v;
  int64_t layer, page, head, token;  // strides in elements
  int32_t n_layers, hkv, d, page_tokens;
  int64_t n_pages;
  const int32_t* tables;  // [rows][width]
  const int32_t* lens;
  int32_t width;
  int32_t* status;  // mapped host words, by StatusBit
};

// Rows and strides of whole 16-byte units.
inline bool vector_rows(const PagedView& c, int esize) {
  const int64_t e = 16 / esize;
  return c.d % e == 0 && c.layer % e == 0 && c.page % e == 0 && c.head % e == 0 && c.token % e == 0 &&
         (reinterpret_cast<uintptr_t>(c.k) & 15) == 0 && (reinterpret_cast<uintptr_t>(c.v) & 15) == 0;
}

// TMA descriptors of the two pools; box: slots of a load, 0 where there are none.
struct PagedMaps {
  CUtensorMap k, v;
  int32_t box;
};

struct PagedAttnArgs {
  PagedView c;
  const void* q;
  void* out;
  int32_t q_dtype, out_dtype;
  int32_t n_seqs, group;  // query heads per kv head
  int32_t layer, window;
  float scale_log2;  // scale * log2(e)
  int32_t min_tiles;
  int32_t box;       // slots of a TMA box
  float* part;       // split partials: [2 * grid] slots of [heads][d + 2]
  int32_t* counters; // one per (sequence, kv head, head group); zero between calls
  float* scores;     // [n_seqs][hkv][score_tokens][group] (log2 domain), or null
  float* stats;      // [n_seqs][hkv * group][2]: the row's max and 1 / sum
  int64_t score_tokens;
};

struct PagedWeightArgs {
  const float* scores;
  const float* stats;
  const float* acc_in;
  float* acc_out;
  const int32_t* lens;
  int64_t score_tokens, acc_stride;
  int32_t n_seqs, hkv, group, window, cap, chunks;
  float decay;
};

struct PagedAppendArgs {
  PagedView c;
  const void* keys;  // [n_seqs][hkv][n_tokens][d]
  const void* values;
  int32_t dtype, pool_dtype, layer, n_seqs;
  int64_t n_tokens;
  int32_t* pos;           // [n_seqs][hkv][pos_stride] or null
  const int32_t* pos0;    // [n_seqs]
  int64_t pos_stride;
};

struct PagedEvictArgs {
  PagedView c;
  int32_t layer, n_seqs, esize;
  int32_t budget, n_sink, n_recent;
  int64_t stride;  // tokens per row of acc and pos
  const float* acc_in;
  const int32_t* pos_in;
  float* acc_out;
  int32_t* pos_out;
  int32_t* list;   // workspace: per row [4][list_cap]: holes, movers, the movers' acc and pos
  int64_t list_cap;
  int32_t* pairs;  // workspace: [rows], the lists' lengths
  int32_t fused;
  uint32_t* keys;  // workspace: [rows][stride], used where a row's keys do not fit shared memory
};

struct PagedReorderArgs {
  PagedView c;
  int32_t n_groups, n_beams, esize;
  const int32_t* parents;
  int32_t* tables_out;
};

struct BeamArgs {
  const void* logits;
  int32_t dtype;
  int64_t row_stride;
  int32_t n_groups, n_beams, n_out, vocab, slices, slice, per;
  const float* scores;
  const uint8_t* finished;  // may be null
  int32_t eos, pad;
  int32_t* status;  // mapped host words, by StatusBit
  float* scores_out;
  int32_t* parents;
  int32_t* tokens;
  uint8_t* finished_out;
  // workspace, by the parts of a row (at most one a slice)
  float* slice_stats;   // [rows][parts][2]: max, sum exp(x - max)
  float* slice_next;    // [rows][parts][2]: the largest logit that is not listed (-inf: none), the least listed
  uint64_t* slice_key;  // [rows][parts][n_out]: (logit, token), best first, 0 for none
  int32_t* counters;    // [n_groups], zero between calls
};

constexpr int kPagedMaxSeqs = 2048;
constexpr int kPagedMaxBlocks = 320;  // of an attention launch
constexpr int kPagedMaxDim = 256;
constexpr int kBeamMaxBeams = 64;
constexpr int kBeamMaxOut = 64;
constexpr int kBeamMaxMerge = 4096;  // candidates of one merge

// Every kernel here is launched with programmatic serialization: its blocks are
// in place when the kernel before it ends, they wait for that one before they
// read or write anything, and let the next kernel's blocks in at once. Calls
// in a row take some 2 us less each: 16 sequences in a window of 1024 went
// from 30.8 to 29.0 us (29.6 since tiles are added by rounding), a batch's
// reorder from 19.4 to 17.7.
void launch_paged_append(const PagedAppendArgs& a, int32_t sms, cudaStream_t s);
// pool_dtype: LC_F32 / LC_BF16 / LC_F16.
void launch_paged_attn(PagedAttnArgs& a, const PagedMaps& maps, int32_t pool_dtype, int32_t device, int32_t sms,
                       cudaStream_t s);
PagedMaps make_paged_maps(const PagedView& c, int32_t dtype);
int64_t paged_part_floats(int32_t sms);
void launch_paged_weights(PagedWeightArgs a, cudaStream_t s);
int paged_evict_cluster(int64_t cap, int rows, int sms);
bool paged_evict_keys_in_smem(int64_t cap, int cluster);
void launch_paged_evict(const PagedEvictArgs& a, int32_t device, int32_t sms, cudaStream_t s);
void launch_paged_reorder(const PagedReorderArgs& a, int32_t sms, cudaStream_t s);
int beam_slice(int32_t dtype);
void launch_beam(BeamArgs a, int32_t device, int32_t sms, cudaStream_t s);

}  // namespace lc
