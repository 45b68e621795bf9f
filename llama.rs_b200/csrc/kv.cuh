// kv.cuh -- the paged KV cache as the operators of kv_ops.cu and
// tree_attention.cu see it (layout: lrs_kv_cache in include/llamars.h).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/llamars.h"
#include "decode.cuh"

namespace lrs {

static_assert(kPageSize == LRS_KV_PAGE, "one page size");

// What an error word (lrs_backend::d_err) holds after a kernel skipped an entry
// that names a slot, position, page or node out of range.  Below
// LRS_ERR_DEVICE_TIMEOUT, which it must not replace: kernels set it by maximum.
constexpr int kErrCacheIndex = 2;
static_assert(kErrCacheIndex < LRS_ERR_DEVICE_TIMEOUT, "the graver error stays");

// Largest magnitude of a Q8_0 cache: 512 * 127, so that d * code is a finite f16.
constexpr float kQ8Limit = 65024.0f;

__host__ __device__ constexpr size_t kv_tile_bytes(uint32_t dtype, int hd) {
  return dtype == LRS_KV_Q8_0 ? (size_t)kPageSize * (hd / 32) * 34
                              : (size_t)kPageSize * hd * (dtype == LRS_KV_BF16 ? 2 : 4);
}
// Byte offsets inside a Q8_0 tile (row r of the page, column c of the head).
__host__ __device__ constexpr int q8_k_code(int r, int c) { return (c / 16 * kPageSize + r) * 16 + c % 16; }
__host__ __device__ constexpr int q8_k_scale(int hd, int r, int b) {
  return kPageSize * hd + (r * (hd / 32) + b) * 2;
}
__host__ __device__ constexpr int q8_v_code(int hd, int r, int c) { return (r / 4 * hd + c) * 4 + r % 4; }
__host__ __device__ constexpr int q8_v_scale(int hd, int r, int b) {
  return kPageSize * hd + (b * kPageSize + r) * 2;
}

struct KvView {
  uint8_t* k;
  uint8_t* v;
  const int* pages;
  int n_pages, n_seqs, max_pages, heads;
  int* err;
};

// Physical page of position `pos` of slot `seq`, or -1 (with the error word
// set) if any of the three is out of range.
__device__ __forceinline__ int kv_page(const KvView& c, int seq, int pos) {
  int page = -1;
  if (seq >= 0 && seq < c.n_seqs && pos >= 0 && pos / kPageSize < c.max_pages)
    page = c.pages[(size_t)seq * c.max_pages + pos / kPageSize];
  if (page < 0 || page >= c.n_pages) {
    atomicMax(c.err, kErrCacheIndex);
    return -1;
  }
  return page;
}

// n rows of K and V, `ld` floats apart, and their slots and positions.
struct KvStoreArgs {
  KvView c;
  const int* seq;
  const int* pos;
  long long n;
  const float* k;
  const float* v;
  long long ld;
};
cudaError_t launch_kv_store(const KvStoreArgs& a, uint32_t dtype, int hd, int sms, cudaStream_t st);

struct KvLoadArgs {
  KvView c;
  const int* seq;
  const int* pos;
  long long n;
  float* k;
  float* v;
  long long ld;
};
cudaError_t launch_kv_load(const KvLoadArgs& a, uint32_t dtype, int hd, int sms, cudaStream_t st);

// lrs_kv_accept, which leaves a skipped tree's error in one of the backend's words.
int32_t kv_accept(lrs_backend* be, const lrs_kv_cache* caches, size_t n_caches, const int32_t* d_seq,
                  const int32_t* d_ctx, const int32_t* d_start, const int32_t* d_nodes, size_t n_trees,
                  size_t n_nodes, int err_word, void* stream);

struct TreeArgs {
  KvView c;
  const int* seq;
  const int* ctx;
  const int* start;
  const unsigned long long* mask;
  int n_trees, n_nodes, max_nodes, max_len;
  const float* q;
  float* out;
  long long q_ld, out_ld;
  int group;      // query heads per KV head
  float scale;
  void* workspace;
};
size_t tree_attention_workspace_bytes(const TreeArgs& a, int hd, int sms);
cudaError_t launch_tree_attention(const TreeArgs& a, uint32_t dtype, int hd, int sms,
                                  cudaStream_t st);

}  // namespace lrs
