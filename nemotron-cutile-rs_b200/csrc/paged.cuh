// paged.cuh — the paged KV cache as the kernels see it: pool geometry, the
// ragged batch, and the checks every kernel makes of device arrays.
#pragma once

#include <atomic>

#include "nk_common.cuh"

namespace nk {

struct PagePool {
  int layers, pages, heads, ps, ps_log2;
  const int32_t *table;
  int64_t table_ld;
  int table_rows;
};

struct PageBatch {
  const int32_t *start, *kv_len, *rows;
  int64_t tokens;
  int seqs, max_new, max_kv;
};

// Host checks of nk_kv_pages / nk_kv_batch shared by the entry points (no
// device work), and their kernel forms.
nk_status check_pages(const nk_kv_pages *kv, int64_t layer);
nk_status check_batch(const nk_kv_pages *kv, const nk_kv_batch *b);
inline PagePool page_pool(const nk_kv_pages &kv) {
  PagePool p{};
  p.layers = (int)kv.layers;
  p.pages = (int)kv.pages;
  p.heads = (int)kv.kv_heads;
  p.ps = (int)kv.page_size;
  p.ps_log2 = __builtin_ctz((unsigned)kv.page_size);
  p.table = kv.table;
  p.table_ld = kv.table_ld;
  p.table_rows = (int)kv.table_rows;
  return p;
}
inline PageBatch page_batch(const nk_kv_batch &b) {
  PageBatch p{};
  p.start = b.start;
  p.kv_len = b.kv_len;
  p.rows = b.rows;
  p.tokens = b.tokens;
  p.seqs = (int)b.seqs;
  p.max_new = (int)b.max_new;
  p.max_kv = (int)b.max_kv;
  return p;
}

// The kernel's dynamic shared memory, set once per device (`prepared`: a bit each).
inline nk_status allow_smem(const void *kernel, int bytes, std::atomic<uint64_t> &prepared) {
  int dev = 0;
  NK_CUDA_TRY(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (prepared.load(std::memory_order_acquire) & bit) return NK_OK;
  NK_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  prepared.fetch_or(bit, std::memory_order_release);
  return NK_OK;
}

// Kernels of this cache often follow one another in a stream (append, scores,
// lists, attention, merge) and are short: each lets the next one be launched
// while it runs (let_next_launch).  A kernel that is launched so (launch_early)
// waits on the device for the end of the one before it (wait_for_previous)
// ahead of its first access to global memory, on every path, and reads nothing
// through the read-only cache.  The wait is for the whole grid and its writes,
// which waited for the grid before it, so the stream's order holds.  Behind any
// other kernel the launch is an ordinary one.
__device__ __forceinline__ void let_next_launch() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void wait_for_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
// cluster > 1: blocks of a cluster.
template <typename... Params, typename... Args>
nk_status launch_early(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, int cluster,
                       cudaStream_t s, const Args &...args) {
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  NK_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, args...));
  return NK_OK;
}

// First error of a kernel stays in the device word.
__device__ __forceinline__ void report(int *err, int code) { atomicCAS(err, 0, code); }

struct SeqView {
  int first, count;      // new tokens: rows first .. first+count-1 of the token buffers
  int len;               // cached tokens, the new ones included
  const int32_t *table;  // the sequence's pages
};

// Sequence s of the batch; false (reported once per calling block by
// `report_it`) when the arrays contradict one another or their bounds.
__device__ __forceinline__ bool load_seq(const PagePool &p, const PageBatch &b, int s, SeqView &v,
                                         int *err, bool report_it) {
  v.first = b.start[s];
  const int end = b.start[s + 1];
  v.count = end - v.first;
  v.len = b.kv_len[s];
  const int row = b.rows ? b.rows[s] : s;
  const bool good = v.first >= 0 && end >= v.first && end <= b.tokens && v.count <= b.max_new &&
                    v.len >= v.count && v.len <= b.max_kv &&
                    (int64_t)v.len <= p.table_ld * (int64_t)p.ps && row >= 0 &&
                    row < p.table_rows;
  if (!good) {
    if (report_it) report(err, NK_INVALID_PARAMS);
    return false;
  }
  v.table = p.table + (int64_t)row * p.table_ld;
  return true;
}

__device__ __forceinline__ bool page_ok(const PagePool &p, int page) {
  return (unsigned)page < (unsigned)p.pages;
}

}  // namespace nk
