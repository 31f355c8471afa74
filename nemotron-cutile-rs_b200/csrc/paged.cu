// paged.cu — the pages of a KV cache: append with key bounds, whole-page
// copies, compaction, and writes of host-planned tables.
//
// All of them move bytes: the floor of each is (bytes read + bytes written) /
// HBM bandwidth, and a decode step's calls are bounded by their launch.  A
// thread moves 16 bytes (8 channels of a token); D/8 neighbouring threads
// hold one token of one head, so every access is a whole 128- or 256-byte row.
#include <algorithm>
#include <vector>

#include "paged.cuh"

namespace nk {

// Channelwise min / max of 8 bf16 channels.  The comparison returns the
// operand that is a number when the other is NaN, so NaN keys leave the
// bounds of their page alone.  Exact: bounds are values of the keys, and do
// not depend on the order of the tokens.
struct Bounds8 {
  __nv_bfloat162 lo[4], hi[4];
  __device__ __forceinline__ void set(const uint4 &x) {
    const __nv_bfloat162 *p = reinterpret_cast<const __nv_bfloat162 *>(&x);
#pragma unroll
    for (int i = 0; i < 4; ++i) lo[i] = hi[i] = p[i];
  }
  __device__ __forceinline__ void add(const uint4 &x) {
    const __nv_bfloat162 *p = reinterpret_cast<const __nv_bfloat162 *>(&x);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo[i] = __hmin2(lo[i], p[i]);
      hi[i] = __hmax2(hi[i], p[i]);
    }
  }
  __device__ __forceinline__ void join(const uint4 &l, const uint4 &h) {
    const __nv_bfloat162 *pl = reinterpret_cast<const __nv_bfloat162 *>(&l);
    const __nv_bfloat162 *ph = reinterpret_cast<const __nv_bfloat162 *>(&h);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo[i] = __hmin2(lo[i], pl[i]);
      hi[i] = __hmax2(hi[i], ph[i]);
    }
  }
  __device__ __forceinline__ uint4 low() const { return *reinterpret_cast<const uint4 *>(lo); }
  __device__ __forceinline__ uint4 high() const { return *reinterpret_cast<const uint4 *>(hi); }
};

// Joins the bounds of the block's token lanes and has lane 0's threads write
// them.  Every thread of the block calls it; `any` = this thread holds a token.
template <int D, int THREADS>
__device__ __forceinline__ void write_bounds(Bounds8 &b, bool any, uint4 *kmin, uint4 *kmax,
                                             uint4 *sh_lo, uint4 *sh_hi, int *sh_any) {
  constexpr int C = D / 8, LANES = THREADS / C;
  const int c = threadIdx.x % C, lane = threadIdx.x / C;
  sh_any[threadIdx.x] = any;
  if (any) {
    sh_lo[threadIdx.x] = b.low();
    sh_hi[threadIdx.x] = b.high();
  }
  __syncthreads();
  if (lane == 0) {
    for (int i = 1; i < LANES; ++i) {
      const int t = i * C + c;
      if (!sh_any[t]) continue;
      if (any) {
        b.join(sh_lo[t], sh_hi[t]);
      } else {
        b.set(sh_lo[t]);
        b.join(sh_lo[t], sh_hi[t]);
        any = true;
      }
    }
    if (any) {
      kmin[c] = b.low();
      kmax[c] = b.high();
    }
  }
}

// Block = (touched page x, head y, sequence z): the new tokens of one page, so
// that the page's bounds have one writer and need no atomics, and a key is read
// once for the copy and the bounds.  For a prefill bound by HBM and by the lookups
// (start, length, row, table) that each block of 16 KB makes ahead of its first
// load (9000 tokens of 8 heads of 128, 74 MB: 16.8 us when the writes reach memory
// too, 10.7 us with all of it in L2; the heads of a page side by side in the grid:
// 18.4 and 10.7), by the launch for a decode step (64 tokens: 2.6 us in a chain of
// calls).
template <int D>
__global__ void __launch_bounds__(128)
    pages_append_kernel(PagePool pool, PageBatch batch, const uint16_t *__restrict__ k_new,
                        int64_t ld_k, const uint16_t *__restrict__ v_new, int64_t ld_v,
                        uint4 *__restrict__ k, uint4 *__restrict__ v, uint4 *__restrict__ k_min,
                        uint4 *__restrict__ k_max, int *err) {
  constexpr int C = D / 8, LANES = 128 / C;
  __shared__ uint4 sh_lo[128], sh_hi[128];
  __shared__ int sh_any[128];
  let_next_launch();
  SeqView s;
  if (!load_seq(pool, batch, blockIdx.z, s, err, threadIdx.x == 0)) return;
  const int p0 = s.len - s.count;  // position of the first new token
  const int j = (p0 >> pool.ps_log2) + (int)blockIdx.x;
  const int page0 = j << pool.ps_log2;
  if (s.count == 0 || page0 >= s.len) return;
  const int page = s.table[j];
  if (!page_ok(pool, page)) {
    if (threadIdx.x == 0) report(err, NK_PAGE_OUT_OF_RANGE);
    return;
  }
  const int h = blockIdx.y;
  const int a = p0 > page0 ? p0 : page0;
  const int e = s.len < page0 + pool.ps ? s.len : page0 + pool.ps;
  const int c = threadIdx.x % C, lane = threadIdx.x / C;
  const int64_t unit = (int64_t)page * pool.heads + h;  // (page, head)
  Bounds8 b;
  bool any = false;
#pragma unroll 4
  for (int t = a + lane; t < e; t += LANES) {
    const int64_t src = (int64_t)s.first + (t - p0);
    const uint4 kx = *reinterpret_cast<const uint4 *>(k_new + src * ld_k + h * D + c * 8);
    const uint4 vx = *reinterpret_cast<const uint4 *>(v_new + src * ld_v + h * D + c * 8);
    const int64_t dst = (unit * pool.ps + (t - page0)) * C + c;
    k[dst] = kx;
    v[dst] = vx;
    if (any) b.add(kx); else b.set(kx);
    any = true;
  }
  if (k_min) {
    uint4 *lo = k_min + unit * C, *hi = k_max + unit * C;
    if (lane == 0 && a > page0) {  // the page held earlier tokens: a lane 0 token exists too
      b.join(lo[c], hi[c]);
    }
    write_bounds<D, 128>(b, any, lo, hi, sh_lo, sh_hi, sh_any);
  }
}

// ------------------------------------------------------------------- copies
// Pairs of pages travel in the kernel's parameters: the host array is read
// before the call returns, nothing is staged, and a captured call keeps them.
template <int N>
struct PagePairs {
  int32_t src[N], dst[N];
};

// Block = (16 KB segment x of a page in one layer, pair y, layer z); the last
// segment carries the bounds.  256 threads with four 16-byte loads each in
// flight; 1531 pairs of pages in two layers, 426 MB read and written: 59 us, 7.2
// TB/s (above the rate of a plain copy, since some writes end in L2).
template <int N>
__global__ void __launch_bounds__(256)
    pages_copy_kernel(const __grid_constant__ PagePairs<N> pairs, int64_t pages, int page_v,
                      int bound_v, uint4 *__restrict__ k, uint4 *__restrict__ v,
                      uint4 *__restrict__ k_min, uint4 *__restrict__ k_max) {
  const int segs = (page_v + 1023) / 1024;
  const int64_t src = (int64_t)blockIdx.z * pages + pairs.src[blockIdx.y];
  const int64_t dst = (int64_t)blockIdx.z * pages + pairs.dst[blockIdx.y];
  int seg = blockIdx.x;
  if (seg < 2 * segs) {
    uint4 *base = seg < segs ? k : v;
    if (seg >= segs) seg -= segs;
    const uint4 *from = base + src * page_v + seg * 1024;
    uint4 *to = base + dst * page_v + seg * 1024;
    const int n = page_v - seg * 1024;  // 16-byte words left in the page
    uint4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (threadIdx.x + 256 * i < n) x[i] = from[threadIdx.x + 256 * i];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (threadIdx.x + 256 * i < n) to[threadIdx.x + 256 * i] = x[i];
  } else {
    for (int i = threadIdx.x; i < bound_v; i += 256) {
      k_min[dst * bound_v + i] = k_min[src * bound_v + i];
      k_max[dst * bound_v + i] = k_max[src * bound_v + i];
    }
  }
}

// -------------------------------------------------------------- host tables
template <int N>
struct TableWrites {
  int64_t offset[N];
  int32_t value[N];
};
template <int N>
struct TableRun {
  int32_t value[N];
};

template <int N>
__global__ void table_scatter_kernel(const __grid_constant__ TableWrites<N> w, int n,
                                     int32_t *__restrict__ dst) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) dst[w.offset[i]] = w.value[i];
}
template <int N>
__global__ void table_run_kernel(const __grid_constant__ TableRun<N> w, int n,
                                 int32_t *__restrict__ dst) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) dst[i] = w.value[i];
}

// ------------------------------------------------------------------ compaction
struct CompactArgs {
  const int32_t *rows, *kv_len, *base, *keep, *n_keep, *dst_table;
  int64_t keep_ld, dst_ld;
  int max_keep;
  int32_t *new_len;
};

struct CompactSeq {
  int len, base, n;
  const int32_t *keep, *src, *dst;
};

__device__ __forceinline__ bool load_compact(const PagePool &p, const CompactArgs &a, int s,
                                             CompactSeq &c, int *err, bool report_it) {
  const int row = a.rows ? a.rows[s] : s;
  c.len = a.kv_len[s];
  c.base = a.base[s];
  c.n = a.n_keep[s];
  const bool good =
      row >= 0 && row < p.table_rows && c.len >= 0 && c.base >= 0 && c.n >= 0 &&
      c.n <= a.max_keep && c.base <= c.len && c.n <= c.len - c.base &&
      (int64_t)c.len <= p.table_ld * (int64_t)p.ps &&
      (!a.dst_table || (int64_t)c.base + c.n <= a.dst_ld * (int64_t)p.ps);
  if (!good) {
    if (report_it) report(err, NK_INVALID_PARAMS);
    return false;
  }
  c.keep = a.keep + s * a.keep_ld;
  c.src = p.table + (int64_t)row * p.table_ld;
  c.dst = a.dst_table ? a.dst_table + s * a.dst_ld : c.src;
  return true;
}

// Position that kept token i comes from, or -1 (reported) for a refused entry.
__device__ __forceinline__ int kept_position(const CompactSeq &c, int i, int *err) {
  const int x = c.keep[i], before = i ? c.keep[i - 1] : -1;
  if (x <= before || x < 0 || x >= c.len - c.base) {
    report(err, NK_INVALID_PARAMS);
    return -1;
  }
  return c.base + x;
}

// Into other pages: block = (destination page x, head and layer y, sequence
// z).  Where each token comes from is looked up first, a thread a token (keep,
// then the page table: two latencies for the page, not two for every few
// tokens); the 128 threads then gather with all their loads in flight.  213 MB:
// 37.7 us, 5.6 TB/s (39 us cold with two lookups for every eight tokens).
template <int D>
__global__ void __launch_bounds__(128)
    pages_compact_kernel(PagePool pool, CompactArgs args, uint4 *__restrict__ k,
                         uint4 *__restrict__ v, uint4 *__restrict__ k_min,
                         uint4 *__restrict__ k_max, int *err) {
  constexpr int C = D / 8, LANES = 128 / C;
  __shared__ uint4 sh_lo[128], sh_hi[128];
  __shared__ int sh_any[128];
  __shared__ int64_t sh_src[128];  // 16-byte word of the token's first channels, -1: none
  CompactSeq s;
  if (!load_compact(pool, args, blockIdx.z, s, err, threadIdx.x == 0)) return;
  const int end = s.base + s.n;
  if (args.new_len && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0)
    args.new_len[blockIdx.z] = end;
  const int j = (s.base >> pool.ps_log2) + (int)blockIdx.x;
  if ((int64_t)j << pool.ps_log2 >= end) return;
  const int page0 = j << pool.ps_log2;
  const int page = s.dst[j];
  if (!page_ok(pool, page)) {
    if (threadIdx.x == 0) report(err, NK_PAGE_OUT_OF_RANGE);
    return;
  }
  const int h = blockIdx.y % pool.heads, layer = blockIdx.y / pool.heads;
  const int64_t lp = (int64_t)layer * pool.pages;
  const int c = threadIdx.x % C, lane = threadIdx.x / C;
  const int64_t unit = (lp + page) * pool.heads + h;
  const int n = end - page0 < pool.ps ? end - page0 : pool.ps;  // tokens of the page
  if ((int)threadIdx.x < n) {
    const int t = page0 + (int)threadIdx.x;
    int64_t src = -1;
    if (t < s.base) {
      src = -2;  // a token below base stays; it belongs to the page's bounds
    } else {
      const int from = kept_position(s, t - s.base, err);
      if (from >= 0) {
        const int fp = s.src[from >> pool.ps_log2];
        if (page_ok(pool, fp))
          src = (((lp + fp) * pool.heads + h) * pool.ps + (from & (pool.ps - 1))) * C;
        else
          report(err, NK_PAGE_OUT_OF_RANGE);
      }
    }
    sh_src[threadIdx.x] = src;
  }
  __syncthreads();
  Bounds8 b;
  bool any = false;
#pragma unroll 1
  for (int t0 = lane; t0 < n; t0 += 4 * LANES) {
    uint4 kx[4], vx[4];
    int64_t src[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int t = t0 + u * LANES;
      src[u] = t < n ? sh_src[t] : -1;
      if (src[u] >= 0) {
        kx[u] = k[src[u] + c];
        vx[u] = v[src[u] + c];
      } else if (src[u] == -2) {
        kx[u] = k[(unit * pool.ps + t) * C + c];
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (src[u] == -1) continue;
      const int64_t dst = (unit * pool.ps + t0 + u * LANES) * C + c;
      if (src[u] >= 0) {
        k[dst] = kx[u];
        v[dst] = vx[u];
      }
      if (any) b.add(kx[u]); else b.set(kx[u]);
      any = true;
    }
  }
  if (k_min) write_bounds<D, 128>(b, any, k_min + unit * C, k_max + unit * C, sh_lo, sh_hi, sh_any);
}

// In place: block = (head and layer x, sequence y).  Token i comes from a
// position at or behind its own (keep is ascending), so rounds of TOK tokens
// that are all read before any is written never read a slot that an earlier
// round has overwritten.  One block keeps that order without flags between
// blocks; the few kept tokens of a verified draft are a round or two, bound by
// two chains of dependent loads, one behind the other (keep, table, key; then for
// the bounds table, keys and the join of the lanes): 9.5 us cold, 6.4 us in a
// chain of calls for 64 sequences of 6 layers and 2 heads.
template <int D>
__global__ void __launch_bounds__(256)
    pages_compact_inplace_kernel(PagePool pool, CompactArgs args, uint4 *k, uint4 *v,
                                 uint4 *__restrict__ k_min, uint4 *__restrict__ k_max, int *err) {
  constexpr int C = D / 8, LANES = 256 / C, TOK = 2 * LANES;
  __shared__ uint4 sh_lo[256], sh_hi[256];
  __shared__ int sh_any[256];
  CompactSeq s;
  if (!load_compact(pool, args, blockIdx.y, s, err, threadIdx.x == 0)) return;
  const int end = s.base + s.n;
  if (args.new_len && blockIdx.x == 0 && threadIdx.x == 0) args.new_len[blockIdx.y] = end;
  const int h = blockIdx.x % pool.heads, layer = blockIdx.x / pool.heads;
  const int64_t lp = (int64_t)layer * pool.pages;
  const int c = threadIdx.x % C, lane = threadIdx.x / C;
  auto slot = [&](int pos) -> int64_t {  // 16-byte word of position pos, or -1
    const int page = s.src[pos >> pool.ps_log2];
    if (!page_ok(pool, page)) {
      report(err, NK_PAGE_OUT_OF_RANGE);
      return -1;
    }
    return (((lp + page) * pool.heads + h) * pool.ps + (pos & (pool.ps - 1))) * C + c;
  };
  for (int i0 = 0; i0 < s.n; i0 += TOK) {
    uint4 kx[2], vx[2];
    int64_t to[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = i0 + u * LANES + lane;
      to[u] = -1;
      if (i < s.n) {
        const int from = kept_position(s, i, err);
        if (from >= 0 && from != s.base + i) {
          const int64_t src = slot(from);
          if (src >= 0) {
            kx[u] = k[src];
            vx[u] = v[src];
            to[u] = slot(s.base + i);
          }
        }
      }
    }
    __syncthreads();  // the round is read
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (to[u] >= 0) {
        k[to[u]] = kx[u];
        v[to[u]] = vx[u];
      }
    __syncthreads();  // and written, before the next reads
  }
  if (!k_min) return;
  for (int j = s.base >> pool.ps_log2; (int64_t)j << pool.ps_log2 < end; ++j) {
    const int page0 = j << pool.ps_log2;
    const int page = s.src[j];
    if (!page_ok(pool, page)) continue;  // uniform over the block, reported above when written
    const int e = end - page0 < pool.ps ? end : page0 + pool.ps;
    const int64_t unit = (lp + page) * pool.heads + h;
    Bounds8 b;
    bool any = false;
    for (int t = page0 + lane; t < e; t += LANES) {
      const uint4 kx = k[(unit * pool.ps + (t - page0)) * C + c];
      if (any) b.add(kx); else b.set(kx);
      any = true;
    }
    write_bounds<D, 256>(b, any, k_min + unit * C, k_max + unit * C, sh_lo, sh_hi, sh_any);
    __syncthreads();
  }
}

// ------------------------------------------------------------------ host checks
nk_status check_pages(const nk_kv_pages *kv, int64_t layer) {
  if (!kv) return fail(NK_INVALID_PARAMS, "kv");
  if (kv->layers <= 0 || kv->pages <= 0 || kv->kv_heads <= 0 || kv->page_size <= 0 ||
      kv->head_dim <= 0)
    return fail(NK_INVALID_SHAPE, "layers, pages, kv_heads, page_size, head_dim > 0");
  if (kv->head_dim != 64 && kv->head_dim != 128)
    return fail(NK_UNSUPPORTED, "head_dim must be 64 or 128");
  if (kv->page_size != 16 && kv->page_size != 32 && kv->page_size != 64 && kv->page_size != 128)
    return fail(NK_UNSUPPORTED, "page_size must be 16, 32, 64 or 128");
  if (kv->kv_heads > 65535 || kv->layers > 65535 || kv->layers * kv->kv_heads > 65535)
    return fail(NK_UNSUPPORTED, "layers * kv_heads must be <= 65535");
  // Token rows are 32-bit coordinates of the tile loads; elements and bytes
  // are 64-bit everywhere.
  if (kv->pages >= (1ll << 31) ||
      kv->pages * kv->layers * kv->kv_heads >= (1ll << 31) / kv->page_size)
    return fail(NK_UNSUPPORTED, "layers * pages * kv_heads * page_size must be < 2^31");
  if (layer < 0 || layer >= kv->layers) return fail(NK_INVALID_PARAMS, "layer out of range");
  if (!kv->k || !kv->v) return fail(NK_INVALID_PARAMS, "k and v are required");
  if (!kv->k_min != !kv->k_max) return fail(NK_INVALID_PARAMS, "k_min and k_max go together");
  if (((uintptr_t)kv->k | (uintptr_t)kv->v | (uintptr_t)kv->k_min | (uintptr_t)kv->k_max) & 15)
    return fail(NK_INVALID_PARAMS, "page pools must be 16-byte aligned");
  return NK_OK;
}

static nk_status check_table(const nk_kv_pages *kv) {
  if (!kv->table || kv->table_rows <= 0 || kv->table_ld <= 0)
    return fail(NK_INVALID_PARAMS, "a page table with rows is required");
  if (kv->table_rows >= (1ll << 31) || kv->table_ld >= (1ll << 31))
    return fail(NK_UNSUPPORTED, "table_rows and table_ld must be < 2^31");
  return NK_OK;
}

nk_status check_batch(const nk_kv_pages *kv, const nk_kv_batch *b) {
  nk_status st = check_table(kv);
  if (st != NK_OK) return st;
  if (!b) return fail(NK_INVALID_PARAMS, "batch");
  if (b->seqs < 0 || b->tokens < 0 || b->max_new < 0 || b->max_kv < 0)
    return fail(NK_INVALID_SHAPE, "seqs, tokens, max_new, max_kv >= 0");
  if (b->seqs > 65535) return fail(NK_UNSUPPORTED, "at most 65535 sequences a call");
  if (b->tokens >= (1ll << 31) || b->max_kv + b->max_new >= (1ll << 31) - 512)
    return fail(NK_UNSUPPORTED, "tokens and max_kv + max_new must be < 2^31 - 512");
  if (b->max_new > b->tokens || b->max_new > b->max_kv)
    return fail(NK_INVALID_PARAMS, "max_new must not exceed tokens or max_kv");
  if (b->seqs > 0 && (!b->start || !b->kv_len))
    return fail(NK_INVALID_PARAMS, "start and kv_len are required");
  if (!b->rows && b->seqs > kv->table_rows)
    return fail(NK_INVALID_PARAMS, "more sequences than table rows");
  return NK_OK;
}

// Whether two arrays of int32 share memory.
static bool overlap(const int32_t *a, int64_t na, const int32_t *b, int64_t nb) {
  return a && b && na > 0 && nb > 0 && (uintptr_t)a < (uintptr_t)(b + nb) &&
         (uintptr_t)b < (uintptr_t)(a + na);
}

static nk_status fail_page(int64_t page, int64_t pages, int64_t index) {
  nk_status st = fail(NK_PAGE_OUT_OF_RANGE, "page id out of range");
  tls_error().actual = (uint64_t)page;
  tls_error().expected = (uint64_t)pages;
  tls_error().index = (uint64_t)index;
  return st;
}

template <int N>
static nk_status launch_copy(const nk_kv_pages &kv, const int32_t *src, const int32_t *dst,
                             int count, cudaStream_t s) {
  PagePairs<N> pairs;
  memcpy(pairs.src, src, sizeof(int32_t) * count);
  memcpy(pairs.dst, dst, sizeof(int32_t) * count);
  const int page_v = (int)(kv.kv_heads * kv.page_size * kv.head_dim / 8);
  const int bound_v = (int)(kv.kv_heads * kv.head_dim / 8);
  const int segs = (page_v + 1023) / 1024;
  const dim3 grid(2 * segs + (kv.k_min ? 1 : 0), (unsigned)count, (unsigned)kv.layers);
  pages_copy_kernel<N><<<grid, 256, 0, s>>>(
      pairs, kv.pages, page_v, bound_v, reinterpret_cast<uint4 *>(kv.k),
      reinterpret_cast<uint4 *>(kv.v), reinterpret_cast<uint4 *>(kv.k_min),
      reinterpret_cast<uint4 *>(kv.k_max));
  return check_launch("pages_copy_kernel");
}

template <int N>
static nk_status launch_table(int32_t *dst, const int64_t *offset, const int32_t *value, int count,
                              cudaStream_t s) {
  if (offset) {
    TableWrites<N> w;
    memcpy(w.offset, offset, sizeof(int64_t) * count);
    memcpy(w.value, value, sizeof(int32_t) * count);
    table_scatter_kernel<N><<<1, 256, 0, s>>>(w, count, dst);
  } else {
    TableRun<N> w;
    memcpy(w.value, value, sizeof(int32_t) * count);
    table_run_kernel<N><<<1, 256, 0, s>>>(w, count, dst);
  }
  return check_launch("table write");
}

}  // namespace nk

using namespace nk;

extern "C" {

nk_status nk_kv_pages_append(const nk_kv_pages *kv, int64_t layer, const nk_kv_batch *batch,
                             const uint16_t *k_new, int64_t ld_k, const uint16_t *v_new,
                             int64_t ld_v, void *stream) {
  nk_status st = check_pages(kv, layer);
  if (st == NK_OK) st = check_batch(kv, batch);
  if (st != NK_OK) return st;
  const int64_t width = kv->kv_heads * kv->head_dim;
  if (ld_k < width || ld_v < width || ld_k % 8 || ld_v % 8)
    return fail(NK_INVALID_PARAMS, "ld_k, ld_v must be multiples of 8 and >= kv_heads * head_dim");
  if (batch->seqs == 0 || batch->tokens == 0 || batch->max_new == 0) return ok();
  if (!k_new || !v_new) return fail(NK_INVALID_PARAMS, "k_new and v_new are required");
  if (((uintptr_t)k_new | (uintptr_t)v_new) & 15)
    return fail(NK_INVALID_PARAMS, "k_new and v_new must be 16-byte aligned");
  int *err = device_error_ptr();
  if (!err) return fail(NK_DEVICE_ERROR, "cannot resolve device error word");
  const PagePool pool = page_pool(*kv);
  const PageBatch b = page_batch(*batch);
  // A run of max_new tokens touches at most this many pages, wherever it starts.
  const int64_t touched = (batch->max_new + kv->page_size - 2) / kv->page_size + 1;
  const dim3 grid((unsigned)touched, (unsigned)kv->kv_heads, (unsigned)batch->seqs);
  const int64_t words = kv->pages * kv->kv_heads * kv->head_dim / 8;  // bounds of one layer
  uint4 *k = reinterpret_cast<uint4 *>(kv->k) + layer * words * kv->page_size;
  uint4 *v = reinterpret_cast<uint4 *>(kv->v) + layer * words * kv->page_size;
  uint4 *lo = kv->k_min ? reinterpret_cast<uint4 *>(kv->k_min) + layer * words : nullptr;
  uint4 *hi = kv->k_max ? reinterpret_cast<uint4 *>(kv->k_max) + layer * words : nullptr;
  cudaStream_t s = as_stream(stream);
  if (kv->head_dim == 128)
    pages_append_kernel<128><<<grid, 128, 0, s>>>(pool, b, k_new, ld_k, v_new, ld_v, k, v, lo, hi,
                                                  err);
  else
    pages_append_kernel<64><<<grid, 128, 0, s>>>(pool, b, k_new, ld_k, v_new, ld_v, k, v, lo, hi,
                                                 err);
  return check_launch("pages_append_kernel");
}

nk_status nk_kv_pages_copy(const nk_kv_pages *kv, const int32_t *src_host,
                           const int32_t *dst_host, int64_t count, void *stream) {
  nk_status st = check_pages(kv, 0);
  if (st != NK_OK) return st;
  if (count < 0) return fail(NK_INVALID_SHAPE, "count >= 0");
  if (count == 0) return ok();
  if (!src_host || !dst_host) return fail(NK_INVALID_PARAMS, "src_host and dst_host are required");
  // Every page is written once and no page is both read and written, so the
  // blocks of one launch need no order.
  for (int64_t i = 0; i < count; ++i) {
    if (src_host[i] < 0 || src_host[i] >= kv->pages) return fail_page(src_host[i], kv->pages, i);
    if (dst_host[i] < 0 || dst_host[i] >= kv->pages) return fail_page(dst_host[i], kv->pages, i);
  }
  int64_t bad = -1;
  try {
    if (kv->pages / 64 <= 1024 + 16 * count) {  // a bit a page
      static thread_local std::vector<uint64_t> written;
      written.assign((size_t)kv->pages / 64 + 1, 0);
      for (int64_t i = 0; i < count && bad < 0; ++i) {
        uint64_t &w = written[dst_host[i] >> 6];
        const uint64_t bit = 1ull << (dst_host[i] & 63);
        if (w & bit) bad = i;
        w |= bit;
      }
      for (int64_t i = 0; i < count && bad < 0; ++i)
        if (written[src_host[i] >> 6] >> (src_host[i] & 63) & 1) bad = i;
    } else {  // few pairs of a huge pool
      std::vector<int32_t> to(dst_host, dst_host + count);
      std::sort(to.begin(), to.end());
      if (std::adjacent_find(to.begin(), to.end()) != to.end())
        for (int64_t i = 1; i < count && bad < 0; ++i)
          if (std::find(dst_host, dst_host + i, dst_host[i]) != dst_host + i) bad = i;
      for (int64_t i = 0; i < count && bad < 0; ++i)
        if (std::binary_search(to.begin(), to.end(), src_host[i])) bad = i;
    }
  } catch (...) {
    return fail(NK_DEVICE_ERROR, "out of host memory");
  }
  if (bad >= 0) {
    st = fail(NK_INVALID_PARAMS, "a destination page appears twice or is a source too");
    tls_error().index = (uint64_t)bad;
    return st;
  }
  cudaStream_t s = as_stream(stream);
  // Parameter blocks of four sizes: a launch copies its parameters, so a
  // single fork should not carry 32 KB of them.
  for (int64_t i = 0; i < count;) {
    const int64_t left = count - i;
    int n;
    if (left <= 16) {
      n = (int)left;
      st = launch_copy<16>(*kv, src_host + i, dst_host + i, n, s);
    } else if (left <= 500) {
      n = (int)left;
      st = launch_copy<500>(*kv, src_host + i, dst_host + i, n, s);
    } else if (left <= 2000) {
      n = (int)left;
      st = launch_copy<2000>(*kv, src_host + i, dst_host + i, n, s);
    } else {
      n = (int)(left < 4000 ? left : 4000);
      st = launch_copy<4000>(*kv, src_host + i, dst_host + i, n, s);
    }
    if (st != NK_OK) return st;
    i += n;
  }
  return ok();
}

nk_status nk_kv_table_write(int32_t *dst, int64_t dst_len, const int64_t *offset_host,
                            const int32_t *value_host, int64_t count, void *stream) {
  if (count < 0 || dst_len < 0) return fail(NK_INVALID_SHAPE, "count, dst_len >= 0");
  if (count == 0) return ok();
  if (!dst || !value_host) return fail(NK_INVALID_PARAMS, "dst and value_host are required");
  if (!offset_host && count > dst_len)
    return fail_length("dst", (uint64_t)count, (uint64_t)dst_len);
  if (offset_host) {
    bool ascending = true;
    for (int64_t i = 0; i < count; ++i) {
      if (offset_host[i] < 0 || offset_host[i] >= dst_len) {
        nk_status st = fail(NK_INVALID_PARAMS, "offset outside dst");
        tls_error().index = (uint64_t)i;
        tls_error().actual = (uint64_t)offset_host[i];
        tls_error().expected = (uint64_t)dst_len;
        return st;
      }
      ascending &= i == 0 || offset_host[i] > offset_host[i - 1];
    }
    if (!ascending) {  // the threads of a launch write in no order
      try {
        std::vector<int64_t> o(offset_host, offset_host + count);
        std::sort(o.begin(), o.end());
        if (std::adjacent_find(o.begin(), o.end()) != o.end())
          return fail(NK_INVALID_PARAMS, "an offset appears twice");
      } catch (...) {
        return fail(NK_DEVICE_ERROR, "out of host memory");
      }
    }
  }
  cudaStream_t s = as_stream(stream);
  for (int64_t i = 0; i < count;) {
    const int64_t left = count - i;
    const int64_t *off = offset_host ? offset_host + i : nullptr;
    int32_t *to = offset_host ? dst : dst + i;
    int n;
    nk_status st;
    if (left <= 64) {
      n = (int)left;
      st = launch_table<64>(to, off, value_host + i, n, s);
    } else {
      n = (int)(left < 2600 ? left : 2600);
      st = launch_table<2600>(to, off, value_host + i, n, s);
    }
    if (st != NK_OK) return st;
    i += n;
  }
  return ok();
}

nk_status nk_kv_pages_compact(const nk_kv_pages *kv, const nk_kv_compact_args *args,
                              void *stream) {
  nk_status st = check_pages(kv, 0);
  if (st == NK_OK) st = check_table(kv);
  if (st != NK_OK) return st;
  if (!args) return fail(NK_INVALID_PARAMS, "args");
  if (args->seqs < 0 || args->max_keep < 0) return fail(NK_INVALID_SHAPE, "seqs, max_keep >= 0");
  if (args->seqs > 65535) return fail(NK_UNSUPPORTED, "at most 65535 sequences a call");
  if (args->max_keep >= (1ll << 31)) return fail(NK_UNSUPPORTED, "max_keep must be < 2^31");
  if (args->max_keep > args->keep_ld)
    return fail(NK_INVALID_PARAMS, "max_keep must not exceed keep_ld");
  if (args->seqs == 0) return ok();
  if (!args->kv_len || !args->base || !args->n_keep || (!args->keep && args->max_keep > 0))
    return fail(NK_INVALID_PARAMS, "kv_len, base, keep and n_keep are required");
  if (!args->rows && args->seqs > kv->table_rows)
    return fail(NK_INVALID_PARAMS, "more sequences than table rows");
  if (args->dst_table && (args->dst_ld <= 0 || args->dst_ld >= (1ll << 31)))
    return fail(NK_INVALID_PARAMS, "dst_ld must be positive and < 2^31");
  if (!args->dst_table && args->dst_ld != 0)
    return fail(NK_INVALID_PARAMS, "dst_ld without dst_table");
  // One block writes a sequence's new length while others still read its arrays.
  const int64_t n = args->seqs;
  if (overlap(args->new_len, n, args->rows, n) || overlap(args->new_len, n, args->kv_len, n) ||
      overlap(args->new_len, n, args->base, n) || overlap(args->new_len, n, args->n_keep, n) ||
      overlap(args->new_len, n, args->keep, (n - 1) * args->keep_ld + args->max_keep) ||
      overlap(args->new_len, n, args->dst_table, n * args->dst_ld) ||
      overlap(args->new_len, n, kv->table, kv->table_rows * kv->table_ld))
    return fail(NK_INVALID_PARAMS, "new_len must not overlap the arrays that the call reads");
  int *err = device_error_ptr();
  if (!err) return fail(NK_DEVICE_ERROR, "cannot resolve device error word");
  const PagePool pool = page_pool(*kv);
  CompactArgs a{};
  a.rows = args->rows;
  a.kv_len = args->kv_len;
  a.base = args->base;
  a.keep = args->keep;
  a.n_keep = args->n_keep;
  a.dst_table = args->dst_table;
  a.keep_ld = args->keep_ld;
  a.dst_ld = args->dst_ld;
  a.max_keep = (int)args->max_keep;
  a.new_len = args->new_len;
  uint4 *k = reinterpret_cast<uint4 *>(kv->k), *v = reinterpret_cast<uint4 *>(kv->v);
  uint4 *lo = reinterpret_cast<uint4 *>(kv->k_min), *hi = reinterpret_cast<uint4 *>(kv->k_max);
  cudaStream_t s = as_stream(stream);
  const unsigned lh = (unsigned)(kv->layers * kv->kv_heads);
  if (args->dst_table) {
    const int64_t touched = (args->max_keep + kv->page_size - 1) / kv->page_size + 1;
    const dim3 grid((unsigned)touched, lh, (unsigned)args->seqs);
    if (kv->head_dim == 128)
      pages_compact_kernel<128><<<grid, 128, 0, s>>>(pool, a, k, v, lo, hi, err);
    else
      pages_compact_kernel<64><<<grid, 128, 0, s>>>(pool, a, k, v, lo, hi, err);
    return check_launch("pages_compact_kernel");
  }
  const dim3 grid(lh, (unsigned)args->seqs);
  if (kv->head_dim == 128)
    pages_compact_inplace_kernel<128><<<grid, 256, 0, s>>>(pool, a, k, v, lo, hi, err);
  else
    pages_compact_inplace_kernel<64><<<grid, 256, 0, s>>>(pool, a, k, v, lo, hi, err);
  return check_launch("pages_compact_inplace_kernel");
}

}  // extern "C"
