// block_select.cu — which blocks of a paged cache each query reads: an upper
// bound of the block's scores from the channel bounds of its keys, then the
// largest top_k of them.
//
// The bound is sum_c q_c * (q_c >= 0 ? k_max_c : k_min_c), per query head;
// the heads that share a KV head share a list, ranked by their largest bound.
// Products of two bf16 values are exact in f64, and sums of head_dim of them
// are exact or off by 2^-53 relative, so the ranking does not depend on the
// order of the sum: a list is the same whatever split or layout computes it.
#include "paged.cuh"

namespace nk {

struct SelectArgs {
  PagePool pool;
  PageBatch batch;
  const uint16_t *q;
  int64_t ld_q;
  int group;
  const uint16_t *k_min, *k_max;  // the layer's
  int top_k, sink, local;
  int64_t score_ld;
  double *scores;  // [tokens, kv_heads, score_ld]
  int32_t *blocks;
  int *err;
};

// Token t of the batch's buffers -> its sequence (start is ascending): -1 when
// no sequence holds it.
__device__ __forceinline__ int sequence_of(const PageBatch &b, int64_t t) {
  int lo = 0, hi = b.seqs;  // start[lo] <= t < start[hi]
  if (t < b.start[0] || t >= b.start[b.seqs]) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (b.start[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

struct Query {
  SeqView seq;
  int pos, blocks;  // position; eligible blocks
  int64_t token;
};

__device__ __forceinline__ bool find_query(const SelectArgs &a, int64_t token, Query &x,
                                           bool report_it) {
  const int s = sequence_of(a.batch, token);
  if (s < 0 || !load_seq(a.pool, a.batch, s, x.seq, a.err, report_it)) return false;
  if (token < x.seq.first || token >= (int64_t)x.seq.first + x.seq.count) return false;
  x.token = token;
  x.pos = x.seq.len - x.seq.count + (int)(token - x.seq.first);
  x.blocks = (x.pos >> a.pool.ps_log2) + 1;
  return true;
}

// Block = (128 eligible blocks x, KV head y, token z): a thread per block, the
// group's queries as f64 in shared memory.
template <int D>
__global__ void __launch_bounds__(128) block_scores_kernel(const SelectArgs a) {
  extern __shared__ double qd[];  // [group][D]
  Query x;
  if (!find_query(a, blockIdx.z, x, threadIdx.x == 0)) return;
  if (x.blocks <= a.top_k) return;  // every block is taken
  const int first = blockIdx.x * 128;
  // the forced blocks need no score
  if (first >= x.blocks - a.local || first + 128 <= a.sink) return;
  const int h = blockIdx.y;
  const uint16_t *q = a.q + x.token * a.ld_q + (int64_t)h * a.group * D;
  for (int i = threadIdx.x; i < a.group * D; i += 128)
    qd[i] = (double)__uint_as_float((uint32_t)q[i] << 16);
  __syncthreads();
  const int j = first + threadIdx.x;
  if (j < a.sink || j >= x.blocks - a.local) return;
  const int page = x.seq.table[j];
  double best = -INFINITY;
  if (page_ok(a.pool, page)) {
    const int64_t at = ((int64_t)page * a.pool.heads + h) * D;
    constexpr int HEADS = 8;  // sums in flight
    for (int g0 = 0; g0 < a.group; g0 += HEADS) {
      double acc[HEADS];
#pragma unroll
      for (int g = 0; g < HEADS; ++g) acc[g] = 0.0;
      for (int c = 0; c < D; c += 8) {
        const uint4 lo4 = *reinterpret_cast<const uint4 *>(a.k_min + at + c);
        const uint4 hi4 = *reinterpret_cast<const uint4 *>(a.k_max + at + c);
        const uint32_t lw[4] = {lo4.x, lo4.y, lo4.z, lo4.w};
        const uint32_t hw[4] = {hi4.x, hi4.y, hi4.z, hi4.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t lb = (e & 1) ? lw[e >> 1] & 0xffff0000u : lw[e >> 1] << 16;
          const uint32_t hb = (e & 1) ? hw[e >> 1] & 0xffff0000u : hw[e >> 1] << 16;
          const double lo = (double)__uint_as_float(lb), hi = (double)__uint_as_float(hb);
#pragma unroll
          for (int g = 0; g < HEADS; ++g)
            if (g0 + g < a.group) {
              const double qv = qd[(g0 + g) * D + c + e];
              acc[g] = fma(qv, qv >= 0.0 ? hi : lo, acc[g]);
            }
        }
      }
#pragma unroll
      for (int g = 0; g < HEADS; ++g)
        if (g0 + g < a.group) best = fmax(best, acc[g]);  // NaN loses
    }
  } else {
    report(a.err, NK_PAGE_OUT_OF_RANGE);
  }
  a.scores[(x.token * a.pool.heads + h) * a.score_ld + j] = best;
}

// f64 -> a whole number of the same order.
__device__ __forceinline__ unsigned long long order_key(double v) {
  v += 0.0;  // -0 ranks as 0
  const unsigned long long b = (unsigned long long)__double_as_longlong(v);
  return b >> 63 ? ~b : b | (1ull << 63);
}

// Block = (KV head x, token y): finds the need-th largest score digit by digit
// (8 bits a pass, stopping once a digit's bin is taken whole), then writes the
// chosen blocks in ascending order.
__global__ void __launch_bounds__(256) block_topk_kernel(const SelectArgs a) {
  __shared__ int hist[256];
  __shared__ int warp_sum[8][2];
  __shared__ int sh_digit, sh_need, sh_count;
  Query x;
  if (!find_query(a, blockIdx.y, x, threadIdx.x == 0)) return;
  const int h = blockIdx.x, n = x.blocks;
  int32_t *out = a.blocks + (x.token * a.pool.heads + h) * (int64_t)a.top_k;
  if (n <= a.top_k) {
    for (int i = threadIdx.x; i < a.top_k; i += 256) out[i] = i < n ? i : -1;
    return;
  }
  const double *sc = a.scores + (x.token * a.pool.heads + h) * a.score_ld;
  const int lo = a.sink, hi = n - a.local;  // free blocks
  int need = a.top_k - a.sink - a.local;
  unsigned long long prefix = 0, mask = 0;  // digits found so far
  bool whole = need == 0;                   // all keys that match the prefix are taken
  for (int shift = 56; shift >= 0 && !whole; shift -= 8) {
    hist[threadIdx.x] = 0;
    __syncthreads();
    for (int j = lo + threadIdx.x; j < hi; j += 256) {
      const unsigned long long key = order_key(sc[j]);
      if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int left = need, d = 255;
      while (d > 0 && hist[d] < left) left -= hist[d--];
      sh_digit = d;
      sh_need = left;
      sh_count = hist[d];
    }
    __syncthreads();
    prefix |= (unsigned long long)sh_digit << shift;
    mask |= 255ull << shift;
    need = sh_need;
    whole = sh_count == need;
    __syncthreads();
  }
  // Above the prefix: taken.  Equal to it: the first `need` by index (all, when
  // the bin is whole).  A contiguous run of blocks per thread keeps the order.
  const int per = (n + 255) / 256;
  const int a0 = threadIdx.x * per < n ? threadIdx.x * per : n;
  const int a1 = a0 + per < n ? a0 + per : n;
  const bool none = a.top_k == a.sink + a.local;
  int above = 0, equal = 0;
  for (int j = a0; j < a1; ++j) {
    if (j < lo || j >= hi) {
      ++above;
    } else if (!none) {
      const unsigned long long key = order_key(sc[j]) & mask;
      above += key > prefix;
      equal += key == prefix;
    }
  }
  // Exclusive sums over the block of both counts.
  int sa = above, se = equal;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int o = 1; o < 32; o <<= 1) {
    const int va = __shfl_up_sync(0xffffffffu, sa, o), ve = __shfl_up_sync(0xffffffffu, se, o);
    if (lane >= o) {
      sa += va;
      se += ve;
    }
  }
  if (lane == 31) {
    warp_sum[warp][0] = sa;
    warp_sum[warp][1] = se;
  }
  __syncthreads();
  for (int w = 0; w < warp; ++w) {
    sa += warp_sum[w][0];
    se += warp_sum[w][1];
  }
  int eq = se - equal;                       // equals before this run
  int at = sa - above + (eq < need ? eq : need);
  for (int j = a0; j < a1; ++j) {
    bool take = j < lo || j >= hi;
    if (!take && !none) {
      const unsigned long long key = order_key(sc[j]) & mask;
      if (key == prefix) take = eq++ < need;
      else take = key > prefix;
    }
    if (take) out[at++] = j;
  }
}

static nk_status check_select(const nk_kv_pages *kv, const nk_kv_batch *b) {
  if (b->tokens > 65535) return fail(NK_UNSUPPORTED, "at most 65535 tokens a call");
  if (!kv->k_min) return fail(NK_INVALID_PARAMS, "k_min and k_max are required");
  return NK_OK;
}

static int64_t score_width(const nk_kv_pages *kv, const nk_kv_batch *b) {
  return ceil_div(b->max_kv > 0 ? b->max_kv : 1, kv->page_size);
}

}  // namespace nk

using namespace nk;

extern "C" {

nk_status nk_kv_block_select_workspace_bytes(const nk_kv_pages *kv, const nk_kv_batch *batch,
                                             size_t *bytes) {
  if (!bytes) return fail(NK_INVALID_PARAMS, "bytes");
  nk_status st = check_pages(kv, 0);
  if (st == NK_OK) st = check_batch(kv, batch);
  if (st == NK_OK) st = check_select(kv, batch);
  if (st != NK_OK) return st;
  *bytes = (size_t)batch->tokens * kv->kv_heads * score_width(kv, batch) * sizeof(double);
  return ok();
}

nk_status nk_kv_block_select(const nk_kv_pages *kv, int64_t layer, const nk_kv_batch *batch,
                             const uint16_t *q, int64_t ld_q, int64_t q_heads, int64_t top_k,
                             int64_t sink, int64_t local, int32_t *blocks, void *workspace,
                             size_t workspace_bytes, void *stream) {
  nk_status st = check_pages(kv, layer);
  if (st == NK_OK) st = check_batch(kv, batch);
  if (st == NK_OK) st = check_select(kv, batch);
  if (st != NK_OK) return st;
  if (q_heads <= 0) return fail(NK_INVALID_SHAPE, "q_heads > 0");
  if (q_heads % kv->kv_heads) {
    st = fail(NK_HEAD_COUNT_MISMATCH, "query heads must be a multiple of KV heads");
    tls_error().expected = (uint64_t)q_heads;
    tls_error().actual = (uint64_t)kv->kv_heads;
    return st;
  }
  const int64_t group = q_heads / kv->kv_heads;
  if (group * kv->head_dim * 8 > 48 * 1024)
    return fail(NK_UNSUPPORTED, "q_heads / kv_heads * head_dim must be <= 6144");
  if (ld_q < q_heads * kv->head_dim)
    return fail(NK_INVALID_PARAMS, "ld_q must be >= q_heads * head_dim");
  if (sink < 0 || local < 1 || top_k < sink + local || top_k > (1 << 20))
    return fail(NK_INVALID_PARAMS, "sink >= 0, local >= 1, sink + local <= top_k <= 2^20");
  if (batch->seqs == 0 || batch->tokens == 0 || batch->max_new == 0) return ok();
  if (!q || !blocks) return fail(NK_INVALID_PARAMS, "q and blocks are required");
  const int64_t width = score_width(kv, batch);
  const size_t need = (size_t)batch->tokens * kv->kv_heads * width * sizeof(double);
  if (workspace_bytes < need || !workspace) {
    st = fail(NK_WORKSPACE_TOO_SMALL, "block selection workspace too small");
    tls_error().expected = need;
    tls_error().actual = workspace_bytes;
    return st;
  }
  if ((uintptr_t)workspace & 15) return fail(NK_INVALID_PARAMS, "workspace must be 16-byte aligned");
  SelectArgs a{};
  a.pool = page_pool(*kv);
  a.batch = page_batch(*batch);
  a.q = q;
  a.ld_q = ld_q;
  a.group = (int)group;
  const int64_t layer_words = kv->pages * kv->kv_heads * kv->head_dim;
  a.k_min = kv->k_min + layer * layer_words;
  a.k_max = kv->k_max + layer * layer_words;
  a.top_k = (int)top_k;
  a.sink = (int)sink;
  a.local = (int)local;
  a.score_ld = width;
  a.scores = static_cast<double *>(workspace);
  a.blocks = blocks;
  a.err = device_error_ptr();
  if (!a.err) return fail(NK_DEVICE_ERROR, "cannot resolve device error word");
  cudaStream_t s = as_stream(stream);
  if (width > top_k) {
    const dim3 grid((unsigned)ceil_div(width, 128), (unsigned)kv->kv_heads,
                    (unsigned)batch->tokens);
    const size_t smem = (size_t)(group * kv->head_dim * 8);
    if (kv->head_dim == 128)
      block_scores_kernel<128><<<grid, 128, smem, s>>>(a);
    else
      block_scores_kernel<64><<<grid, 128, smem, s>>>(a);
    st = check_launch("block_scores_kernel");
    if (st != NK_OK) return st;
  }
  block_topk_kernel<<<dim3((unsigned)kv->kv_heads, (unsigned)batch->tokens), 256, 0, s>>>(a);
  return check_launch("block_topk_kernel");
}

}  // extern "C"
