// block_select.cu — which blocks of a paged cache each query reads: an upper
// bound of the block's scores from the channel bounds of its keys, then the
// largest top_k of them.
//
// The score is sum_c q_c * (q_c >= 0 ? k_max_c : k_min_c), per query head; the
// heads that share a KV head share a list, ranked by their largest score.  A
// list must not depend on the order of a sum, so it is defined by 64-bit sums
// (products of two bf16 values are exact in f64).  f64 arithmetic over every
// block measured 42 us for 4 sequences of 131072 tokens, so the first pass is
// f32 with a bound of its error: each block gets an interval that holds its
// score, the intervals settle nearly every block, and only those that straddle
// the border are summed again in 64 bits.
#include <atomic>

#include "paged.cuh"

namespace nk {

typedef unsigned long long u64;

struct SelectArgs {
  PagePool pool;
  PageBatch batch;
  const uint16_t *q;
  int64_t ld_q;
  int group;
  const uint16_t *k_min, *k_max;  // the layer's
  int top_k, sink, local;
  int64_t score_ld;
  float2 *range;   // [tokens, kv_heads, score_ld]: the score lies in it
  double *exact;   // the same shape: 64-bit scores of the blocks in doubt
  int32_t *blocks;
  int *err;
};

// Token t of the batch's buffers -> its sequence (start is ascending), -1 when
// no sequence holds it.  A warp halves the range 32-fold a load; every lane
// returns the result.
__device__ __forceinline__ int sequence_of(const PageBatch &b, int64_t t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = b.seqs + 1;  // the last start <= t lies in lo .. lo+n-1
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int at = lo + lane * step;
    const bool le = lane * step < n && b.start[at] <= t;
    const uint32_t hit = __ballot_sync(0xffffffffu, le);
    if (!hit) return -1;
    const int last = 31 - __clz(hit);
    const int left = n - last * step;
    lo += last * step;
    n = left < step ? left : step;
  }
  return b.start[lo] <= t && lo < b.seqs ? lo : -1;
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

__device__ __forceinline__ float bf16_f32(uint16_t x) {
  return __uint_as_float((uint32_t)x << 16);
}

// Two f32 FMAs in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(*reinterpret_cast<u64 *>(&d))
      : "l"(*reinterpret_cast<const u64 *>(&a)), "l"(*reinterpret_cast<const u64 *>(&b)),
        "l"(*reinterpret_cast<const u64 *>(&c)));
  return d;
}

// Block = (128 eligible blocks x, KV head y, token z): each of 8 warps takes an
// eighth of the channels, a lane 4 blocks, so that a query value is one
// broadcast read of shared memory for 128 blocks (a broadcast moves 4 bytes a
// cycle: with a block a lane those reads took 12000 cycles, 6 us); HEADS query
// heads at a time.
//   s_g = sum_c max(q, 0) * k_max + min(q, 0) * k_min   (f32 FMAs)
//   A   = sum_c max_g|q| * max(|k_min|, |k_max|)        >= sum of any head's |terms|
// A lane adds D/8 terms (the other product of a channel is 0) and the eighths
// are joined in three more steps, each off by at most 2^-24 of a partial sum,
// itself at most A: |s_g - score| <= (D/8 + 3) * 2^-24 A.  The interval takes
// (D/8 + 7) * 2^-24 A: one more covers the roundings of its own ends, another
// the relative error of A ((D/8 + 4) * 2^-24, times D/8 + 3), and 1e-38 results
// that underflow.  Where a sum is not finite (0 * inf is NaN here, not in the
// definition) the interval is everything.
// The loop is not unrolled beyond two channels: a warp runs through it a few
// times only, and straight-line code of this kernel spent its time on
// instruction fetch (47 us against 19 for the same sums).
// 4 sequences of 131072 tokens, 2048 blocks of 2 heads of 128, 16 query heads a
// KV head, 8.4 MB of bounds: 13.8 us cold.  Bound by latency and issue: one round
// of loads, then two multiply-adds a head, channel and block, then the join.
constexpr int kScoreBlocks = 128, kScoreWarps = 8;

template <int D>
struct ScoreShared {
  static constexpr int kRow = D * 2 + 4;  // bytes of a block's bounds: 4 apart in banks
  static constexpr int kBounds = 2 * kScoreBlocks * kRow;
  static constexpr int kSums = kScoreWarps * kScoreBlocks * 4;  // of a head: [warp][block] f32
  // The sums of a pass lie over the bounds when it is the only one.
  static size_t bytes(int64_t wide, int heads) {
    const size_t sums = (size_t)(heads + 1) * kSums, queries = (size_t)wide * D * 8 + D * 4;
    if (wide > heads) return kBounds + queries + sums;
    return queries + (sums > (size_t)kBounds ? sums : (size_t)kBounds);
  }
};

template <int D, int HEADS>
__global__ void __launch_bounds__(32 * kScoreWarps) block_scores_kernel(const SelectArgs a) {
  using S = ScoreShared<D>;
  constexpr int NB = kScoreBlocks / 32;  // blocks of a lane
  constexpr int C = D / 8;               // 16-byte words of a row
  constexpr int T = 32 * kScoreWarps;
  extern __shared__ __align__(16) uint8_t smem[];
  const int wide = (a.group + HEADS - 1) / HEADS * HEADS;
  // [D][wide/2]: q+ of two heads, q- of both
  float4 *qs = reinterpret_cast<float4 *>(smem);
  float *qm = reinterpret_cast<float *>(qs + D * wide / 2);  // [D]: max_g |q|
  uint8_t *bounds = reinterpret_cast<uint8_t *>(qm + D);     // [low, high][block][kRow]
  const bool once = wide == HEADS;                           // one pass
  float *sums = reinterpret_cast<float *>(bounds + (once ? 0 : S::kBounds));
                                                             // [HEADS + 1][warp][block]
  let_next_launch();
  wait_for_previous();
  const int h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // The first 8 channels of this thread's queries are on their way while the
  // sequence is found.
  const uint4 *q =
      reinterpret_cast<const uint4 *>(a.q + blockIdx.z * a.ld_q + (int64_t)h * a.group * D);
  uint4 qw = make_uint4(0, 0, 0, 0);
  if ((int)threadIdx.x < a.group * C) qw = q[threadIdx.x];
  Query x;
  if (!find_query(a, blockIdx.z, x, threadIdx.x == 0)) return;
  if (x.blocks <= a.top_k) return;  // every block is taken
  const int first = blockIdx.x * kScoreBlocks;
  // the forced blocks need no score
  if (first >= x.blocks - a.local || first + kScoreBlocks <= a.sink) return;
  // Bounds: a warp copies the rows of 16 blocks, whole 128- or 256-byte rows a
  // load.  (Rows lie 4 bytes past a multiple of 128: words go in by fours.)
  {
    constexpr int ROWS = kScoreBlocks / kScoreWarps;
    const int mine = first + warp * ROWS + lane % ROWS;
    int page = -1;
    if (mine >= a.sink && mine < x.blocks - a.local) {
      page = x.seq.table[mine];
      if (!page_ok(a.pool, page)) {
        report(a.err, NK_PAGE_OUT_OF_RANGE);
        page = -1;
      }
    }
#pragma unroll
    for (int r = 0; r < ROWS; r += 32 / C) {
      const int row = r + lane / C;
      const int pg = __shfl_sync(0xffffffffu, page, row);
      const int64_t at = ((int64_t)(pg < 0 ? 0 : pg) * a.pool.heads + h) * C + lane % C;
      const uint4 lo = reinterpret_cast<const uint4 *>(a.k_min)[at];
      const uint4 hi = reinterpret_cast<const uint4 *>(a.k_max)[at];
      uint32_t *to = reinterpret_cast<uint32_t *>(bounds + (warp * ROWS + row) * S::kRow) +
                     (lane % C) * 4;
      to[0] = lo.x, to[1] = lo.y, to[2] = lo.z, to[3] = lo.w;
      to += kScoreBlocks * S::kRow / 4;
      to[0] = hi.x, to[1] = hi.y, to[2] = hi.z, to[3] = hi.w;
    }
  }
  bool odd = false;  // a NaN query is dropped by fmaxf and fminf
  for (int i = threadIdx.x; i < wide * C; i += T) {
    const int g = i / C, c = (i % C) * 8;
    if (i >= T) qw = i < a.group * C ? q[i] : make_uint4(0, 0, 0, 0);
    const uint32_t w[4] = {qw.x, qw.y, qw.z, qw.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = __uint_as_float((e & 1) ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
      odd |= v != v;
      float *to = reinterpret_cast<float *>(qs + (c + e) * (wide / 2) + g / 2) + (g & 1);
      to[0] = fmaxf(v, 0.0f);
      to[2] = fminf(v, 0.0f);
    }
  }
  odd = __syncthreads_or(odd);
  for (int c = threadIdx.x; c < D; c += T) {
    const float4 *row = qs + c * (wide / 2);
    float mx = 0.0f;
#pragma unroll 4
    for (int g = 0; g < wide / 2; ++g)
      mx = fmaxf(mx, fmaxf(fmaxf(row[g].x, row[g].y), fmaxf(-row[g].z, -row[g].w)));
    qm[c] = mx;
  }
  __syncthreads();
  const uint8_t *low_row = bounds + lane * S::kRow + warp * (D / kScoreWarps * 2);
  const int jb = threadIdx.x >> 1, j = first + jb;  // block of this thread's join
  auto joined = [&](int g) {
    const float *v = sums + g * kScoreWarps * kScoreBlocks + jb;
    float s[kScoreWarps];
#pragma unroll
    for (int w = 0; w < kScoreWarps; ++w) s[w] = v[w * kScoreBlocks];
    return ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
  };
  float mag[NB], best = -INFINITY;
#pragma unroll
  for (int i = 0; i < NB; ++i) mag[i] = 0.0f;
#pragma unroll 1
  for (int g0 = 0; g0 < wide; g0 += HEADS) {
    float2 acc[NB][HEADS / 2];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int g = 0; g < HEADS / 2; ++g) acc[i][g] = make_float2(0.0f, 0.0f);
    const float4 *qc = qs + warp * (D / kScoreWarps) * (wide / 2) + g0 / 2;
    const float *qa = qm + warp * (D / kScoreWarps);
#pragma unroll 1
    for (int c = 0; c < D / kScoreWarps; c += 2) {
      uint32_t lw[NB], hw[NB];
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const uint8_t *at = low_row + i * 32 * S::kRow + c * 2;
        lw[i] = *reinterpret_cast<const uint32_t *>(at);
        hw[i] = *reinterpret_cast<const uint32_t *>(at + kScoreBlocks * S::kRow);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e, qc += wide / 2) {
        float l[NB], u[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          l[i] = __uint_as_float(e ? lw[i] & 0xffff0000u : lw[i] << 16);
          u[i] = __uint_as_float(e ? hw[i] & 0xffff0000u : hw[i] << 16);
        }
#pragma unroll
        for (int g = 0; g < HEADS / 2; ++g) {
          const float4 v = qc[g];
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            acc[i][g] = fma2(make_float2(v.x, v.y), make_float2(u[i], u[i]), acc[i][g]);
            acc[i][g] = fma2(make_float2(v.z, v.w), make_float2(l[i], l[i]), acc[i][g]);
          }
        }
        if (g0 == 0) {
          const float m = qa[c + e];
#pragma unroll
          for (int i = 0; i < NB; ++i) mag[i] = fmaf(m, fmaxf(fabsf(l[i]), fabsf(u[i])), mag[i]);
        }
      }
    }
    if (once) __syncthreads();  // the bounds are read
#pragma unroll
    for (int g = 0; g < HEADS / 2; ++g)
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        float *to = sums + (2 * g * kScoreWarps + warp) * kScoreBlocks + i * 32 + lane;
        to[0] = acc[i][g].x;
        to[kScoreWarps * kScoreBlocks] = acc[i][g].y;
      }
    if (g0 == 0)
#pragma unroll
      for (int i = 0; i < NB; ++i)
        sums[(HEADS * kScoreWarps + warp) * kScoreBlocks + i * 32 + lane] = mag[i];
    __syncthreads();
    // Join the eighths: two neighbouring threads a block, every other head each.
    for (int g = threadIdx.x & 1; g < HEADS && g0 + g < a.group; g += 2) {
      const float v = joined(g);
      odd |= !(fabsf(v) < INFINITY);
      best = fmaxf(best, v);
    }
    if (g0 + HEADS < wide) __syncthreads();  // before the next pass writes its sums
  }
  best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 1));
  odd |= __shfl_xor_sync(0xffffffffu, (int)odd, 1) != 0;
  if ((threadIdx.x & 1) == 0 && j >= a.sink && j < x.blocks - a.local) {
    const float e = fmaf(joined(HEADS), (D / 8 + 7) * 0x1p-24f, 1e-38f);
    float2 r = make_float2(best - e, best + e);
    if (odd || !(e < INFINITY)) r = make_float2(-INFINITY, INFINITY);
    if (!page_ok(a.pool, x.seq.table[j])) r = make_float2(-INFINITY, -INFINITY);
    a.range[(x.token * a.pool.heads + h) * a.score_ld + j] = r;
  }
}

// The score by its definition, by one warp (every lane returns it): a lane sums
// D / 32 neighbouring channels.
template <int D>
__device__ __forceinline__ double exact_score(const SelectArgs &a, const Query &x, int h, int j) {
  constexpr int V = D / 32;
  struct alignas(2 * V) Chunk { uint16_t v[V]; };
  const int c0 = (threadIdx.x & 31) * V;
  const int page = x.seq.table[j];
  double best = -INFINITY;
  if (!page_ok(a.pool, page)) return best;
  const int64_t at = ((int64_t)page * a.pool.heads + h) * D + c0;
  const Chunk lo = *reinterpret_cast<const Chunk *>(a.k_min + at);
  const Chunk hi = *reinterpret_cast<const Chunk *>(a.k_max + at);
  const uint16_t *q = a.q + x.token * a.ld_q + (int64_t)h * a.group * D + c0;
#pragma unroll 4
  for (int g = 0; g < a.group; ++g) {
    double s = 0.0;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const float v = bf16_f32(q[g * D + c]);
      s = fma((double)v, (double)bf16_f32(v >= 0.0f ? hi.v[c] : lo.v[c]), s);
    }
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    best = fmax(best, s);  // NaN loses
  }
  return best;
}

// A float or double -> a whole number of the same order (-0 ranks as 0), above 0.
__device__ __forceinline__ u64 order_key(double v) {
  v += 0.0;
  const u64 b = (u64)__double_as_longlong(v);
  return b >> 63 ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ uint32_t order_key(float v) {
  v += 0.0f;
  const uint32_t b = __float_as_uint(v);
  return b >> 31 ? ~b : b | 0x80000000u;
}

template <int T>
struct TopShared {
  static constexpr int kWarps = T / 32, kDoubt = 128;
  int hist[256];
  u64 doubt_key[kDoubt], from;
  int doubt[kDoubt], doubts, ties;
  u64 ends[2][kWarps];
  int above[kWarps], equal[kWarps];
  int digit, need, whole;
};

__device__ __forceinline__ uint32_t warp_min(uint32_t v) {
  return __reduce_min_sync(0xffffffffu, v);
}
__device__ __forceinline__ uint32_t warp_max(uint32_t v) {
  return __reduce_max_sync(0xffffffffu, v);
}
__device__ __forceinline__ u64 warp_min(u64 v) {
  for (int o = 16; o > 0; o >>= 1) {
    const u64 w = __shfl_xor_sync(0xffffffffu, v, o);
    v = w < v ? w : v;
  }
  return v;
}
__device__ __forceinline__ u64 warp_max(u64 v) {
  for (int o = 16; o > 0; o >>= 1) {
    const u64 w = __shfl_xor_sync(0xffffffffu, v, o);
    v = w > v ? w : v;
  }
  return v;
}

// Sum over the block; ends with a barrier behind which `sh` may be reused.
template <int T>
__device__ __forceinline__ int block_sum(int v, int *sh) {
  v = __reduce_add_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < T / 32; ++w) total += sh[w];
  __syncthreads();
  return total;
}

// The need-th largest of the keys at(j), j = j0, j0+32, .. < j1 of all threads
// (0: no key; 1 <= need <= keys): a t that the need-th key reaches and the next
// smaller one does not (`whole`), or, when keys tie there, their value.  A pass
// spreads the keys that are left over 256 bins between the smallest and the
// largest of them, so one or two passes end most searches among a few thousand.
template <typename K, int T, typename At>
__device__ __forceinline__ K nth_largest(int j0, int j1, At at, int need, TopShared<T> &sh,
                                         bool &whole) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  K least = ~(K)0, most = 0;
#pragma unroll 4
  for (int j = j0; j < j1; j += 32) {
    const K k = at(j);
    if (k) {
      least = k < least ? k : least;
      most = k > most ? k : most;
    }
  }
  least = warp_min(least);
  most = warp_max(most);
  if (lane == 0) {
    sh.ends[0][warp] = least;
    sh.ends[1][warp] = most;
  }
  for (int i = threadIdx.x; i < 256; i += T) sh.hist[i] = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < T / 32; ++w) {
    least = (K)sh.ends[0][w] < least ? (K)sh.ends[0][w] : least;
    most = (K)sh.ends[1][w] > most ? (K)sh.ends[1][w] : most;
  }
  for (;;) {
    const int bits = 64 - __clzll((long long)(u64)(most - least));
    const int shift = bits > 8 ? bits - 8 : 0;
#pragma unroll 4
    for (int j = j0; j < j1; j += 32) {
      const K k = at(j);
      if (k >= least && k <= most) atomicAdd(&sh.hist[(int)((k - least) >> shift)], 1);
    }
    __syncthreads();
    if (warp == 0) {  // lane: bins 8*lane .. +7; higher bins hold larger keys
      int c[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += c[i] = sh.hist[lane * 8 + i];
      int up = sum;  // bins of this lane and the lanes above
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_down_sync(0xffffffffu, up, o);
        if (lane + o < 32) up += v;
      }
      int before = up - sum;
      if (before < need && up >= need) {  // one lane
#pragma unroll
        for (int i = 7; i >= 0; --i)
          if (before < need) {
            before += c[i];
            if (before >= need) {
              sh.digit = lane * 8 + i;
              sh.need = need - (before - c[i]);
              sh.whole = before == need;
              before = need;  // found
            }
          }
      }
    }
    __syncthreads();
    least += (K)sh.digit << shift;
    need = sh.need;
    whole = sh.whole != 0;
    for (int i = threadIdx.x; i < 256; i += T) sh.hist[i] = 0;
    __syncthreads();  // the shared words are read, the bins are empty
    if (whole || shift == 0) return least;
    // The end of the bin, not past the largest key: least + span can pass the
    // type's end (an infinite score's key is close to it).
    const K span = ((K)1 << shift) - 1;
    if (most - least > span) most = least + span;
  }
}

// Block = (KV head x, token y).  With L the need-th largest lower end of the
// intervals: a block whose upper end is below L is out, and when exactly `need`
// upper ends reach L they are the list.  If not, with H the largest upper end of
// a block whose lower end is L or less, a block whose lower end is above H is in
// (only blocks whose lower end is above L could beat it, `need` with itself at
// most) and those in between are scored in 64 bits.  Then the list is written in
// ascending order: a warp holds a contiguous run of blocks, 32 neighbours at a
// time.  T threads: 128 up to 1024 blocks, 512 beyond (400 lists of 190, scores and
// attention included: 63 us a call with 512 threads, most of them idle, 58 with
// 128).  Bound by the chain of the search's barriers: 8 lists of 2048 blocks 10 us
// cold, 400 of 190 12 us.  Blocks in doubt add 5 us to a call; with a second search
// for H and a third for the 64-bit scores it was 12.
template <int D, int T>
__global__ void __launch_bounds__(T, 1024 / T) block_topk_kernel(const SelectArgs a) {
  __shared__ TopShared<T> sh;
  let_next_launch();
  wait_for_previous();
  Query x;
  if (!find_query(a, blockIdx.y, x, threadIdx.x == 0)) return;
  const int h = blockIdx.x, n = x.blocks;
  int32_t *out = a.blocks + (x.token * a.pool.heads + h) * (int64_t)a.top_k;
  if (n <= a.top_k) {
    for (int i = threadIdx.x; i < a.top_k; i += T) out[i] = i < n ? i : -1;
    return;
  }
  const int64_t row = (x.token * a.pool.heads + h) * a.score_ld;
  const float2 *range = a.range + row;
  double *exact = a.exact + row;
  const int lo = a.sink, hi = n - a.local;  // free blocks
  const int need = a.top_k - a.sink - a.local;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int run = ((n + T - 1) / T) * 32;
  const int j0 = warp * run + lane, j1 = (warp + 1) * run < n ? (warp + 1) * run : n;
  auto is_free = [&](int j) { return j >= lo && j < hi; };
  uint32_t low = 0xffffffffu;
  if (need > 0) {
    bool whole;
    // A `whole` result may lie below L: the blocks it keeps in play are more.
    low = nth_largest<uint32_t, T>(
        j0, j1, [&](int j) { return is_free(j) ? order_key(range[j].x) : 0u; }, need, sh, whole);
  }
  // The forced blocks and those that reach L: the list, if they are top_k.
  auto reaches = [&](int j) {
    return j < j1 && (!is_free(j) || order_key(range[j].y) >= low);
  };
  const uint32_t below = (1u << lane) - 1;
  uint32_t kept = 0;  // of the first 32 blocks of this thread
  int mine = 0;
#pragma unroll 1
  for (int j = j0, i = 0; j - lane < j1; j += 32, ++i) {
    const bool r = reaches(j);
    if (i < 32) kept |= (uint32_t)r << i;
    mine += __popc(__ballot_sync(0xffffffffu, r));
  }
  if (lane == 0) sh.above[warp] = mine;
  __syncthreads();
  int reach = 0, at = 0;  // of the block, and before this warp's run
#pragma unroll
  for (int w = 0; w < T / 32; ++w) {
    if (w < warp) at += sh.above[w];
    reach += sh.above[w];
  }
  if (reach == a.top_k) {
#pragma unroll 1
    for (int j = j0, i = 0; j - lane < j1; j += 32, ++i) {
      const bool take = i < 32 ? kept >> i & 1 : reaches(j);
      const uint32_t taken = __ballot_sync(0xffffffffu, take);
      const int to = at + __popc(taken & below);
      if (take && to < a.top_k) out[to] = j;
      at += __popc(taken);
    }
    return;
  }
  __syncthreads();
  // H
  uint32_t top = 0, high;
#pragma unroll 4
  for (int j = j0; j < j1; j += 32) {
    if (!is_free(j)) continue;
    const uint32_t k = order_key(range[j].y);
    if (k >= low && order_key(range[j].x) <= low && k > top) top = k;
  }
  top = warp_max(top);
  if (lane == 0) sh.above[warp] = (int)top;
  if (threadIdx.x == 0) sh.doubts = 0;
  __syncthreads();
  for (int w = 0; w < T / 32; ++w)
    top = (uint32_t)sh.above[w] > top ? (uint32_t)sh.above[w] : top;
  high = top;
  __syncthreads();
  // 0: out, 1: in, 2: in doubt.
  auto kind = [&](int j) {
    if (!is_free(j)) return 1;
    const float2 r = range[j];
    if (order_key(r.y) < low) return 0;
    return order_key(r.x) > high ? 1 : 2;
  };
  int in = 0;
  for (int j = j0; j < j1; j += 32) {
    const int k = kind(j);
    in += k == 1 && is_free(j);
    if (k == 2) {
      const int i = atomicAdd(&sh.doubts, 1);
      if (i < TopShared<T>::kDoubt) sh.doubt[i] = j;
    }
  }
  const int left = need - block_sum<T>(in, sh.above), doubts = sh.doubts;
  // Blocks in doubt: taken above `from`, and the first by index of those equal to
  // it.  (No score is that large: it would be a NaN's.)
  u64 from = ~0ull;
  bool ties = false;
  if (left > 0 && doubts <= TopShared<T>::kDoubt) {
    // A few: a warp each, and a thread each to rank it among them.
    for (int i = warp; i < doubts; i += T / 32) {
      const double v = exact_score<D>(a, x, h, sh.doubt[i]);
      if (lane == 0) {
        exact[sh.doubt[i]] = v;
        sh.doubt_key[i] = order_key(v);
      }
    }
    __syncthreads();
    if ((int)threadIdx.x < doubts) {
      const u64 own = sh.doubt_key[threadIdx.x];
      int larger = 0, as_large = 0;
#pragma unroll 2
      for (int i = 0; i < doubts; ++i) {
        const u64 k = sh.doubt_key[i];
        larger += k > own;
        as_large += k >= own;
      }
      if (larger < left && left <= as_large) {  // one value
        sh.from = own;
        sh.ties = as_large > left;
      }
    }
    __syncthreads();
    from = sh.from;
    ties = sh.ties != 0;
  } else if (left > 0) {
    for (int j = j0; j - lane < j1; j += 32)
      for (uint32_t doubt = __ballot_sync(0xffffffffu, j < j1 && kind(j) == 2); doubt;
           doubt &= doubt - 1) {
        const int b = j - lane + __ffs(doubt) - 1;
        const double v = exact_score<D>(a, x, h, b);
        if (b == j) exact[b] = v;  // read again by this thread only
      }
    bool whole;
    from = nth_largest<u64, T>(
        j0, j1, [&](int j) { return kind(j) == 2 ? order_key(exact[j]) : 0ull; }, left, sh,
        whole);
    ties = !whole;
  }
  // How a block counts: 0 out, 1 taken, 2 equal to the last score taken.
  auto verdict = [&](int j) {
    const int k = kind(j);
    if (k != 2) return k;
    const u64 e = order_key(exact[j]);
    return e == from ? (ties ? 2 : 1) : (e > from ? 1 : 0);
  };
  int above = 0, equal = 0;
  kept = 0;  // the verdicts of the first 16 blocks of this thread
  for (int j = j0, i = 0; j - lane < j1; j += 32, ++i) {
    const int v = j < j1 ? verdict(j) : 0;
    if (i < 16) kept |= (uint32_t)v << (2 * i);
    above += __popc(__ballot_sync(0xffffffffu, v == 1));
    equal += __popc(__ballot_sync(0xffffffffu, v == 2));
  }
  if (lane == 0) {
    sh.above[warp] = above;
    sh.equal[warp] = equal;
  }
  __syncthreads();
  int eq = 0, all_above = 0;  // before this warp's run
  at = 0;
#pragma unroll
  for (int w = 0; w < T / 32; ++w) {
    all_above += sh.above[w];
    if (w < warp) {
      at += sh.above[w];
      eq += sh.equal[w];
    }
  }
  const int room = a.top_k - all_above;  // equals that are taken
  at += eq < room ? eq : room;
  for (int j = j0, i = 0; j - lane < j1; j += 32, ++i) {
    const int v = i < 16 ? (kept >> (2 * i)) & 3 : (j < j1 ? verdict(j) : 0);
    const uint32_t same = __ballot_sync(0xffffffffu, v == 2);
    const bool take = v == 1 || (v == 2 && eq + __popc(same & below) < room);
    const uint32_t taken = __ballot_sync(0xffffffffu, take);
    const int to = at + __popc(taken & below);
    if (take && to < a.top_k) out[to] = j;
    at += __popc(taken);
    eq += __popc(same);
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

template <int D, int HEADS>
static nk_status launch_scores_heads(const SelectArgs &a, dim3 grid, cudaStream_t s) {
  static std::atomic<uint64_t> prepared{0};  // a bit per device
  nk_status st = allow_smem(reinterpret_cast<const void *>(block_scores_kernel<D, HEADS>),
                            227 * 1024, prepared);
  if (st != NK_OK) return st;
  const int64_t wide = ceil_div(a.group, HEADS) * HEADS;
  const size_t bytes = ScoreShared<D>::bytes(wide, HEADS);
  return launch_early(block_scores_kernel<D, HEADS>, grid, dim3(32 * kScoreWarps), bytes, 1, s, a);
}

// Heads of a pass: as many as a list has, up to 16.
template <int D>
static nk_status launch_scores(const SelectArgs &a, dim3 grid, cudaStream_t s) {
  return a.group <= 2   ? launch_scores_heads<D, 2>(a, grid, s)
         : a.group <= 4 ? launch_scores_heads<D, 4>(a, grid, s)
         : a.group <= 8 ? launch_scores_heads<D, 8>(a, grid, s)
                        : launch_scores_heads<D, 16>(a, grid, s);
}

static size_t select_bytes(const nk_kv_pages *kv, const nk_kv_batch *b) {
  return (size_t)b->tokens * kv->kv_heads * score_width(kv, b) * (sizeof(float2) + sizeof(double));
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
  *bytes = select_bytes(kv, batch);
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
  if (group > 64) return fail(NK_UNSUPPORTED, "q_heads / kv_heads must be <= 64");
  if (ld_q < q_heads * kv->head_dim || ld_q % 8)
    return fail(NK_INVALID_PARAMS, "ld_q must be a multiple of 8 and >= q_heads * head_dim");
  if (sink < 0 || local < 1 || top_k < sink + local || top_k > (1 << 20))
    return fail(NK_INVALID_PARAMS, "sink >= 0, local >= 1, sink + local <= top_k <= 2^20");
  if (batch->seqs == 0 || batch->tokens == 0 || batch->max_new == 0) return ok();
  if (!q || !blocks) return fail(NK_INVALID_PARAMS, "q and blocks are required");
  if ((uintptr_t)q & 15) return fail(NK_INVALID_PARAMS, "q must be 16-byte aligned");
  const int64_t width = score_width(kv, batch);
  const size_t need = select_bytes(kv, batch);
  if (workspace_bytes < need || !workspace) {
    st = fail(NK_WORKSPACE_TOO_SMALL, "block selection workspace too small");
    tls_error().expected = need;
    tls_error().actual = workspace_bytes;
    return st;
  }
  if ((uintptr_t)workspace & 15)
    return fail(NK_INVALID_PARAMS, "workspace must be 16-byte aligned");
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
  a.exact = static_cast<double *>(workspace);
  a.range = reinterpret_cast<float2 *>(a.exact + batch->tokens * kv->kv_heads * width);
  a.blocks = blocks;
  a.err = device_error_ptr();
  if (!a.err) return fail(NK_DEVICE_ERROR, "cannot resolve device error word");
  cudaStream_t s = as_stream(stream);
  if (width > top_k) {
    const dim3 grid((unsigned)ceil_div(width, kScoreBlocks), (unsigned)kv->kv_heads,
                    (unsigned)batch->tokens);
    st = kv->head_dim == 128 ? launch_scores<128>(a, grid, s) : launch_scores<64>(a, grid, s);
    if (st != NK_OK) return st;
  }
  const bool small = width <= 1024;
  const dim3 grid((unsigned)kv->kv_heads, (unsigned)batch->tokens), block(small ? 128 : 512);
  if (kv->head_dim == 128)
    st = launch_early(small ? block_topk_kernel<128, 128> : block_topk_kernel<128, 512>, grid,
                      block, 0, 1, s, a);
  else
    st = launch_early(small ? block_topk_kernel<64, 128> : block_topk_kernel<64, 512>, grid, block,
                      0, 1, s, a);
  if (st != NK_OK) return st;
  return ok();
}

}  // extern "C"
