// attention_paged.cu — attention of new tokens over the pages of their
// sequences: single tokens, prefill chunks, trees of drafted tokens, and
// lists of chosen blocks.
//
// The rows of one KV head are the new tokens times the query heads that share
// it (r = token * G + g), so one read of K and V serves them all.  A block
// takes a tile of those rows and a range of keys (split) of one sequence, and
// runs the softmax in one pass: with m the running row maximum, l the running
// sum and O the running output,
//   m' = max(m, max_j s_j),  c = exp(m - m'),  p_j = exp(s_j - m'),
//   l' = c l + sum_j p_j,    O' = c O + sum_j p_j v_j,
// out = O / l at the end.  Ranges are joined by the same rule.  Statistics and
// sums are f32; p is rounded to bf16 (relative error 2^-8 at most) for the
// value product, as the operand type of the tensor cores asks, while l sums the
// unrounded p.
//
// Tiles of 128 keys come by TMA (boxes of 64 channels x the keys of one page)
// into a ring of shared-memory stages, in the 128-byte swizzle that ldmatrix
// reads without bank conflicts.
#include <cudaTypedefs.h>

#include <atomic>

#include "gemm_tc.h"
#include "paged.cuh"

namespace nk {

constexpr int kTile = 128;  // keys of a stage

struct PagedAttn {
  PagePool pool;
  PageBatch batch;
  const uint16_t *q, *v;  // v: the value pool, for poison()
  int64_t ld_q;
  int q_heads, group;
  int64_t layer_row;  // first token row of the layer in the pools
  const uint64_t *mask;
  const int32_t *blocks;
  int max_blocks;
  float scale_log2;  // scale * log2(e): exp(scale * s) = 2^(scale_log2 * s)
  void *out;
  int out_f32;
  float *part_o;          // [2 * blocks][row tile][head_dim], unnormalised
  float2 *part_ml;        // [2 * blocks][row tile]: m (in log2 units), l
  struct MergeJob *jobs;  // [blocks]
  int cluster, units_most;  // clusters of blocks share a unit (see below): their
                            // size, and the units a sequence has at most
  int *err;
};

// ---------------------------------------------------------------- fragments
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two f32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(*reinterpret_cast<unsigned long long *>(&d))
      : "l"(*reinterpret_cast<const unsigned long long *>(&a)),
        "l"(*reinterpret_cast<const unsigned long long *>(&b)),
        "l"(*reinterpret_cast<const unsigned long long *>(&c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(*reinterpret_cast<unsigned long long *>(&d))
      : "l"(*reinterpret_cast<const unsigned long long *>(&a)),
        "l"(*reinterpret_cast<const unsigned long long *>(&b)));
  return d;
}
__device__ __forceinline__ float ld_cluster(uint32_t cluster_addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t *>(&v);
}

// Byte offset of (row, column) in a matrix of ROWS rows of bf16 held as strips
// of 64 columns: 128-byte rows, 16-byte chunks XORed with the row (TMA's
// 128-byte swizzle, which ldmatrix reads without bank conflicts).
template <int ROWS>
__device__ __forceinline__ uint32_t strip_offset(int row, int col) {
  return (uint32_t)((col >> 6) * (ROWS * 128) + row * 128 + (((col & 63) * 2) ^ ((row & 7) * 16)));
}

// --------------------------------------------------------------- scheduling
// A unit is one row tile of one KV head of one sequence; it costs a tile per
// 128 keys.  Blocks are persistent and share the tiles of all units evenly:
// block c takes tiles c*per .. (c+1)*per-1 of the list (sequence, unit, key
// tile), so ragged lengths leave no block idle and the loader streams across
// unit borders.  The first and the last unit of a block may be parts; parts go
// to slots of the workspace (2c for the block's first piece, 2c+1 for a later
// one) and the block in which a split unit begins describes it to the merge.
struct Piece {
  SeqView seq;
  int head;        // KV head
  int row0, rows;  // rows row0 .. row0+rows-1 of the sequence's count * group
  int prefix;      // cached tokens before the new ones
  int keys;        // keys of the unit: positions (dense), list slots * page size
  int pos;         // block lists: the token's position
  const int32_t *list;
  int t0, t1;      // key tiles of this piece
  bool first, last;  // it holds the unit's first / last tile
  int unit_at;       // list index of the unit's first tile
};

struct MergeJob {
  int slot0, parts;  // parts: blocks that the unit is split over, 0: none begins here
  int first_token, row0, rows, head;
  int pad[2];
};

// Units of a sequence and tiles of each; 0 units when the arrays contradict.
template <int R>
__device__ __forceinline__ void seq_units(const PagedAttn &a, int b, SeqView &seq, int &units,
                                          int &tiles, bool report_it) {
  units = tiles = 0;
  if (!load_seq(a.pool, a.batch, b, seq, a.err, report_it) || seq.count == 0) return;
  if (a.blocks) {
    units = a.pool.heads * seq.count * ((a.group + R - 1) / R);
    const int held = (seq.len + a.pool.ps - 1) >> a.pool.ps_log2;
    const int nb = held < a.max_blocks ? held : a.max_blocks;
    tiles = ((nb << a.pool.ps_log2) + kTile - 1) / kTile;
  } else {
    units = a.pool.heads * ((seq.count * a.group + R - 1) / R);
    tiles = (seq.len + kTile - 1) / kTile;
  }
}

template <int R>
struct Cursor {
  int b, unit, units, tiles, t;
  int left, at;  // tiles left to the block; list index of the next tile
  int parts;     // blocks a unit is split over when it is known beforehand, else 0
  SeqView seq;

  // The next piece; false at the end of the block's share.  Every lane of a
  // warp takes the same steps.
  __device__ __forceinline__ bool next(const PagedAttn &a, Piece &p) {
    if (left <= 0) return false;
    while (unit >= units) {
      if (++b >= a.batch.seqs) return false;
      seq_units<R>(a, b, seq, units, tiles, false);
      unit = 0;
      t = 0;
    }
    const int n = tiles - t < left ? tiles - t : left;
    p.seq = seq;
    p.prefix = seq.len - seq.count;
    p.t0 = t;
    p.t1 = t + n;
    p.first = t == 0;
    p.last = t + n == tiles;
    p.unit_at = at - t;
    // Head-major: the row tiles that read the same keys run side by side.
    int tile = 0;
    p.head = unit;
    if (units != a.pool.heads) {
      const int per_head = units / a.pool.heads;
      p.head = unit / per_head;
      tile = unit - p.head * per_head;
    }
    if (a.blocks) {
      const int gt = (a.group + R - 1) / R;
      const int token = tile / gt, g0 = (tile % gt) * R;
      p.row0 = token * a.group + g0;
      p.rows = a.group - g0 < R ? a.group - g0 : R;
      p.pos = p.prefix + token;
      p.list = a.blocks + ((int64_t)(seq.first + token) * a.pool.heads + p.head) * a.max_blocks;
      // Entries behind the last block hold -1: no tiles for them.  The unit's
      // tiles count an entry a block of the sequence; blocks that skipped entries
      // push behind those belong to its last piece.
      const int e0 = (int)(((int64_t)p.t0 * kTile) >> a.pool.ps_log2);
      int64_t e1 = ((int64_t)p.t1 * kTile + a.pool.ps - 1) >> a.pool.ps_log2;
      if (p.last || e1 > a.max_blocks) e1 = a.max_blocks;
      int n_list = 0;
      for (int e = e0; e < e1; e += 32) {
        const int x = e + (int)(threadIdx.x & 31);
        const uint32_t hit = __ballot_sync(0xffffffffu, x < e1 && p.list[x] >= 0);
        if (hit) n_list = e + 32 - __clz(hit);
      }
      p.keys = n_list << a.pool.ps_log2;
    } else {
      const int total = seq.count * a.group;
      p.row0 = tile * R;
      p.rows = total - p.row0 < R ? total - p.row0 : R;
      p.pos = 0;
      p.list = nullptr;
      p.keys = seq.len;
      if (!a.mask) {  // causal: up to the row tile's last token
        const int lim = p.prefix + (p.row0 + p.rows - 1) / a.group + 1;
        if (lim < p.keys) p.keys = lim;
      }
    }
    const int have = (p.keys + kTile - 1) / kTile;
    if (p.t1 > have || (p.list && p.last)) p.t1 = have > p.t0 ? have : p.t0;
    left -= n;
    at += n;
    t += n;
    if (t == tiles) {
      t = 0;
      ++unit;
    }
    return true;
  }
};

// The block's share of the tile list, in `share`.  Called by all THREADS
// threads; ends with a barrier.  The host has checked that the list is shorter
// than 2^31.
template <int R, int THREADS>
__device__ __forceinline__ void find_share(const PagedAttn &a, Cursor<R> &share, int *sh_per) {
  __shared__ int warp_total[THREADS / 32];
  const int n = a.batch.seqs;
  const int chunk = n <= THREADS ? 1 : (n + THREADS - 1) / THREADS;
  const int b0 = threadIdx.x * chunk, b1 = b0 + chunk < n ? b0 + chunk : n;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int sum = 0;
  Cursor<R> c;
  c.units = c.tiles = 0;
  for (int b = b0; b < b1; ++b) {
    seq_units<R>(a, b, c.seq, c.units, c.tiles, blockIdx.x == 0);
    sum += c.units * c.tiles;
  }
  int scan = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += v;
  }
  if (lane == 31) warp_total[warp] = scan;
  if (threadIdx.x == 0) share.left = 0;
  __syncthreads();
  int total = 0, before = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += warp_total[w];
    total += warp_total[w];
  }
  before += scan - sum;
  const int per = (int)(((unsigned)total + gridDim.x - 1) / gridDim.x);
  const unsigned begin = (unsigned)per * blockIdx.x;
  if (begin >= (unsigned)before && begin < (unsigned)before + sum) {
    // One thread's sequences hold it.
    int at = before, b = b0;
    if (chunk > 1)
      for (; b < b1; ++b) {
        seq_units<R>(a, b, c.seq, c.units, c.tiles, false);
        const int w = c.units * c.tiles;
        if ((int)begin < at + w) break;
        at += w;
      }
    c.b = b;
    c.at = (int)begin;
    c.left = total - (int)begin < per ? total - (int)begin : per;
    const int off = (int)begin - at;
    c.unit = (int)((unsigned)off / (unsigned)c.tiles);
    c.t = off - c.unit * c.tiles;
    c.parts = 0;
    share = c;
    *sh_per = per;
  }
  __syncthreads();
}

// A share of one piece: units split evenly over whole blocks, as many blocks
// each as the shortest share allows that fits the grid.  Wide units (256 rows)
// pay for every piece with a load of their queries and a pass of results
// through memory, which weighs more than a perfect balance.  Falls back to
// find_share when there are more units than blocks.  scratch: 2 * THREADS words
// of shared memory.
template <int R, int THREADS>
__device__ __forceinline__ void find_piece(const PagedAttn &a, Cursor<R> &share, int *sh_per,
                                           int *scratch) {
  __shared__ int warp_total[THREADS / 32], best;
  int *sh_units = scratch, *sh_tiles = scratch + THREADS;
  const int n = a.batch.seqs;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (n > THREADS) {
    find_share<R, THREADS>(a, share, sh_per);
    return;
  }
  Cursor<R> c;
  c.units = c.tiles = 0;
  if ((int)threadIdx.x < n) seq_units<R>(a, threadIdx.x, c.seq, c.units, c.tiles, blockIdx.x == 0);
  sh_units[threadIdx.x] = c.units;
  sh_tiles[threadIdx.x] = c.tiles;
  if (threadIdx.x == 0) {
    best = 0x7fffffff;
    share.left = 0;
  }
  __syncthreads();
  // A warp tries a share length: blocks that it takes.
  int total = 0, longest = 0, units = 0;
  for (int b = lane; b < n; b += 32) {
    total += sh_units[b] * sh_tiles[b];
    units += sh_units[b];
    longest = sh_tiles[b] > longest ? sh_tiles[b] : longest;
  }
  total = __reduce_add_sync(0xffffffffu, total);
  units = __reduce_add_sync(0xffffffffu, units);
  longest = __reduce_max_sync(0xffffffffu, longest);
  if (units > (int)gridDim.x) {  // the same in every warp
    find_share<R, THREADS>(a, share, sh_per);
    return;
  }
  const int least = (int)(((unsigned)total + gridDim.x - 1) / gridDim.x);
  for (int x = least + warp; x < longest + THREADS / 32; x += THREADS / 32) {
    int blocks = 0;
    for (int b = lane; b < n; b += 32)
      blocks += sh_units[b] * (int)(((unsigned)sh_tiles[b] + x - 1) / (unsigned)x);
    blocks = __reduce_add_sync(0xffffffffu, blocks);
    const bool fits = blocks <= (int)gridDim.x;
    if (fits && lane == 0) atomicMin(&best, x);
    __syncthreads();  // all warps make the same number of rounds
    if (best != 0x7fffffff) break;
    __syncthreads();
  }
  __syncthreads();
  const int len = best;
  int parts = 0, each = 0;
  if (c.tiles > 0) {
    parts = (c.tiles + len - 1) / len;
    each = (c.tiles + parts - 1) / parts;
    parts = (c.tiles + each - 1) / each;
  }
  const int sum = c.units * parts;
  int scan = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += v;
  }
  if (lane == 31) warp_total[warp] = scan;
  __syncthreads();
  int before = scan - sum;
  for (int w = 0; w < warp; ++w) before += warp_total[w];
  const int off = (int)blockIdx.x - before;
  if (off >= 0 && off < sum) {
    c.b = threadIdx.x;
    c.unit = off / parts;
    c.t = (off - c.unit * parts) * each;
    c.left = c.tiles - c.t < each ? c.tiles - c.t : each;
    c.at = 0;
    c.parts = parts;
    share = c;
    *sh_per = each;
  }
  __syncthreads();
}

// Output row of row r of a piece: (token, query head).
__device__ __forceinline__ int64_t out_row(const PagedAttn &a, int first_token, int head, int x) {
  return ((int64_t)first_token + x / a.group) * a.q_heads + head * a.group + x % a.group;
}

__device__ __forceinline__ void store_out(const PagedAttn &a, int64_t at, float x, float y) {
  if (a.out_f32)
    *reinterpret_cast<float2 *>(static_cast<float *>(a.out) + at) = make_float2(x, y);
  else
    *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(a.out) + at) = pack_bf16(x, y);
}

// Up to 32 rows: warp products on the whole block.  8 compute warps work on
// one tile of 128 keys together:
//   scores   warp w takes keys 16w .. 16w+15 for all rows,
//   maximum  a row's maximum over the warps meets in shared memory,
//   weights  each warp writes its 16 columns of P (bf16),
//   values   warp w takes columns w*D/8 .. of the output over all 128 keys,
// so an output lives in one place (D/8 columns a warp: 8 or 4 registers a row
// tile), K, V and P are read from shared memory by whole tiles, and there is
// nothing to join over the warps at the end but l.  A ninth warp loads.  Rings
// of 192 KB an SM cover HBM's latency several times: one block with heads of
// 128 (64 KB a tile, whose chain of three barriers is shorter than its load),
// two with heads of 64, where a tile is half the bytes but the same chain (400
// block lists of 48 pages of 32: one block 46 us, two 37 us).
//
// As a tile list it is bound by HBM: 64 contexts of up to 8192 tokens, 2 heads of
// 128, 328 MB: 60.5 us cold, 5.4 TB/s; of that some 5 us pass before the first
// tile lands (share, page lookup, HBM) and 2 at the end.  Two loader warps, one
// for K and one for V, were no faster (61 us).
template <int D, int MT>
struct Cfg {
  static constexpr int kRows = 16 * MT;
  static constexpr int kBlocks = D == 128 ? 1 : 2;  // of an SM
  static constexpr int kStages = 3;
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kQBytes = kRows * D * 2;
  static constexpr int kPBytes = kRows * kTile * 2;
  static constexpr int kSmem = kStages * kStageBytes + kQBytes + kPBytes + 1024;
  static constexpr int kThreads = 288;
};

// Producer warp of both attention kernels: streams the block's tiles into the
// ring.  Lane = (page of the tile, channel strip, K or V): up to 32 boxes of 64
// channels x one page.  Pages are looked up 32 at a time, a lane each, one
// batch ahead of the loads.  SPLIT: K and V of a tile are stages of their own
// (2i and 2i+1), else they share one.  limits[i % LIMITS] gets the keys of tile
// i that any row may see, by groups of 16.
template <int D, int R, int STAGES, bool SPLIT, int LIMITS>
__device__ __forceinline__ void load_tiles(const PagedAttn &a, Cursor<R> cur,
                                           const CUtensorMap *kmap, const CUtensorMap *vmap,
                                           uint8_t *ring, uint64_t *full, uint64_t *empty,
                                           int (*limits)[8], int *abort_flag,
                                           uint64_t *queries = nullptr) {
  constexpr int kTileBytes = kTile * D * 2;
  const int lane = threadIdx.x & 31;
  const int box_rows = a.pool.ps, npg = kTile >> a.pool.ps_log2;  // pages of a tile
  const int boxes = npg * (D / 64) * 2;
  const int c = lane & (npg - 1), strip = (lane / npg) % (D / 64), is_v = lane / (npg * (D / 64));
  fence_proxy_async_global();  // what the kernel before stored, ahead of the tile loads
  Piece p;
  int i = 0;
  while (cur.next(a, p)) {
    const int last = (p.keys - 1) >> a.pool.ps_log2;  // last block or list entry
    int page_ahead, block_ahead;
    auto lookup = [&](int e) {  // block e + lane of the unit
      e += lane;
      int b = e <= last ? e : -1;
      if (p.list && b >= 0) {
        b = p.list[e];
        if (b > (p.pos >> a.pool.ps_log2) || (e > 0 && b <= p.list[e - 1])) b = -1;
      }
      block_ahead = b;
      page_ahead = b >= 0 ? p.seq.table[b] : -1;
    };
    int base = p.t0 * npg;  // block of lane 0; a tile's blocks lie in one batch
    int page_now = 0, block_now = 0;
    lookup(base);
    base -= 32;
    for (int t = p.t0; t < p.t1; ++t, ++i) {
      const int e = t * npg + c;
      if (t * npg - base >= 32) {  // the same for all lanes
        base += 32;
        page_now = page_ahead;
        block_now = block_ahead;
        if (base + 32 <= last) lookup(base + 32);
      }
      int page = __shfl_sync(0xffffffffu, page_now, (e - base) & 31);
      const int block = __shfl_sync(0xffffffffu, block_now, (e - base) & 31);
      if (block >= 0 && !page_ok(a.pool, page)) {
        report(a.err, NK_PAGE_OUT_OF_RANGE);
        page = -1;
      }
      const bool have = block >= 0 && page >= 0;
      const bool load = have && lane < boxes;
      const int64_t row =
          a.layer_row + (((int64_t)page * a.pool.heads + p.head) << a.pool.ps_log2);
#pragma unroll
      for (int half = 0; half < (SPLIT ? 2 : 1); ++half) {
        const int stage = SPLIT ? 2 * i + half : i, s = stage % STAGES;
        // The ring's first fill would go ahead of the queries in the memory
        // system, and nothing starts without them.  (No second phase of this
        // barrier can begin before the first values are loaded.)
        if (SPLIT && stage == 1 &&
            !__all_sync(0xffffffffu, mbar_wait(queries, 0, abort_flag)))
          return;
        const bool room = stage < STAGES ||
                          mbar_wait(&empty[s], ((stage / STAGES) - 1) & 1, abort_flag);
        if (!__all_sync(0xffffffffu, room)) return;  // the lanes leave together
        if (half == 0 && lane < npg) {
          // Keys of the box that the rows may see: up to the last position.
          int n = 0;
          if (have) {
            n = p.list ? p.pos + 1 - (block << a.pool.ps_log2) : p.keys - (e << a.pool.ps_log2);
            n = n < 0 ? 0 : (n > box_rows ? box_rows : n);
          }
          for (int g = 0; g < box_rows / 16; ++g)
            limits[i % LIMITS][c * (box_rows / 16) + g] =
                n - 16 * g < 0 ? 0 : (n - 16 * g > 16 ? 16 : n - 16 * g);
        }
        const bool now = load && (!SPLIT || is_v == half);
        const uint32_t mine = __ballot_sync(0xffffffffu, now);
        __syncwarp();  // the limits of all lanes, ahead of the arrival that shows them
        if (lane == 0)
          mbar_arrive_expect_tx(&full[s], (uint32_t)__popc(mine) * (uint32_t)box_rows * 128u);
        __syncwarp();
        if (now) {
          uint8_t *dst = ring + s * (SPLIT ? 1 : 2) * kTileBytes +
                         (SPLIT ? 0 : is_v * kTileBytes) + strip * (kTile * 128) +
                         c * box_rows * 128;
          tma_load_2d(dst, is_v ? vmap : kmap, &full[s], strip * 64, (int)row);
        }
      }
    }
  }
}

// After an abort: the copies in flight land (or 1 ms passes) before the
// block's memory is given up.
__device__ __forceinline__ void drain_ring(uint64_t *full, int stages) {
  for (int s = 0; s < stages; ++s)
    for (int ph = 0; ph < 2; ++ph) {
      const uint64_t start = nk_globaltimer();
      while (!mbar_try_wait(&full[s], ph) && nk_globaltimer() - start < 1000000ull) {
      }
    }
}

// Positions from here on are not seen by every row of the piece.
__device__ __forceinline__ int seen_by_all(const PagedAttn &a, const Piece &p) {
  return p.list ? 0x7fffffff : (a.mask ? p.prefix : p.prefix + p.row0 / a.group + 1);
}
// Whether the new token `tok` sees position pos < keys of its sequence.
__device__ __forceinline__ bool sees(const PagedAttn &a, const Piece &p, int tok, int pos) {
  if (!a.mask) return pos <= p.prefix + tok;
  return pos < p.prefix ||
         (tok < p.seq.count && ((a.mask[p.seq.first + tok] >> (pos - p.prefix)) & 1) != 0);
}

// A weight of 0 must leave no trace, and 0 * inf is NaN.  One of PARTS threads
// of a key's row in the value tile: what lies behind the last key becomes 0, and
// of the keys from `shared` on, which only some rows see, the infinities and
// NaN become 0.  True when it found one: the piece's end puts them back for the
// rows that see them (poison).  The weights are signalled behind this, so the
// product reads the tile as it is then.
template <int D>
__device__ __forceinline__ bool clean_values(uint8_t *vt, int key, int part, int parts,
                                             const int *limits, int shared) {
  const bool dead = (key & 15) >= limits[key >> 4];
  if (!dead && key < shared) return false;
  bool found = false;
#pragma unroll 1
  for (int c = part * 8; c < D; c += parts * 8) {
    uint4 *x = reinterpret_cast<uint4 *>(vt + strip_offset<kTile>(key, c));
    if (dead) {
      *x = make_uint4(0, 0, 0, 0);
      continue;
    }
    const uint4 y = *x;
    uint32_t word[4] = {y.x, y.y, y.z, y.w};
    bool hit = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if ((word[j] & 0x7f80u) == 0x7f80u) {
        word[j] &= 0xffff0000u;
        hit = true;
      }
      if ((word[j] & 0x7f800000u) == 0x7f800000u) {
        word[j] &= 0x0000ffffu;
        hit = true;
      }
    }
    if (hit) *x = make_uint4(word[0], word[1], word[2], word[3]);
    found |= hit;
  }
  fence_proxy_async_smem();  // before the stage is loaded again, or read by an MMA
  return found;
}

// What a row's output channel gains from infinities and NaN that clean_values
// took out: their sum over the keys of the piece that the row sees.
__device__ __noinline__ float poison(const PagedAttn &a, const Piece &p, const uint16_t *v,
                                     int head_dim, int tok, int chan) {
  float sum = 0.0f;
  int from = seen_by_all(a, p);
  if (from < p.t0 * kTile) from = p.t0 * kTile;
  const int to = p.keys < p.t1 * kTile ? p.keys : p.t1 * kTile;
  for (int pos = from; pos < to; ++pos) {
    if (!sees(a, p, tok, pos)) continue;
    const int page = p.seq.table[pos >> a.pool.ps_log2];
    if (!page_ok(a.pool, page)) continue;
    const int64_t row = a.layer_row +
                        (((int64_t)page * a.pool.heads + p.head) << a.pool.ps_log2) +
                        (pos & (a.pool.ps - 1));
    const float x = __uint_as_float((uint32_t)v[row * head_dim + chan] << 16);
    if (!(fabsf(x) < INFINITY)) sum += x;
  }
  return sum;
}

// Barrier of the 256 compute threads that also ORs a flag.
__device__ __forceinline__ bool compute_vote(bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 256, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)x)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void compute_sync() {
  asm volatile("bar.sync 1, 256;" ::: "memory");
}

// CLUSTER: few units of few tiles (a short context, a small batch) run without a
// list, a workspace and a merge launch: a cluster of blocks takes a unit, a
// block each an even run of its tiles, and the blocks join through distributed
// shared memory.  Bound by the chain launch, lengths, page, tile, softmax, join:
// one sequence of 1025 tokens 7.9 us in a chain of calls (as a list with a
// merge 8.8, and 4 us more on the host).
template <int D, int MT, bool CLUSTER>
__global__ void __launch_bounds__(288, Cfg<D, MT>::kBlocks)
    paged_attn_kernel(const __grid_constant__ CUtensorMap kmap,
                      const __grid_constant__ CUtensorMap vmap,
                      const __grid_constant__ PagedAttn a) {
  using C = Cfg<D, MT>;
  constexpr int R = C::kRows, STAGES = C::kStages;
  constexpr int COLS = D / 8, ON = COLS / 8;  // output columns of a warp
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~uintptr_t(1023));
  uint8_t *qs = smem + STAGES * C::kStageBytes;
  uint8_t *ps = qs + C::kQBytes;
  __shared__ uint64_t full[STAGES], empty[STAGES];
  __shared__ __align__(16) int limits[STAGES][8];  // seen keys of each 16-key group
  __shared__ __align__(16) float red[R][8];        // a value per row and warp
  __shared__ int odd;  // a value that only some rows see is no finite number
  __shared__ int abort_flag;
  __shared__ Cursor<R> share;
  __shared__ int per;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  let_next_launch();
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 8);
    }
    fence_mbar_init();
    abort_flag = 0;
  }
  if (threadIdx.x == 256) {
    tma_prefetch_desc(&kmap);
    tma_prefetch_desc(&vmap);
  }
  wait_for_previous();
  if (threadIdx.x == 0 && a.jobs) a.jobs[blockIdx.x].parts = 0;
  Cursor<R> cur;
  if (CLUSTER) {
    cur.b = blockIdx.x / (a.cluster * a.units_most);
    cur.unit = blockIdx.x / a.cluster - cur.b * a.units_most;
    seq_units<R>(a, cur.b, cur.seq, cur.units, cur.tiles,
                 cur.unit == 0 && blockIdx.x % a.cluster == 0 && threadIdx.x == 0);
    if (cur.unit >= cur.units) return;  // the whole cluster
    const int each = (cur.tiles + a.cluster - 1) / a.cluster;
    cur.t = (int)(blockIdx.x % a.cluster) * each;
    cur.left = cur.tiles - cur.t < each ? cur.tiles - cur.t : each;
    cur.at = cur.parts = 0;
    __syncthreads();
  } else {
    find_share<R, C::kThreads>(a, share, &per);
    if (share.left <= 0) return;
    cur = share;
  }
  const Cursor<R> start = cur;
  // CLUSTER: this block's part, over the ring once its tiles are used.
  float *part_o = reinterpret_cast<float *>(smem);
  float2 *part_ml = reinterpret_cast<float2 *>(smem + R * D * 4);

  if (warp == 8) {
    load_tiles<D, R, STAGES, false, STAGES>(a, cur, &kmap, &vmap, smem, full, empty, limits,
                                            &abort_flag);
    if (*(volatile int *)&abort_flag) drain_ring(full, STAGES);
  } else {
    const int quad = lane >> 2, qc = (lane & 3) * 2;
    Piece p;
    int i = 0;      // tiles so far
    int piece = 0;  // pieces so far
    bool live = true;
    while (live && cur.next(a, p)) {
      // Queries to shared memory, 16 bytes a thread; rows of no token are 0.
      // (The last reads of the old ones lie before the last tile's barriers.)
      for (int x = threadIdx.x; x < R * D / 8; x += 256) {
        const int r = x / (D / 8), c = (x % (D / 8)) * 8;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < p.rows) {
          const int y = p.row0 + r, tok = y / a.group;
          v = *reinterpret_cast<const uint4 *>(
              a.q + ((int64_t)p.seq.first + tok) * a.ld_q +
              ((int64_t)p.head * a.group + (y - tok * a.group)) * D + c);
        }
        *reinterpret_cast<uint4 *>(qs + strip_offset<R>(r, c)) = v;
      }
      // Rows of this lane: quad and quad + 8 of each row tile.
      int tok_row[MT][2];
      float m[MT][2], l[MT][2], o[MT][ON][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          tok_row[mt][hh] = (p.row0 + mt * 16 + quad + hh * 8) / a.group;
          m[mt][hh] = -INFINITY;
          l[mt][hh] = 0.0f;
        }
#pragma unroll
        for (int n = 0; n < ON; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[mt][n][j] = 0.0f;
      }
      const int all_see = seen_by_all(a, p);
      if (threadIdx.x == 0) odd = 0;
      compute_sync();  // the queries are there

      for (int t = p.t0; t < p.t1; ++t, ++i) {
        const int s = i % STAGES;
        const bool got = mbar_wait(&full[s], (i / STAGES) & 1, &abort_flag);
        if (compute_vote(!got)) {  // all warps leave together
          live = false;
          break;
        }
        uint8_t *kt = smem + s * C::kStageBytes, *vt = kt + C::kTileBytes;
        const int4 la = *reinterpret_cast<const int4 *>(&limits[s][0]);
        const int4 lb = *reinterpret_cast<const int4 *>(&limits[s][4]);
        const bool tail = la.x + la.y + la.z + la.w + lb.x + lb.y + lb.z + lb.w < kTile;
        const bool partial = !p.list && (t + 1) * kTile > all_see;
        if (tail || partial) {
          if (clean_values<D>(vt, threadIdx.x >> 1, threadIdx.x & 1, 2, limits[s],
                              partial ? all_see - t * kTile : kTile))
            odd = 1;
        }

        // Scores of the warp's 16 keys.
        float sc[MT][2][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) sc[mt][n][j] = 0.0f;
        const uint32_t kb = smem_u32(kt), vb = smem_u32(vt), qb = smem_u32(qs),
                       pb = smem_u32(ps);
        const int mtx = lane >> 3;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          uint32_t b[4];
          ldsm4(b, kb + strip_offset<kTile>(warp * 16 + (mtx >> 1) * 8 + (lane & 7),
                                            k * 16 + (mtx & 1) * 8));
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            uint32_t q4[4];
            ldsm4(q4, qb + strip_offset<R>(mt * 16 + (mtx & 1) * 8 + (lane & 7),
                                           k * 16 + (mtx >> 1) * 8));
            mma16816(sc[mt][0], q4, b[0], b[1]);
            mma16816(sc[mt][1], q4, b[2], b[3]);
          }
        }
        if (tail || partial) {
          const int lim = limits[s][warp];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int key = n * 8 + qc + (j & 1);
                bool ok = key < lim;
                if (ok && partial)
                  ok = sees(a, p, tok_row[mt][j >> 1], t * kTile + warp * 16 + key);
                if (!ok) sc[mt][n][j] = -INFINITY;
              }
        }
        // A row's maximum over the warp's keys, then over the warps.
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            float mx = fmaxf(fmaxf(sc[mt][0][2 * hh], sc[mt][0][2 * hh + 1]),
                             fmaxf(sc[mt][1][2 * hh], sc[mt][1][2 * hh + 1]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            if ((lane & 3) == 0) red[mt * 16 + quad + hh * 8][warp] = mx;
          }
        compute_sync();
        float mu[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            const float4 *x = reinterpret_cast<const float4 *>(red[mt * 16 + quad + hh * 8]);
            const float4 x0 = x[0], x1 = x[1];
            const float mx = fmaxf(fmaxf(fmaxf(x0.x, x0.y), fmaxf(x0.z, x0.w)),
                                   fmaxf(fmaxf(x1.x, x1.y), fmaxf(x1.z, x1.w)));
            const float mn = fmaxf(m[mt][hh], mx * a.scale_log2);
            // No key so far: any finite shift will do, and keeps -inf - -inf out.
            mu[mt][hh] = mn == -INFINITY ? 0.0f : mn;
            const float corr = exp2_approx(m[mt][hh] - mu[mt][hh]);
            m[mt][hh] = mn;
            float sum = 0.0f;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              const float w0 = exp2_approx(sc[mt][n][2 * hh] * a.scale_log2 - mu[mt][hh]);
              const float w1 = exp2_approx(sc[mt][n][2 * hh + 1] * a.scale_log2 - mu[mt][hh]);
              sum += w0 + w1;
              *reinterpret_cast<uint32_t *>(
                  ps + strip_offset<R>(mt * 16 + quad + hh * 8, warp * 16 + n * 8 + qc)) =
                  pack_bf16(w0, w1);
            }
            l[mt][hh] = l[mt][hh] * corr + sum;
#pragma unroll
            for (int n = 0; n < ON; ++n) {
              o[mt][n][2 * hh] *= corr;
              o[mt][n][2 * hh + 1] *= corr;
            }
          }
        compute_sync();  // the weights are there

        // O += P V for the warp's columns.
        if (ON == 2) {
#pragma unroll
          for (int k = 0; k < kTile / 16; ++k) {
            uint32_t b[4];
            ldsm4_t(b, vb + strip_offset<kTile>(k * 16 + (mtx & 1) * 8 + (lane & 7),
                                                warp * COLS + (mtx >> 1) * 8));
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              uint32_t p4[4];
              ldsm4(p4, pb + strip_offset<R>(mt * 16 + (mtx & 1) * 8 + (lane & 7),
                                             k * 16 + (mtx >> 1) * 8));
              mma16816(o[mt][0], p4, b[0], b[1]);
              mma16816(o[mt][ON - 1], p4, b[2], b[3]);
            }
          }
        } else {
#pragma unroll
          for (int k = 0; k < kTile / 16; k += 2) {
            uint32_t b[4];  // 32 keys x 8 columns
            ldsm4_t(b, vb + strip_offset<kTile>(k * 16 + mtx * 8 + (lane & 7), warp * COLS));
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                uint32_t p4[4];
                ldsm4(p4, pb + strip_offset<R>(mt * 16 + (mtx & 1) * 8 + (lane & 7),
                                               (k + u) * 16 + (mtx >> 1) * 8));
                mma16816(o[mt][0], p4, b[2 * u], b[2 * u + 1]);
              }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
      }
      if (!live) break;

      // l over the quad's lanes, then over the warps, in their order.
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          float x = l[mt][hh];
          x += __shfl_xor_sync(0xffffffffu, x, 1);
          x += __shfl_xor_sync(0xffffffffu, x, 2);
          if ((lane & 3) == 0) red[mt * 16 + quad + hh * 8][warp] = x;
        }
      compute_sync();
      const int slot = 2 * (int)blockIdx.x + (piece > 0);
      const bool whole = p.first && p.last;
      if (odd) {  // rare
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int hh = 0; hh < 2; ++hh)
#pragma unroll
            for (int n = 0; n < ON; ++n)
#pragma unroll
              for (int j = 0; j < 2; ++j)
                o[mt][n][2 * hh + j] += poison(a, p, a.v, D, tok_row[mt][hh],
                                               warp * COLS + n * 8 + qc + j);
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int r = mt * 16 + quad + hh * 8;
          if (r >= p.rows) continue;
          float sum = 0.0f;
#pragma unroll
          for (int w = 0; w < 8; ++w) sum += red[r][w];
          if (CLUSTER) {
            if (warp == 0 && (lane & 3) == 0) part_ml[r] = make_float2(m[mt][hh], sum);
#pragma unroll
            for (int n = 0; n < ON; ++n)
              *reinterpret_cast<float2 *>(part_o + r * D + warp * COLS + n * 8 + qc) =
                  make_float2(o[mt][n][2 * hh], o[mt][n][2 * hh + 1]);
          } else if (whole) {
            const int64_t at =
                out_row(a, p.seq.first, p.head, p.row0 + r) * D + warp * COLS + qc;
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
            for (int n = 0; n < ON; ++n)
              store_out(a, at + n * 8, o[mt][n][2 * hh] * inv, o[mt][n][2 * hh + 1] * inv);
          } else {
            const int64_t at = (int64_t)slot * R + r;
            if (warp == 0 && (lane & 3) == 0) a.part_ml[at] = make_float2(m[mt][hh], sum);
#pragma unroll
            for (int n = 0; n < ON; ++n)
              *reinterpret_cast<float2 *>(a.part_o + at * D + warp * COLS + n * 8 + qc) =
                  make_float2(o[mt][n][2 * hh], o[mt][n][2 * hh + 1]);
          }
        }
      if (!CLUSTER && threadIdx.x == 0 && p.first && !p.last) {
        MergeJob j{};
        j.slot0 = slot;
        j.parts = (p.unit_at + cur.tiles - 1) / per - (int)blockIdx.x + 1;
        j.first_token = p.seq.first;
        j.row0 = p.row0;
        j.rows = p.rows;
        j.head = p.head;
        a.jobs[blockIdx.x] = j;
      }
      ++piece;
      compute_sync();  // red and odd are read before the next piece writes them
    }
    if (CLUSTER && start.left <= 0 && threadIdx.x < R)
      part_ml[threadIdx.x] = make_float2(-INFINITY, 0.0f);
  }
  if (CLUSTER) {
    // Rows rank, rank + cluster, .. are joined here, a column a thread, from the
    // parts of all blocks in their order.
    Cursor<R> any = start;  // the unit's rows, whatever this block's tiles
    any.t = 0;
    any.left = 1;
    Piece p;
    any.next(a, p);
    const int rank = (int)(blockIdx.x % a.cluster);
    cluster_sync();
    if (threadIdx.x < 256 && !abort_flag) {
      const uint32_t mine_o = smem_u32(part_o), mine_ml = smem_u32(part_ml);
      const int col = threadIdx.x % D;
      for (int r = rank + a.cluster * (int)(threadIdx.x / D); r < p.rows;
           r += a.cluster * (256 / D)) {
        float mx = -INFINITY, sum = 0.0f, x = 0.0f;
        for (int k = 0; k < a.cluster; ++k)
          mx = fmaxf(mx, ld_cluster(mapa_cta(mine_ml + r * 8, k)));
        const float mu = mx == -INFINITY ? 0.0f : mx;
#pragma unroll 4
        for (int k = 0; k < a.cluster; ++k) {
          const uint32_t ml = mapa_cta(mine_ml + r * 8, k);
          const float lk = ld_cluster(ml + 4), c = exp2_approx(ld_cluster(ml) - mu);
          const float ok = ld_cluster(mapa_cta(mine_o + (r * D + col) * 4, k));
          if (lk != 0.0f) {  // else the block had no key: nothing is written there
            sum += lk * c;
            x += ok * c;
          }
        }
        x *= sum == 0.0f ? 0.0f : 1.0f / sum;
        const int64_t at = out_row(a, p.seq.first, p.head, p.row0 + r) * D + col;
        if (a.out_f32)
          static_cast<float *>(a.out)[at] = x;
        else
          static_cast<__nv_bfloat16 *>(a.out)[at] = __float2bfloat16_rn(x);
      }
    }
    cluster_sync();  // the other blocks have read this one's part
  } else {
    __syncthreads();
  }
  if (abort_flag && threadIdx.x == 0) report(a.err, NK_TIMEOUT);
}

// ------------------------------------------------------- more than 32 rows
// tcgen05 products.  A unit is up to 256 rows: two tiles of 128 (A and B) that
// share every K and V tile of 128 keys.  Per key tile and row tile
//   S = Q K^T  128 x 128 x D, f32 in tensor memory,
//   P          exp2 of the scaled scores, bf16, written over S,
//   O += P V   P from tensor memory, V as it lies (MN-major), f32 in tensor memory.
// Warps 0-3 turn A's scores into weights, a row a thread (its 128 scores stay in
// registers), warps 4-7 B's, warp 8 issues the products, warp 9 loads.  While
// one row tile's weights are computed the tensor cores work for the other.  A
// block's products run in the order of their issue, so the next scores may be
// issued behind the product that reads the weights they go over.
// Bound by the chain of a row tile: 2350 cycles for a tile's weights (1024 of
// them the exponential unit's, shared by both row tiles), 1300 for the value
// product's second half and the next scores: 3650 cycles a key tile, against
// 2 x 1024 tensor cycles.  8 trees of up to 64 drafts over up to 8192 tokens,
// 16 query heads a KV head: 72 us cold, 41 GFLOP; half of the exponentials left out
// (to time the rest) gained 4 us.  Scores in halves of 64 keys with
// buffers of their own were slower (5300 cycles: products of 64 columns cost
// nearly as much to issue and run as those of 128), as was one f32 mma.sync
// kernel for all rows (185 us).
// The running maximum moves only when it grows by more than 2^8 (weights stay
// below 2^8, sums and bf16 lose nothing by that), so O is hardly ever rescaled.
template <int D>
struct TcCfg {
  static constexpr int kRows = 256;
  static constexpr int kStages = 5;  // K and V tiles of their own: K0 V0 K1 V1 ..
  static constexpr int kLimits = 4;  // the loader is at most 3 tiles ahead
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kQBytes = 2 * 128 * D * 2;
  static constexpr int kSmem = kStages * kTileBytes + kQBytes + 1024;
  static constexpr int kThreads = 320;
  static constexpr uint32_t kO = 256;  // tensor memory columns: S/P A, S/P B, O A, O B
};

// All lanes or none: a wait whose outcome the warp shares.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t phase, int *abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, phase, abort_flag));
}

template <int D>
__global__ void __launch_bounds__(320, 1)
    paged_attn_tc_kernel(const __grid_constant__ CUtensorMap kmap,
                         const __grid_constant__ CUtensorMap vmap,
                         const __grid_constant__ PagedAttn a) {
  using C = TcCfg<D>;
  constexpr int R = C::kRows, STAGES = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~uintptr_t(1023));
  uint8_t *qs = ring + STAGES * C::kTileBytes;  // [A, B][strips][128 rows][128 bytes]
  __shared__ uint64_t full[STAGES], empty[STAGES];
  __shared__ uint64_t q_full[2], s_full[2], p_full[2][2], o_full[2], e_done[2], drain;
  __shared__ __align__(16) int limits[C::kLimits][8];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ int odd;  // some piece so far: a value that only some rows see is no finite number
  __shared__ Cursor<R> share;
  __shared__ int per;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  let_next_launch();
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(&q_full[g], 4);
      mbar_init(&s_full[g], 1);
      mbar_init(&p_full[g][0], 4);  // the weights of keys 0-63
      mbar_init(&p_full[g][1], 4);  // and of keys 64-127
      mbar_init(&o_full[g], 1);
      mbar_init(&e_done[g], 4);
    }
    mbar_init(&drain, 1);
    fence_mbar_init();
    abort_flag = 0;
    odd = 0;
  }
  if (threadIdx.x == 288) {
    tma_prefetch_desc(&kmap);
    tma_prefetch_desc(&vmap);
  }
  wait_for_previous();
  if (threadIdx.x == 0 && a.jobs) a.jobs[blockIdx.x].parts = 0;
  if (warp == 8) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  find_piece<R, C::kThreads>(a, share, &per, reinterpret_cast<int *>(qs));
  tc_fence_after();
  if (share.left <= 0) {
    if (warp == 8) tmem_dealloc(tmem_slot, 512);
    return;
  }
  Cursor<R> cur = share;
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);

  if (warp == 9) {
    load_tiles<D, R, STAGES, true, C::kLimits>(a, cur, &kmap, &vmap, ring, full, empty, limits,
                                               &abort_flag, &q_full[0]);
    if (*(volatile int *)&abort_flag) drain_ring(full, STAGES);
  } else if (warp == 8) {
    // --------------------------------------------------------------- products
    const uint32_t idesc_s = idesc_bf16_f32(128, 128);
    const uint32_t idesc_o = idesc_bf16_f32(128, D) | (1u << 16);  // B (the values) MN-major
    int i = 0;           // tiles before this piece
    int pieces[2] = {};  // pieces with rows in A / B
    int tiles[2] = {};   // tiles of A / B so far
    bool live = true;
    Piece p;
    // The whole warp walks through the products (one lane is elected to issue
    // each), so that descriptors stay in uniform registers: under a branch on
    // the lane a product cost 90 to 180 cycles to issue, more than it takes.
    const uint64_t dk = smem_desc_sw128(smem_u32(ring));
    const uint64_t dv = smem_desc_sw128_mn(smem_u32(ring), kTile * 128);
    const uint64_t dq = smem_desc_sw128(smem_u32(qs));
    auto scores = [&](int g, int tile) {
      const uint32_t q = (uint32_t)dq + g * (128 * D * 2 >> 4);
      const uint32_t k = (uint32_t)dk + (2 * tile) % STAGES * (C::kTileBytes >> 4);
#pragma unroll
      for (int x = 0; x < D / 16; ++x) {
        const uint32_t off = ((x >> 2) * (128 * 128) + (x & 3) * 32) >> 4;
        tc_mma_bf16_warp(tmem + g * 128, q + off, (uint32_t)(dq >> 32), k + off,
                         (uint32_t)(dk >> 32), idesc_s, x > 0);
      }
      tc_commit_warp(&s_full[g]);
    };
    auto values = [&](int g, int half, int tile, bool more) {
      const uint32_t v = (uint32_t)dv + (2 * tile + 1) % STAGES * (C::kTileBytes >> 4) +
                         half * (kTile / 2 * 128 >> 4);
      const uint32_t o = tmem + C::kO + g * 128, w = tmem + g * 128 + half * 32;
#pragma unroll
      for (int x = 0; x < kTile / 32; ++x)
        tc_mma_bf16_ta_warp(o, w + x * 8, v + x * (2048 >> 4), (uint32_t)(dv >> 32), idesc_o,
                            (uint32_t)more + x);
    };
    auto loaded = [&](int stage) {
      return warp_wait(&full[stage % STAGES], (stage / STAGES) & 1, &abort_flag);
    };
    while (live && cur.next(a, p)) {
      const int n = p.t1 - p.t0;
      if (n <= 0) continue;
      const int groups = p.rows > 128 ? 2 : 1;
      for (int g = 0; live && g < groups; ++g)
        live = warp_wait(&q_full[g], pieces[g] & 1, &abort_flag);
      live = live && loaded(2 * i);
      if (!live) break;
      tc_fence_after();
      for (int g = 0; g < groups; ++g) scores(g, i);
      tc_commit_warp(&empty[(2 * i) % STAGES]);
      for (int x = 0; live && x < n; ++x) {
        const int tile = i + x;
        const bool again = x + 1 < n;
        for (int g = 0; live && g < groups; ++g) {
          // The weights of this row tile come in halves; its next scores go
          // over them, behind the products that read them.
          live = warp_wait(&p_full[g][0], tiles[g] & 1, &abort_flag) && loaded(2 * tile + 1);
          if (!live) break;
          tc_fence_after();
          values(g, 0, tile, x > 0);
          live = warp_wait(&p_full[g][1], tiles[g] & 1, &abort_flag);
          if (live && again) live = loaded(2 * tile + 2);
          if (!live) break;
          ++tiles[g];
          tc_fence_after();
          values(g, 1, tile, true);
          if (g == groups - 1) tc_commit_warp(&empty[(2 * tile + 1) % STAGES]);
          if (again) scores(g, tile + 1);
          else tc_commit_warp(&o_full[g]);
          if (again && g == groups - 1) tc_commit_warp(&empty[(2 * tile + 2) % STAGES]);
        }
      }
      for (int g = 0; g < groups; ++g) ++pieces[g];
      i += n;
    }
    if (*(volatile int *)&abort_flag) {  // products in flight end before the memory goes
      __syncwarp();
      tc_commit_warp(&drain);
      const uint64_t start = nk_globaltimer();
      while (!mbar_try_wait(&drain, 0) && nk_globaltimer() - start < 10000000ull) {
      }
    }
  } else {
    // ---------------------------------------------------------------- weights
    const int g = warp >> 2;
    const int r = threadIdx.x;  // row of the unit
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + g * 128 + lanes, to = tmem + C::kO + g * 128 + lanes;
    int i = 0, pieces_g = 0, tiles_g = 0, ends_g = 0, piece = 0;
    bool live = true;
    Piece p;
    while (live && cur.next(a, p)) {
      const int n = p.t1 - p.t0;
      const bool mine = g == 0 || p.rows > 128;  // the row tile holds rows
      const bool ok_row = r < p.rows;
      const int tok0 = p.row0 / a.group, tok = (p.row0 + r) / a.group;
      const int all_see = seen_by_all(a, p);
      float m = -INFINITY, l = 0.0f;
      // The warps of a row tile leave the shared memory of its last results
      // together.
      if (mine && ends_g > 0 && !warp_wait(&e_done[g], (ends_g - 1) & 1, &abort_flag)) break;
      if (mine && n > 0) {
        // Queries: neighbouring threads load neighbouring 16 bytes of a row, 8
        // rows' loads in flight.
        uint8_t *qt = qs + g * (128 * D * 2);
        constexpr int RP = 128 / (D / 8);  // rows of a pass over the threads
        const int q0 = (threadIdx.x & 127) / (D / 8), qc = (threadIdx.x % (D / 8)) * 8;
        const int over = p.row0 - tok0 * a.group;  // row0 = tok0 * group + over
        const float inv_group = 1.0f / (float)a.group;
#pragma unroll 1
        for (int x0 = 0; x0 < 128; x0 += 8 * RP) {
          uint4 v[8];
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const int y = g * 128 + x0 + x * RP + q0;  // row of the unit
            v[x] = make_uint4(0, 0, 0, 0);
            if (y < p.rows) {
              // (over + y) / group: the half keeps the product off whole numbers
              const int t = (int)(((float)(over + y) + 0.5f) * inv_group);
              v[x] = *reinterpret_cast<const uint4 *>(
                  a.q + ((int64_t)p.seq.first + tok0 + t) * a.ld_q +
                  ((int64_t)p.head * a.group + (over + y - t * a.group)) * D + qc);
            }
          }
#pragma unroll
          for (int x = 0; x < 8; ++x)
            *reinterpret_cast<uint4 *>(qt + strip_offset<128>(x0 + x * RP + q0, qc)) = v[x];
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[g]);
        const uint64_t tree =
            a.mask && ok_row && tok < p.seq.count ? a.mask[p.seq.first + tok] : 0;

        for (int t = p.t0; t < p.t1; ++t) {
          const int tile = i + t - p.t0;
          live = warp_wait(&s_full[g], tiles_g & 1, &abort_flag);
          if (!live) break;
          ++tiles_g;
          tc_fence_after();
          const int *lim = limits[tile % C::kLimits];
          const int4 la = *reinterpret_cast<const int4 *>(lim);
          const int4 lb = *reinterpret_cast<const int4 *>(lim + 4);
          const bool tail = la.x + la.y + la.z + la.w + lb.x + lb.y + lb.z + lb.w < kTile;
          const bool partial = !p.list && (t + 1) * kTile > all_see;
          if (g == 0 && (tail || partial)) {
            const int stage = 2 * tile + 1;
            live = warp_wait(&full[stage % STAGES], (stage / STAGES) & 1, &abort_flag);
            if (!live) break;
            if (clean_values<D>(ring + stage % STAGES * C::kTileBytes, r, 0, 1, lim,
                                partial ? all_see - t * kTile : kTile))
              odd = 1;
            __syncwarp();
          }
          // Keys of a chunk of 32 that this row sees, a bit each.
          auto seen = [&](int c) -> uint32_t {
            const int l0 = lim[2 * c], l1 = lim[2 * c + 1];
            uint32_t bits = ((1u << l0) - 1) | ((1u << l1) - 1) << 16;
            if (partial) {
              const int k0 = t * kTile + c * 32;
              if (a.mask) {
                // positions below the prefix, then the tree's bits
                const int d = k0 - p.prefix;  // draft of the chunk's first key
                uint32_t see;
                if (d >= 0) see = d < 64 ? (uint32_t)(tree >> d) : 0u;
                else if (d > -32) see = (uint32_t)(tree << -d) | ((1u << -d) - 1);
                else see = 0xffffffffu;
                bits &= see;
              } else {
                const int last = p.prefix + tok - k0;  // last key seen
                bits &= last >= 31 ? 0xffffffffu : (last < 0 ? 0u : (2u << last) - 1);
              }
            }
            return bits;
          };
          const bool masked = tail || partial;
          // The row's 128 scores stay in registers from here to the weights.
          uint32_t sv[128];
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32_issue(ts + c * 32, sv + c * 32);
          tmem_wait_ld();
          if (masked) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const uint32_t bits = seen(c);
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (!((bits >> j) & 1)) sv[c * 32 + j] = 0xff800000u;
            }
          }
          float mx = -INFINITY, mx1 = -INFINITY;
#pragma unroll
          for (int j = 0; j < 128; j += 4) {
            mx = fmaxf(mx, fmaxf(__uint_as_float(sv[j]), __uint_as_float(sv[j + 1])));
            mx1 = fmaxf(mx1, fmaxf(__uint_as_float(sv[j + 2]), __uint_as_float(sv[j + 3])));
          }
          const float mn = fmaxf(mx, mx1) * a.scale_log2;
          // First keys of the row, or a maximum that has outgrown the old one.
          const bool grow = mn > m + 8.0f || (m == -INFINITY && mn > m);
          const float corr = grow ? exp2_approx(m - mn) : 1.0f;  // 0 for the first keys
          if (grow) {
            m = mn;
            l *= corr;
          }
          const bool rescale = t > p.t0 && __any_sync(0xffffffffu, grow);
          const float mu = m == -INFINITY ? 0.0f : m;
          const float2 scale2 = make_float2(a.scale_log2, a.scale_log2);
          const float2 mu2 = make_float2(-mu, -mu);
          float2 sum2 = make_float2(0.0f, 0.0f);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int c = 2 * half; c < 2 * half + 2; ++c) {
              uint32_t w[16];
#pragma unroll
              for (int j = 0; j < 32; j += 2) {
                float2 x = make_float2(__uint_as_float(sv[c * 32 + j]),
                                       __uint_as_float(sv[c * 32 + j + 1]));
                x = fma2(x, scale2, mu2);
                x.x = exp2_approx(x.x);
                x.y = exp2_approx(x.y);
                sum2 = add2(sum2, x);
                w[j / 2] = pack_bf16(x.x, x.y);
              }
              tmem_st16(ts + c * 16, w);  // over scores that have been read
            }
            // O follows the maximum; here the first half's registers are free.
            if (half == 0 && rescale) {
#pragma unroll 1
              for (int c = 0; c < D / 16; ++c) {
                float v[16];
                tmem_ld16(to + c * 16, v);
                uint32_t w[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) w[j] = __float_as_uint(v[j] * corr);
                tmem_st16(to + c * 16, w);
              }
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[g][half]);
          }
          l += sum2.x + sum2.y;
        }
        live = live && warp_wait(&o_full[g], pieces_g & 1, &abort_flag);
        if (!live) break;
        ++pieces_g;
        tc_fence_after();
      }
      const int slot = 2 * (int)blockIdx.x + (piece > 0);
      const bool whole = p.first && p.last;
      if (mine) {
        const float f = whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
        if (!whole && ok_row) a.part_ml[(int64_t)slot * R + r] = make_float2(m, l);
        // One flag, never cleared: A may be any number of pieces ahead of B, which
        // skips pieces without rows of its own.  For a piece that took nothing out
        // poison adds 0.
        const bool bad = n > 0 && odd;
        // Through shared memory (the queries' tile is free): a thread holds a
        // row, a store instruction writes 4 rows of 32 columns.
        float4 *stage = reinterpret_cast<float4 *>(qs + g * (128 * D * 2) + (warp & 3) * 4096);
        const int er = lane >> 3, ec = lane & 7;
        const int first_row = r - lane;
        const int over = p.row0 - tok0 * a.group;
        const float inv_group = 1.0f / (float)a.group;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          float v[32];
          __syncwarp();
          if (n > 0) {
            tmem_ld32(to + c * 32, v);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0.0f;
          }
          if (bad && ok_row) {  // rare
#pragma unroll 1
            for (int j = 0; j < 32; ++j) {
              const float x = poison(a, p, a.v, D, tok, c * 32 + j);
#pragma unroll
              for (int y = 0; y < 32; ++y)
                if (y == j) v[y] += x;
            }
          }
#pragma unroll
          for (int j = 0; j < 8; ++j)
            stage[lane * 8 + (j ^ (lane & 7))] =
                make_float4(v[4 * j] * f, v[4 * j + 1] * f, v[4 * j + 2] * f, v[4 * j + 3] * f);
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int lr = k * 4 + er, y = first_row + lr;  // row of the unit
            const float4 x = stage[lr * 8 + (ec ^ (lr & 7))];
            if (y >= p.rows) continue;
            if (!whole) {
              *reinterpret_cast<float4 *>(a.part_o + ((int64_t)slot * R + y) * D + c * 32 +
                                          ec * 4) = x;
              continue;
            }
            const int t = (int)(((float)(over + y) + 0.5f) * inv_group);
            const int64_t at = (((int64_t)p.seq.first + tok0 + t) * a.q_heads +
                                p.head * a.group + (over + y - t * a.group)) * D + c * 32 + ec * 4;
            if (a.out_f32)
              *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + at) = x;
            else
              *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + at) =
                  make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
          }
        }
        __syncwarp();
        tc_fence_before();  // O is read before the next piece's weights are signalled
        if (lane == 0) mbar_arrive(&e_done[g]);
        ++ends_g;
      }
      if (threadIdx.x == 0 && p.first && !p.last) {
        MergeJob j{};
        j.slot0 = slot;
        j.parts = cur.parts ? cur.parts
                            : (p.unit_at + cur.tiles - 1) / per - (int)blockIdx.x + 1;
        j.first_token = p.seq.first;
        j.row0 = p.row0;
        j.rows = p.rows;
        j.head = p.head;
        a.jobs[blockIdx.x] = j;
      }
      ++piece;
      i += n > 0 ? n : 0;
    }
  }
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(tmem, 512);
  if (abort_flag && threadIdx.x == 0) report(a.err, NK_TIMEOUT);
}

// Joins the parts of the unit that begins in block blockIdx.x of the
// attention, in their order.  SPLIT warps a row sum every SPLIT-th part and
// meet in shared memory: 4 for units of few rows, whose parts are many, 1 for
// wide units.  Bound by latency (job, statistics, parts: three dependent loads):
// 7 us cold by itself, of which its early launch hides about half; 18 MB of
// parts of wide trees 13 us cold.
template <int D, int SPLIT>
__global__ void __launch_bounds__(512)
    paged_merge_kernel(const __grid_constant__ PagedAttn a, int R) {
  constexpr int V = D / 32, ROWS = 16 / SPLIT;
  __shared__ float sum[SPLIT > 1 ? SPLIT - 1 : 1][ROWS][32][V + 1];
  wait_for_previous();
  const MergeJob j = a.jobs[blockIdx.x];
  const int lane = threadIdx.x & 31, row = (threadIdx.x >> 5) % ROWS;
  const int part = threadIdx.x / (32 * ROWS);
  const int r = blockIdx.y * ROWS + row;
  if (j.parts <= 0 || (int)blockIdx.y * ROWS >= j.rows) return;  // the whole block
  const bool live = r < j.rows;
  // Part i > 0 is the first piece of block blockIdx.x + i.
  auto row_of = [&](int i) {
    return (int64_t)(i ? 2 * ((int)blockIdx.x + i) : j.slot0) * R + r;
  };
  float mx = -INFINITY, l = 0.0f, o[V];
#pragma unroll
  for (int k = 0; k < V; ++k) o[k] = 0.0f;
  if (live) {
    for (int i = lane; i < j.parts; i += 32) mx = fmaxf(mx, a.part_ml[row_of(i)].x);
    for (int k = 16; k > 0; k >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
    const float mu = mx == -INFINITY ? 0.0f : mx;
#pragma unroll 4
    for (int i = part; i < j.parts; i += SPLIT) {
      const float2 ml = a.part_ml[row_of(i)];
      const float c = exp2_approx(ml.x - mu);
      l += ml.y * c;
      const float *p = a.part_o + row_of(i) * D + lane * V;
#pragma unroll
      for (int k = 0; k < V; k += 2) {
        const float2 x = *reinterpret_cast<const float2 *>(p + k);
        o[k] += x.x * c;
        o[k + 1] += x.y * c;
      }
    }
  }
  if (SPLIT > 1) {
    if (part > 0) {
#pragma unroll
      for (int k = 0; k < V; ++k) sum[part - 1][row][lane][k] = o[k];
      sum[part - 1][row][lane][V] = l;
    }
    __syncthreads();
    if (part > 0) return;
#pragma unroll
    for (int w = 0; w < SPLIT - 1; ++w) {
#pragma unroll
      for (int k = 0; k < V; ++k) o[k] += sum[w][row][lane][k];
      l += sum[w][row][lane][V];
    }
  }
  if (!live) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int64_t at = out_row(a, j.first_token, j.head, j.row0 + r) * D + lane * V;
#pragma unroll
  for (int k = 0; k < V; k += 2) store_out(a, at + k, o[k] * inv, o[k + 1] * inv);
}

// ------------------------------------------------------------------- host
// Row tile and blocks of a call, from its bounds alone.
struct AttnPlan {
  int row_tiles;  // 16 * row_tiles rows a unit (1, 2, or 16: tensor memory)
  double tiles;   // the longest list
  int unit_rows;  // rows that a unit holds at most
  int blocks;
  bool merge;     // a unit may be split over blocks
  int cluster;    // blocks that share a unit and join it among them, 0: a tile list
  int units_most; // units of a sequence at most
  size_t o_bytes, ml_bytes, bytes;
};

// Clusters of c blocks that the current device holds at once.  Asked once a
// device: a GPC holds whole clusters only, so this is less than the SMs' number
// over c (16 clusters of 8 with one block an SM do not fit 148 SMs).
template <int D, int MT>
static int resident_clusters(int c) {
  using C = Cfg<D, MT>;
  static std::atomic<int> known[64][4];  // 1 + the answer
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  std::atomic<int> &slot = known[dev & 63][__builtin_ctz((unsigned)c)];
  const int seen = slot.load(std::memory_order_relaxed);
  if (seen) return seen - 1;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)c;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)c);
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const auto kernel = paged_attn_kernel<D, MT, true>;
  int n = 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) !=
          cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
    cudaGetLastError();
    n = 0;
  }
  slot.store(n + 1, std::memory_order_relaxed);
  return n;
}

static AttnPlan plan_attention(const nk_kv_pages &kv, const nk_kv_batch &b,
                               const nk_paged_attention_args &a) {
  AttnPlan p{};
  const int64_t group = a.q_heads / kv.kv_heads;
  const int64_t rows = a.blocks ? group : b.max_new * group;
  p.row_tiles = rows <= 16 ? 1 : (rows <= 32 ? 2 : 16);
  const int64_t r = 16 * p.row_tiles;
  p.unit_rows = (int)(rows < r ? rows : r);
  const int64_t units = a.blocks ? b.max_new * ceil_div(group, r) : ceil_div(rows, r);
  int64_t keys = b.max_kv;
  if (a.blocks && a.max_blocks < ceil_div(keys, kv.page_size)) keys = a.max_blocks * kv.page_size;
  const int64_t tiles = ceil_div(ceil_div(keys, kv.page_size) * kv.page_size, kTile);
  // As many blocks as are resident, or fewer when there are not as many tiles.
  p.tiles = (double)b.seqs * kv.kv_heads * units * tiles;
  const int most = num_sms() * (kv.head_dim == 64 && p.row_tiles <= 2 ? Cfg<64, 1>::kBlocks : 1);
  p.blocks = p.tiles < most ? (p.tiles < 1 ? 1 : (int)p.tiles) : most;
  p.units_most = (int)(kv.kv_heads * units < (1 << 30) ? kv.kv_heads * units : 1 << 30);
  // Clusters, when every unit gets a block for four of its tiles or fewer and all
  // clusters are resident at once: one launch, no workspace (1 sequence of 4096,
  // 8 heads of 128: 9.7 us, 13.4 with the call's host time, as a list 10.2 and
  // 17; 4 of 2048: 9.9 and 12.2).  Block lists of more than 16 tiles run as a
  // tile list: its start hides behind the selection, and few SMs are slower on
  // pages that lie far apart (64 pages of 131072 tokens: 34 us as clusters, 28).
  // (Clusters of 16 found no room side by side: 8 units of 32 tiles 22 us.)
  if (p.row_tiles <= 2 && tiles > 1 && tiles <= (a.blocks ? 16 : 32)) {
    const double all = (double)b.seqs * p.units_most;
    int c = 8;
    while (c / 2 >= tiles) c /= 2;
    for (; c * 4 >= tiles && c > 0; c /= 2) {
      const int room = kv.head_dim == 128
                           ? (p.row_tiles == 1 ? resident_clusters<128, 1>(c)
                                               : resident_clusters<128, 2>(c))
                           : (p.row_tiles == 1 ? resident_clusters<64, 1>(c)
                                               : resident_clusters<64, 2>(c));
      if (all > room) continue;
      p.cluster = c;
      p.blocks = (int)b.seqs * p.units_most * c;
      return p;
    }
  }
  p.merge = tiles > 1;
  if (p.merge) {
    p.o_bytes = (size_t)2 * p.blocks * r * kv.head_dim * 4;
    p.ml_bytes = (size_t)2 * p.blocks * r * 8;
    p.bytes = p.o_bytes + p.ml_bytes + (size_t)p.blocks * sizeof(MergeJob);
  }
  return p;
}

static nk_status check_attention(const nk_kv_pages *kv, const nk_kv_batch *b,
                                 const nk_paged_attention_args *a) {
  if (!a) return fail(NK_INVALID_PARAMS, "args");
  if (a->q_heads <= 0) return fail(NK_INVALID_SHAPE, "q_heads > 0");
  if (a->q_heads % kv->kv_heads) {
    nk_status st = fail(NK_HEAD_COUNT_MISMATCH, "query heads must be a multiple of KV heads");
    tls_error().expected = (uint64_t)a->q_heads;
    tls_error().actual = (uint64_t)kv->kv_heads;
    return st;
  }
  const float sc = a->has_scale ? a->scale : 1.0f / sqrtf((float)kv->head_dim);
  if (!isfinite(sc) || sc <= 0.0f) {
    nk_status st = fail(NK_INVALID_SCALE, "softmax scale must be finite and > 0");
    tls_error().value = sc;
    return st;
  }
  if (a->ld_q < a->q_heads * kv->head_dim || a->ld_q % 8)
    return fail(NK_INVALID_PARAMS, "ld_q must be a multiple of 8 and >= q_heads * head_dim");
  if (a->out_dtype != NK_DTYPE_F32 && a->out_dtype != NK_DTYPE_BF16)
    return fail(NK_INVALID_PARAMS, "out_dtype must be NK_DTYPE_F32 or NK_DTYPE_BF16");
  if (a->tree_mask && a->blocks)
    return fail(NK_UNSUPPORTED, "tree_mask and blocks do not go together");
  if (a->tree_mask && b->max_new > 64)
    return fail(NK_UNSUPPORTED, "a tree holds at most 64 drafted tokens");
  if (a->blocks && (a->max_blocks <= 0 || a->max_blocks > (1 << 20)))
    return fail(NK_INVALID_PARAMS, "max_blocks must lie in 1 .. 2^20");
  if (!a->blocks && a->max_blocks != 0)
    return fail(NK_INVALID_PARAMS, "max_blocks without blocks");
  if (b->max_new * a->q_heads >= (1ll << 31) - 64)
    return fail(NK_UNSUPPORTED, "max_new * q_heads must be < 2^31 - 64");
  if (plan_attention(*kv, *b, *a).tiles >= 2147000000.0)
    return fail(NK_UNSUPPORTED, "too much work for one call: split the batch");
  return NK_OK;
}

// [rows, D] bf16 as boxes of 64 channels x box_rows tokens, 128-byte swizzle.
static nk_status page_map(const uint16_t *base, int64_t rows, int64_t d, int box_rows,
                          CUtensorMap *map) {
  static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> known{nullptr};  // calls of many threads
  PFN_cuTensorMapEncodeTiled_v12000 fn = known.load(std::memory_order_relaxed);
  if (!fn) {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) !=
            cudaSuccess || q != cudaDriverEntryPointSuccess)
      return fail(NK_DEVICE_ERROR, "cuTensorMapEncodeTiled unavailable");
    fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    known.store(fn, std::memory_order_relaxed);
  }
  const cuuint64_t dims[2] = {(cuuint64_t)d, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)d * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
  const cuuint32_t ones[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<uint16_t *>(base),
                        dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(NK_DEVICE_ERROR, "cuTensorMapEncodeTiled failed");
  return NK_OK;
}

template <typename Kernel>
static nk_status launch_attention(Kernel kernel, int smem, int threads,
                                  std::atomic<uint64_t> &prepared, const CUtensorMap &km,
                                  const CUtensorMap &vm, const PagedAttn &a, const AttnPlan &p,
                                  cudaStream_t s) {
  nk_status st = allow_smem(reinterpret_cast<const void *>(kernel), smem, prepared);
  if (st != NK_OK) return st;
  st = launch_early(kernel, dim3((unsigned)p.blocks), dim3((unsigned)threads), (size_t)smem,
                    p.cluster, s, km, vm, a);
  return st != NK_OK ? st : ok();
}

template <int D, int MT>
static nk_status launch_rows(const CUtensorMap &km, const CUtensorMap &vm, const PagedAttn &a,
                             const AttnPlan &p, cudaStream_t s) {
  using C = Cfg<D, MT>;
  static std::atomic<uint64_t> list{0}, clusters{0};  // a bit per device
  if (!p.cluster)
    return launch_attention(paged_attn_kernel<D, MT, false>, C::kSmem, C::kThreads, list, km, vm,
                            a, p, s);
  return launch_attention(paged_attn_kernel<D, MT, true>, C::kSmem, C::kThreads,
                          clusters, km, vm, a, p, s);
}

template <int D>
static nk_status launch_attention(const CUtensorMap &km, const CUtensorMap &vm,
                                  const PagedAttn &a, const AttnPlan &p, cudaStream_t s) {
  static std::atomic<uint64_t> prepared{0};
  nk_status st =
      p.row_tiles == 1   ? launch_rows<D, 1>(km, vm, a, p, s)
      : p.row_tiles == 2 ? launch_rows<D, 2>(km, vm, a, p, s)
                         : launch_attention(paged_attn_tc_kernel<D>, TcCfg<D>::kSmem,
                                            TcCfg<D>::kThreads, prepared, km, vm, a, p, s);
  if (st != NK_OK || !p.merge) return st;
  const bool wide = p.row_tiles > 2;
  const dim3 grid((unsigned)p.blocks, (unsigned)ceil_div(p.unit_rows, wide ? 16 : 4));
  st = launch_early(wide ? paged_merge_kernel<D, 1> : paged_merge_kernel<D, 4>, grid, dim3(512), 0,
                    1, s, a, 16 * p.row_tiles);
  return st != NK_OK ? st : ok();
}

}  // namespace nk

using namespace nk;

extern "C" {

nk_status nk_attention_paged_workspace_bytes(const nk_kv_pages *kv, const nk_kv_batch *batch,
                                             const nk_paged_attention_args *args, size_t *bytes) {
  if (!bytes) return fail(NK_INVALID_PARAMS, "bytes");
  nk_status st = check_pages(kv, 0);
  if (st == NK_OK) st = check_batch(kv, batch);
  if (st == NK_OK) st = check_attention(kv, batch, args);
  if (st != NK_OK) return st;
  *bytes = plan_attention(*kv, *batch, *args).bytes;
  return ok();
}

nk_status nk_attention_paged(const nk_kv_pages *kv, int64_t layer, const nk_kv_batch *batch,
                             const nk_paged_attention_args *args, void *workspace,
                             size_t workspace_bytes, void *stream) {
  nk_status st = check_pages(kv, layer);
  if (st == NK_OK) st = check_batch(kv, batch);
  if (st == NK_OK) st = check_attention(kv, batch, args);
  if (st != NK_OK) return st;
  if (batch->seqs == 0 || batch->tokens == 0 || batch->max_new == 0) return ok();
  if (!args->q || !args->out) return fail(NK_INVALID_PARAMS, "q and out are required");
  if (((uintptr_t)args->q | (uintptr_t)args->out | (uintptr_t)workspace) & 15)
    return fail(NK_INVALID_PARAMS, "q, out and workspace must be 16-byte aligned");
  const AttnPlan p = plan_attention(*kv, *batch, *args);
  if (workspace_bytes < p.bytes || (p.bytes && !workspace)) {
    st = fail(NK_WORKSPACE_TOO_SMALL, "attention workspace too small");
    tls_error().expected = p.bytes;
    tls_error().actual = workspace_bytes;
    return st;
  }
  PagedAttn a{};
  a.pool = page_pool(*kv);
  a.batch = page_batch(*batch);
  a.q = args->q;
  a.v = kv->v;
  a.ld_q = args->ld_q;
  a.q_heads = (int)args->q_heads;
  a.group = (int)(args->q_heads / kv->kv_heads);
  a.layer_row = layer * kv->pages * kv->kv_heads * kv->page_size;
  a.mask = args->tree_mask;
  a.blocks = args->blocks;
  a.max_blocks = (int)args->max_blocks;
  const float sc = args->has_scale ? args->scale : 1.0f / sqrtf((float)kv->head_dim);
  a.scale_log2 = sc * 1.44269504088896340736f;
  a.out = args->out;
  a.out_f32 = args->out_dtype == NK_DTYPE_F32;
  a.cluster = p.cluster;
  a.units_most = p.units_most;
  if (p.merge) {
    uint8_t *w = static_cast<uint8_t *>(workspace);
    a.part_o = reinterpret_cast<float *>(w);
    a.part_ml = reinterpret_cast<float2 *>(w + p.o_bytes);
    a.jobs = reinterpret_cast<MergeJob *>(w + p.o_bytes + p.ml_bytes);
  }
  a.err = device_error_ptr();
  if (!a.err) return fail(NK_DEVICE_ERROR, "cannot resolve device error word");
  const int64_t rows = kv->layers * kv->pages * kv->kv_heads * kv->page_size;
  const int box = (int)kv->page_size;
  CUtensorMap km, vm;
  st = page_map(kv->k, rows, kv->head_dim, box, &km);
  if (st == NK_OK) st = page_map(kv->v, rows, kv->head_dim, box, &vm);
  if (st != NK_OK) return st;
  cudaStream_t s = as_stream(stream);
  return kv->head_dim == 128 ? launch_attention<128>(km, vm, a, p, s)
                             : launch_attention<64>(km, vm, a, p, s);
}

}  // extern "C"
