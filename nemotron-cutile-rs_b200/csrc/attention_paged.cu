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
// sums are f32; p is rounded to bf16 (relative error 2^-9) for the value
// product, as the operand type of the tensor cores asks, while l sums the
// unrounded p.
//
// Tiles of 64 keys come by TMA (boxes of 64 channels x the keys of one page)
// into a ring of shared-memory stages, in the 128-byte swizzle that ldmatrix
// reads without bank conflicts.
#include <cudaTypedefs.h>

#include "gemm_tc.h"
#include "paged.cuh"

namespace nk {

constexpr int kTile = 64;  // keys of a stage

struct PagedAttn {
  PagePool pool;
  PageBatch batch;
  const uint16_t *q;
  int64_t ld_q;
  int q_heads, group;
  int64_t layer_row;  // first token row of the layer in the pools
  const uint64_t *mask;
  const int32_t *blocks;
  int max_blocks;
  float scale_log2;  // scale * log2(e): exp(scale * s) = 2^(scale_log2 * s)
  void *out;
  int out_f32;
  int splits, split_tiles;  // key tiles of a split
  float *part_o;            // [splits][tokens * q_heads][head_dim], unnormalised
  float2 *part_ml;          // [splits][tokens * q_heads]: m (in log2 units), l
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
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t *>(&v);
}

// Byte offset of (key, channel) in a tile: halves of 64 channels, 128-byte
// rows, 16-byte chunks XORed with the row (TMA's 128-byte swizzle).
__device__ __forceinline__ uint32_t tile_offset(int key, int chan) {
  return (uint32_t)((chan >> 6) * (kTile * 128) + key * 128 +
                    (((chan & 63) * 2) ^ ((key & 7) * 16)));
}

// What a block works on.
struct Work {
  SeqView seq;
  int head;         // KV head
  int row0, rows;   // rows row0 .. row0+rows-1 of the sequence's count * group
  int prefix;       // cached tokens before the new ones
  int keys;         // keys 0 .. keys-1 (dense) or list slots * page size (blocks)
  int pos;          // blocks: the token's position
  const int32_t *list;
};

template <int R>
__device__ __forceinline__ bool find_work(const PagedAttn &a, Work &w, bool report_it) {
  if (!load_seq(a.pool, a.batch, blockIdx.z, w.seq, a.err, report_it)) return false;
  w.prefix = w.seq.len - w.seq.count;
  const int heads = a.pool.heads;
  w.head = blockIdx.y % heads;
  const int tile = blockIdx.y / heads;
  if (a.blocks) {
    const int gt = (a.group + R - 1) / R;
    const int token = tile / gt, g0 = (tile % gt) * R;
    if (token >= w.seq.count) return false;
    w.row0 = token * a.group + g0;
    w.rows = a.group - g0 < R ? a.group - g0 : R;
    w.pos = w.prefix + token;
    w.list = a.blocks + ((int64_t)(w.seq.first + token) * heads + w.head) * a.max_blocks;
    w.keys = a.max_blocks << a.pool.ps_log2;
  } else {
    const int total = w.seq.count * a.group;
    w.row0 = tile * R;
    if (w.row0 >= total) return false;
    w.rows = total - w.row0 < R ? total - w.row0 : R;
    w.pos = 0;
    w.list = nullptr;
    w.keys = w.seq.len;
    if (!a.mask) {  // causal: up to the tile's last token
      const int last = w.prefix + (w.row0 + w.rows - 1) / a.group + 1;
      if (last < w.keys) w.keys = last;
    }
  }
  return true;
}

// Output row of row r of the block's tile: (token, query head).
__device__ __forceinline__ int64_t out_row(const PagedAttn &a, const Work &w, int r) {
  const int x = w.row0 + r;
  return ((int64_t)w.seq.first + x / a.group) * a.q_heads + w.head * a.group + x % a.group;
}

// Warps: 4 compute warps, RW of them over rows (16 each) and 4/RW over the
// keys of a tile; warp 4 loads.
template <int D, int RW, int STAGES>
struct Cfg {
  static constexpr int kRows = 16 * RW;
  static constexpr int kKeyWarps = 4 / RW;
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kSmem = STAGES * kStageBytes + 1024;
};

template <int D, int RW, int STAGES>
__global__ void __launch_bounds__(160, (D == 128 && STAGES > 3) ? 1 : 2)
    paged_attn_kernel(const __grid_constant__ CUtensorMap kmap,
                      const __grid_constant__ CUtensorMap vmap, const PagedAttn a) {
  using C = Cfg<D, RW, STAGES>;
  constexpr int R = C::kRows, KW = C::kKeyWarps;
  constexpr int NK = kTile / KW;  // keys of a warp per tile
  constexpr int NT = NK / 8;      // score fragments
  constexpr int OT = D / 8;       // output fragments
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~uintptr_t(1023));
  __shared__ uint64_t full[STAGES], empty[STAGES];
  __shared__ __align__(16) int limits[STAGES][4];  // written keys of each 16-key group
  __shared__ int abort_flag, list_len;
  __shared__ uint32_t odd_keys[2];   // keys of the tile that hold an infinity or NaN

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Work w;
  if (!find_work<R>(a, w, threadIdx.x == 0)) return;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 4);
    }
    fence_mbar_init();
    abort_flag = 0;
    list_len = 0;
  }
  __syncthreads();
  if (w.list) {  // entries behind the last block hold -1: no tiles for them
    int n = 0;
    for (int i = threadIdx.x; i < a.max_blocks; i += blockDim.x)
      if (w.list[i] >= 0) n = i + 1;
    atomicMax(&list_len, n);
    __syncthreads();
    w.keys = list_len << a.pool.ps_log2;
  }
  const int tiles_all = (w.keys + kTile - 1) / kTile;
  const int t0 = blockIdx.x * a.split_tiles;
  const int t1 = t0 + a.split_tiles < tiles_all ? t0 + a.split_tiles : tiles_all;

  float o[OT][4];
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < OT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;

  if (warp == 4) {
    // ------------------------------------------------------------- loader
    // Lane = (page of the tile, channel half, K or V): up to 16 boxes.
    const int per = a.pool.ps >= kTile ? 1 : kTile >> a.pool.ps_log2;  // pages of a tile
    const int box_rows = a.pool.ps < kTile ? a.pool.ps : kTile;
    const int boxes = per * (D / 64) * 2;
    const int c = lane % per, half = (lane / per) % (D / 64), is_v = lane / (per * (D / 64));
    int page_next = 0, block_next = 0;
    auto lookup = [&](int t) {  // block and page of this lane's box of tile t
      const int key0 = t * kTile + c * box_rows;
      int b = key0 >> a.pool.ps_log2;
      page_next = -1;
      block_next = -1;
      if (lane >= boxes || key0 >= w.keys) return;
      if (w.list) {
        const int e = b;
        b = w.list[e];
        if (b < 0 || b > (w.pos >> a.pool.ps_log2) || (e > 0 && b <= w.list[e - 1])) return;
      }
      block_next = b;
      const int page = w.seq.table[b];
      if (page_ok(a.pool, page)) page_next = page;
      else report(a.err, NK_PAGE_OUT_OF_RANGE);
    };
    if (t0 < t1) lookup(t0);
    for (int t = t0, i = 0; t < t1; ++t, ++i) {
      const int s = i % STAGES;
      const int page = page_next, block = block_next;
      if (t + 1 < t1) lookup(t + 1);  // in flight while this tile waits
      if (i >= STAGES && !mbar_wait(&empty[s], ((i / STAGES) - 1) & 1, &abort_flag)) break;
      const bool load = page >= 0;
      const int within = a.pool.ps > kTile ? (t * kTile) & (a.pool.ps - 1) : 0;
      if (lane < per && half == 0 && is_v == 0) {
        // Keys of the box that the rows may see: up to the last position.
        int n = 0;
        if (load) {
          n = w.list ? w.pos + 1 - ((block << a.pool.ps_log2) + within)
                     : w.keys - (t * kTile + c * box_rows);
          n = n < 0 ? 0 : (n > box_rows ? box_rows : n);
        }
        for (int g = 0; g < box_rows / 16; ++g)
          limits[s][c * (box_rows / 16) + g] = n - 16 * g < 0 ? 0 : (n - 16 * g > 16 ? 16 : n - 16 * g);
      }
      const uint32_t mine = __ballot_sync(0xffffffffu, load);
      __syncwarp();
      if (lane == 0)
        mbar_arrive_expect_tx(&full[s], (uint32_t)__popc(mine) * (uint32_t)box_rows * 128u);
      __syncwarp();
      if (load) {
        uint8_t *dst = smem + s * C::kStageBytes + is_v * C::kTileBytes + half * (kTile * 128) +
                       c * box_rows * 128;
        const int64_t row = a.layer_row +
                            (((int64_t)page * a.pool.heads + w.head) << a.pool.ps_log2) + within;
        tma_load_2d(dst, is_v ? &vmap : &kmap, &full[s], half * 64, (int)row);
      }
    }
    // The copies in flight land before the block's memory is given up.
    const int issued = t1 - t0;
    if (abort_flag && issued > 0) {
      for (int s = 0; s < STAGES; ++s)
        for (int ph = 0; ph < 2; ++ph) {
          const uint64_t start = nk_globaltimer();
          while (!mbar_try_wait(&full[s], ph) && nk_globaltimer() - start < 1000000ull) {
          }
        }
    }
  } else {
    // ------------------------------------------------------------ compute
    const int rw = warp % RW, kw = warp / RW;
    const int quad = lane >> 2, qc = (lane & 3) * 2;
    // Rows of this lane: quad and quad + 8 of the warp's 16.
    uint32_t qf[D / 16][4];
    int pos_row[2];       // causal: last position the row sees
    uint64_t tree[2];
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const int r = rw * 16 + quad + hh * 8;
      const bool live = r < w.rows;
      const int x = w.row0 + r;
      const uint16_t *qr =
          a.q + ((int64_t)w.seq.first + x / a.group) * a.ld_q +
          ((int64_t)w.head * a.group + x % a.group) * D;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        qf[k][hh] = live ? *reinterpret_cast<const uint32_t *>(qr + k * 16 + qc) : 0u;
        qf[k][hh + 2] = live ? *reinterpret_cast<const uint32_t *>(qr + k * 16 + 8 + qc) : 0u;
      }
      pos_row[hh] = w.prefix + x / a.group;
      tree[hh] = a.mask && live ? a.mask[w.seq.first + x / a.group] : 0;
    }
    // Positions from here on are not seen by every row of the tile.
    const int all_see = w.list ? 0x7fffffff
                               : (a.mask ? w.prefix : w.prefix + w.row0 / a.group + 1);
    auto allowed = [&](int hh, int p) {  // p < keys
      if (a.mask) return p < w.prefix || ((tree[hh] >> (p - w.prefix)) & 1) != 0;
      return p <= pos_row[hh];
    };

    for (int t = t0, i = 0; t < t1; ++t, ++i) {
      const int s = i % STAGES;
      if (!mbar_wait(&full[s], (i / STAGES) & 1, &abort_flag)) break;
      uint8_t *kt = smem + s * C::kStageBytes, *vt = kt + C::kTileBytes;
      const int4 lim = *reinterpret_cast<const int4 *>(limits[s]);
      const bool tail = (lim.x + lim.y + lim.z + lim.w) < kTile;
      const bool partial = (t + 1) * kTile > all_see && !w.list;
      uint64_t odd = 0;
      if (tail || partial) {
        // Values that a row may not see are multiplied by a weight of 0, so
        // what lies behind the last key becomes 0, and keys that only some
        // rows see are searched for infinities and NaN (0 * inf is NaN).
        if (threadIdx.x < 2) odd_keys[threadIdx.x] = 0;
        asm volatile("bar.sync 1, 128;" ::: "memory");
        const int key = threadIdx.x >> 1, part = threadIdx.x & 1;  // half of the key's channels
        const int g = key >> 4;
        const int lg = g == 0 ? lim.x : (g == 1 ? lim.y : (g == 2 ? lim.z : lim.w));
        const bool dead = (key & 15) >= lg;
        const bool some = partial && !dead && t * kTile + key >= all_see;
        bool found = false;
        if (dead || some) {
#pragma unroll
          for (int ch = 0; ch < D / 16; ++ch) {
            uint4 *p = reinterpret_cast<uint4 *>(vt + tile_offset(key, part * (D / 2) + ch * 8));
            if (dead) {
              *p = make_uint4(0, 0, 0, 0);
            } else {
              const uint4 x = *p;
              const uint32_t word[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
              for (int j = 0; j < 4; ++j)
                found |= (word[j] & 0x7f80u) == 0x7f80u ||
                         (word[j] & 0x7f800000u) == 0x7f800000u;
            }
          }
        }
        if (found) atomicOr(&odd_keys[key >> 5], 1u << (key & 31));
        if (dead) fence_proxy_async_smem();  // before the stage is loaded again
        asm volatile("bar.sync 1, 128;" ::: "memory");
        odd = (uint64_t)odd_keys[1] << 32 | odd_keys[0];
        asm volatile("bar.sync 1, 128;" ::: "memory");  // read by all before the next tile's reset
      }

      // Scores of the warp's NK keys.
      float sc[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[n][j] = 0.0f;
      const uint32_t kb = smem_u32(kt), vb = smem_u32(vt);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
          uint32_t b[4];
          const int mtx = lane >> 3;
          ldsm4(b, kb + tile_offset(kw * NK + n * 8 + (mtx >> 1) * 8 + (lane & 7),
                                    k * 16 + (mtx & 1) * 8));
          mma16816(sc[n], qf[k], b[0], b[1]);
          mma16816(sc[n + 1], qf[k], b[2], b[3]);
        }
      }
      if (tail || partial) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = kw * NK + n * 8 + qc + (j & 1);
            const int g = key >> 4;
            const int lg = g == 0 ? lim.x : (g == 1 ? lim.y : (g == 2 ? lim.z : lim.w));
            bool ok = (key & 15) < lg;
            if (ok && partial) ok = allowed(j >> 1, t * kTile + key);
            if (!ok) sc[n][j] = -INFINITY;
          }
      }
      // Running maximum and sum, two rows a lane, four lanes a row.
      float corr[2], mu[2];
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        float mx = -INFINITY;
#pragma unroll
        for (int n = 0; n < NT; ++n) mx = fmaxf(mx, fmaxf(sc[n][2 * hh], sc[n][2 * hh + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m[hh], mx * a.scale_log2);
        // No key so far: any finite shift will do, and keeps -inf - -inf out.
        mu[hh] = mn == -INFINITY ? 0.0f : mn;
        corr[hh] = exp2_approx(m[hh] - mu[hh]);
        m[hh] = mn;
        l[hh] *= corr[hh];
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p = exp2_approx(sc[n][j] * a.scale_log2 - mu[j >> 1]);
          sc[n][j] = p;
          l[j >> 1] += p;
        }
#pragma unroll
      for (int n = 0; n < OT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n][j] *= corr[j >> 1];

      if (odd) {
        // Rare: an infinity or NaN in a key that some rows see.  Its terms are
        // added by hand for the rows that see it, then its values become 0.
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int key = kw * NK + n * 8 + e;
            if (!((odd >> key) & 1)) continue;
            const int src = (lane & ~3) | (e >> 1);
            const float p0 = __shfl_sync(0xffffffffu, sc[n][e & 1], src);
            const float p1 = __shfl_sync(0xffffffffu, sc[n][2 + (e & 1)], src);
            const int p = t * kTile + key;
            const bool see0 = allowed(0, p), see1 = allowed(1, p);
#pragma unroll
            for (int f = 0; f < OT; ++f)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const float v = __bfloat162float(*reinterpret_cast<const __nv_bfloat16 *>(
                    vt + tile_offset(key, f * 8 + qc + j)));
                if (see0) o[f][j] += p0 * v;
                if (see1) o[f][2 + j] += p1 * v;
              }
          }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        const int key = threadIdx.x >> 1, part = threadIdx.x & 1;
        if ((odd >> key) & 1) {
#pragma unroll
          for (int ch = 0; ch < D / 16; ++ch)
            *reinterpret_cast<uint4 *>(vt + tile_offset(key, part * (D / 2) + ch * 8)) =
                make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
      }

      // O += P V
#pragma unroll
      for (int kk = 0; kk < NK / 16; ++kk) {
        const uint32_t pa[4] = {pack_bf16(sc[2 * kk][0], sc[2 * kk][1]),
                                pack_bf16(sc[2 * kk][2], sc[2 * kk][3]),
                                pack_bf16(sc[2 * kk + 1][0], sc[2 * kk + 1][1]),
                                pack_bf16(sc[2 * kk + 1][2], sc[2 * kk + 1][3])};
#pragma unroll
        for (int n = 0; n < OT; n += 2) {
          uint32_t b[4];
          const int mtx = lane >> 3;
          ldsm4_t(b, vb + tile_offset(kw * NK + kk * 16 + (mtx & 1) * 8 + (lane & 7),
                                      n * 8 + (mtx >> 1) * 8));
          mma16816(o[n], pa, b[0], b[1]);
          mma16816(o[n + 1], pa, b[2], b[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      l[hh] += __shfl_xor_sync(0xffffffffu, l[hh], 1);
      l[hh] += __shfl_xor_sync(0xffffffffu, l[hh], 2);
    }
  }
  __syncthreads();  // every tile is read: the ring is free
  if (abort_flag) {
    if (threadIdx.x == 0) report(a.err, NK_TIMEOUT);
    return;
  }

  if (KW > 1) {
    // Join the key warps of each row group through shared memory, in order.
    const int rw = warp % RW, kw = warp / RW;
    float *buf = reinterpret_cast<float *>(smem);  // [KW-1][RW][32 lanes][OT*4+4]
    constexpr int W = OT * 4 + 4;
    if (warp < 4 && kw > 0) {
      float *p = buf + (((kw - 1) * RW + rw) * W) * 32 + lane;
#pragma unroll
      for (int n = 0; n < OT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) p[(n * 4 + j) * 32] = o[n][j];
      p[(OT * 4) * 32] = m[0];
      p[(OT * 4 + 1) * 32] = m[1];
      p[(OT * 4 + 2) * 32] = l[0];
      p[(OT * 4 + 3) * 32] = l[1];
    }
    __syncthreads();
    if (warp < 4 && kw == 0) {
      for (int x = 1; x < KW; ++x) {
        const float *p = buf + (((x - 1) * RW + rw) * W) * 32 + lane;
        float ca[2], cb[2];
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const float mo = p[(OT * 4 + hh) * 32];
          const float mn = fmaxf(m[hh], mo);
          const float mu = mn == -INFINITY ? 0.0f : mn;
          ca[hh] = exp2_approx(m[hh] - mu);
          cb[hh] = exp2_approx(mo - mu);
          m[hh] = mn;
          l[hh] = l[hh] * ca[hh] + p[(OT * 4 + 2 + hh) * 32] * cb[hh];
        }
#pragma unroll
        for (int n = 0; n < OT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            o[n][j] = o[n][j] * ca[j >> 1] + p[(n * 4 + j) * 32] * cb[j >> 1];
      }
    }
  }
  if (warp < RW) {
    const int quad = lane >> 2, qc = (lane & 3) * 2;
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const int r = warp * 16 + quad + hh * 8;
      if (r >= w.rows) continue;
      const int64_t row = out_row(a, w, r);
      if (a.splits > 1) {
        const int64_t at = (int64_t)blockIdx.x * a.batch.tokens * a.q_heads + row;
        if ((lane & 3) == 0) a.part_ml[at] = make_float2(m[hh], l[hh]);
        if (t0 >= t1) continue;  // no key in the range: l = 0 says so
        float *p = a.part_o + at * D + qc;
#pragma unroll
        for (int n = 0; n < OT; ++n)
          *reinterpret_cast<float2 *>(p + n * 8) = make_float2(o[n][2 * hh], o[n][2 * hh + 1]);
      } else {
        const float inv = l[hh] == 0.0f ? 0.0f : 1.0f / l[hh];
#pragma unroll
        for (int n = 0; n < OT; ++n) {
          const float x = o[n][2 * hh] * inv, y = o[n][2 * hh + 1] * inv;
          if (a.out_f32)
            *reinterpret_cast<float2 *>(static_cast<float *>(a.out) + row * D + n * 8 + qc) =
                make_float2(x, y);
          else
            *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(a.out) + row * D + n * 8 + qc) =
                pack_bf16(x, y);
        }
      }
    }
  }
}

// Joins the splits of a row in their order: warp per (token, query head).
// Only rows that belong to a sequence are written.
template <int D>
__global__ void __launch_bounds__(128) paged_merge_kernel(const PagedAttn a) {
  const int s = blockIdx.y, lane = threadIdx.x & 31;
  SeqView seq;
  if (!load_seq(a.pool, a.batch, s, seq, a.err, false)) return;
  const int x = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (x >= seq.count * a.q_heads) return;
  const int64_t rows = a.batch.tokens * a.q_heads;
  const int64_t row = (int64_t)seq.first * a.q_heads + x;
  constexpr int V = D / 32;
  float mx = -INFINITY;
  for (int i = lane; i < a.splits; i += 32) mx = fmaxf(mx, a.part_ml[i * rows + row].x);
  for (int k = 16; k > 0; k >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
  const float mu = mx == -INFINITY ? 0.0f : mx;
  float l = 0.0f, o[V];
#pragma unroll
  for (int j = 0; j < V; ++j) o[j] = 0.0f;
#pragma unroll 4
  for (int i = 0; i < a.splits; ++i) {
    const float2 ml = a.part_ml[i * rows + row];
    const float c = exp2_approx(ml.x - mu);
    if (ml.y == 0.0f) continue;  // the split had no key
    l += ml.y * c;
    const float *p = a.part_o + (i * rows + row) * D + lane * V;
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] += p[j] * c;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int64_t at = row * D + lane * V + j;
    if (a.out_f32)
      static_cast<float *>(a.out)[at] = o[j] * inv;
    else
      static_cast<__nv_bfloat16 *>(a.out)[at] = __float2bfloat16_rn(o[j] * inv);
  }
}

// ------------------------------------------------------------------- host
// Row tile and key split of a call, from its bounds alone.
struct AttnPlan {
  int row_warps;   // 16 * row_warps rows a block
  int row_tiles;   // blocks over the rows of a sequence and head
  int splits, split_tiles;
  size_t bytes;
};

static AttnPlan plan_attention(const nk_kv_pages &kv, const nk_kv_batch &b,
                               const nk_paged_attention_args &a) {
  AttnPlan p{};
  const int64_t group = a.q_heads / kv.kv_heads;
  const int64_t rows = a.blocks ? group : b.max_new * group;
  p.row_warps = rows <= 16 ? 1 : (rows <= 32 ? 2 : 4);
  const int64_t r = 16 * p.row_warps;
  p.row_tiles = (int)(a.blocks ? b.max_new * ceil_div(group, r) : ceil_div(rows, r));
  const int64_t keys = a.blocks ? a.max_blocks * kv.page_size : b.max_kv;
  const int64_t tiles = ceil_div(keys > 0 ? keys : 1, kTile);
  const int64_t units = b.seqs * kv.kv_heads * p.row_tiles;
  // Two blocks a SM; ragged lengths want a few blocks more to even out.
  int64_t want = ceil_div(2 * 2 * 148, units > 0 ? units : 1);
  int64_t per = ceil_div(tiles, want);
  if (per < 2) per = 2;  // a range shorter than two tiles costs more to join than to read
  p.split_tiles = (int)per;
  p.splits = (int)ceil_div(tiles, per);
  if (p.splits > 1)
    p.bytes = (size_t)p.splits * b.tokens * a.q_heads * (kv.head_dim * 4 + 8);
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
  const int64_t group = a->q_heads / kv->kv_heads;
  if (b->max_new * a->q_heads >= (1ll << 31) - 64 || b->tokens * a->q_heads >= (1ll << 40))
    return fail(NK_UNSUPPORTED, "max_new * q_heads must be < 2^31 - 64");
  const AttnPlan p = plan_attention(*kv, *b, *a);
  if ((a->blocks ? b->max_new * ceil_div(group, 16 * p.row_warps) : (int64_t)p.row_tiles) *
          kv->kv_heads > 65535)
    return fail(NK_UNSUPPORTED, "too many query rows in one sequence: split the chunk");
  return NK_OK;
}

// [rows, D] bf16 as boxes of 64 channels x box_rows tokens, 128-byte swizzle.
static nk_status page_map(const uint16_t *base, int64_t rows, int64_t d, int box_rows,
                          CUtensorMap *map) {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  if (!fn) {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) !=
            cudaSuccess || q != cudaDriverEntryPointSuccess)
      return fail(NK_DEVICE_ERROR, "cuTensorMapEncodeTiled unavailable");
    fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
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

template <int D, int RW, int STAGES>
static nk_status launch_attention(const CUtensorMap &km, const CUtensorMap &vm,
                                  const PagedAttn &a, dim3 grid, cudaStream_t s) {
  using C = Cfg<D, RW, STAGES>;
  NK_CUDA_TRY(cudaFuncSetAttribute(paged_attn_kernel<D, RW, STAGES>,
                                   cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
  paged_attn_kernel<D, RW, STAGES><<<grid, 160, C::kSmem, s>>>(km, vm, a);
  return check_launch("paged_attn_kernel");
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
  a.splits = p.splits;
  a.split_tiles = p.split_tiles;
  a.part_o = static_cast<float *>(workspace);
  a.part_ml = reinterpret_cast<float2 *>(a.part_o + (int64_t)p.splits * batch->tokens *
                                                        args->q_heads * kv->head_dim);
  a.err = device_error_ptr();
  if (!a.err) return fail(NK_DEVICE_ERROR, "cannot resolve device error word");
  const int64_t rows = kv->layers * kv->pages * kv->kv_heads * kv->page_size;
  const int box = kv->page_size < kTile ? (int)kv->page_size : kTile;
  CUtensorMap km, vm;
  st = page_map(kv->k, rows, kv->head_dim, box, &km);
  if (st == NK_OK) st = page_map(kv->v, rows, kv->head_dim, box, &vm);
  if (st != NK_OK) return st;
  cudaStream_t s = as_stream(stream);
  const dim3 grid((unsigned)p.splits, (unsigned)(p.row_tiles * kv->kv_heads),
                  (unsigned)batch->seqs);
  if (kv->head_dim == 128) {
    st = p.row_warps == 1   ? launch_attention<128, 1, 3>(km, vm, a, grid, s)
         : p.row_warps == 2 ? launch_attention<128, 2, 3>(km, vm, a, grid, s)
                            : launch_attention<128, 4, 3>(km, vm, a, grid, s);
  } else {
    st = p.row_warps == 1   ? launch_attention<64, 1, 6>(km, vm, a, grid, s)
         : p.row_warps == 2 ? launch_attention<64, 2, 6>(km, vm, a, grid, s)
                            : launch_attention<64, 4, 6>(km, vm, a, grid, s);
  }
  if (st != NK_OK || p.splits == 1) return st;
  const dim3 mg((unsigned)ceil_div(batch->max_new * args->q_heads, 4), (unsigned)batch->seqs);
  if (kv->head_dim == 128)
    paged_merge_kernel<128><<<mg, 128, 0, s>>>(a);
  else
    paged_merge_kernel<64><<<mg, 128, 0, s>>>(a);
  return check_launch("paged_merge_kernel");
}

}  // extern "C"
