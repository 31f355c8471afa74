"""A paged cache built on the host and the plain 64-bit forms of the operators
that read it, for the GPU tests."""
import numpy as np
import torch

import nk


def bf16(a):
    """f64 -> the nearest bf16, as f32 values."""
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).bfloat16().float().numpy()


class Paged:
    """Random pools and shuffled tables.  Slots behind a sequence's end and
    pages of no sequence hold `filler`."""

    def __init__(self, seed, lens, heads, ps, d, *, layers=1, spare=3, width=None,
                 filler=np.nan, max_rows=None):
        r = np.random.default_rng(seed)
        self.rng, self.lens = r, np.asarray(lens, np.int64)
        self.heads, self.ps, self.d, self.layers = heads, ps, d, layers
        blocks = -(-self.lens // ps)
        pages = int(blocks.sum()) + spare
        self.n_pages = pages
        order = r.permutation(pages)
        rows = max_rows or max(1, len(lens))
        self.table = np.full((rows, max(1, width or int(blocks.max(initial=1)))), -1, np.int32)
        at = 0
        for i, b in enumerate(blocks):
            self.table[i, :b] = order[at:at + b]
            at += b
        self.spare = order[at:]
        self.k = bf16(r.standard_normal((layers, pages, heads, ps, d)))
        self.v = bf16(r.standard_normal((layers, pages, heads, ps, d)))
        for x in (self.k, self.v):
            x[:, self.spare] = filler
            for i, n in enumerate(self.lens):
                if n % ps:
                    x[:, self.table[i, n // ps], :, n % ps:] = filler
        self.lo, self.hi = np.zeros((2, layers, pages, heads, d), np.float32)
        self.refresh_bounds()

    def refresh_bounds(self, seqs=None, lens=None):
        lens = self.lens if lens is None else lens
        for i, n in enumerate(lens):
            for j in range(-(-int(n) // self.ps)):
                p, m = self.table[i, j], min(self.ps, int(n) - j * self.ps)
                self.lo[:, p] = self.k[:, p, :, :m].min(2)
                self.hi[:, p] = self.k[:, p, :, :m].max(2)

    def slot(self, s, pos):
        return self.table[s, pos // self.ps], pos % self.ps

    def tokens(self, pool, s, layer=0):
        """[heads, len, d] of a sequence in position order."""
        n = int(self.lens[s])
        pos = np.arange(n)
        return pool[layer, self.table[s, pos // self.ps], :, pos % self.ps].transpose(1, 0, 2)

    def device(self):
        t = lambda a: torch.from_numpy(a).bfloat16().cuda()  # noqa: E731
        return nk.KvPages(t(self.k), t(self.v), torch.from_numpy(self.table).cuda(),
                          k_min=t(self.lo), k_max=t(self.hi))


def same(device_pool, host_pool):
    """Equal values, NaN in the same places."""
    return np.array_equal(device_pool.float().cpu().numpy(), host_pool, equal_nan=True)


def ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


def starts(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def attention(q, k, v, seen, scale):
    """q [T, H, d], k, v [Hkv, L, d], seen [T, Hkv or 1, L] truth values ->
    (out, mean |v| under the weights), both [T, H, d], in 64 bits.  Positions
    that are not seen are left out before anything is multiplied."""
    T, H, d = q.shape
    G = H // k.shape[0]
    out, mag = np.zeros((T, H, d)), np.zeros((T, H, d))
    for t in range(T):
        for h in range(H):
            use = np.flatnonzero(seen[t, min(h // G, seen.shape[1] - 1)])
            if use.size == 0:
                continue
            with np.errstate(invalid="ignore", over="ignore"):
                s = (k[h // G, use].astype(np.float64) @ q[t, h].astype(np.float64)) * scale
                w = np.exp(s - s.max())
                vv = v[h // G, use].astype(np.float64)
                out[t, h] = (w[:, None] * vv).sum(0) / w.sum()
                mag[t, h] = (w[:, None] * np.abs(vv)).sum(0) / w.sum()
    return out, mag


def tree_masks(rng, n):
    """A random tree of n drafts: (words int64, seen [n, n])."""
    seen = np.zeros((n, n), bool)
    for i in range(n):
        if i and rng.random() < 0.9:
            seen[i] = seen[int(rng.integers(0, i))]
        seen[i, i] = True
    words = [sum(1 << int(j) for j in np.flatnonzero(row)) for row in seen]
    return np.array(words, np.uint64).view(np.int64), seen


def chosen_blocks(q, lo, hi, n, top_k, sink, local):
    """Blocks of one token and KV head: q [G, d], bounds [n, d], in 64 bits."""
    with np.errstate(invalid="ignore"):
        s = np.stack([np.where(x >= 0, hi, lo).astype(np.float64) @ x.astype(np.float64)
                      for x in q])
    s = np.where(np.isnan(s), -np.inf, s).max(0)
    must = (np.arange(n) < sink) | (np.arange(n) >= n - local)
    order = np.lexsort((np.arange(n), -s, ~must))
    return np.sort(order[:top_k])
