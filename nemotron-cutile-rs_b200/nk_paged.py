"""nk_paged.py — a KV cache of pages for sequences of their own lengths.

The reference's KvCache (cache.rs:74-110) and nk.KvCache hold one length for
the whole batch.  PagedKvCache keeps the keys and values of every sequence in
pages of one pool (nk.KvPages, shared by the layers), so that sequences grow,
fork, drop tokens and end on their own:

    cache = PagedKvCache(pages, kv_heads, head_dim, max_seqs=.., max_len=..)
    s = cache.new_sequence()
    step = cache.step([s], [T])            # reserves the step's slots
    cache.append(step, k, v, layer=i)      # per layer
    o = cache.attend(q, step, q_heads, layer=i)
    child = cache.fork(s)                  # shares full pages
    cache.accept(step, [[0, 3, 7]])        # keeps a drafted branch
    cache.free(s)

Which page belongs to whom is host bookkeeping (reference counts and a stack
of free pages); the device sees page tables and lengths that it uploads
through kernel parameters, so no call waits for the GPU.  Calls must be issued
on one stream, or on streams that the caller orders: a freed page is handed
out again at once, and the stream's order keeps its readers ahead of its next
writer.
"""
from __future__ import annotations

import numpy as np

import nk


class PagedStep:
    """The ragged batch of one step: device arrays for the kernels (start,
    kv_len, rows) and what the host knows of them."""

    def __init__(self, seqs, counts, lens, arrays):
        n = len(seqs)
        self.seqs, self.counts, self.lens = list(seqs), list(counts), list(lens)
        self.start, self.kv_len, self.rows = arrays[:n + 1], arrays[n + 1:2 * n + 1], \
            arrays[2 * n + 1:]
        self.tokens = int(sum(counts))
        self.max_new = int(max(counts, default=0))
        self.max_kv = int(max(lens, default=0))


class PagedKvCache:
    """KV pages of up to max_seqs sequences of up to max_len tokens.

    pages: pages of the pool, page_size: tokens of a page (16, 32, 64 or 128),
    layers: attention layers that share the tables, bounds: keep the key
    bounds that attend_sparse needs."""

    def __init__(self, pages, kv_heads, head_dim, *, max_seqs, max_len, page_size=64, layers=1,
                 bounds=True, device="cuda"):
        import torch

        if pages <= 0 or max_seqs <= 0 or max_len <= 0:
            raise ValueError("pages, max_seqs and max_len must be positive")
        self.page_size, self.layers, self.max_len = page_size, layers, max_len
        self.width = -(-max_len // page_size)
        shape = (layers, pages, kv_heads, page_size, head_dim)
        k = torch.empty(shape, dtype=torch.bfloat16, device=device)
        v = torch.empty_like(k)
        lo = hi = None
        if bounds:
            lo = torch.zeros(layers, pages, kv_heads, head_dim, dtype=torch.bfloat16,
                             device=device)
            hi = torch.zeros_like(lo)
        table = torch.zeros(max_seqs, self.width, dtype=torch.int32, device=device)
        self._init_host(pages, max_seqs)
        self._bounds = bool(bounds)
        self._bind(k, v, table, lo, hi)

    _bounds = True  # key bounds are kept

    def _bind(self, k, v, table, lo, hi):
        self.pages = nk.KvPages(k, v, table, k_min=lo, k_max=hi)

    def _init_host(self, pages, max_seqs):
        self._refs = np.zeros(pages, np.int32)
        self._free = list(range(pages - 1, -1, -1))  # a stack: the last freed page is used next
        self._table = np.full((max_seqs, self.width), -1, np.int32)
        self._len = np.zeros(max_seqs, np.int64)
        self._live = np.zeros(max_seqs, bool)

    # ---- device work the bookkeeping asks for (one method each) -------------
    def _copy_pages(self, src, dst, stream):
        nk.kv_pages_copy(self.pages, src, dst, stream=stream)

    def _write_table(self, offsets, values, stream):
        nk.kv_table_write(self.pages.table, values, offsets, stream=stream)

    def _compact(self, step, base, keep, n_keep, stream):
        nk.kv_pages_compact(self.pages, step.kv_len, base, keep, n_keep, rows=step.rows,
                            stream=stream)

    def _upload(self, values, stream):
        import torch

        out = nk._empty(len(values), torch.int32, self.pages.device, stream)
        nk.kv_table_write(out, values, stream=stream)
        return out

    # ---- state ------------------------------------------------------------------
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq) -> int:
        return int(self._len[self._check(seq)])

    def page_ids(self, seq):
        """The sequence's pages in order (host ints)."""
        self._check(seq)
        return self._table[seq, :self._blocks(self._len[seq])].tolist()

    def refcount(self, page) -> int:
        return int(self._refs[page])

    def _blocks(self, length) -> int:
        return -(-int(length) // self.page_size)

    def _check(self, seq):
        if not 0 <= seq < len(self._live) or not self._live[seq]:
            raise ValueError(f"no sequence {seq}")
        return seq

    def _take(self, n):
        if n > len(self._free):
            raise RuntimeError(f"out of pages: {n} needed, {len(self._free)} free")
        out = [self._free.pop() for _ in range(n)]
        self._refs[out] = 1
        return out

    def _drop(self, ids):
        """Gives up one reference to each page; the last one frees it."""
        for p in ids:
            self._refs[p] -= 1
            if self._refs[p] == 0:
                self._free.append(int(p))

    # ---- sequences --------------------------------------------------------------
    def new_sequence(self) -> int:
        """An empty sequence: the row of the page table that it owns."""
        free = np.flatnonzero(~self._live)
        if free.size == 0:
            raise RuntimeError("out of sequences")
        s = int(free[0])
        self._live[s], self._len[s] = True, 0
        return s

    def free(self, seq) -> None:
        """Ends the sequence and gives its pages back."""
        self._check(seq)
        self._drop(self._table[seq, :self._blocks(self._len[seq])][::-1])
        self._table[seq] = -1
        self._live[seq], self._len[seq] = False, 0

    def fork(self, seq, stream=None) -> int:
        """A new sequence with the same tokens: full pages are shared, the
        partial last page is copied (both sequences may append to it)."""
        self._check(seq)
        length = int(self._len[seq])
        full, blocks = length // self.page_size, self._blocks(length)
        if blocks > full and not self._free:
            raise RuntimeError("out of pages: 1 needed, 0 free")
        child = self.new_sequence()
        ids = self._table[seq, :blocks].copy()
        self._refs[ids[:full]] += 1
        if blocks > full:
            fresh = self._take(1)[0]
            self._copy_pages([int(ids[full])], [fresh], stream)
            ids[full] = fresh
        self._table[child, :blocks], self._len[child] = ids, length
        if blocks:
            self._write_table(child * self.width + np.arange(blocks), ids, stream)
        return child

    # ---- steps ------------------------------------------------------------------
    def step(self, seqs, counts, stream=None) -> PagedStep:
        """Reserves slots for counts[i] new tokens of seqs[i] and returns the
        step.  A shared page that would be written is copied first.  Nothing
        changes when pages run out."""
        seqs, counts = [int(s) for s in seqs], [int(c) for c in counts]
        if len(seqs) != len(counts):
            raise ValueError("seqs and counts must have one length")
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence appears twice in one step")
        if any(c < 0 for c in counts):
            raise ValueError("counts must not be negative")
        need, last = 0, {}  # writers of a shared page: the last one keeps it
        for s, c in zip(seqs, counts):
            self._check(s)
            if self._len[s] + c > self.max_len:
                raise ValueError(f"sequence {s} would pass max_len {self.max_len}")
            need += self._blocks(self._len[s] + c) - self._blocks(self._len[s])
            page = self._partial_page(s, c)
            if page is not None:
                left = last.get(page, int(self._refs[page]))
                if left > 1:
                    need += 1
                    last[page] = left - 1
        if need > len(self._free):
            raise RuntimeError(f"out of pages: {need} needed, {len(self._free)} free")
        src, dst, offsets, values = [], [], [], []
        for s, c in zip(seqs, counts):
            old = int(self._len[s])
            page = self._partial_page(s, c)
            if page is not None and self._refs[page] > 1:
                self._replace(s, old // self.page_size, src, dst, offsets, values)
            b0, b1 = self._blocks(old), self._blocks(old + c)
            if b1 > b0:
                fresh = self._take(b1 - b0)
                self._table[s, b0:b1] = fresh
                offsets += range(s * self.width + b0, s * self.width + b1)
                values += fresh
            self._len[s] = old + c
        self._flush(src, dst, offsets, values, stream)
        lens = [int(self._len[s]) for s in seqs]
        start = np.concatenate([[0], np.cumsum(counts)]) if counts else np.zeros(1)
        arrays = self._upload(np.concatenate([start, lens, seqs]).astype(np.int32), stream)
        return PagedStep(seqs, counts, lens, arrays)

    def _partial_page(self, s, c):
        """The page that c new tokens of s would share with older ones."""
        old = int(self._len[s])
        return int(self._table[s, old // self.page_size]) if c and old % self.page_size else None

    def _replace(self, s, block, src, dst, offsets, values):
        """Gives s a copy of a shared page of its own."""
        page = int(self._table[s, block])
        fresh = self._take(1)[0]
        self._refs[page] -= 1
        self._table[s, block] = fresh
        src.append(page)
        dst.append(fresh)
        offsets.append(s * self.width + block)
        values.append(fresh)

    def _flush(self, src, dst, offsets, values, stream):
        if src:
            self._copy_pages(src, dst, stream)
        if offsets:
            # one entry a slot: a page replaced and then extended appears once
            self._write_table(np.array(offsets, np.int64), values, stream)

    def append(self, step: PagedStep, k_new, v_new, layer=0, stream=None) -> None:
        """Stores the step's keys and values (bf16 [tokens, kv_heads * head_dim])."""
        nk.kv_pages_append(self.pages, k_new, v_new, step.start, step.kv_len,
                           max_new=step.max_new, max_kv=step.max_kv, rows=step.rows, layer=layer,
                           stream=stream)

    def attend(self, q, step: PagedStep, q_heads, *, layer=0, tree_mask=None, scale=None,
               out_dtype=nk.BF16, out=None, workspace=None, stream=None):
        """nk.attention_paged of the step's queries (drafts with tree_mask)."""
        return nk.attention_paged(q, self.pages, step.start, step.kv_len, q_heads,
                                  max_q=step.max_new, max_kv=step.max_kv, tree_mask=tree_mask,
                                  rows=step.rows, layer=layer, scale=scale, out_dtype=out_dtype,
                                  out=out, workspace=workspace, stream=stream)

    def attend_sparse(self, q, step: PagedStep, q_heads, top_k, *, sink=1, local=1, layer=0,
                      scale=None, out_dtype=nk.BF16, out=None, stream=None):
        """nk.attention_paged_sparse of the step's queries: (out, blocks)."""
        return nk.attention_paged_sparse(q, self.pages, step.start, step.kv_len, q_heads, top_k,
                                         sink=sink, local=local, max_q=step.max_new,
                                         max_kv=step.max_kv, rows=step.rows, layer=layer,
                                         scale=scale, out_dtype=out_dtype, out=out, stream=stream)

    def accept(self, step: PagedStep, keep, stream=None) -> None:
        """Keeps, of each of the step's sequences, the new tokens keep[i]
        (ascending indexes within the step: the accepted path of a draft tree)
        and drops the others: the kept ones close up behind the older tokens
        and pages that empty are given back.  Every sequence must still have
        the length that the step left it with."""
        if len(keep) != len(step.seqs):
            raise ValueError("keep must have a list for each sequence of the step")
        keep = [[int(x) for x in row] for row in keep]
        for s, c, length, row in zip(step.seqs, step.counts, step.lens, keep):
            self._check(s)
            if self._len[s] != length:
                raise ValueError(f"sequence {s} has changed since the step")
            if any(b <= a for a, b in zip([-1] + row, row)) or (row and row[-1] >= c):
                raise ValueError("kept indexes must be ascending and within the step")
        n = len(keep)
        if n == 0:
            return
        # Slots and bounds that the move writes must not be shared with a fork.
        jobs, need, left = [], 0, {}
        for s, c, length, row in zip(step.seqs, step.counts, step.lens, keep):
            base = length - c
            first, end = base // self.page_size, self._blocks(base + len(row))
            if not row and not self._bounds:
                end = first
            for b in range(first, end):
                page = int(self._table[s, b])
                refs = left.get(page, int(self._refs[page]))
                if refs > 1:
                    jobs.append((s, b))
                    need += 1
                    left[page] = refs - 1
        if need > len(self._free):
            raise RuntimeError(f"out of pages: {need} needed, {len(self._free)} free")
        src, dst, offsets, values = [], [], [], []
        for s, b in jobs:
            self._replace(s, b, src, dst, offsets, values)
        self._flush(src, dst, offsets, values, stream)
        width = max(1, max(len(row) for row in keep))
        packed = np.zeros((n, width), np.int32)
        for i, row in enumerate(keep):
            packed[i, :len(row)] = row
        base = np.array(step.lens) - np.array(step.counts)
        counts = np.array([len(row) for row in keep])
        arrays = self._upload(np.concatenate([base, counts, packed.reshape(-1)]).astype(np.int32),
                              stream)
        self._compact(step, arrays[:n], arrays[2 * n:].reshape(n, width), arrays[n:2 * n], stream)
        for s, b, c in zip(step.seqs, base, counts):
            self._shorten(s, int(b + c))

    def _shorten(self, s, length):
        b0, b1 = self._blocks(length), self._blocks(self._len[s])
        self._drop(self._table[s, b0:b1][::-1])
        self._table[s, b0:b1] = -1
        self._len[s] = length

    def truncate(self, seq, length, stream=None) -> None:
        """Drops the tokens from position `length` on; the bounds of the last
        page left are taken anew over what it still holds (in a copy, which
        takes a free page, when a fork shares it)."""
        self._check(seq)
        old = int(self._len[seq])
        if not 0 <= length <= old:
            raise ValueError(f"length must lie in 0 .. {old}")
        arrays = self._upload(np.array([0, old - length, old, seq], np.int32), stream)
        self.accept(PagedStep([seq], [old - length], [old], arrays), [[]], stream)
