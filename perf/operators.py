"""Paged KV cache operators: what is measured.

Five operators of the serving path, each in a plain form (elementary torch
operations) and as the framework's call:

    append   new keys and values of ragged sequences into their pages, with
             the per-page channel bounds of the keys
    copy     whole pages to other pages in every layer (copy on write, forks)
    compact  kept tokens moved together (accepted drafts in place, evicted
             contexts into fresh pages)
    tree     attention of drafted tokens (or of one token) over paged caches
    sparse   blocks chosen for each query by an upper bound of its scores,
             then attention over those blocks

Layout: k, v bf16 [layers, pages, kv_heads, page_size, head_dim]; k_min,
k_max bf16 [layers, pages, kv_heads, head_dim]; table int32 [sequences,
blocks]: the token at position p of sequence s is slot p % page_size of page
table[s, p // page_size].
"""
import math
import os
import sys
import zlib

import numpy as np
import torch

own = False

DEV = "cuda"


def _nk():
    """The framework's binding, from the repository that is the working folder."""
    path = os.path.join(os.getcwd(), "nemotron-cutile-rs_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import nk

    return nk


# ------------------------------------------------------------------- cases
def listed():
    return [
        # One sampled branch leaves a shared prompt: its partial page is copied
        # in the decoder's six attention layers (2 KV heads of 128).
        dict(name="copy_one_fork", op="copy", layers=6, pages=512, kv_heads=2, page_size=64,
             head_dim=128, pairs=1),
        # Beam search over a full batch: many pages copied at once.
        dict(name="copy_beams", op="copy", layers=2, pages=4096, kv_heads=8, page_size=16,
             head_dim=128, pairs=1531),
        # A decode step of 64 sequences: one token each, ragged positions.
        dict(name="append_decode", op="append", seqs=64, kv_heads=2, page_size=64, head_dim=128,
             max_new=1, max_prev=1279),
        # Prompts of up to 1024 tokens written by a prefill, some behind a
        # cached prefix.
        dict(name="append_prefill", op="append", seqs=16, kv_heads=8, page_size=32, head_dim=128,
             max_new=1024, max_prev=517),
        # Drafts verified: the accepted path of each tree closes up in place.
        dict(name="compact_accept", op="compact", seqs=64, layers=6, kv_heads=2, page_size=64,
             head_dim=128, max_len=1280, draft=32, max_keep=6, in_place=True),
        # Long contexts thinned to a quarter of their tokens, into fresh pages.
        dict(name="compact_evict", op="compact", seqs=4, layers=1, kv_heads=8, page_size=64,
             head_dim=128, max_len=32768, draft=0, max_keep=8192, in_place=False),
        # One user, one token: latency over a short context.
        dict(name="decode_one", op="tree", seqs=1, q_heads=32, kv_heads=2, page_size=64,
             head_dim=128, max_draft=1, max_len=1025, tree=False),
        # The decode step of the decoder's batch over long ragged contexts.
        dict(name="decode_batch", op="tree", seqs=64, q_heads=32, kv_heads=2, page_size=64,
             head_dim=128, max_draft=1, max_len=8192, tree=False),
        # Small trees, small pages, few query heads to a KV head.
        dict(name="tree_small", op="tree", seqs=5, q_heads=16, kv_heads=4, page_size=16,
             head_dim=64, max_draft=7, max_len=777, tree=True),
        # Wide trees of 64 drafts over long contexts: the largest products.
        dict(name="tree_wide", op="tree", seqs=8, q_heads=32, kv_heads=2, page_size=64,
             head_dim=128, max_draft=64, max_len=8192, tree=True),
        # Long documents, one token each: bounds of 2048 blocks, 64 are read.
        dict(name="sparse_long", op="sparse", seqs=4, q_heads=32, kv_heads=2, page_size=64,
             head_dim=128, max_draft=1, max_len=131072, top_k=64, sink=1, local=2),
        # A batch of medium contexts with two tokens a step and small blocks.
        dict(name="sparse_batch", op="sparse", seqs=32, q_heads=32, kv_heads=8, page_size=32,
             head_dim=64, max_draft=2, max_len=9000, top_k=48, sink=1, local=1),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["copy", "append", "compact", "tree", "tree", "sparse"])
    ps = rng.choice([16, 32, 64, 128])
    d = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 8])
    if op == "copy":
        layers = rng.randint(1, 6)
        pages = _log(rng, 8, 4096 * 2 * 8 * 16 * 128 // (layers * kv * ps * d))
        return dict(op=op, layers=layers, pages=pages, kv_heads=kv, page_size=ps, head_dim=d,
                    pairs=_log(rng, 1, max(1, min(1531, pages * 3 // 8))))
    if op == "append":
        seqs = _log(rng, 1, 64)
        new = _log(rng, 1, 1024)
        while seqs * new * kv * d > 16 * 1024 * 8 * 128:
            new = max(1, new // 2)
        return dict(op=op, seqs=seqs, kv_heads=kv, page_size=ps, head_dim=d, max_new=new,
                    max_prev=_log(rng, 1, 2048))
    if op == "compact":
        if rng.random() < 0.5:
            return dict(op=op, seqs=_log(rng, 1, 64), layers=rng.randint(1, 6), kv_heads=min(kv, 2),
                        page_size=ps, head_dim=d, max_len=_log(rng, 65, 1280),
                        draft=rng.randint(2, 64), max_keep=rng.randint(1, 12), in_place=True)
        length = _log(rng, 64, 32768)
        return dict(op=op, seqs=rng.randint(1, 4), layers=1, kv_heads=kv, page_size=ps, head_dim=d,
                    max_len=length, draft=0, max_keep=max(1, int(length * rng.uniform(0.05, 0.25))),
                    in_place=False)
    group = rng.choice([1, 2, 4, 8, 16])
    kv = min(kv, max(1, 32 // group))
    seqs = _log(rng, 1, 64)
    if op == "tree":
        draft = _log(rng, 1, 64)
        length = _log(rng, draft + 1, 8192)
        # at most the widest listed tree's products and the largest listed cache
        while seqs > 1 and (seqs * draft * group * kv * d * length > 8 * 64 * 32 * 128 * 8192 or
                            seqs * kv * d * length > 64 * 2 * 128 * 8192):
            seqs = max(1, seqs // 2)
        return dict(op=op, seqs=seqs, q_heads=kv * group, kv_heads=kv, page_size=ps, head_dim=d,
                    max_draft=draft, max_len=length, tree=draft > 1 and rng.random() < 0.8)
    length = _log(rng, 256, 131072)
    while seqs > 1 and seqs * kv * d * length > 4 * 2 * 128 * 131072:
        seqs = max(1, seqs // 2)
    while seqs * kv * d * length > 4 * 2 * 128 * 131072:
        length //= 2
    sink, local = rng.randint(0, 2), rng.randint(1, 3)
    return dict(op=op, seqs=seqs, q_heads=kv * group, kv_heads=kv, page_size=ps, head_dim=d,
                max_draft=rng.randint(1, 3), max_len=length, top_k=rng.randint(sink + local, 64),
                sink=sink, local=local)


# ------------------------------------------------------------------ inputs
class _State:
    """What a serving program holds before the call."""


def _lengths(rng, n, lo, hi):
    """n whole numbers in [lo, hi]; the first is hi."""
    out = rng.integers(lo, hi + 1, n).astype(np.int32)
    out[0] = hi
    return out


def _counts(case):
    """The ragged lengths of a case's sequences: they belong to the case, so
    that inputs of another seed have the same shapes."""
    text = repr(sorted((key, x) for key, x in case.items() if key != "name"))
    rng = np.random.default_rng(zlib.crc32(text.encode()))
    n, op = case["seqs"], case["op"]
    c = {}
    if op == "append":
        c["prev"] = rng.integers(0, case["max_prev"] + 1, n).astype(np.int32)
        c["new"] = _lengths(rng, n, 1, case["max_new"])
        c["lens"] = c["prev"] + c["new"]
    elif op == "compact" and case["in_place"]:
        room = max(1, case["max_len"] - case["draft"])
        c["base"] = rng.integers(1, room + 1, n).astype(np.int32)
        c["lens"] = c["base"] + case["draft"]
        # the kept drafts lie behind the slots that they close up to
        most = max(1, min(case["max_keep"], (case["draft"] + 1) // 2))
        c["n_keep"] = rng.integers(1, most + 1, n).astype(np.int32)
    elif op == "compact":
        c["base"] = np.zeros(n, np.int32)
        c["lens"] = _lengths(rng, n, max(1, case["max_len"] // 2), case["max_len"])
        c["n_keep"] = np.minimum(_lengths(rng, n, max(1, case["max_keep"] // 2), case["max_keep"]),
                                 c["lens"])
    else:
        c["draft"] = _lengths(rng, n, 1, case["max_draft"])
        low = max(case["max_draft"], case["max_len"] // 4)
        c["lens"] = _lengths(rng, n, low, case["max_len"])
    return c


def _table(rng, blocks, pages, width):
    """Distinct random pages for sequences of blocks[i] blocks each."""
    order = rng.permutation(pages).astype(np.int32)
    table = np.zeros((len(blocks), width), np.int32)
    at = 0
    for i, b in enumerate(blocks):
        table[i, :b] = order[at:at + b]
        at += int(b)
    return table


def _pools(case, gen, layers, pages):
    shape = (layers, pages, case["kv_heads"], case["page_size"], case["head_dim"])
    k = torch.empty(shape, dtype=torch.bfloat16, device=DEV).normal_(generator=gen)
    v = torch.empty(shape, dtype=torch.bfloat16, device=DEV).normal_(generator=gen)
    return k, v


def _bounds(k, table, lens, ps):
    """Channel bounds of the valid slots of every sequence's pages (others 0)."""
    layers, pages, heads, _, d = k.shape
    k_min = torch.zeros(layers, pages, heads, d, dtype=k.dtype, device=k.device)
    k_max = torch.zeros_like(k_min)
    for row, length in zip(table, lens):
        n = -(-int(length) // ps)
        if n == 0:
            continue
        ids = torch.as_tensor(row[:n].astype(np.int64), device=k.device)
        part = k[:, ids]
        lo, hi = part.amin(3), part.amax(3)
        tail = int(length) - (n - 1) * ps
        lo[:, n - 1] = part[:, n - 1, :, :tail].amin(2)
        hi[:, n - 1] = part[:, n - 1, :, :tail].amax(2)
        k_min[:, ids] = lo
        k_max[:, ids] = hi
    return k_min, k_max


def _starts(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def _dev(a):
    return torch.as_tensor(a, device=DEV)


def _tree_masks(rng, counts):
    """Bit j of a draft's word: it attends draft j (its ancestors and itself)."""
    words = []
    for t in counts:
        masks = []
        for i in range(int(t)):
            m = 1 << i
            if i:
                m |= masks[int(rng.integers(0, i))]
            masks.append(m)
        words += masks
    return np.array(words, np.uint64).view(np.int64)


def _accepted(rng, draft, n):
    """A path of n drafts: the root, then drafts behind the kept slots."""
    rest = n + np.sort(rng.choice(draft - n, n - 1, replace=False)) if n > 1 else []
    return np.concatenate([[0], rest]).astype(np.int32)


def prepare(case, seed):
    s = _State()
    s.case = case
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    op, ps = case["op"], case["page_size"]
    if op == "copy":
        s.k, s.v = _pools(case, gen, case["layers"], case["pages"])
        s.k_min, s.k_max = s.k.amin(3), s.k.amax(3)
        ids = rng.permutation(case["pages"]).astype(np.int32)
        s.dst = ids[:case["pairs"]]
        # several branches may leave one page
        s.src = rng.choice(ids[case["pairs"]:], case["pairs"]).astype(np.int32)
        s.table = np.zeros((1, 1), np.int32)
    else:
        c = _counts(case)
        n, s.kv_len = case["seqs"], c["lens"]
        blocks = -(-s.kv_len // ps)
        fresh = np.zeros(0, np.int64)
        if op == "compact" and not case["in_place"]:
            fresh = -(-c["n_keep"] // ps)
        pages = int(blocks.sum() + fresh.sum()) + 8
        both = _table(rng, np.concatenate([blocks, fresh]).astype(int), pages, int(blocks.max()))
        s.table, s.dst_table = both[:n], both[n:] if len(fresh) else None
        s.k, s.v = _pools(case, gen, case.get("layers", 1), pages)
        s.k_min = s.k_max = None
    if op == "append":
        s.k_min, s.k_max = _bounds(s.k, s.table, c["prev"], ps)
        s.start, s.max_new = _starts(c["new"]), int(c["new"].max())
        kvd = case["kv_heads"] * case["head_dim"]
        # the K and V projections write one fused row
        fused = torch.empty(int(s.start[-1]), 2 * kvd, dtype=torch.bfloat16,
                            device=DEV).normal_(generator=gen)
        s.k_new, s.v_new = fused[:, :kvd], fused[:, kvd:]
    elif op == "compact":
        s.base, s.n_keep = c["base"], c["n_keep"]
        s.keep = np.full((n, case["max_keep"]), -1, np.int32)
        for i, m in enumerate(s.n_keep):
            s.keep[i, :m] = _accepted(rng, case["draft"], int(m)) if case["in_place"] else \
                np.sort(rng.choice(int(s.kv_len[i]), m, replace=False))
        s.k_min, s.k_max = _bounds(s.k, s.table, s.kv_len, ps)
    elif op in ("tree", "sparse"):
        s.start, s.max_draft, s.max_kv = _starts(c["draft"]), int(c["draft"].max()), \
            int(s.kv_len.max())
        s.q = torch.empty(int(s.start[-1]), case["q_heads"] * case["head_dim"],
                          dtype=torch.bfloat16, device=DEV).normal_(generator=gen)
        s.tree_mask = _tree_masks(rng, c["draft"]) if case.get("tree") else None
        if op == "sparse":
            s.k_min, s.k_max = _bounds(s.k, s.table, s.kv_len, ps)
    s.table_host = s.table
    s.table = _dev(s.table)
    for name in ("start", "kv_len", "base", "n_keep", "keep", "tree_mask", "dst_table"):
        a = getattr(s, name, None)
        setattr(s, name + "_host", a)
        setattr(s, name, None if a is None else _dev(a))
    if own:
        s.nk = _nk()
        s.pages = s.nk.KvPages(s.k, s.v, s.table, k_min=s.k_min, k_max=s.k_max)
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    op = state.case["op"]
    return (_OWN if own else _PLAIN)[op](state)


def _own_copy(s):
    s.nk.kv_pages_copy(s.pages, s.src, s.dst)
    return s.k, s.v, s.k_min, s.k_max


def _own_append(s):
    s.nk.kv_pages_append(s.pages, s.k_new, s.v_new, s.start, s.kv_len, max_new=s.max_new)
    return s.k, s.v, s.k_min, s.k_max


def _own_compact(s):
    new_len = s.nk.kv_pages_compact(s.pages, s.kv_len, s.base, s.keep, s.n_keep,
                                    dst_table=s.dst_table)
    return s.k, s.v, s.k_min, s.k_max, new_len


def _own_tree(s):
    return s.nk.attention_paged(s.q, s.pages, s.start, s.kv_len, s.case["q_heads"],
                                max_q=s.max_draft, max_kv=s.max_kv, tree_mask=s.tree_mask)


def _own_sparse(s):
    c = s.case
    return s.nk.attention_paged_sparse(s.q, s.pages, s.start, s.kv_len, c["q_heads"], c["top_k"],
                                       sink=c["sink"], local=c["local"], max_q=s.max_draft,
                                       max_kv=s.max_kv)


def _plain_copy(s):
    src = torch.as_tensor(s.src.astype(np.int64), device=DEV)
    dst = torch.as_tensor(s.dst.astype(np.int64), device=DEV)
    for t in (s.k, s.v, s.k_min, s.k_max):
        t[:, dst] = t[:, src]
    return s.k, s.v, s.k_min, s.k_max


def _page_bounds(k, ids, valid):
    """Bounds of pages ids over their first valid slots (valid > 0)."""
    part = k[:, ids].float()
    dead = torch.arange(k.shape[3], device=k.device)[None, :] >= valid[:, None]
    dead = dead[None, :, None, :, None]
    lo = part.masked_fill(dead, float("inf")).amin(3)
    hi = part.masked_fill(dead, float("-inf")).amax(3)
    return lo.to(k.dtype), hi.to(k.dtype)


def _plain_append(s):
    ps, d = s.case["page_size"], s.case["head_dim"]
    heads = s.case["kv_heads"]
    start, lens = s.start_host, s.kv_len_host
    new = np.diff(start)
    seq = np.repeat(np.arange(len(new)), new)
    pos = np.arange(start[-1]) - start[seq] + (lens - new)[seq]
    page = torch.as_tensor(s.table_host[seq, pos // ps].astype(np.int64), device=DEV)
    slot = torch.as_tensor(pos % ps, device=DEV)
    s.k[0, page, :, slot] = s.k_new.reshape(-1, heads, d)
    s.v[0, page, :, slot] = s.v_new.reshape(-1, heads, d)
    ids, valid = [], []
    for b in range(len(new)):
        first, last = (lens[b] - new[b]) // ps, (lens[b] - 1) // ps
        for j in range(first, last + 1):
            ids.append(int(s.table_host[b, j]))
            valid.append(min(ps, int(lens[b]) - j * ps))
    ids = torch.tensor(ids, device=DEV)
    s.k_min[:, ids], s.k_max[:, ids] = _page_bounds(s.k, ids, torch.tensor(valid, device=DEV))
    return s.k, s.v, s.k_min, s.k_max


def _plain_compact(s):
    ps = s.case["page_size"]
    to = s.table_host if s.dst_table_host is None else s.dst_table_host
    sp, ss, dp, ds, ids, valid = [], [], [], [], [], []
    for b in range(s.case["seqs"]):
        base, n = int(s.base_host[b]), int(s.n_keep_host[b])
        src = base + s.keep_host[b, :n].astype(np.int64)
        dst = base + np.arange(n)
        sp.append(s.table_host[b, src // ps])
        ss.append(src % ps)
        dp.append(to[b, dst // ps])
        ds.append(dst % ps)
        for j in range(base // ps, -(-(base + n) // ps)):
            ids.append(int(to[b, j]))
            valid.append(min(ps, base + n - j * ps))
    sp, ss, dp, ds = (torch.as_tensor(np.concatenate(x).astype(np.int64), device=DEV)
                      for x in (sp, ss, dp, ds))
    for t in (s.k, s.v):
        t[:, dp, :, ds] = t[:, sp, :, ss]
    ids = torch.tensor(ids, device=DEV)
    s.k_min[:, ids], s.k_max[:, ids] = _page_bounds(s.k, ids, torch.tensor(valid, device=DEV))
    return s.k, s.v, s.k_min, s.k_max, s.base + s.n_keep


def _gather(pool, row, length):
    """Tokens 0..length-1 of a sequence, [kv_heads, length, head_dim]."""
    ps = pool.shape[3]
    ids = row[:-(-length // ps)].long()
    x = pool[0, ids].transpose(0, 1)
    return x.reshape(x.shape[0], -1, x.shape[-1])[:, :length]


def _softmax_sum(scores, v):
    """Rows of softmax(scores) times v; rows with no allowed key give 0."""
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top) & (top < 0), torch.zeros_like(top), top)
    w = torch.exp(scores - top)
    total = w.sum(-1, keepdim=True)
    out = w @ v
    return torch.where(total == 0, torch.zeros_like(out), out / total)


def _plain_tree(s):
    c = s.case
    heads, kv, d = c["q_heads"], c["kv_heads"], c["head_dim"]
    group = heads // kv
    out = torch.empty_like(s.q)
    shift = torch.arange(64, device=DEV)
    for b in range(c["seqs"]):
        a, e, length = int(s.start_host[b]), int(s.start_host[b + 1]), int(s.kv_len_host[b])
        t = e - a
        k = _gather(s.k, s.table[b], length).float()
        v = _gather(s.v, s.table[b], length).float()
        q = s.q[a:e].float().reshape(t, kv, group, d).permute(1, 0, 2, 3).reshape(kv, t * group, d)
        allowed = torch.ones(t, length, dtype=torch.bool, device=DEV)
        if s.tree_mask is not None:
            allowed[:, length - t:] = ((s.tree_mask[a:e, None] >> shift[:t]) & 1) != 0
        else:
            place = torch.arange(length, device=DEV)
            allowed = place[None, :] <= length - t + torch.arange(t, device=DEV)[:, None]
        scores = (q @ k.transpose(1, 2)) * (1.0 / math.sqrt(d))
        scores = scores.reshape(kv, t, group, length)
        scores = scores.masked_fill(~allowed[None, :, None, :], float("-inf"))
        o = _softmax_sum(scores.reshape(kv, t * group, length), v)
        out[a:e] = o.reshape(kv, t, group, d).permute(1, 0, 2, 3).reshape(t, heads * d)
    return out


def _plain_sparse(s):
    c = s.case
    heads, kv, d, ps = c["q_heads"], c["kv_heads"], c["head_dim"], c["page_size"]
    group, top_k = heads // kv, c["top_k"]
    out = torch.empty_like(s.q)
    lists = torch.full((s.q.shape[0], kv, top_k), -1, dtype=torch.int32, device=DEV)
    for b in range(c["seqs"]):
        a, e, length = int(s.start_host[b]), int(s.start_host[b + 1]), int(s.kv_len_host[b])
        t = e - a
        ids = s.table[b, :-(-length // ps)].long()
        lo, hi = s.k_min[0, ids].double(), s.k_max[0, ids].double()  # [blocks, kv, d]
        k = _gather(s.k, s.table[b], length).float()
        v = _gather(s.v, s.table[b], length).float()
        for i in range(t):
            pos = length - t + i
            n = pos // ps + 1
            q = s.q[a + i].reshape(kv, group, d)
            # the largest product over a block's bounds, 64-bit sums: a list
            # must not hang on the order of a sum
            pos_q, neg_q = q.double().clamp(min=0), q.double().clamp(max=0)
            score = torch.einsum("hgd,jhd->hgj", pos_q, hi[:n]) + \
                torch.einsum("hgd,jhd->hgj", neg_q, lo[:n])
            score = score.amax(1)
            block = torch.arange(n, device=DEV)
            forced = (block < c["sink"]) | (block >= n - c["local"])
            score = score.masked_fill(forced[None, :], float("inf"))
            m = min(top_k, n)
            # a stable descending sort: ties go to the lower index
            order = torch.sort(score, dim=1, descending=True, stable=True)[1][:, :m]
            order = torch.sort(order, dim=1)[0]
            lists[a + i, :, :m] = order.int()
            allowed = torch.zeros(kv, n, dtype=torch.bool, device=DEV).scatter_(1, order, True)
            allowed = allowed.repeat_interleave(ps, 1)[:, :pos + 1]
            sc = (q.float() @ k[:, :pos + 1].transpose(1, 2)) * (1.0 / math.sqrt(d))
            sc = sc.masked_fill(~allowed[:, None, :], float("-inf"))
            out[a + i] = _softmax_sum(sc, v[:, :pos + 1]).reshape(-1)
    return out, lists


_PLAIN = dict(copy=_plain_copy, append=_plain_append, compact=_plain_compact, tree=_plain_tree,
              sparse=_plain_sparse)
_OWN = dict(copy=_own_copy, append=_own_append, compact=_own_compact, tree=_own_tree,
            sparse=_own_sparse)


# ---------------------------------------------------------------------- work
def work(case):
    op, kv, ps, d = case["op"], case["kv_heads"], case["page_size"], case["head_dim"]
    bounds = 2 * kv * d * 2  # one page's
    token = 2 * kv * d * 2   # one token's key and value
    if op == "copy":
        return {"bytes": 2 * case["pairs"] * case["layers"] * (ps * token + bounds), "flops": 0}
    c = _counts(case)
    if op == "append":
        pages = (c["lens"] - 1) // ps - c["prev"] // ps + 1
        return {"bytes": int(2 * c["new"].sum() * token + pages.sum() * bounds), "flops": 0}
    if op == "compact":
        pages = -(-(c["base"] + c["n_keep"]) // ps) - c["base"] // ps
        return {"bytes": int(case["layers"] * (2 * c["n_keep"].sum() * token +
                                               pages.sum() * bounds)), "flops": 0}
    heads, lens, draft = case["q_heads"], c["lens"].astype(np.int64), c["draft"].astype(np.int64)
    io = int(2 * draft.sum() * heads * d * 2)
    if op == "tree":
        return {"bytes": int(lens.sum()) * token + io,
                "flops": int(4 * heads * d * (draft * lens).sum())}
    blocks = -(-lens // ps)
    chosen = np.minimum(case["top_k"], blocks)
    # a sequence's queries may choose the same blocks: each is read at least once
    return {"bytes": int(blocks.sum()) * bounds + int(chosen.sum()) * ps * token + io,
            "flops": int(4 * heads * d * (draft * (chosen * ps + blocks)).sum())}


# --------------------------------------------------------------------- exact
def exact(case, seed):
    """Attention outputs by the definition, in 64 bits, one KV head of one
    sequence at a time; copies and moves have no computed value."""
    op = case["op"]
    if op not in ("tree", "sparse"):
        return None
    s = prepare(case, seed)
    kv, d, ps = case["kv_heads"], case["head_dim"], case["page_size"]
    group = case["q_heads"] // kv
    result = torch.zeros(s.q.shape, dtype=torch.float64, device=DEV)
    lists = np.full((s.q.shape[0], kv, case.get("top_k", 1)), -1, np.int32)
    table, lens, start = s.table_host, s.kv_len_host, s.start_host
    for b in range(case["seqs"]):
        length, first, end = int(lens[b]), int(start[b]), int(start[b + 1])
        count = end - first
        at = torch.arange(length, device=DEV)
        page = torch.as_tensor(table[b].astype(np.int64), device=DEV)[at // ps]
        # seen[i, j]: token i's query may attend position j
        seen = np.tri(count, length, length - count, dtype=bool)
        if op == "tree" and s.tree_mask_host is not None:
            for i in range(count):
                word = int(s.tree_mask_host[first + i]) & (2 ** 64 - 1)
                for j in range(count):
                    seen[i, length - count + j] = bool(word >> j & 1)
        for h in range(kv):
            keys = s.k[0, page, h, at % ps].double()
            values = s.v[0, page, h, at % ps].double()
            cols = slice(h * group * d, (h + 1) * group * d)
            q = s.q[first:end, cols].double().reshape(count, group, d)
            use = seen
            if op == "sparse":
                use = seen.copy()
                for i in range(count):
                    use[i] &= np.repeat(_chosen(case, s, b, h, q[i], length - count + i,
                                                lists[first + i, h]),
                                        ps)[:length]
            hidden = ~torch.as_tensor(use, device=DEV)[:, None, :]
            logits = torch.einsum("igd,jd->igj", q, keys) / math.sqrt(d)
            logits.masked_fill_(hidden, -math.inf)
            weight = torch.softmax(logits, -1).masked_fill_(hidden, 0.0)
            result[first:end, cols] = (weight @ values).reshape(count, group * d)
    return result if op == "tree" else (result, torch.as_tensor(lists, device=DEV))


def _chosen(case, s, b, h, q, pos, row):
    """The blocks that the query heads q [group, d] at position pos read;
    writes their list into row and returns them as truth values."""
    ps = case["page_size"]
    last = pos // ps
    page = torch.as_tensor(s.table_host[b, :last + 1].astype(np.int64), device=DEV)
    low, high = s.k_min[0, page, h].double(), s.k_max[0, page, h].double()
    bound = np.max([(torch.where(x >= 0, high, low) @ x).cpu().numpy() for x in q], axis=0)
    block = np.arange(last + 1)
    must = (block < case["sink"]) | (block > last - case["local"])
    order = np.lexsort((block, -bound, ~must))
    take = np.sort(order[:case["top_k"]])
    row[:len(take)] = take
    hit = np.zeros(s.table_host.shape[1], bool)
    hit[take] = True
    return hit
