"""Attention over paged caches on the B200 against the formula in 64 bits.

Tolerance, element by element.  With weights w (sum 1) and values v the
kernel rounds each weight to bf16 (at most 2^-8 of it, so 2^-8 sum w|v| in
all), sums 128 exact products of a score in f32 (128 * 2^-22 * sum|q k| *
scale <= 2^-11 relative in a weight for unit-variance inputs, which also
covers the exponential and the f32 sums), and rounds a bf16 result once
(2^-8 of it):  |error| <= (2^-8 + 2^-11) sum w|v| + [bf16] 2^-8 |out|."""
import numpy as np
import pytest
import torch

import nk
import nk_model
import nk_paged
from gpu_util import dev, host, rel_err, rng
from paged_ref import Paged, attention, bf16, chosen_blocks, ints, starts, tree_masks

pytestmark = pytest.mark.gpu


def _close(got, want, mag, f32=False):
    got = got.double().cpu().numpy().reshape(want.shape)
    tol = (2.0**-8 + 2.0**-11) * mag + (0 if f32 else 2.0**-8) * np.abs(want)
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    bad = ~same & ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], tol[bad][:4])


def _reference(c, q, counts, q_heads, kind, masks=None, lists=None, scale=None, layer=0):
    """[tokens, q_heads, d] and magnitudes for the whole batch."""
    outs, mags, at = [], [], 0
    for s, t in enumerate(counts):
        n = int(c.lens[s])
        seen = np.zeros((t, c.heads if lists is not None else 1, n), bool)
        for i in range(t):
            pos = n - t + i
            if kind == "tree":
                seen[i, 0, :n - t] = True
                seen[i, 0, n - t:] = masks[s][i]
            elif kind == "blocks":
                for h in range(c.heads):
                    for b in lists[at + i][h]:
                        if 0 <= b <= pos // c.ps:
                            seen[i, h, b * c.ps:min(pos + 1, (b + 1) * c.ps)] = True
            else:
                seen[i, 0, :pos + 1] = True
        k, v = c.tokens(c.k, s, layer), c.tokens(c.v, s, layer)
        o, m = attention(q[at:at + t], k, v, seen, c.d ** -0.5 if scale is None else scale)
        outs.append(o)
        mags.append(m)
        at += t
    return np.concatenate(outs), np.concatenate(mags)


CASES = [  # ps, d, kv heads, group, lens, counts
    (16, 64, 1, 1, [1], [1]),                                   # one token in all
    (64, 128, 2, 16, [1025], [1]),                              # split over keys
    (64, 128, 2, 16, [64, 63, 65, 700, 1], [1, 1, 1, 1, 1]),    # page and tile edges
    (32, 64, 4, 4, [777, 31, 200], [7, 3, 0]),                  # a sequence without queries
    (16, 128, 3, 5, [129, 300], [9, 64]),                       # odd heads, 45 and 320 rows
    (128, 64, 2, 8, [513, 1000, 128], [64, 33, 2]),
    (128, 128, 1, 32, [640], [5]),
    (16, 64, 2, 2, [2000], [1]),
    (64, 128, 1, 1, [90, 5000], [64, 17])]


@pytest.mark.parametrize("ps,d,kv,group,lens,counts", CASES)
@pytest.mark.parametrize("kind", ["causal", "tree"])
def test_matches_the_formula(cuda, ps, d, kv, group, lens, counts, kind):
    c = Paged(ps + d + len(lens), lens, kv, ps, d)  # NaN wherever no token is
    H, T = kv * group, sum(counts)
    q = bf16(c.rng.standard_normal((T, H, d)))
    pages = c.device()
    masks, words = [], []
    for t in counts:
        w, seen = tree_masks(c.rng, t)
        masks.append(seen)
        words.append(w)
    tree = torch.from_numpy(np.concatenate(words)).cuda() if kind == "tree" else None
    want, mag = _reference(c, q, counts, H, kind, masks)
    # close bounds (short contexts: a cluster of blocks a unit) and loose ones (a
    # list of tiles that is split anywhere)
    for dt, max_kv in ((nk.BF16, max(lens)), (nk.F32, max(lens)), (nk.BF16, 20000),
                       (nk.F32, 20000)):
        got = nk.attention_paged(dev(q.reshape(T, H * d)).bfloat16(), pages, ints(starts(counts)),
                                 ints(lens), H, max_q=max(counts), max_kv=max_kv,
                                 tree_mask=tree, out_dtype=dt)
        nk.device_status()
        _close(got, want, mag, dt == nk.F32)


@pytest.mark.parametrize("ps,d,kv,group,lens,count", [
    (64, 128, 2, 4, [300], 300), (16, 64, 2, 2, [1000, 257], 257), (32, 128, 1, 8, [190], 130)])
def test_prefill_chunks(cuda, ps, d, kv, group, lens, count):
    c = Paged(3, lens, kv, ps, d)
    counts = [min(count, n) for n in lens]
    T, H = sum(counts), kv * group
    q = bf16(c.rng.standard_normal((T, H, d)))
    got = nk.attention_paged(dev(q.reshape(T, -1)).bfloat16(), c.device(), ints(starts(counts)),
                             ints(lens), H, max_q=max(counts), max_kv=max(lens))
    nk.device_status()
    want, mag = _reference(c, q, counts, H, "causal")
    _close(got, want, mag)


def test_loose_bounds_layers_scale_and_strided_queries(cuda):
    """max_q and max_kv far above what the batch holds, the second of two
    layers, rows of other sequences between, q a view of a fused projection,
    and rows behind the last sequence that keep what they held."""
    c = Paged(8, [100, 40, 333], 2, 32, 64, layers=2, width=40)
    H, d = 4, 64
    counts, rows = [3, 2], [2, 0]
    q = bf16(c.rng.standard_normal((8, H, d)))
    wide = torch.randn(8, H * d + 128, device="cuda").bfloat16()
    wide[:, 64:64 + H * d] = dev(q.reshape(8, -1)).bfloat16()
    out = torch.full((8, H * d), 5.0, device="cuda")
    got = nk.attention_paged(wide[:, 64:64 + H * d], c.device(), ints(starts(counts)),
                             ints([333, 100]), H, rows=ints(rows), layer=1, scale=0.3, out=out)
    nk.device_status()
    o = Paged.__new__(Paged)
    o.__dict__.update(c.__dict__)
    o.table, o.lens = c.table[rows], c.lens[rows]
    want, mag = _reference(o, q, counts, H, "causal", scale=0.3, layer=1)
    # the score error bound scales with the scale: 0.3 / 0.125 of the default's
    _close(got[:5], want, mag * (1 + 2.0**-3), True)
    assert (got[5:] == 5.0).all()


def test_rows_that_see_nothing_are_zero(cuda):
    c = Paged(2, [5, 9], 1, 16, 64)
    q = bf16(c.rng.standard_normal((7, 2, 64)))
    words = [0, 1, 0b11, 0, 0b10000, 0, 0]  # five drafts without a prefix, then two with one
    got = nk.attention_paged(dev(q.reshape(7, -1)).bfloat16(), c.device(), ints([0, 5, 7]),
                             ints([5, 9]), 2, max_q=5, max_kv=9, out_dtype=nk.F32,
                             tree_mask=torch.tensor(words, device="cuda"))
    nk.device_status()
    seen = [np.array([[w >> j & 1 for j in range(5)] for w in words[:5]], bool),
            np.zeros((2, 2), bool)]
    want, mag = _reference(c, q, [5, 2], 2, "tree", seen)
    _close(got, want, mag, True)
    assert not got[0].any() and not got[3].any() and got[5].any()


@pytest.mark.parametrize("group,T", [(1, 6), (8, 6), (16, 9)])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_masked_infinities_and_nan_do_not_reach_a_row(cuda, value, group, T):
    """One branch's draft holds an infinity or NaN in its key, another in its
    value: rows of other branches are exact, rows that see them get what the
    formula gives."""
    c = Paged(6, [70 + T], 2, 16, 64)
    H = 2 * group
    words, seen = tree_masks(c.rng, T)
    seen[:] = np.eye(T, dtype=bool)
    seen[4, 1] = True
    words = np.array([sum(1 << int(j) for j in np.flatnonzero(r)) for r in seen], np.int64)
    p, s = c.slot(0, 70 + 1)
    c.v[0, p, 0, s, 3] = value            # seen by drafts 1 and 4
    p, s = c.slot(0, 70 + 2)
    c.k[0, p, 1, s, 5] = value            # seen by draft 2
    q = bf16(np.abs(c.rng.standard_normal((T, H, 64))) + 0.1)
    got = nk.attention_paged(dev(q.reshape(T, -1)).bfloat16(), c.device(), ints([0, T]),
                             ints([70 + T]), H, max_q=T, max_kv=70 + T, out_dtype=nk.F32,
                             tree_mask=torch.from_numpy(words).cuda())
    nk.device_status()
    want, mag = _reference(c, q, [T], H, "tree", [seen])
    clean = [0, 3] + list(range(5, T))
    assert np.isfinite(want[clean]).all()
    mag = np.where(np.isfinite(mag), mag, 0)
    _close(got, want, mag, True)


def test_causal_chunk_with_an_infinite_value(cuda):
    c = Paged(7, [90], 1, 32, 128)
    p, s = c.slot(0, 60)
    c.v[0, p, 0, s, 100] = np.inf
    q = bf16(c.rng.standard_normal((50, 2, 128)))
    got = nk.attention_paged(dev(q.reshape(50, -1)).bfloat16(), c.device(), ints([0, 50]),
                             ints([90]), 2, max_q=50, max_kv=90)
    nk.device_status()
    want, mag = _reference(c, q, [50], 2, "causal")
    assert np.isfinite(want[:20]).all() and np.isinf(want[20:, :, 100]).all()
    _close(got, want, np.where(np.isfinite(mag), mag, 0))


def test_minus_infinite_scores_leave_no_weight(cuda):
    # every key of the sequence scores -inf: as if nothing were seen
    c = Paged(1, [40], 1, 16, 64)
    c.k[0, c.table[0]] = -np.inf
    q = np.ones((1, 1, 64), np.float32)
    got = nk.attention_paged(dev(q.reshape(1, -1)).bfloat16(), c.device(), ints([0, 1]),
                             ints([40]), 1, max_q=1, max_kv=40)
    nk.device_status()
    assert not got.any()


@pytest.mark.parametrize("start,kv_len,rows,edit,code", [
    ([0, 2], [65], None, None, nk.INVALID_PARAMS), ([0, 2], [1], None, None, nk.INVALID_PARAMS),
    ([2, 0], [40], None, None, nk.INVALID_PARAMS), ([0, 3], [40], None, None, nk.INVALID_PARAMS),
    ([0, 2], [40], [1], None, nk.INVALID_PARAMS),
    ([0, 2], [40], None, 10**6, nk.PAGE_OUT_OF_RANGE),
    ([0, 2], [40], None, -1, nk.PAGE_OUT_OF_RANGE)])
def test_contradicting_batches_are_reported(cuda, start, kv_len, rows, edit, code):
    c = Paged(1, [40], 2, 16, 64, width=4)
    if edit is not None:
        c.table[0, 1] = edit
    pages = c.device()
    q = torch.randn(2, 256, device="cuda").bfloat16()
    out = torch.full((2, 256), 9.0, device="cuda")
    r = None if rows is None else ints(rows)
    nk.attention_paged(q, pages, ints(start), ints(kv_len), 4, max_q=2, max_kv=64, rows=r, out=out)
    with pytest.raises(nk.NkError) as e:
        nk.device_status()
    assert e.value.code == code
    if code == nk.INVALID_PARAMS:
        assert (out == 9.0).all()
    else:
        assert torch.isfinite(out).all()  # the page is not read
    lists = torch.full((2, 2, 3), 7, dtype=torch.int32, device="cuda")
    nk.kv_block_select(q, pages, ints(start), ints(kv_len), 4, 3, max_q=2, max_kv=64, rows=r,
                       out=lists)
    try:
        nk.device_status()
    except nk.NkError as e2:
        assert e2.code == code
    if code == nk.INVALID_PARAMS:
        assert (lists == 7).all()


@pytest.mark.parametrize("lens,T,H,kv,bound", [
    ([2000], 1, 32, 2, 2000), ([300, 1200, 64], 2, 8, 8, 1200), ([700], 64, 16, 1, 700),
    ([2000, 37], 1, 32, 2, 20000), ([300, 1200, 64], 2, 8, 8, 9000), ([900, 20], 9, 8, 2, 9000)])
def test_captured_and_on_another_stream(cuda, lens, T, H, kv, bound):
    """Two graphs with workspaces of their own replayed in turn on new inputs,
    and two calls in flight on two streams."""
    c = Paged(4, lens, kv, 64, 64)
    pages, counts = c.device(), [T] * len(lens)
    args = (ints(starts(counts)), ints(lens), H)
    kw = dict(max_q=T, max_kv=bound)
    n = T * len(lens)
    qs = [torch.randn(n, H * 64, device="cuda").bfloat16() for _ in range(4)]
    want = [nk.attention_paged(q, pages, *args, **kw) for q in qs]
    static = [torch.empty_like(qs[0]) for _ in range(2)]
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(nk.attention_paged(static[i], pages, *args, **kw))
        graphs.append(g)
    for pair in ((0, 1), (2, 3)):
        for i in range(2):
            static[i].copy_(qs[pair[i]])
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], want[pair[i]])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [nk.attention_paged(qs[i], pages, *args, stream=streams[i % 2], **kw)
           for i in range(4)]
    torch.cuda.synchronize()
    for i in range(4):
        assert torch.equal(got[i], want[i])
    nk.device_status()


def test_captured_behind_copies_and_other_streams(cuda):
    """Calls captured behind a copy, a fill, an append and a join of two streams:
    each sees what was written before it, at every replay."""
    heads, d, ps, lens = 2, 64, 16, [700, 333]
    H = heads * 4
    c = Paged(21, lens, heads, ps, d)
    pages = c.device()
    start, kv_len = ints([0, 1, 2]), ints(lens)
    kw = dict(max_q=1, max_kv=9000)
    source = torch.zeros(2, H * d, dtype=torch.bfloat16, device="cuda")
    q, q2 = torch.zeros_like(source), torch.zeros_like(source)
    new = torch.zeros(2, 2, heads * d, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    nk.attention_paged(q, pages, start, kv_len, H, **kw)  # workspaces of the first call
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q.copy_(source)
        behind_copy = nk.attention_paged(q, pages, start, kv_len, H, **kw)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            q2.zero_()
            q2.add_(source, alpha=2)
        nk.kv_pages_append(pages, new[0], new[1], start, kv_len, max_new=1, max_kv=9000)
        torch.cuda.current_stream().wait_stream(side)
        joined = nk.attention_paged(q2, pages, start, kv_len, H, **kw)
        sparse, blocks = nk.attention_paged_sparse(q2, pages, start, kv_len, H, 6, **kw)
        again = nk.attention_paged(q, pages, start, kv_len, H, **kw)
    for _ in range(6):
        source.copy_(torch.from_numpy(bf16(c.rng.standard_normal((2, H * d)))))
        new.copy_(torch.from_numpy(bf16(c.rng.standard_normal((2, 2, heads * d)))))
        want_first = nk.attention_paged(source, pages, start, kv_len, H, **kw)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        twice = source * 2
        assert torch.equal(behind_copy, want_first)
        assert torch.equal(joined, nk.attention_paged(twice, pages, start, kv_len, H, **kw))
        assert torch.equal(again, nk.attention_paged(source, pages, start, kv_len, H, **kw))
        want = nk.attention_paged_sparse(twice, pages, start, kv_len, H, 6, **kw)
        assert torch.equal(sparse, want[0]) and torch.equal(blocks, want[1])
    nk.device_status()


@pytest.mark.parametrize("group,top_k", [(4, 3), (40, 9)])
def test_steps_issued_back_to_back(cuda, group, top_k):
    """Appends, attention and block lists of many steps in flight at once give
    what the same steps give with a wait for the GPU after each call."""
    heads, d, ps, steps, lens = 2, 64, 16, 60, [100, 31, 250]
    n, H = len(lens), heads * group
    results = []
    for wait in (True, False):
        c = Paged(31, [x + steps for x in lens], heads, ps, d)
        pages = c.device()
        start = ints(starts([1] * n))
        now = [ints([x + i + 1 for x in lens]) for i in range(steps)]
        gen = torch.Generator(device="cuda").manual_seed(5)
        new = torch.empty(steps, 2, n, heads * d, dtype=torch.bfloat16,
                          device="cuda").normal_(generator=gen)
        q = torch.empty(steps, n, H * d, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
        got = []
        torch.cuda.synchronize()

        def done():
            if wait:
                torch.cuda.synchronize()
        for i in range(steps):
            kw = dict(max_q=1, max_kv=400)
            nk.kv_pages_append(pages, new[i, 0], new[i, 1], start, now[i], max_new=1, max_kv=400)
            done()
            got.append(nk.attention_paged(q[i], pages, start, now[i], H, **kw))
            done()
            got += nk.attention_paged_sparse(q[i], pages, start, now[i], H, top_k, **kw)
            done()
        torch.cuda.synchronize()
        nk.device_status()
        results.append(got)
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_explicit_workspace(cuda):
    c = Paged(4, [3000], 2, 64, 64)
    pages, q = c.device(), torch.randn(1, 256, device="cuda").bfloat16()
    need = nk.attention_paged_workspace_bytes(pages, 1, 1, 4, max_q=1, max_kv=9000)
    assert need > 0
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    args = (q, pages, ints([0, 1]), ints([3000]), 4)
    a = nk.attention_paged(*args, max_q=1, max_kv=9000, workspace=ws)
    b = nk.attention_paged(*args, max_q=1, max_kv=9000)
    assert torch.equal(a, b)
    with pytest.raises(nk.NkError) as e:
        nk.attention_paged(*args, max_q=1, max_kv=9000, workspace=ws[:need - 16])
    assert e.value.code == nk.WORKSPACE_TOO_SMALL


# -------------------------------------------------------------- block lists
SELECT = [  # ps, d, kv, group, lens, counts, top_k, sink, local
    (16, 64, 1, 1, [5], [1], 3, 1, 1),                       # one block, a longer list
    (64, 128, 2, 16, [4000, 64, 65], [1, 1, 1], 8, 1, 2),
    (32, 64, 8, 4, [900, 333], [2, 3], 9, 2, 1),
    (16, 128, 2, 3, [5000, 15], [1, 2], 64, 0, 1),
    (128, 64, 1, 8, [20000], [1], 5, 1, 1),
    (16, 64, 2, 2, [700], [40], 6, 3, 3)]                    # nothing left to rank


@pytest.mark.parametrize("ps,d,kv,group,lens,counts,top_k,sink,local", SELECT)
def test_block_select_and_sparse_attention(cuda, ps, d, kv, group, lens, counts, top_k, sink,
                                           local):
    c = Paged(ps + d + top_k, lens, kv, ps, d)
    H, T = kv * group, sum(counts)
    q = bf16(c.rng.standard_normal((T, H, d)))
    lists = np.full((T, kv, top_k), -1, np.int32)
    at = 0
    for s, t in enumerate(counts):
        for i in range(t):
            n = (int(lens[s]) - t + i) // ps + 1
            for h in range(kv):
                x = chosen_blocks(q[at, h * group:(h + 1) * group], c.lo[0, c.table[s, :n], h],
                                  c.hi[0, c.table[s, :n], h], n, top_k, sink, local)
                lists[at, h, :len(x)] = x
            at += 1
    want, mag = _reference(c, q, counts, H, "blocks", lists=lists)
    out, blocks = nk.attention_paged_sparse(dev(q.reshape(T, -1)).bfloat16(), c.device(),
                                            ints(starts(counts)), ints(lens), H, top_k, sink=sink,
                                            local=local, max_q=max(counts), max_kv=max(lens))
    nk.device_status()
    assert np.array_equal(blocks.cpu().numpy(), lists)
    _close(out, want, mag)


def test_block_select_ties_and_nan(cuda):
    """Equal scores go to the lower block; a block whose score is NaN is last."""
    ps, d = 16, 64
    c = Paged(0, [16 * 40], 1, ps, d)
    c.lo[:], c.hi[:] = -1.0, 1.0                    # every block ties
    c.hi[0, c.table[0, 20]] = np.nan
    c.lo[0, c.table[0, 20]] = np.nan
    c.hi[0, c.table[0, 33], 0, 2] = 50.0
    q = np.ones((1, 1, d), np.float32)
    q[0, 0, 1::2] = -1
    pages = c.device()
    args = (dev(q.reshape(1, -1)).bfloat16(), pages, ints([0, 1]), ints([16 * 40]), 1)
    got = nk.kv_block_select(*args, 6, sink=1, local=1, max_q=1, max_kv=640)
    assert got.cpu().numpy()[0, 0].tolist() == [0, 1, 2, 3, 33, 39]
    got = nk.kv_block_select(*args, 39, sink=0, local=1, max_q=1, max_kv=640)
    assert got.cpu().numpy()[0, 0].tolist() == [j for j in range(40) if j != 20]
    nk.device_status()


def test_lists_with_repeated_and_foreign_blocks(cuda):
    """Entries that are negative, repeated or past the token are skipped."""
    c = Paged(3, [100, 50], 2, 16, 64)
    q = bf16(c.rng.standard_normal((2, 4, 64)))
    lists = np.array([[[0, 0, 3, 3, 6, 9], [-1, 2, 2, 5, 4, 10**6]],
                      [[-7, -1, -1, -1, -1, -1], [1, 3, 3, 4, 4, 5]]], np.int32)
    clean = [[[0, 3, 6], [2, 5]], [[], [1, 3]]]
    got = nk.attention_paged(dev(q.reshape(2, -1)).bfloat16(), c.device(), ints([0, 1, 2]),
                             ints([100, 50]), 4, max_q=1, max_kv=100, out_dtype=nk.F32,
                             blocks=ints(lists))
    nk.device_status()
    want, mag = _reference(c, q, [1, 1], 4, "blocks", lists=clean)
    _close(got, want, mag, True)
    assert not got[1, :128].any()


# ------------------------------------------------------- together, as in use
def test_drafting_and_sparse_reading_over_one_cache(cuda):
    """Prefill of two prompts, a fork, a drafted tree verified and accepted,
    then a sparse step: each attention equals the formula over the tokens that
    the sequence holds by then."""
    heads, d, ps, group = 2, 64, 16, 4
    H = heads * group
    r = np.random.default_rng(1)
    cache = nk_paged.PagedKvCache(80, heads, d, max_seqs=4, max_len=400, page_size=ps)
    kv = {}

    def feed(seqs, counts):
        step = cache.step(seqs, counts)
        k, v, q = (bf16(r.standard_normal((step.tokens, n, d))) for n in (heads, heads, H))
        t = lambda a: dev(a.reshape(step.tokens, -1)).bfloat16()  # noqa: E731
        cache.append(step, t(k), t(v))
        at = 0
        for s, c in zip(seqs, counts):
            old = kv.get(s, np.zeros((2, 0, heads, d), np.float32))
            kv[s] = np.concatenate([old, np.stack([k[at:at + c], v[at:at + c]])], 1)
            at += c
        return step, q, t(q)

    def check(got, q, step, masks=None, lists=None):
        at = 0
        for s, c in zip(step.seqs, step.counts):
            n = kv[s].shape[1]
            seen = np.tri(c, n, n - c, dtype=bool)[:, None]
            if masks is not None:
                seen[:, 0, n - c:] = masks[s]
            if lists is not None:
                seen = np.repeat(seen, heads, 1)
                for i in range(c):
                    for h in range(heads):
                        hit = np.isin(np.arange(n) // ps, lists[at + i, h])
                        seen[i, h] &= hit
            o, m = attention(q[at:at + c], kv[s][0].transpose(1, 0, 2),
                             kv[s][1].transpose(1, 0, 2), seen, d**-0.5)
            _close(got[at:at + c], o, m)
            at += c

    a, b = cache.new_sequence(), cache.new_sequence()
    step, q, qd = feed([a, b], [130, 75])
    check(cache.attend(qd, step, H), q, step)
    c = cache.fork(a)
    kv[c] = kv[a].copy()
    words, masks, seqs = [], {}, [b, c, a]
    for s in seqs:
        w, masks[s] = tree_masks(r, 11)
        words.append(w)
    step, q, qd = feed(seqs, [11, 11, 11])
    tree = torch.from_numpy(np.concatenate(words)).cuda()
    check(cache.attend(qd, step, H, tree_mask=tree), q, step, masks)
    keep = [sorted(np.flatnonzero(masks[s][10]).tolist()) for s in seqs]
    cache.accept(step, keep)
    for s, row in zip(seqs, keep):
        n = kv[s].shape[1] - 11
        kv[s] = kv[s][:, list(range(n)) + [n + i for i in row]]
    for _ in range(3):
        step, q, qd = feed([c, a, b], [1, 2, 1])
        out, lists = cache.attend_sparse(qd, step, H, 4, sink=1, local=1)
        check(out, q, step, lists=lists.cpu().numpy())
    nk.device_status()


def test_decoder_over_pages_matches_the_contiguous_cache(cuda):
    """The hybrid decoder, prefill and steps, over both caches: the same
    projections, weights of the softmax rounded to bf16 in both (the contiguous
    path normalises before the rounding), so the logits agree within the
    decoder's own bar."""
    tiny = dict(vocab=512, hidden=128, pattern="M*E*", mamba_heads=4, mamba_head_dim=32,
                mamba_groups=2, mamba_state=32, conv_kernel=4, experts=8, top_k=2, moe_inter=64,
                shared_inter=128, q_heads=4, kv_heads=2, head_dim=64, std=0.08)
    model = nk_model.Decoder(nk_model.DecoderConfig(**tiny))
    B, T, steps = 3, 21, 4
    toks = rng(4).integers(0, 512, (B, T + steps)).astype(np.int32)
    plain, paged = model.new_state(B, T + steps), model.new_state(B, T + steps, page_size=16)
    feed = [(toks[:, :T], T)] + [(toks[:, T + s:T + s + 1], 1) for s in range(steps)]
    for ids, n in feed:
        ids = dev(ids.reshape(-1).copy())
        x = model.forward(ids, B, n, plain)
        y = model.forward(ids, B, n, paged)
        assert rel_err(host(y), host(x)) <= 2e-2
    nk.device_status()
    out = model.generate(dev(toks[:, :T].copy()), steps, page_size=32)
    assert out.shape == (B, steps) and int(out.min()) >= 0 and int(out.max()) < 512


@pytest.mark.parametrize("ps,d,group,n,top_k,step", [
    (16, 64, 2, 700, 40, 0.0), (16, 128, 16, 5000, 64, 2.0**-16), (32, 64, 1, 300, 7, 2.0**-30),
    (16, 128, 3, 4099, 1000, 2.0**-22), (16, 64, 17, 130, 64, 1.0)])
def test_block_select_with_scores_that_nearly_tie(cuda, ps, d, group, n, top_k, step):
    """Bounds that differ from block to block by a last place somewhere, so
    that f32 sums cannot tell them apart, and many that are equal: the list is
    the one of 64-bit sums, ties by index."""
    c = Paged(n, [n * ps - 3], 1, ps, d)
    r = c.rng
    base = bf16(r.standard_normal(d))
    c.lo[0], c.hi[0] = base, base
    order = r.permutation(n)
    for rank, j in enumerate(order):
        ch = int(r.integers(0, d))
        c.hi[0, c.table[0, j], 0, ch] = bf16(np.array([base[ch] + step * (rank // 3)]))[0]
    q = bf16(r.standard_normal((1, group, d)))
    want = chosen_blocks(q[0], c.lo[0, c.table[0, :n], 0], c.hi[0, c.table[0, :n], 0], n, top_k, 1,
                         1)
    got = nk.kv_block_select(dev(q.reshape(1, -1)).bfloat16(), c.device(), ints([0, 1]),
                             ints([n * ps - 3]), group, top_k, max_q=1, max_kv=n * ps)
    nk.device_status()
    assert got.cpu().numpy()[0, 0].tolist() == want.tolist()


@pytest.mark.parametrize("n", [500, 1700])
@pytest.mark.parametrize("alike", [2, 127, 128, 129, 300])
@pytest.mark.parametrize("distinct", [False, True])
def test_block_select_with_few_and_many_blocks_at_the_border(cuda, n, alike, distinct):
    """Clear winners, clear losers, and `alike` blocks at the border that f32 sums
    cannot tell apart: equal ones, or ones that differ by 2^-26 of a term."""
    ps, d, winners = 16, 128, 9
    c = Paged(n + alike, [n * ps], 1, ps, d)
    order = 1 + c.rng.permutation(n - 2)  # the first and the last block are forced
    low = np.full((n, d), -1.0, np.float32)
    high = np.full((n, d), 1.0, np.float32)
    high[order[:winners]] = 3.0
    high[order[winners + alike:]] = 0.5
    if distinct:  # q = 1 but for channel 7, where it is 2^-20
        high[order[winners:winners + alike], 7] = bf16(
            1 + np.arange(alike) % 64 / 64.0)[c.rng.permutation(alike)]
    c.lo[0, c.table[0, :n], 0], c.hi[0, c.table[0, :n], 0] = low, high
    q = np.ones((1, 2, d), np.float32)
    q[..., 7] = 2.0**-20
    for top_k in (2 + winners + 1, 2 + winners + alike - 1):
        want = chosen_blocks(q[0], low, high, n, top_k, 1, 1)
        got = nk.kv_block_select(dev(q.reshape(1, -1)).bfloat16(), c.device(), ints([0, 1]),
                                 ints([n * ps]), 2, top_k, max_q=1, max_kv=n * ps)
        nk.device_status()
        assert got.cpu().numpy()[0, 0].tolist() == want.tolist()


@pytest.mark.parametrize("n,heads,seqs", [
    (2000, 1, 1), (2000, 8, 2), (2000, 2, 4), (4096, 1, 1), (4096, 8, 2), (4096, 2, 4),
    (1000, 8, 8), (500, 8, 16), (130, 8, 18), (600, 8, 18), (600, 8, 19)])
def test_clusters_of_several_tiles_a_block(cuda, n, heads, seqs):
    """Units of 2 to 32 tiles, which clusters of one to eight blocks take up to
    four tiles a block where they fit, and a tile list where not; lengths end
    inside tiles."""
    lens = [max(1, n - 37 * s - 1) for s in range(seqs)]
    c = Paged(heads + seqs, lens, heads, 64, 128)
    H = heads * 2
    q = bf16(c.rng.standard_normal((seqs, H, 128)))
    got = nk.attention_paged(dev(q.reshape(seqs, -1)).bfloat16(), c.device(),
                             ints(starts([1] * seqs)), ints(lens), H, max_q=1, max_kv=n)
    nk.device_status()
    want, mag = _reference(c, q, [1] * seqs, H, "causal")
    _close(got, want, mag)


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_block_select_with_infinite_bounds_and_queries(cuda, value):
    """What the definition makes of infinities and NaN, in a bound and in a
    query: no f32 interval holds such a score."""
    n, ps, d = 200, 16, 64
    for where in ("hi", "lo", "q"):
        c = Paged(5, [n * ps], 1, ps, d)
        q = bf16(c.rng.standard_normal((1, 2, d)))
        if where == "q":
            q[0, 1, 9] = value
        else:
            for j in (3, 50, 51, 120):
                getattr(c, where)[0, c.table[0, j], 0, 9] = value
        q[0, 0, 9] = 0.0
        want = chosen_blocks(q[0], c.lo[0, c.table[0, :n], 0], c.hi[0, c.table[0, :n], 0], n, 20,
                             1, 1)
        got = nk.kv_block_select(dev(q.reshape(1, -1)).bfloat16(), c.device(), ints([0, 1]),
                                 ints([n * ps]), 2, 20, max_q=1, max_kv=n * ps)
        nk.device_status()
        assert got.cpu().numpy()[0, 0].tolist() == want.tolist(), where


@pytest.mark.parametrize("bound", [512, 8192])
def test_captured_decode_steps_follow_the_device_lengths(cuda, bound):
    """A decode step (append, attention, block lists, sparse attention) captured
    once and replayed while the lengths and the table grow on the device."""
    heads, group, d, ps, top_k = 2, 4, 64, 16, 5
    H, lens = heads * group, [100, 31]
    c = Paged(12, [n + 40 for n in lens], heads, ps, d, width=bound // ps)
    pages = c.device()
    k, v = torch.zeros(2, 2, heads * d, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros(2, H * d, dtype=torch.bfloat16, device="cuda")
    start, kv_len = ints([0, 1, 2]), ints(lens)
    kw = dict(max_q=1, max_kv=bound)

    def step():
        nk.kv_pages_append(pages, k, v, start, kv_len, max_new=1, max_kv=bound)
        return nk.attention_paged(q, pages, start, kv_len, H, **kw), \
            nk.attention_paged_sparse(q, pages, start, kv_len, H, top_k, **kw)

    # bounds of the cached tokens alone
    c.lens = np.array(lens) - 1
    c.lo[:], c.hi[:] = 0, 0
    c.refresh_bounds()
    pages.k_min.copy_(torch.from_numpy(c.lo))
    pages.k_max.copy_(torch.from_numpy(c.hi))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        full, (sparse, blocks) = step()
    for _ in range(36):
        new = bf16(c.rng.standard_normal((2, 2, heads, d)))
        qh = bf16(c.rng.standard_normal((2, H, d)))
        k.copy_(torch.from_numpy(new[0].reshape(2, -1)))
        v.copy_(torch.from_numpy(new[1].reshape(2, -1)))
        q.copy_(torch.from_numpy(qh.reshape(2, -1)))
        c.lens = c.lens + 1
        kv_len.copy_(ints(c.lens))
        for s in range(2):
            page, slot = c.slot(s, int(c.lens[s]) - 1)
            c.k[0, page, :, slot], c.v[0, page, :, slot] = new[0, s], new[1, s]
        c.refresh_bounds()
        g.replay()
        torch.cuda.synchronize()
        want, mag = _reference(c, qh, [1, 1], H, "causal")
        _close(full, want, mag)
        lists = np.full((2, heads, top_k), -1, np.int32)
        for s in range(2):
            n = -(-int(c.lens[s]) // ps)
            for h in range(heads):
                x = chosen_blocks(qh[s, h * group:(h + 1) * group], c.lo[0, c.table[s, :n], h],
                                  c.hi[0, c.table[s, :n], h], n, top_k, 1, 1)
                lists[s, h, :len(x)] = x
        assert np.array_equal(blocks.cpu().numpy(), lists)
        want, mag = _reference(c, qh, [1, 1], H, "blocks", lists=lists)
        _close(sparse, want, mag)
    nk.device_status()


@pytest.mark.parametrize("group,kv,T", [(64, 1, 1), (40, 2, 3)])
def test_many_query_heads_to_a_kv_head(cuda, group, kv, T):
    """Block lists whose rows fill tensor-memory tiles, and the selection's limit."""
    c = Paged(group, [700, 90], kv, 16, 128)
    H, n = group * kv, 2 * T
    q = bf16(c.rng.standard_normal((n, H, 128)))
    out, blocks = nk.attention_paged_sparse(dev(q.reshape(n, -1)).bfloat16(), c.device(),
                                            ints([0, T, n]), ints([700, 90]), H, 9, max_q=T,
                                            max_kv=700)
    nk.device_status()
    lists = blocks.cpu().numpy()
    for s in range(2):
        for i in range(T):
            m = (int(c.lens[s]) - T + i) // 16 + 1
            for h in range(kv):
                x = chosen_blocks(q[s * T + i, h * group:(h + 1) * group],
                                  c.lo[0, c.table[s, :m], h], c.hi[0, c.table[s, :m], h], m, 9,
                                  1, 1)
                assert lists[s * T + i, h, :len(x)].tolist() == x.tolist()
    want, mag = _reference(c, q, [T, T], H, "blocks", lists=lists)
    _close(out, want, mag)


def test_large_magnitudes_rescale(cuda):
    """Scores that grow by hundreds along the sequence: the running maximum
    moves and the sums so far shrink, in every kernel."""
    for H, kv, T in ((2, 1, 1), (16, 1, 2), (8, 1, 20)):
        c = Paged(H, [1000], kv, 64, 128)
        ramp = np.linspace(0.01, 12.0, 1000)
        for p in range(1000):
            page, slot = c.slot(0, p)
            c.k[0, page, :, slot] = bf16(c.k[0, page, :, slot] * ramp[p])
        q = bf16(c.rng.standard_normal((T, H, 128)))
        for bound in (1000, 9000):
            got = nk.attention_paged(dev(q.reshape(T, -1)).bfloat16(), c.device(), ints([0, T]),
                                     ints([1000]), H, max_q=T, max_kv=bound, out_dtype=nk.F32)
            nk.device_status()
            want, mag = _reference(c, q, [T], H, "causal")
            # keys up to 12 times unit variance: 12 times the score's error bound
            _close(got, want, mag * (1 + 12 * 2.0**-3), True)


@pytest.mark.parametrize("n,infinite,top_k", [(800, 200, 32), (1900, 129, 130), (1900, 700, 202),
                                              (300, 200, 250)])
@pytest.mark.parametrize("low", [8.0, 40.0, 2.0**100])
def test_block_select_with_many_infinite_scores_among_finite_ones(cuda, n, infinite, top_k, low):
    """A key channel that overflowed in many pages: more than 128 blocks in doubt, +inf
    for some of them and large finite scores for the others, so that the search's
    bins reach the last of the 64-bit keys.  Nothing is written behind a list."""
    ps, d = 16, 64
    c = Paged(n, [n * ps] * 2, 1, ps, d)
    r = c.rng
    low_, high = np.full((n, d), -1.0, np.float32), np.full((n, d), 0.0, np.float32)
    high[:, 3] = bf16(low * (1 + r.random(n)))
    high[1 + r.permutation(n - 2)[:infinite], 5] = np.inf
    for s in range(2):
        c.lo[0, c.table[s], 0], c.hi[0, c.table[s], 0] = low_, high
    q = np.zeros((1, 2, d), np.float32)
    q[:, :, 3], q[:, :, 5] = 1.0, 0.5
    want = chosen_blocks(q[0], low_, high, n, top_k, 1, 1)
    lists = torch.full((4, 1, top_k), -7, dtype=torch.int32, device="cuda")
    nk.kv_block_select(dev(np.repeat(q.reshape(1, -1), 2, 0)).bfloat16(), c.device(),
                       ints([0, 1, 2]), ints([n * ps] * 2), 2, top_k, max_q=1, max_kv=n * ps,
                       out=lists[:2])
    nk.device_status()
    got = lists.cpu().numpy()
    for s in range(2):
        assert got[s, 0].tolist() == want.tolist()
    assert (got[2:] == -7).all()


@pytest.mark.parametrize("call", ["attend", "select", "sparse", "compact", "step", "accept"])
def test_a_call_on_another_stream_takes_no_memory_of_the_current_one(cuda, call):
    """Blocks of every size the call needs are freed on the current stream while a
    copy of them is still queued there; the call runs at once on its own stream."""
    heads, d, ps, H, top_k, lens = 2, 64, 16, 8, 4, [9000, 333]
    c = Paged(3, lens, heads, ps, d)
    pages = c.device()
    side = torch.cuda.Stream()
    start, kv_len = ints([0, 1, 2]), ints(lens)
    keep, n_keep, base = ints([[0], [0]]), ints([1, 1]), ints([n - 1 for n in lens])
    q = torch.randn(2, H * d, device="cuda").bfloat16()
    kw = dict(max_q=1, max_kv=9008)
    sizes = [2 * H * d * 2, 2 * heads * top_k * 4, 8, 40, 4 * 7, 4 * 6,
             nk.attention_paged_workspace_bytes(pages, 2, 2, H, max_q=1, max_kv=9008),
             nk.attention_paged_workspace_bytes(pages, 2, 2, H, max_q=1, max_kv=9008,
                                                max_blocks=top_k),
             pages._select_bytes(pages.batch(start, kv_len, 2, 1, 9008))]
    cache = nk_paged.PagedKvCache(9, heads, d, max_seqs=2, max_len=64, page_size=ps)
    seqs = [cache.new_sequence(), cache.new_sequence()]
    step = cache.step(seqs, [2, 2])

    def run(stream):
        if call == "attend":
            return nk.attention_paged(q, pages, start, kv_len, H, stream=stream, **kw)
        if call == "select":
            return nk.kv_block_select(q, pages, start, kv_len, H, top_k, stream=stream, **kw)
        if call == "sparse":
            return nk.attention_paged_sparse(q, pages, start, kv_len, H, top_k, stream=stream, **kw)
        if call == "compact":
            return nk.kv_pages_compact(pages, kv_len, base, keep, n_keep, stream=stream)
        if call == "step":
            return cache.step(seqs, [1, 1], stream=stream)
        return cache.accept(step, [[1], [0]], stream=stream)

    planted = [torch.full((max(n, 1),), 90, dtype=torch.uint8, device="cuda")
               for n in sizes for _ in range(2)]
    copies = [torch.zeros_like(x) for x in planted]
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)  # some 100 ms
    for x, y in zip(planted, copies):
        y.copy_(x)
    del planted, x
    got = run(side)
    torch.cuda.synchronize()
    nk.device_status()
    assert all(bool((y == 90).all()) for y in copies)
    del got


def test_results_of_another_stream_live_until_they_are_read(cuda):
    c = Paged(4, [700], 2, 16, 64)
    pages, side = c.device(), torch.cuda.Stream()
    qs = [torch.randn(1, 512, device="cuda").bfloat16() for _ in range(2)]
    args, kw = (pages, ints([0, 1]), ints([700]), 8), dict(max_q=1, max_kv=700)
    want = nk.attention_paged(qs[0], *args, **kw)
    read = torch.empty_like(want)
    torch.cuda.synchronize()
    out = nk.attention_paged(qs[0], *args, stream=side, **kw)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda._sleep(200_000_000)
    read.copy_(out)
    del out
    again = nk.attention_paged(qs[1], *args, stream=side, **kw)
    torch.cuda.synchronize()
    assert torch.equal(read, want) and not torch.equal(again, want)


@pytest.mark.parametrize("rows", [1, 2, 4, 7])
@pytest.mark.parametrize("bound", [64, 512, 9000])
def test_projections_behind_attention_read_what_it_wrote(cuda, rows, bound):
    """Attention into one buffer and the projection of it, many times back to back
    (the projection is launched while the attention runs), give what they give with
    a wait for the GPU between them."""
    heads, H, d, steps = 2, 32, 128, 100
    lens = [min(1 + 13 * s, bound) for s in range(rows)] if bound == 64 else [400 - 31 * s for s in range(rows)]
    c = Paged(rows, lens, heads, 64, d)
    pages, start, kv_len = c.device(), ints(starts([1] * rows)), ints(lens)
    w = torch.randn(256, H * d, device="cuda").mul_(0.02).bfloat16()
    qs = torch.randn(steps, rows, H * d, device="cuda").bfloat16()
    out = torch.empty(rows, H * d, dtype=torch.bfloat16, device="cuda")
    results = []
    for wait in (True, False):
        ys = []
        for q in qs:
            nk.attention_paged(q, pages, start, kv_len, H, max_q=1, max_kv=bound, out=out)
            if wait:
                torch.cuda.synchronize()
            ys.append(nk.gemm(out, w, out_dtype=torch.float32))
        torch.cuda.synchronize()
        results.append(torch.stack(ys))
    nk.device_status()
    assert torch.equal(*results)
    if max(lens) > 1:  # a single cached token is the output whatever the query
        assert not torch.equal(results[0][0], results[0][1])


@pytest.mark.parametrize("B", [1, 2])
def test_decoder_of_one_and_two_rows_over_pages(cuda, B):
    """Decode steps whose projections stream the weights: the same bar as for more
    rows, and the same bits when each step waits for the one before."""
    tiny = dict(vocab=512, hidden=128, pattern="*E*M", mamba_heads=4, mamba_head_dim=32,
                mamba_groups=2, mamba_state=32, conv_kernel=4, experts=8, top_k=2, moe_inter=64,
                shared_inter=128, q_heads=4, kv_heads=2, head_dim=64, std=0.08)
    model = nk_model.Decoder(nk_model.DecoderConfig(**tiny))
    T, steps = 21, 12
    toks = dev(rng(5).integers(0, 512, (B, T + steps)).astype(np.int32))
    feed = [(toks[:, :T].reshape(-1).contiguous(), T)] + \
        [(toks[:, T + s].contiguous(), 1) for s in range(steps)]
    plain = model.new_state(B, T + steps)
    want = [model.forward(ids, B, n, plain) for ids, n in feed]
    got = []
    for wait in (True, False):
        state = model.new_state(B, T + steps, page_size=16)
        torch.cuda.synchronize()
        got.append([])
        for ids, n in feed:
            got[-1].append(model.forward(ids, B, n, state))
            if wait:
                torch.cuda.synchronize()
    nk.device_status()
    for x, y, z in zip(want, *got):
        assert rel_err(host(y), host(x)) <= 2e-2 and torch.equal(y, z)


@pytest.mark.parametrize("bound", [0, 9000])
@pytest.mark.parametrize("ps,d,kv,group,lens", [
    (128, 64, 2, 4, [256, 130, 1]), (16, 64, 2, 3, [700, 40, 333]), (64, 128, 1, 16, [1300, 64]),
    (32, 64, 1, 40, [500, 77])])
def test_lists_whose_blocks_stand_behind_skipped_entries(cuda, ps, d, kv, group, lens, bound):
    """Negative, foreign and repeated entries before and between the blocks push
    them past as many entries as the sequence has blocks, a tile or several."""
    c = Paged(ps + group, lens, kv, ps, d)
    n, H, r = len(lens), kv * group, c.rng
    most = max(-(-x // ps) for x in lens)
    width = 3 * most + 130
    lists = np.full((n, kv, width), -1, np.int32)
    clean = []
    for s, x in enumerate(lens):
        clean.append([])
        held = -(-x // ps)
        for h in range(kv):
            keep = np.sort(r.choice(held, max(1, held // 2), replace=False))
            at = np.sort(r.choice(width, len(keep), replace=False))
            if h == 0:  # all of them at the list's end
                at = np.arange(width - len(keep), width)
            lists[s, h, at] = keep
            if h and at[0] > 3:  # foreign ones in front
                lists[s, h, :2] = [held, 10**6]
            clean[-1].append(keep.tolist())
    if lens[0] == 256:
        lists[0, 0, :3], lists[0, 0, 3:], clean[0][0] = [-1, 0, 1], -1, [0, 1]
        lists[1, 0, :4], lists[1, 0, 4:], clean[1][0] = [0, 0, 0, 1], -1, [0, 1]
    q = bf16(r.standard_normal((n, H, d)))
    got = nk.attention_paged(dev(q.reshape(n, -1)).bfloat16(), c.device(), ints(starts([1] * n)),
                             ints(lens), H, max_q=1, max_kv=bound or max(lens), out_dtype=nk.F32,
                             blocks=ints(lists))
    nk.device_status()
    want, mag = _reference(c, q, [1] * n, H, "blocks", lists=clean)
    _close(got, want, mag, True)


def test_empty_lists_and_tables_are_refused(cuda):
    """A list of no entries is not attention without lists, a table of no columns
    not a compaction in place."""
    c = Paged(2, [40, 9], 2, 16, 64)
    pages, start, kv_len = c.device(), ints([0, 1, 2]), ints([40, 9])
    q = torch.randn(2, 256, device="cuda").bfloat16()
    with pytest.raises(ValueError, match="an entry"):
        nk.attention_paged(q, pages, start, kv_len, 4, max_q=1, max_kv=40,
                           blocks=torch.empty(2, 2, 0, dtype=torch.int32, device="cuda"))
    before = pages.k.clone()
    with pytest.raises(ValueError, match="a column"):
        nk.kv_pages_compact(pages, kv_len, ints([30, 0]), ints([[5], [1]]), ints([1, 1]),
                            dst_table=torch.empty(2, 0, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(before.nan_to_num(), pages.k.nan_to_num())
    # no tokens, no sequences: nothing to do
    none, no = torch.empty(0, 256, dtype=torch.bfloat16, device="cuda"), ints([])
    for lists in (None, torch.empty(0, 2, 8, dtype=torch.int32, device="cuda")):
        out = nk.attention_paged(none, pages, ints([0, 0, 0]), kv_len, 4, max_q=0, blocks=lists)
        assert out.shape == (0, 256)
    out, lists = nk.attention_paged_sparse(none, pages, ints([0]), no, 4, 3, max_q=0)
    assert out.shape == (0, 256) and lists.shape == (0, 2, 3)
    got = nk.kv_pages_compact(pages, no, no, torch.empty(0, 3, dtype=torch.int32, device="cuda"),
                              no, dst_table=torch.empty(0, 4, dtype=torch.int32, device="cuda"))
    assert got.numel() == 0
    nk.device_status()


@pytest.mark.parametrize("ps,d,group", [(16, 64, 4), (32, 128, 16), (16, 128, 40), (64, 64, 48)])
def test_tiles_without_pages_between_full_ones(cuda, ps, d, group):
    """Lists whose tiles change between whole ones, ones with a page or two, ones
    that end inside a page and ones with nothing to load (whose keys are counted
    by the loader alone): the formula's result, the same bits fifty times."""
    lens = [128 * 9 - 3, 128 * 5 + 1]
    c = Paged(group, lens, 2, ps, d)
    H, per, r = 2 * group, 128 // ps, c.rng
    width = 12 * per
    lists, clean = np.full((2, 2, width), -1, np.int32), [[], []]
    for s, n in enumerate(lens):
        held = -(-n // ps)
        for h in range(2):
            tiles = [x for x in range(12) if x % 3 != h]
            slots = np.array([t * per + i for t in tiles for i in range(per)
                              if t % 4 != 1 or i % per == t % per])[:held]
            keep = np.sort(r.choice(held - 1, min(len(slots), held) - 1, replace=False)).tolist()
            keep.append(held - 1)  # the sequence's last block, partly filled
            lists[s, h, slots[:len(keep)]] = keep
            clean[s].append(keep)
    q = bf16(r.standard_normal((2, H, d)))
    want, mag = _reference(c, q, [1, 1], H, "blocks", lists=clean)
    args = (dev(q.reshape(2, -1)).bfloat16(), c.device(), ints([0, 1, 2]), ints(lens), H)
    kw = dict(max_q=1, out_dtype=nk.F32, blocks=ints(lists))
    for bound in (max(lens), 9000):
        got = [nk.attention_paged(*args, max_kv=bound, **kw) for _ in range(50)]
        nk.device_status()
        _close(got[0], want, mag, True)
        assert all(torch.equal(got[0], x) for x in got[1:])


@pytest.mark.parametrize("value", [1.0, np.inf, np.nan])
@pytest.mark.parametrize("kind", ["tree", "causal"])
def test_more_wide_units_than_blocks(cuda, kind, value):
    """Units of up to 256 rows, several to a block one after the other, whole ones
    and parts, two row tiles and one in turn; a value of some drafts is no finite
    number, which rows of other branches and earlier tokens do not see."""
    kv, group, d, ps = 2, 4, 64, 32
    counts = [(64, 3, 64, 20, 1, 33, 9, 64, 0, 40)[s % 10] for s in range(110)]
    r = np.random.default_rng(11)
    lens = [t + int(r.integers(0, 300)) for t in counts]
    lens[17] = 2500
    c = Paged(77, [max(1, n) for n in lens], kv, ps, d)
    lens = c.lens
    H, T = kv * group, sum(counts)
    masks, words = [], []
    for s, t in enumerate(counts):
        w, seen = tree_masks(c.rng, t)
        masks.append(seen)
        words.append(w)
        if t and s % 3 == 0:
            p, x = c.slot(s, int(lens[s]) - t + t // 2)
            c.v[0, p, s % kv, x, s % d] = value
    q = bf16(c.rng.standard_normal((T, H, d)))
    tree = torch.from_numpy(np.concatenate(words)).cuda() if kind == "tree" else None
    want, mag = _reference(c, q, counts, H, kind, masks)
    args = (dev(q.reshape(T, -1)).bfloat16(), c.device(), ints(starts(counts)), ints(lens), H)
    got = [nk.attention_paged(*args, max_q=64, max_kv=2500, tree_mask=tree, out_dtype=nk.F32)
           for _ in range(3)]
    nk.device_status()
    _close(got[0], want, np.where(np.isfinite(mag), mag, 0), True)
    assert all(torch.equal(got[0].nan_to_num(7.0), x.nan_to_num(7.0)) for x in got[1:])


def test_default_bounds_of_a_batch_longer_than_a_sequence(cuda):
    """More tokens in all than one sequence can hold, without bounds given."""
    lens = [16, 7, 1] * 8
    c = Paged(9, lens, 2, 16, 64)
    n, H = len(lens), 4
    q = bf16(c.rng.standard_normal((n, H, 64)))
    args = (dev(q.reshape(n, -1)).bfloat16(), c.device(), ints(starts([1] * n)), ints(lens), H)
    want, mag = _reference(c, q, [1] * n, H, "causal")
    _close(nk.attention_paged(*args), want, mag)
    out, blocks = nk.attention_paged_sparse(*args, 2)
    _close(out, want, mag)
    assert torch.equal(blocks, nk.kv_block_select(*args, 2))
    _close(nk.attention_paged(*args, max_kv=20, out_dtype=nk.F32), want, mag, True)
    nk.device_status()
    # trees of 30 drafts, 90 in all
    c, counts = Paged(10, [100, 30, 64], 2, 16, 64), [30, 30, 30]
    trees = [tree_masks(c.rng, 30) for _ in counts]
    q = bf16(c.rng.standard_normal((90, H, 64)))
    got = nk.attention_paged(dev(q.reshape(90, -1)).bfloat16(), c.device(), ints(starts(counts)),
                             ints([100, 30, 64]), H,
                             tree_mask=torch.from_numpy(np.concatenate([w for w, _ in trees])).cuda())
    nk.device_status()
    want, mag = _reference(c, q, counts, H, "tree", [m for _, m in trees])
    _close(got, want, mag)


def test_workspace_sizes_kept_are_bounded(cuda):
    """A bound that grows with every step does not grow the host's memory, and the
    sizes are those that the library asks for."""
    pages = Paged(1, [20], 1, 16, 64).device()
    start, kv_len = ints([0, 1]), ints([20])
    for n in range(1, 9001):
        assert pages._select_bytes(pages.batch(start, kv_len, 1, 1, n)) == -(-n // 16) * 16
        assert len(pages._bytes) <= 4097
    sizes = [nk.attention_paged_workspace_bytes(pages, 1, 1, 2, max_q=1, max_kv=n)
             for n in (100, 5000, 100)]
    assert sizes[0] == sizes[2] == 0 < sizes[1]


def test_workspaces_of_another_device_or_type_are_refused(cuda):
    c = Paged(4, [300], 1, 16, 64)
    pages, q = c.device(), torch.randn(1, 128, device="cuda").bfloat16()
    args, kw = (q, pages, ints([0, 1]), ints([300]), 2), dict(max_q=1, max_kv=9000)
    need = nk.attention_paged_workspace_bytes(pages, 1, 1, 2, max_q=1, max_kv=9000)
    for bad in (torch.empty(need, dtype=torch.uint8), torch.empty(need, device="cuda"),
                torch.empty(2 * need, dtype=torch.uint8, device="cuda")[::2]):
        with pytest.raises(ValueError, match="workspace"):
            nk.attention_paged(*args, workspace=bad, **kw)
        with pytest.raises(ValueError, match="workspace"):
            nk.kv_block_select(*args, 3, workspace=bad, **kw)
    ws = torch.empty(need + (1 << 20), dtype=torch.uint8, device="cuda")
    assert torch.equal(nk.attention_paged(*args, workspace=ws, **kw),
                       nk.attention_paged(*args, **kw))
    assert torch.equal(nk.kv_block_select(*args, 3, workspace=ws, **kw),
                       nk.kv_block_select(*args, 3, **kw))
    nk.device_status()


@pytest.mark.parametrize("kv,group,bound", [(2, 4, 0), (2, 4, 9000), (1, 24, 9000), (1, 40, 0),
                                            (2, 40, 9000)])
def test_more_sequences_than_threads(cuda, kv, group, bound):
    """700 sequences, whose tiles the threads of a block count in runs of two or
    three; some have no new token, one is much longer than the others."""
    n, d, ps = 700, 64, 16
    r = np.random.default_rng(kv + group)
    lens = 1 + r.integers(0, 150, n)
    lens[[0, 333, 699]] = [129, 1900, 64]
    counts = [0 if s % 7 == 3 else 1 for s in range(n)]
    c = Paged(group, lens, kv, ps, d)
    H, T = kv * group, sum(counts)
    q = bf16(c.rng.standard_normal((T, H, d)))
    want, mag = _reference(c, q, counts, H, "causal")
    got = nk.attention_paged(dev(q.reshape(T, -1)).bfloat16(), c.device(), ints(starts(counts)),
                             ints(lens), H, max_q=1, max_kv=bound or 1900)
    nk.device_status()
    _close(got, want, mag)
    out, blocks = nk.attention_paged_sparse(dev(q.reshape(T, -1)).bfloat16(), c.device(),
                                            ints(starts(counts)), ints(lens), H, 3, max_q=1,
                                            max_kv=bound or 1900)
    nk.device_status()
    want, mag = _reference(c, q, counts, H, "blocks", lists=blocks.cpu().numpy())
    _close(out, want, mag)


@pytest.mark.parametrize("kv,group,d,ps,lens,counts", [
    (2, 16, 64, 64, [1300], [1300]),                        # one prompt, 164 units
    (1, 8, 128, 32, [700, 1, 2100, 900], [700, 1, 600, 899]),  # behind cached prefixes too
    (4, 16, 64, 16, [200] * 12 + [31, 1], [200] * 12 + [30, 1])])
def test_prompts_of_more_units_than_blocks(cuda, kv, group, d, ps, lens, counts):
    """Prompt chunks whose row tiles outnumber the SMs: a block runs several
    units, whole ones and parts, each up to its own causal limit."""
    c = Paged(kv + d, lens, kv, ps, d)
    H, T = kv * group, sum(counts)
    q = bf16(c.rng.standard_normal((T, H, d)))
    args = (dev(q.reshape(T, -1)).bfloat16(), c.device(), ints(starts(counts)), ints(lens), H)
    kw = dict(max_q=max(counts), max_kv=max(lens))
    outs = [nk.attention_paged(*args, **kw) for _ in range(2)]
    nk.device_status()
    assert torch.equal(*outs)
    got, at = outs[0].view(T, H, d), 0
    for s, t in enumerate(counts):
        n = int(lens[s])
        k, v = c.tokens(c.k, s).astype(np.float64), c.tokens(c.v, s).astype(np.float64)
        seen = np.tri(t, n, n - t, dtype=bool)
        for h in range(H):
            x = q[at:at + t, h].astype(np.float64) @ k[h // group].T * d**-0.5
            w = np.where(seen, np.exp(x - np.where(seen, x, -np.inf).max(1, keepdims=True)), 0)
            w /= w.sum(1, keepdims=True)
            _close(got[at:at + t, h], w @ v[h // group], w @ np.abs(v[h // group]))
        at += t


def test_lists_follow_lengths_written_just_before(cuda):
    """The batch's arrays are rewritten by the kernel ahead of each selection, in
    the same memory: every kernel of the call reads the new ones."""
    heads, H, ps, top_k, steps = 2, 8, 16, 6, 80
    results = []
    for wait in (True, False):
        c = Paged(13, [400, 1500, 900], heads, ps, 64)
        pages = c.device()
        gen = torch.Generator(device="cuda").manual_seed(3)
        q = torch.empty(steps, 3, H * 64, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
        start, kv_len, rows = ints([0, 1, 2, 3]), ints([200, 700, 20]), ints([0, 1, 2])
        got = []
        torch.cuda.synchronize()
        for i in range(steps):
            kv_len.add_(1 + i % 3)
            rows.copy_(rows.roll(1) if i % 16 == 15 else rows)
            kv_len.clamp_(max=400)
            for _ in range(3):
                got.append(nk.kv_block_select(q[i], pages, start, kv_len, H, top_k, rows=rows,
                                              max_q=1, max_kv=1500))
                if wait:
                    torch.cuda.synchronize()
        torch.cuda.synchronize()
        nk.device_status()
        results.append(got)
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert not torch.equal(results[0][0], results[0][-1])


def test_captured_on_a_stream_that_joins_the_capture(cuda):
    """Calls captured with stream= on a stream forked from the capturing one, their
    results read behind the join; replayed on new inputs with other graphs between."""
    lens, H = [700, 90, 333], 8
    c = Paged(14, lens, 2, 16, 64)
    pages, start, kv_len = c.device(), ints([0, 1, 2, 3]), ints(lens)
    kw = dict(max_q=1, max_kv=9000)
    q = torch.zeros(3, H * 64, dtype=torch.bfloat16, device="cuda")
    side, graphs = torch.cuda.Stream(), []
    nk.attention_paged_sparse(q, pages, start, kv_len, H, 5, stream=side, **kw)
    torch.cuda.synchronize()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            side.wait_stream(torch.cuda.current_stream())
            full = nk.attention_paged(q, pages, start, kv_len, H, stream=side, **kw)
            out, blocks = nk.attention_paged_sparse(q, pages, start, kv_len, H, 5, stream=side,
                                                    **kw)
            torch.cuda.current_stream().wait_stream(side)
            both = full + out
        graphs.append((g, both, blocks))
    for i in range(4):
        q.normal_()
        full = nk.attention_paged(q, pages, start, kv_len, H, **kw)
        out, blocks = nk.attention_paged_sparse(q, pages, start, kv_len, H, 5, **kw)
        g, both, lists = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(both, full + out) and torch.equal(lists, blocks)
    nk.device_status()


def test_calls_of_two_threads_at_once(cuda):
    """Two host threads, a stream each, over one cache."""
    import threading

    lens, H = [2000, 64, 700], 8
    c = Paged(15, lens, 2, 16, 64)
    pages, start, kv_len = c.device(), ints([0, 1, 2, 3]), ints(lens)
    q = torch.randn(2, 40, 3, H * 64, device="cuda").bfloat16()

    def calls(x, i, stream=None):
        kw = dict(max_q=1, max_kv=2000 + 64 * i, stream=stream)
        full = nk.attention_paged(x, pages, start, kv_len, H, **kw)
        return [full, *nk.attention_paged_sparse(x, pages, start, kv_len, H, 3 + i % 4, **kw)]

    want = [[calls(x, i) for i, x in enumerate(q[t])] for t in range(2)]
    torch.cuda.synchronize()
    got, failed = [None, None], []

    def work(t):
        try:
            s = torch.cuda.Stream()
            got[t] = [calls(x, i, s) for i, x in enumerate(q[t])]
            s.synchronize()
        except Exception as e:  # noqa: BLE001
            failed.append(e)
    threads = [threading.Thread(target=work, args=(t,)) for t in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed
    for a, b in zip(want, got):
        for x, y in zip(a, b):
            assert all(torch.equal(m, n) for m, n in zip(x, y))
    nk.device_status()
