"""Page operations of the KV cache on the B200: appends, whole-page copies,
compaction and table writes move values and take minima and maxima, so every
pool is compared for equality with a host copy, the untouched slots too."""
import numpy as np
import pytest
import torch

import nk
import nk_paged
from paged_ref import Paged, bf16, ints, same, starts

pytestmark = pytest.mark.gpu


def _append_host(c, counts, kn, vn, layer):
    """kn, vn [tokens, heads, d] at the last positions of each sequence."""
    at = 0
    for s, t in enumerate(counts):
        n = int(c.lens[s])
        for p in range(n - t, n):
            page, slot = c.slot(s, p)
            c.k[layer, page, :, slot] = kn[at]
            c.v[layer, page, :, slot] = vn[at]
            at += 1
    for s, t in enumerate(counts):
        if not t:
            continue
        n = int(c.lens[s])
        for j in range((n - t) // c.ps, (n - 1) // c.ps + 1):
            p, m = c.table[s, j], min(c.ps, n - j * c.ps)
            c.lo[layer, p] = c.k[layer, p, :, :m].min(1)
            c.hi[layer, p] = c.k[layer, p, :, :m].max(1)


@pytest.mark.parametrize("ps,d,heads,lens,counts,layers,layer", [
    (16, 64, 1, [1], [1], 1, 0),                       # the first token of a cache
    (16, 64, 3, [16, 17, 31], [1, 1, 1], 2, 1),        # last slot, new page, inside a page
    (32, 128, 2, [100, 33, 64, 5], [37, 0, 64, 5], 1, 0),
    (64, 128, 2, [300, 1, 129, 64], [300, 1, 70, 63], 2, 0),
    (128, 128, 4, [513, 127], [257, 127], 1, 0),
    (128, 64, 8, [128, 1000], [128, 999], 1, 0)])
def test_append(cuda, ps, d, heads, lens, counts, layers, layer):
    c = Paged(ps + d, lens, heads, ps, d, layers=layers, filler=7.5)
    # bounds before the append: over the older tokens
    old = np.array(lens) - counts
    c.refresh_bounds(lens=old)
    pages = c.device()
    T = sum(counts)
    kn, vn = bf16(c.rng.standard_normal((2, T, heads, d)))
    # a fused projection row: k and v are strided views of it
    fused = torch.from_numpy(np.concatenate([kn.reshape(T, -1), vn.reshape(T, -1)], 1)) \
        .bfloat16().cuda()
    w = heads * d
    nk.kv_pages_append(pages, fused[:, :w], fused[:, w:], ints(starts(counts)), ints(lens),
                       max_new=max(counts), layer=layer)
    nk.device_status()
    _append_host(c, counts, kn, vn, layer)
    for got, want in ((pages.k, c.k), (pages.v, c.v), (pages.k_min, c.lo), (pages.k_max, c.hi)):
        assert same(got, want)


def test_append_nan_keys_leave_the_bounds(cuda):
    c = Paged(0, [20], 1, 16, 64, filler=0.0)
    c.refresh_bounds(lens=[10])
    pages = c.device()
    kn, vn = bf16(c.rng.standard_normal((2, 10, 1, 64)))
    kn[3] = np.nan
    kn[5, 0, 7] = np.inf
    nk.kv_pages_append(pages, torch.from_numpy(kn.reshape(10, 64)).bfloat16().cuda(),
                       torch.from_numpy(vn.reshape(10, 64)).bfloat16().cuda(), ints([0, 10]),
                       ints([20]), max_new=10)
    nk.device_status()
    c.k[0, c.table[0, 0], :, 10:] = kn[:6].transpose(1, 0, 2)
    p = c.table[0, 0]
    assert np.array_equal(pages.k_min[0, p, 0].float().cpu().numpy(),
                          np.nanmin(c.k[0, p, 0], 0))
    assert np.array_equal(pages.k_max[0, p, 0].float().cpu().numpy(),
                          np.nanmax(c.k[0, p, 0], 0))


def test_append_rows_and_rows_behind_the_last_sequence(cuda):
    # sequences in other table rows; token buffers longer than the batch
    c = Paged(5, [40, 9, 33], 2, 32, 64, filler=1.0)
    pages = c.device()
    before = [t.clone() for t in (pages.k, pages.v, pages.k_min, pages.k_max)]
    kn, vn = bf16(c.rng.standard_normal((2, 6, 2, 64)))
    t = lambda a: torch.from_numpy(a.reshape(6, -1)).bfloat16().cuda()  # noqa: E731
    nk.kv_pages_append(pages, t(kn), t(vn), ints([0, 1, 3]), ints([33, 40]), max_new=2,
                       rows=ints([2, 0]))
    nk.device_status()
    for i, (row, pos) in enumerate([(2, 32), (0, 38), (0, 39)]):
        page, slot = c.slot(row, pos)
        assert np.array_equal(pages.k[0, page, :, slot].float().cpu().numpy(), kn[i])
        assert np.array_equal(pages.v[0, page, :, slot].float().cpu().numpy(), vn[i])
        before[0][0, page, :, slot] = pages.k[0, page, :, slot]
        before[1][0, page, :, slot] = pages.v[0, page, :, slot]
        for x, y in ((before[2], pages.k_min), (before[3], pages.k_max)):
            x[0, page] = y[0, page]
    for x, y in zip(before, (pages.k, pages.v, pages.k_min, pages.k_max)):
        assert torch.equal(x, y)


BAD_STEPS = [  # (start, kv_len, rows, table edit, code)
    ([0, 2], [65], None, None, nk.INVALID_PARAMS),      # past max_kv and the table
    ([0, 2], [1], None, None, nk.INVALID_PARAMS),       # fewer cached than new
    ([2, 0], [40], None, None, nk.INVALID_PARAMS),      # start descends
    ([0, 3], [40], None, None, nk.INVALID_PARAMS),      # past the buffers
    ([-1, 1], [40], None, None, nk.INVALID_PARAMS),
    ([0, 2], [40], [1], None, nk.INVALID_PARAMS),       # rows outside the table
    ([0, 2], [40], [-1], None, nk.INVALID_PARAMS),
    ([0, 2], [40], None, 10**6, nk.PAGE_OUT_OF_RANGE),
    ([0, 2], [40], None, -1, nk.PAGE_OUT_OF_RANGE)]


@pytest.mark.parametrize("start,kv_len,rows,edit,code", BAD_STEPS)
def test_contradicting_batches_write_nothing(cuda, start, kv_len, rows, edit, code):
    c = Paged(1, [40], 1, 16, 64, width=4, filler=0.0)
    if edit is not None:
        c.table[0, 2] = edit
    pages = c.device()
    before = [t.clone() for t in (pages.k, pages.v, pages.k_min, pages.k_max)]
    new = torch.ones(2, 64, dtype=torch.bfloat16, device="cuda")
    nk.kv_pages_append(pages, new, new, ints(start), ints(kv_len), max_new=2,
                       rows=None if rows is None else ints(rows))
    with pytest.raises(nk.NkError) as e:
        nk.device_status()
    assert e.value.code == code
    nk.device_status()  # reading cleared it
    for x, y in zip(before, (pages.k, pages.v, pages.k_min, pages.k_max)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("ps,d,heads,layers,pages,pairs,bounds", [
    (16, 64, 1, 1, 2, 1, True), (64, 128, 2, 6, 40, 9, True), (16, 128, 8, 2, 1300, 501, True),
    (128, 64, 3, 1, 64, 17, False), (32, 64, 1, 1, 9000, 4100, True)])
def test_copy(cuda, ps, d, heads, layers, pages, pairs, bounds):
    g = torch.Generator(device=cuda).manual_seed(pages)
    shape = (layers, pages, heads, ps, d)
    k, v = (torch.randn(shape, device=cuda, generator=g).bfloat16() for _ in range(2))
    lo, hi = (torch.randn(layers, pages, heads, d, device=cuda, generator=g).bfloat16()
              for _ in range(2)) if bounds else (None, None)
    want = [None if t is None else t.clone() for t in (k, v, lo, hi)]
    r = np.random.default_rng(pairs)
    ids = r.permutation(pages)
    dst, src = ids[:pairs], r.choice(ids[pairs:], pairs)  # a source may serve many
    kv = nk.KvPages(k, v, torch.zeros(1, 1, dtype=torch.int32, device=cuda), k_min=lo, k_max=hi)
    nk.kv_pages_copy(kv, src, dst)
    nk.device_status()
    for t, got in zip(want, (k, v, lo, hi)):
        if t is not None:
            t[:, torch.from_numpy(dst).cuda()] = t[:, torch.from_numpy(src).cuda()]
            assert torch.equal(t, got)


def test_table_write(cuda):
    r = np.random.default_rng(0)
    for n in (1, 64, 65, 2600, 2601, 6000):
        dst = torch.full((8000,), -1, dtype=torch.int32, device=cuda)
        want = dst.cpu().numpy()
        off, val = r.permutation(8000)[:n], r.integers(-2**31, 2**31, n)
        nk.kv_table_write(dst, val, off)
        want[off] = val
        assert np.array_equal(dst.cpu().numpy(), want)
        nk.kv_table_write(dst, val)
        want[:n] = val
        assert np.array_equal(dst.cpu().numpy(), want)


def _compact_host(c, lens, base, keeps, dst=None):
    """Sequentially, as the formula says; bounds of the touched pages anew."""
    table = c.table if dst is None else dst
    for s, row in enumerate(keeps):
        old = [(c.k[:, p, :, x].copy(), c.v[:, p, :, x].copy())
               for p, x in (c.slot(s, base[s] + i) for i in row)]
        for i, (kk, vv) in enumerate(old):
            pos = base[s] + i
            p = table[s, pos // c.ps]
            c.k[:, p, :, pos % c.ps], c.v[:, p, :, pos % c.ps] = kk, vv
        end = base[s] + len(row)
        for j in range(base[s] // c.ps, -(-end // c.ps)):
            p, m = table[s, j], min(c.ps, end - j * c.ps)
            c.lo[:, p] = c.k[:, p, :, :m].min(2)
            c.hi[:, p] = c.k[:, p, :, :m].max(2)


def _keep_array(keeps, width=None):
    out = np.full((len(keeps), max(1, width or max(len(x) for x in keeps))), -9, np.int32)
    for i, x in enumerate(keeps):
        out[i, :len(x)] = x
    return out


@pytest.mark.parametrize("ps,d,heads,layers,lens,news,keep_n", [
    (16, 64, 1, 1, [5], [4], 2), (64, 128, 2, 6, [130, 64, 65, 20], [32, 64, 1, 20], 9),
    (16, 128, 3, 2, [77, 16, 200], [64, 3, 50], 40), (128, 64, 2, 1, [300, 129], [64, 2], 33),
    (32, 128, 2, 1, [1500], [1400], 700)])
def test_compact_in_place(cuda, ps, d, heads, layers, lens, news, keep_n):
    c = Paged(ps * 3 + d, lens, heads, ps, d, layers=layers, filler=3.0)
    pages = c.device()
    keeps = []
    for i, t in enumerate(news):
        n = min(t, keep_n if i != 2 else 0)  # the third sequence keeps nothing
        keeps.append(np.sort(c.rng.choice(t, n, replace=False)))
    base = np.array(lens) - news
    got = nk.kv_pages_compact(pages, ints(lens), ints(base), ints(_keep_array(keeps)),
                              ints([len(x) for x in keeps]))
    nk.device_status()
    _compact_host(c, lens, base, keeps)
    assert got.tolist() == [int(b) + len(x) for b, x in zip(base, keeps)]
    for x, want in ((pages.k, c.k), (pages.v, c.v), (pages.k_min, c.lo), (pages.k_max, c.hi)):
        assert same(x, want)


@pytest.mark.parametrize("ps,d,heads,layers,lens,base,n_keep", [
    (16, 64, 2, 1, [40, 16], [0, 0], [7, 16]), (64, 128, 2, 2, [700, 65], [0, 3], [130, 62]),
    (32, 64, 1, 1, [300, 90, 33], [70, 0, 32], [111, 0, 1]), (128, 128, 4, 1, [513], [0], [300])])
def test_compact_into_other_pages(cuda, ps, d, heads, layers, lens, base, n_keep):
    need = [-(-(b + n) // ps) for b, n in zip(base, n_keep)]
    c = Paged(ps + 11, lens, heads, ps, d, layers=layers, filler=2.0, spare=sum(need) + 2)
    dst = np.full((len(lens), max(need) + 1), -1, np.int32)
    at = 0
    for i, m in enumerate(need):
        dst[i, :m] = c.spare[at:at + m]
        at += m
    pages = c.device()
    keeps = [np.sort(c.rng.choice(n - b, m, replace=False))
             for n, b, m in zip(lens, base, n_keep)]
    rows = list(range(len(lens)))[::-1]  # batch order is not table order
    pick = lambda a: [a[i] for i in rows]  # noqa: E731
    got = nk.kv_pages_compact(pages, ints(pick(lens)), ints(pick(base)),
                              ints(_keep_array(pick(keeps), max(n_keep) + 3)),
                              ints(pick(n_keep)), rows=ints(rows), dst_table=ints(dst[rows]))
    nk.device_status()
    _compact_host(c, lens, base, keeps, dst)
    assert got.tolist() == [base[i] + n_keep[i] for i in rows]
    for x, want in ((pages.k, c.k), (pages.v, c.v), (pages.k_min, c.lo), (pages.k_max, c.hi)):
        assert same(x, want)


@pytest.mark.parametrize("keep,n,kv_len,base,code", [
    ([0, 1], 3, 40, 30, nk.INVALID_PARAMS),    # more than max_keep
    ([0, 1], -1, 40, 30, nk.INVALID_PARAMS), ([0, 1], 2, 40, 39, nk.INVALID_PARAMS),
    ([0, 1], 2, 40, -1, nk.INVALID_PARAMS), ([0, 1], 2, 70, 30, nk.INVALID_PARAMS)])
@pytest.mark.parametrize("in_place", [True, False])
def test_compact_refused_on_the_device(cuda, keep, n, kv_len, base, code, in_place):
    c = Paged(3, [40], 1, 16, 64, width=4, spare=6, filler=0.0)
    pages = c.device()
    before = [t.clone() for t in (pages.k, pages.v, pages.k_min, pages.k_max)]
    dst = None if in_place else ints(c.spare[:4].reshape(1, 4))
    nk.kv_pages_compact(pages, ints([kv_len]), ints([base]), ints([keep]), ints([n]),
                        dst_table=dst)
    with pytest.raises(nk.NkError) as e:
        nk.device_status()
    assert e.value.code == code
    for x, y in zip(before, (pages.k, pages.v, pages.k_min, pages.k_max)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("in_place", [True, False])
def test_compact_bad_entries_stay_in_bounds(cuda, in_place):
    # entries that do not ascend or lie past the end leave their slot unwritten
    c = Paged(4, [40], 1, 16, 64, width=4, spare=6, filler=0.0)
    pages = c.device()
    dst = None if in_place else ints(c.spare[:4].reshape(1, 4))
    nk.kv_pages_compact(pages, ints([40]), ints([30]), ints([[2, 2, 2**30, -5]]), ints([4]),
                        dst_table=dst)
    with pytest.raises(nk.NkError) as e:
        nk.device_status()
    assert e.value.code == nk.INVALID_PARAMS
    table = c.table if in_place else np.concatenate([c.table[:, :0], c.spare[:4].reshape(1, 4)], 1)
    page, slot = table[0, 1], 14
    src = c.slot(0, 32)
    assert np.array_equal(pages.k[0, page, :, slot].float().cpu().numpy(),
                          c.k[0, src[0], :, src[1]])
    kept = c.k[0, table[0, 1], :, 15]  # slot of the refused second entry
    assert np.array_equal(pages.k[0, table[0, 1], :, 15].float().cpu().numpy(), kept)


def test_captured_calls_replay(cuda):
    """Append, copy, table write and compaction in one CUDA graph: host arrays
    are read at capture, device arrays at each replay."""
    c = Paged(9, [40, 20], 2, 16, 64, spare=6, filler=0.0)
    pages = c.device()
    kn, vn = torch.randn(2, 4, 128, device="cuda").bfloat16()
    start, lens = ints([0, 2, 4]), ints([40, 20])
    base, keep, n_keep = ints([38, 18]), ints([[1], [0]]), ints([1, 0])
    new_len, table = ints([0, 0]), torch.zeros(8, dtype=torch.int32, device="cuda")
    src, dst = [int(c.table[0, 0])], [int(c.spare[0])]
    nk.device_status()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        nk.kv_pages_append(pages, kn, vn, start, lens, max_new=2)
        nk.kv_pages_copy(pages, src, dst)
        nk.kv_table_write(table, [5, 6], [1, 7])
        nk.kv_pages_compact(pages, lens, base, keep, n_keep, new_len=new_len)
    for _ in range(2):
        kn.normal_()
        vn.normal_()
        table.zero_()
        g.replay()
        torch.cuda.synchronize()
        page, slot = c.slot(0, 38)  # the second new token has closed up
        assert torch.equal(pages.k[0, page, :, slot].reshape(-1), kn[1])
        assert torch.equal(pages.v[0, page, :, slot].reshape(-1), vn[1])
        assert torch.equal(pages.k[:, dst[0]], pages.k[:, src[0]])
        assert table.tolist() == [0, 5, 0, 0, 0, 0, 0, 6] and new_len.tolist() == [39, 18]
    nk.device_status()


def test_offsets_past_32_bits(cuda):
    # 2^31 + channels of a pool: the last pages of the second layer
    pages, heads, ps, d = 70000, 2, 64, 128
    k = torch.zeros(2, pages, heads, ps, d, dtype=torch.bfloat16, device=cuda)
    v = torch.zeros_like(k)
    table = ints([[pages - 1, pages - 2]])
    kv = nk.KvPages(k, v, table)
    new = torch.randn(70, heads * d, device=cuda).bfloat16()
    nk.kv_pages_append(kv, new, new, ints([0, 70]), ints([70]), max_new=70, layer=1)
    nk.kv_pages_copy(kv, [pages - 1], [3])
    nk.kv_pages_compact(kv, ints([70]), ints([0]), ints([[5, 69]]), ints([2]))
    q = torch.randn(1, heads * d, device=cuda).bfloat16()
    out = nk.attention_paged(q, kv, ints([0, 1]), ints([2]), heads, layer=1)
    nk.device_status()
    want = new[:64].view(64, heads, d).transpose(0, 1)
    assert torch.equal(k[1, 3], want) and torch.equal(v[1, 3], want)
    assert torch.equal(k[1, pages - 1, :, 0].reshape(-1), new[5])
    assert torch.equal(k[1, pages - 1, :, 1].reshape(-1), new[69])
    assert not k[0].any() and not v[0].any()
    two = torch.stack([new[5], new[69]]).double().view(2, heads, d)
    w = torch.softmax((two * q.double().view(heads, d)).sum(-1) / d**0.5, 0)
    ref = (w[:, :, None] * two).sum(0).reshape(1, -1)
    mag = (w[:, :, None] * two.abs()).sum(0).reshape(1, -1)
    # weights rounded to bf16 (2^-8 each) and the bf16 result
    assert ((out.double() - ref).abs() <= (2**-8 + 2**-11) * mag + 2**-8 * ref.abs()).all()


# ---------------------------------------------------- the cache as it is used
def test_cache_grows_forks_and_frees(cuda):
    """Prefill, fork, drafts, acceptance, truncation and reuse of freed pages:
    the pages of every sequence hold the tokens that a list holds."""
    heads, d, ps, layers = 2, 64, 16, 2
    r = np.random.default_rng(0)
    cache = nk_paged.PagedKvCache(40, heads, d, max_seqs=6, max_len=200, page_size=ps,
                                  layers=layers)
    model = {}

    def feed(seqs, counts):
        step = cache.step(seqs, counts)
        new = torch.randn(layers, 2, step.tokens, heads * d, device="cuda").bfloat16()
        for i in range(layers):
            cache.append(step, new[i, 0], new[i, 1], layer=i)
        at = 0
        for s, c in zip(seqs, counts):
            model[s] = torch.cat([model[s], new[:, :, at:at + c]], 2)
            at += c
        return step

    def check():
        nk.device_status()
        for s, t in model.items():
            assert cache.length(s) == t.shape[2]
            ids = torch.tensor(cache.page_ids(s), device="cuda", dtype=torch.long)
            row = cache.pages.table[s, :len(ids)].long()
            assert torch.equal(ids, row)
            for j, pool in enumerate((cache.pages.k, cache.pages.v)):
                x = pool[:, ids].transpose(2, 3).reshape(layers, -1, heads * d)
                assert torch.equal(x[:, :t.shape[2]], t[:, j])
            for b in range(len(ids)):
                m = min(ps, t.shape[2] - b * ps)
                x = cache.pages.k[:, ids[b], :, :m]
                assert torch.equal(cache.pages.k_min[:, ids[b]], x.amin(2))
                assert torch.equal(cache.pages.k_max[:, ids[b]], x.amax(2))

    for _ in range(3):
        s = cache.new_sequence()
        model[s] = torch.zeros(layers, 2, 0, heads * d, dtype=torch.bfloat16, device="cuda")
    feed([0, 1, 2], [37, 16, 5])
    check()
    for parent in (0, 1, 0):
        model[cache.fork(parent)] = model[parent].clone()
    check()
    for _ in range(6):
        seqs = [int(x) for x in r.permutation(sorted(model))]
        counts = [int(x) for x in r.integers(0, 12, len(seqs))]
        step = feed(seqs, counts)
        check()
        keep = [sorted(r.choice(c, r.integers(0, c + 1), replace=False).tolist()) for c in counts]
        cache.accept(step, keep)
        for s, c, row in zip(seqs, counts, keep):
            n = model[s].shape[2] - c
            index = torch.tensor(list(range(n)) + [n + i for i in row], device="cuda")
            model[s] = model[s][:, :, index]
        check()
    cache.truncate(0, 20)
    model[0] = model[0][:, :, :20]
    cache.free(1)
    del model[1]
    check()
    s = cache.new_sequence()
    model[s] = torch.zeros(layers, 2, 0, heads * d, dtype=torch.bfloat16, device="cuda")
    feed([s, 0], [33, 1])
    check()
    for s in sorted(model):
        cache.free(s)
    assert cache.free_pages == 40


def test_new_lengths_beside_the_other_arrays(cuda):
    """The batch arrays of a call cut from one buffer, new_len next to them."""
    c = Paged(5, [40, 30], 1, 16, 64, filler=0.0)
    buf = ints([40, 30, 38, 20, 1, 2, -1, -1, 1, 0, 0, 9])
    kv_len, base, n_keep, new_len = (buf[i:i + 2] for i in (0, 2, 4, 6))
    got = nk.kv_pages_compact(c.device(), kv_len, base, buf[8:].view(2, 2), n_keep,
                              new_len=new_len)
    nk.device_status()
    assert got.data_ptr() == new_len.data_ptr()
    assert buf.tolist() == [40, 30, 38, 20, 1, 2, 39, 22, 1, 0, 0, 9]
    with pytest.raises(nk.NkError) as e:
        nk.kv_pages_compact(c.device(), kv_len, base, buf[8:].view(2, 2), n_keep, new_len=kv_len)
    assert e.value.code == nk.INVALID_PARAMS


def _apart(a, extra, device="cuda"):
    """The table as columns of a wider buffer, whose other entries are valid pages."""
    wide = torch.zeros(a.shape[0], a.shape[1] + extra, dtype=torch.int32, device=device)
    wide[:, :a.shape[1]] = ints(a)
    return wide[:, :a.shape[1]]


def test_tables_whose_rows_lie_apart(cuda):
    """The same results as with a table of its own, and lengths past the table's
    columns are refused although its rows are longer in memory."""
    lens, base, n_keep = [60, 33], [20, 0], [18, 30]
    c = Paged(4, lens, 1, 16, 64, spare=12, width=4, filler=0.0)
    dst = c.spare[:8].reshape(2, 4)
    keeps = ints([sorted(c.rng.choice(n - b, 30, replace=False)) for n, b in zip(lens, base)])
    kn, vn = torch.randn(2, 5, 64, device="cuda").bfloat16()
    q = torch.randn(5, 128, device="cuda").bfloat16()
    pools = []
    for apart in (False, True):
        pages = c.device()
        if apart:
            pages = nk.KvPages(pages.k, pages.v, _apart(c.table, 7), k_min=pages.k_min,
                               k_max=pages.k_max)
        nk.kv_pages_append(pages, kn, vn, ints([0, 2, 5]), ints(lens), max_new=3, max_kv=100)
        out = nk.attention_paged(q, pages, ints([0, 2, 5]), ints(lens), 2, max_q=3, max_kv=100)
        sparse = nk.attention_paged_sparse(q, pages, ints([0, 2, 5]), ints(lens), 2, 2, max_q=3)
        moved = nk.kv_pages_compact(pages, ints(lens), ints(base), keeps, ints(n_keep),
                                    dst_table=_apart(dst, 5) if apart else ints(dst))
        nk.device_status()
        pools.append([pages.k, pages.v, pages.k_min, pages.k_max, out, *sparse, moved])
        nk.kv_pages_compact(pages, ints(lens), ints(base), keeps, ints(n_keep))
        nk.device_status()
        # 66 tokens do not fit four columns of 16
        before = [x.clone() for x in pools[-1]]
        for call in (
                lambda: nk.kv_pages_append(pages, kn, vn, ints([0, 2, 5]), ints([33, 66]),
                                           max_new=3, max_kv=100, rows=ints([0, 1])),
                lambda: nk.kv_pages_compact(pages, ints([66, 66]), ints([60, 60]), ints([[5], [5]]),
                                            ints([1, 1])),
                lambda: nk.kv_pages_compact(pages, ints([60, 33]), ints([0, 0]),
                                            ints([list(range(40))] * 2), ints([0, 33]),
                                            dst_table=_apart(dst[:, :2], 9)),
                lambda: nk.attention_paged(q, pages, ints([0, 2, 5]), ints([66, 66]), 2, max_q=3,
                                           max_kv=100, out=pools[-1][4]),
                lambda: nk.kv_block_select(q, pages, ints([0, 2, 5]), ints([66, 66]), 2, 2, max_q=3,
                                           max_kv=100, out=pools[-1][6])):
            call()
            with pytest.raises(nk.NkError) as e:
                nk.device_status()
            assert e.value.code == nk.INVALID_PARAMS
        assert all(torch.equal(x, y) for x, y in zip(before[4:], pools[-1][4:]))
    for x, y in zip(*pools):
        assert torch.equal(x, y)


def test_truncation_of_forks_with_and_without_bounds(cuda):
    """A fork cut back inside a shared page and grown again leaves the other alone."""
    for bounds in (True, False):
        cache = nk_paged.PagedKvCache(8, 1, 64, max_seqs=3, max_len=64, page_size=16, bounds=bounds)
        a = cache.new_sequence()
        first = torch.randn(2, 32, 64, device="cuda").bfloat16()
        cache.append(cache.step([a], [32]), first[0], first[1])
        b = cache.fork(a)
        cache.truncate(b, 20)
        assert cache.free_pages == (5 if bounds else 6)
        more = torch.randn(2, 5, 64, device="cuda").bfloat16()
        cache.append(cache.step([b], [5]), more[0], more[1])
        nk.device_status()
        for s, want in ((a, first), (b, torch.cat([first[:, :20], more], 1))):
            ids = torch.tensor(cache.page_ids(s), device="cuda")
            n = want.shape[1]
            for pool, x in ((cache.pages.k, want[0]), (cache.pages.v, want[1])):
                assert torch.equal(pool[0, ids, 0].reshape(-1, 64)[:n], x)
            if bounds:
                for j in range(2):
                    x = want[0, 16 * j:16 * j + 16]
                    assert torch.equal(cache.pages.k_min[0, ids[j], 0], x.amin(0))
                    assert torch.equal(cache.pages.k_max[0, ids[j], 0], x.amax(0))
