"""The paged KV cache without a GPU: the entry points' refusals (argument
checks come before any device call) and the host bookkeeping of
nk_paged.PagedKvCache (pages, reference counts, copies before writes) driven
through random steps against sequences kept as plain lists."""
import ctypes

import numpy as np
import pytest

import nk
import nk_paged


# ------------------------------------------------------------- C ABI refusals
def _pages(**kw):
    f = dict(layers=1, pages=8, kv_heads=2, page_size=16, head_dim=64, k=4096, v=8192,
             k_min=None, k_max=None, table=256, table_rows=4, table_ld=4)
    f.update(kw)
    return nk.NkKvPages(*(f[n] for n, _ in nk.NkKvPages._fields_))


def _batch(**kw):
    f = dict(seqs=2, tokens=4, start=256, kv_len=256, rows=None, max_new=2, max_kv=64)
    f.update(kw)
    return nk.NkKvBatch(*(f[n] for n, _ in nk.NkKvBatch._fields_))


def _attn(**kw):
    f = dict(q=4096, ld_q=256, q_heads=4, tree_mask=None, blocks=None, max_blocks=0, has_scale=0,
             scale=0.0, out=4096, out_dtype=nk.BF16)
    f.update(kw)
    return nk.NkPagedAttentionArgs(*(f[n] for n, _ in nk.NkPagedAttentionArgs._fields_))


def _r(x):
    return ctypes.byref(x)


BAD_PAGES = [
    (dict(layers=0), nk.INVALID_SHAPE), (dict(pages=0), nk.INVALID_SHAPE),
    (dict(kv_heads=-1), nk.INVALID_SHAPE), (dict(page_size=0), nk.INVALID_SHAPE),
    (dict(head_dim=96), nk.UNSUPPORTED), (dict(page_size=48), nk.UNSUPPORTED),
    (dict(page_size=256), nk.UNSUPPORTED), (dict(kv_heads=70000), nk.UNSUPPORTED),
    (dict(pages=2**26, kv_heads=2), nk.UNSUPPORTED),  # token rows pass 2^31
    (dict(k=None), nk.INVALID_PARAMS), (dict(v=None), nk.INVALID_PARAMS),
    (dict(k=4104), nk.INVALID_PARAMS), (dict(k_min=4096), nk.INVALID_PARAMS),
]
BAD_TABLE = [(dict(table=None), nk.INVALID_PARAMS), (dict(table_rows=0), nk.INVALID_PARAMS),
             (dict(table_ld=0), nk.INVALID_PARAMS)]
BAD_BATCH = [
    (dict(seqs=-1), nk.INVALID_SHAPE), (dict(tokens=-1), nk.INVALID_SHAPE),
    (dict(max_new=-1), nk.INVALID_SHAPE), (dict(max_kv=-1), nk.INVALID_SHAPE),
    (dict(seqs=65536, rows=256), nk.UNSUPPORTED), (dict(tokens=2**31), nk.UNSUPPORTED),
    (dict(max_kv=2**31 - 512), nk.UNSUPPORTED), (dict(max_new=5), nk.INVALID_PARAMS),
    (dict(max_new=3, max_kv=2), nk.INVALID_PARAMS), (dict(start=None), nk.INVALID_PARAMS),
    (dict(kv_len=None), nk.INVALID_PARAMS), (dict(seqs=5), nk.INVALID_PARAMS),
]


@pytest.mark.parametrize("kw,code", BAD_PAGES + BAD_TABLE)
def test_bad_pools_are_refused_by_every_entry_point(kw, code):
    lib, kv, b, n = nk.lib(), _pages(**kw), _batch(), ctypes.c_size_t()
    assert lib.nk_kv_pages_append(_r(kv), 0, _r(b), 4096, 128, 4096, 128, None) == code
    assert lib.nk_attention_paged_workspace_bytes(_r(kv), _r(b), _r(_attn()), _r(n)) == code
    assert lib.nk_attention_paged(_r(kv), 0, _r(b), _r(_attn()), None, 0, None) == code
    if "k_min" not in kw:
        kv.k_min, kv.k_max = 4096, 4096
    assert lib.nk_kv_block_select(_r(kv), 0, _r(b), 4096, 256, 4, 4, 1, 1, 4096, None, 0,
                                  None) == code
    a = nk.NkKvCompactArgs(1, None, 256, 256, 256, 4, 256, 4, None, 0, None)
    assert lib.nk_kv_pages_compact(_r(kv), _r(a), None) == code
    if (kw, code) in BAD_PAGES:
        ids = (ctypes.c_int32 * 2)(0, 1)
        assert lib.nk_kv_pages_copy(_r(kv), ids, ids, 1, None) == code


@pytest.mark.parametrize("kw,code", BAD_BATCH)
def test_bad_batches_are_refused(kw, code):
    lib, kv, b = nk.lib(), _pages(k_min=4096, k_max=4096), _batch(**kw)
    assert lib.nk_kv_pages_append(_r(kv), 0, _r(b), 4096, 128, 4096, 128, None) == code
    assert lib.nk_attention_paged(_r(kv), 0, _r(b), _r(_attn()), None, 0, None) == code
    assert lib.nk_kv_block_select(_r(kv), 0, _r(b), 4096, 256, 4, 4, 1, 1, 4096, None, 0,
                                  None) == code


def test_append_refusals_and_empty_calls():
    lib, kv, b = nk.lib(), _pages(), _batch()
    call = lib.nk_kv_pages_append
    assert call(None, 0, _r(b), 4096, 128, 4096, 128, None) == nk.INVALID_PARAMS
    assert call(_r(kv), 1, _r(b), 4096, 128, 4096, 128, None) == nk.INVALID_PARAMS
    assert call(_r(kv), -1, _r(b), 4096, 128, 4096, 128, None) == nk.INVALID_PARAMS
    assert call(_r(kv), 0, None, 4096, 128, 4096, 128, None) == nk.INVALID_PARAMS
    assert call(_r(kv), 0, _r(b), 4096, 120, 4096, 128, None) == nk.INVALID_PARAMS
    assert call(_r(kv), 0, _r(b), 4096, 128, 4096, 132, None) == nk.INVALID_PARAMS
    assert call(_r(kv), 0, _r(b), None, 128, 4096, 128, None) == nk.INVALID_PARAMS
    assert call(_r(kv), 0, _r(b), 4098, 128, 4096, 128, None) == nk.INVALID_PARAMS
    for empty in (dict(seqs=0), dict(tokens=0, max_new=0), dict(max_new=0)):
        assert call(_r(kv), 0, _r(_batch(**empty)), None, 128, None, 128, None) == nk.OK


def test_copy_refusals():
    lib, kv = nk.lib(), _pages()

    def call(src, dst, n=None):
        a, b = (ctypes.c_int32 * 8)(*src), (ctypes.c_int32 * 8)(*dst)
        return lib.nk_kv_pages_copy(_r(kv), a, b, len(src) if n is None else n, None)

    assert call([0], [8]) == nk.PAGE_OUT_OF_RANGE
    e = nk.last_error()
    assert (e.actual, e.expected, e.index) == (8, 8, 0)
    assert call([0, -1], [2, 3]) == nk.PAGE_OUT_OF_RANGE
    assert call([0, 1], [2, 2]) == nk.INVALID_PARAMS  # one destination twice
    assert nk.last_error().index == 1
    assert call([0, 2], [2, 3]) == nk.INVALID_PARAMS  # a destination that is a source
    assert call([1], [1]) == nk.INVALID_PARAMS
    kv.pages = 2**26  # a pool too large for a bit a page
    kv.kv_heads = 1
    assert call([0, 1, 2], [9, 2**25, 9]) == nk.INVALID_PARAMS
    assert nk.last_error().index == 2
    assert call([0, 2**25 + 7], [2**25 + 7, 3]) == nk.INVALID_PARAMS
    assert nk.last_error().index == 1
    assert call([0, 2**26], [2, 3]) == nk.PAGE_OUT_OF_RANGE
    kv.pages, kv.kv_heads = 8, 2
    assert call([], [], -1) == nk.INVALID_SHAPE
    assert call([], []) == nk.OK
    assert lib.nk_kv_pages_copy(_r(kv), None, None, 1, None) == nk.INVALID_PARAMS


def test_table_write_refusals():
    lib = nk.lib()
    v, o = (ctypes.c_int32 * 4)(1, 2, 3, 4), (ctypes.c_int64 * 4)(0, 2, 1, 2)
    assert lib.nk_kv_table_write(4096, 4, None, v, 5, None) == nk.LENGTH_MISMATCH
    assert lib.nk_kv_table_write(4096, 2, o, v, 2, None) == nk.INVALID_PARAMS
    assert (nk.last_error().index, nk.last_error().actual) == (1, 2)
    assert lib.nk_kv_table_write(4096, 4, o, v, 4, None) == nk.INVALID_PARAMS  # 2 twice
    assert lib.nk_kv_table_write(None, 4, None, v, 4, None) == nk.INVALID_PARAMS
    assert lib.nk_kv_table_write(4096, 4, None, v, -1, None) == nk.INVALID_SHAPE
    assert lib.nk_kv_table_write(None, 0, None, None, 0, None) == nk.OK


def test_compact_refusals():
    lib, kv = nk.lib(), _pages()

    def call(**kw):
        f = dict(seqs=2, rows=None, kv_len=256, base=256, keep=256, keep_ld=4, n_keep=256,
                 max_keep=4, dst_table=None, dst_ld=0, new_len=None)
        f.update(kw)
        a = nk.NkKvCompactArgs(*(f[n] for n, _ in nk.NkKvCompactArgs._fields_))
        return lib.nk_kv_pages_compact(_r(kv), _r(a), None)

    assert lib.nk_kv_pages_compact(_r(kv), None, None) == nk.INVALID_PARAMS
    assert call(seqs=-1) == nk.INVALID_SHAPE
    assert call(max_keep=-1) == nk.INVALID_SHAPE
    assert call(seqs=65536, rows=256) == nk.UNSUPPORTED
    assert call(max_keep=5) == nk.INVALID_PARAMS
    assert call(seqs=5) == nk.INVALID_PARAMS
    for name in ("kv_len", "base", "keep", "n_keep"):
        assert call(**{name: None}) == nk.INVALID_PARAMS
    assert call(dst_table=256) == nk.INVALID_PARAMS  # no width
    assert call(seqs=0) == nk.OK


def test_attention_refusals():
    lib, kv = nk.lib(), _pages()
    n = ctypes.c_size_t()

    def call(b=None, ws=None, ws_bytes=0, **kw):
        return lib.nk_attention_paged(_r(kv), 0, _r(b or _batch()), _r(_attn(**kw)), ws, ws_bytes,
                                      None)

    assert lib.nk_attention_paged(_r(kv), 0, _r(_batch()), None, None, 0, None) == \
        nk.INVALID_PARAMS
    assert call(q_heads=0) == nk.INVALID_SHAPE
    assert call(q_heads=3) == nk.HEAD_COUNT_MISMATCH
    assert (nk.last_error().expected, nk.last_error().actual) == (3, 2)
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        assert call(has_scale=1, scale=bad) == nk.INVALID_SCALE
    assert call(ld_q=248) == nk.INVALID_PARAMS
    assert call(ld_q=260) == nk.INVALID_PARAMS
    assert call(out_dtype=7) == nk.INVALID_PARAMS
    assert call(tree_mask=256, blocks=256, max_blocks=1) == nk.UNSUPPORTED
    assert call(_batch(tokens=200, max_new=65, max_kv=300), tree_mask=256) == nk.UNSUPPORTED
    assert call(blocks=256, max_blocks=0) == nk.INVALID_PARAMS
    assert call(q=None) == nk.INVALID_PARAMS
    assert call(out=None) == nk.INVALID_PARAMS
    assert call(q=4104) == nk.INVALID_PARAMS
    long = _batch(max_kv=100000)
    assert lib.nk_attention_paged_workspace_bytes(_r(kv), _r(long), _r(_attn()), None) == \
        nk.INVALID_PARAMS
    assert lib.nk_attention_paged_workspace_bytes(_r(kv), _r(long), _r(_attn()), _r(n)) == nk.OK
    assert n.value > 0
    assert call(long, 4096, n.value - 1) == nk.WORKSPACE_TOO_SMALL
    assert nk.last_error().expected == n.value
    assert call(long, None, n.value) == nk.WORKSPACE_TOO_SMALL
    for empty in (dict(seqs=0), dict(tokens=0, max_new=0), dict(max_new=0)):
        assert call(_batch(**empty), q=None, out=None) == nk.OK


def test_block_select_refusals():
    lib, kv = nk.lib(), _pages(k_min=4096, k_max=4096)

    def call(kv=kv, b=None, q=4096, ld=256, heads=4, top_k=4, sink=1, local=1, out=4096, ws=4096,
             n=1 << 20):
        return lib.nk_kv_block_select(_r(kv), 0, _r(b or _batch()), q, ld, heads, top_k, sink,
                                      local, out, ws, n, None)

    assert call(kv=_pages()) == nk.INVALID_PARAMS  # no bounds kept
    assert call(heads=0) == nk.INVALID_SHAPE
    assert call(heads=5) == nk.HEAD_COUNT_MISMATCH
    assert call(ld=255) == nk.INVALID_PARAMS
    assert call(sink=-1) == nk.INVALID_PARAMS
    assert call(local=0) == nk.INVALID_PARAMS
    assert call(sink=2, local=3) == nk.INVALID_PARAMS
    assert call(b=_batch(tokens=65536)) == nk.UNSUPPORTED
    assert call(q=None) == nk.INVALID_PARAMS
    assert call(out=None) == nk.INVALID_PARAMS
    assert call(n=1) == nk.WORKSPACE_TOO_SMALL
    assert call(ws=None) == nk.WORKSPACE_TOO_SMALL
    assert call(b=_batch(seqs=0), q=None, out=None, ws=None, n=0) == nk.OK


def test_binding_refuses_host_tensors():
    import torch

    k = torch.zeros(1, 2, 1, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        nk.KvPages(k, k.clone(), torch.zeros(1, 2, dtype=torch.int32))
    with pytest.raises(TypeError):
        nk.KvPages(k.float(), k, torch.zeros(1, 2, dtype=torch.int32))


# ---------------------------------------------------------------- bookkeeping
class HostCache(nk_paged.PagedKvCache):
    """The bookkeeping over numpy pools: what each device call does, in plain
    Python.  A token is one number."""

    def __init__(self, pages, max_seqs, max_len, page_size):
        self.page_size, self.layers, self.max_len = page_size, 1, max_len
        self.width = -(-max_len // page_size)
        self._init_host(pages, max_seqs)
        self.pool = np.full((pages, page_size), -1, np.int64)
        self.device_table = np.zeros((max_seqs, self.width), np.int32)

    def _copy_pages(self, src, dst, stream):
        assert len(set(dst)) == len(dst) and not set(dst) & set(src)
        self.pool[dst] = self.pool[src]

    def _write_table(self, offsets, values, stream):
        assert len(set(np.asarray(offsets).tolist())) == len(offsets)
        self.device_table.reshape(-1)[np.asarray(offsets)] = values

    def _upload(self, values, stream):
        return np.asarray(values)

    def slot(self, row, pos):
        return self.device_table[row, pos // self.page_size], pos % self.page_size

    def write(self, step, tokens):
        at = 0
        for s, c, n in zip(step.seqs, step.counts, step.lens):
            for p in range(n - c, n):
                page, slot = self.slot(s, p)
                assert self._refs[page] == 1, "a shared page is written"
                self.pool[page, slot] = tokens[at]
                at += 1

    def _compact(self, step, base, keep, n_keep, stream):
        for i, s in enumerate(step.seqs):
            first, end = base[i] // self.page_size, self._blocks(base[i] + n_keep[i])
            for b in range(first, end):  # pages whose slots or bounds are written
                assert self._refs[self.device_table[s, b]] == 1
            for j in range(n_keep[i]):
                fp, fs = self.slot(s, base[i] + keep[i][j])
                tp, ts = self.slot(s, base[i] + j)
                self.pool[tp, ts] = self.pool[fp, fs]

    def read(self, s):
        return [int(self.pool[self.slot(s, p)]) for p in range(self.length(s))]


def _check(cache, model):
    for s, tokens in model.items():
        assert cache.read(s) == tokens, s
    # every page is free or counted once for each sequence that holds it
    refs = np.zeros(len(cache._refs), int)
    for s in model:
        for p in cache.page_ids(s):
            refs[p] += 1
    assert (refs == cache._refs).all()
    assert sorted(cache._free) == np.flatnonzero(refs == 0).tolist()


@pytest.mark.parametrize("seed,page_size", [(0, 4), (1, 1), (2, 16), (3, 3)])
def test_random_steps_keep_every_sequence(seed, page_size):
    rng = np.random.default_rng(seed)
    cache, model, count = HostCache(60, 9, 60, page_size), {}, 0
    for _ in range(600):
        what = rng.integers(0, 6)
        live = sorted(model)
        try:
            if what == 0:
                s = cache.new_sequence()
                model[s] = []
            elif what == 1 and live:
                s = int(rng.choice(live))
                child = cache.fork(s)
                model[child] = list(model[s])
            elif what == 2 and len(live) > 3:
                s = int(rng.choice(live))
                cache.free(s)
                del model[s]
            elif what == 3 and live:
                s = int(rng.choice(live))
                n = int(rng.integers(0, len(model[s]) + 1))
                cache.truncate(s, n)
                model[s] = model[s][:n]
            elif live:
                seqs = [int(x) for x in rng.permutation(live)[:rng.integers(1, len(live) + 1)]]
                counts = [int(x) for x in rng.integers(0, 9, len(seqs))]
                step = cache.step(seqs, counts)
                new = list(range(count, count + step.tokens))
                count += step.tokens
                cache.write(step, new)
                at = 0
                for s, c in zip(seqs, counts):
                    model[s] = model[s] + new[at:at + c]
                    at += c
                if what == 5:  # some of the step's tokens are accepted
                    if rng.integers(0, 2):  # a fork of the drafted state keeps them all
                        child = cache.fork(seqs[0])
                        model[child] = list(model[seqs[0]])
                    keep = [sorted(rng.choice(c, rng.integers(0, c + 1), replace=False).tolist())
                            for c in counts]
                    try:
                        cache.accept(step, keep)
                    except RuntimeError as e:
                        assert "out of pages" in str(e)
                    else:
                        for s, c, row in zip(seqs, counts, keep):
                            t = model[s]
                            model[s] = t[:len(t) - c] + [t[len(t) - c + i] for i in row]
        except RuntimeError as e:
            assert "out of" in str(e)
        except ValueError as e:
            assert "max_len" in str(e)
        _check(cache, model)
    assert count > 500


def test_fork_shares_full_pages_and_copies_before_a_write():
    c = HostCache(8, 4, 32, 4)
    a = c.new_sequence()
    c.write(c.step([a], [10]), list(range(10)))
    b = c.fork(a)
    assert c.page_ids(a)[:2] == c.page_ids(b)[:2] and c.page_ids(a)[2] != c.page_ids(b)[2]
    assert [c.refcount(p) for p in c.page_ids(a)] == [2, 2, 1]
    d = c.fork(a)
    c.truncate(d, 6)  # its last page is shared with a and b, and now partial
    assert c.read(d) == list(range(6)) and c.read(a) == list(range(10))
    c.write(c.step([d], [1]), [99])
    assert c.read(d) == list(range(6)) + [99] and c.read(b) == list(range(10))
    for s in (a, b, d):
        c.free(s)
    assert c.free_pages == 8


def test_bookkeeping_refusals_change_nothing():
    c = HostCache(3, 2, 12, 4)
    a = c.new_sequence()
    c.write(c.step([a], [9]), list(range(9)))
    with pytest.raises(RuntimeError, match="out of pages"):
        c.fork(a)
    with pytest.raises(ValueError, match="max_len"):
        c.step([a], [4])
    with pytest.raises(ValueError, match="twice"):
        c.step([a, a], [1, 1])
    with pytest.raises(ValueError, match="negative"):
        c.step([a], [-1])
    with pytest.raises(ValueError, match="one length"):
        c.step([a], [])
    with pytest.raises(ValueError, match="no sequence"):
        c.step([1], [1])
    with pytest.raises(ValueError, match="no sequence"):
        c.length(-1)
    with pytest.raises(ValueError):
        c.truncate(a, 10)
    b = c.new_sequence()
    with pytest.raises(RuntimeError, match="out of pages"):
        c.step([a, b], [1, 1])
    with pytest.raises(RuntimeError, match="out of sequences"):
        c.new_sequence()
    step = c.step([a], [3])
    for bad in ([[0, 0]], [[2, 1]], [[3]], [[-1]], [[], []]):
        with pytest.raises(ValueError):
            c.accept(step, bad)
    c.truncate(a, 11)
    with pytest.raises(ValueError, match="changed"):
        c.accept(step, [[0]])
    assert c.read(a)[:9] == list(range(9)) and c.length(a) == 11
    _check(c, {a: c.read(a), b: []})


def test_host_arrays_that_do_not_fit_are_refused():
    """A 64-bit page id or a fraction must not turn into another page."""
    for bad in (np.array([2**32 + 1]), np.array([-2**31 - 1]), np.array([1.5])):
        with pytest.raises(ValueError):
            nk._host_ints(bad, np.int32)
    with pytest.raises(OverflowError):
        nk._host_ints([2**32 + 1], np.int32)
    for good in ([], [3, 4], np.array([3, 4]), np.array([3, 4], np.int32)[::-1], np.zeros(0)):
        got = nk._host_ints(good, np.int32)
        assert got.dtype == np.int32 and got.flags.c_contiguous
        assert got.tolist() == list(map(int, good))


def test_a_width_without_its_array_is_refused():
    """An empty list or table has no address, which would mean none was given."""
    lib, kv, n = nk.lib(), _pages(), ctypes.c_size_t()
    for width in (1, 8, -1):
        a = _attn(max_blocks=width)
        assert lib.nk_attention_paged(_r(kv), 0, _r(_batch()), _r(a), None, 0, None) == \
            nk.INVALID_PARAMS
        assert lib.nk_attention_paged_workspace_bytes(_r(kv), _r(_batch()), _r(a), _r(n)) == \
            nk.INVALID_PARAMS
        c = nk.NkKvCompactArgs(2, None, 256, 256, 256, 4, 256, 4, None, width, None)
        assert lib.nk_kv_pages_compact(_r(kv), _r(c), None) == nk.INVALID_PARAMS


@pytest.mark.parametrize("name,at", [
    ("kv_len", 0), ("kv_len", 8), ("kv_len", -8), ("base", 0), ("n_keep", 4), ("rows", -4),
    ("keep", 0), ("keep", 36), ("dst_table", 56), ("table", 60)])
def test_new_lengths_over_an_array_that_is_read_are_refused(name, at):
    lib, kv = nk.lib(), _pages()
    f = dict(seqs=3, rows=2048, kv_len=4096, base=8192, keep=16384, keep_ld=4, n_keep=32768,
             max_keep=2, dst_table=65536, dst_ld=5)
    f["new_len"] = (256 if name == "table" else f[name]) + at
    a = nk.NkKvCompactArgs(*(f[n] for n, _ in nk.NkKvCompactArgs._fields_))
    assert lib.nk_kv_pages_compact(_r(kv), _r(a), None) == nk.INVALID_PARAMS
    assert b"new_len" in nk.last_error().message


@pytest.mark.parametrize("bad", [
    [1.5], [1, 2.0], (0.0,), [np.float32(3)], [None], ["1"], [2**70], [[1], [2.5]],
    np.array([2.5], object), np.array([True])])
def test_host_lists_that_are_no_whole_numbers_are_refused(bad):
    """A list of fractions must not turn into the pages below them."""
    with pytest.raises((ValueError, OverflowError, TypeError)):
        nk._host_ints(bad, np.int32)
    for good in ([1, np.int64(2)], (3,), range(4), [], 7, [2**31 - 1, -2**31]):
        assert nk._host_ints(good, np.int32).tolist() == np.atleast_1d(good).tolist()
    with pytest.raises(OverflowError):
        nk._host_ints([2**31], np.int32)
    assert nk._host_ints([2**40], np.int64).tolist() == [2**40]


def test_truncation_without_bounds_takes_no_page():
    """Nothing of a shared page is written when no bounds are kept."""
    class NoBounds(HostCache):
        _bounds = False

        def _compact(self, step, base, keep, n_keep, stream):
            for i, s in enumerate(step.seqs):
                for j in range(n_keep[i]):
                    assert self._refs[self.slot(s, base[i] + j)[0]] == 1
            self.moved = n_keep

    for kind, need in ((NoBounds, 0), (HostCache, 1)):
        c = kind(4, 3, 32, 4)
        a = c.new_sequence()
        c.write(c.step([a], [12]), list(range(12)))
        b = c.fork(a)  # three shared pages, one free
        d = c.new_sequence()
        c.write(c.step([d], [1 - need]), [77][need:])
        if need:
            assert c.free_pages == 1
        c.truncate(b, 6)
        assert c.free_pages == 0 and c.read(b) == list(range(6))
        _check(c, {a: list(range(12)), b: list(range(6)), d: c.read(d)})
        if not need:  # a write asks for the page
            with pytest.raises(RuntimeError, match="out of pages"):
                c.step([b], [1])
