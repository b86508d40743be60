"""The pages of the paged cache (apk_pages_*) against a model in plain Python (tests/paged_util.py), the copies of pages, and
a whole run of them: extend, rotary rows, K/V store, attention, fork, truncate, compact."""
import numpy as np
import pytest

from tests.paged_util import PageModel, attention64, ceil_div

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def be():
    import allpaka_amd as apk

    b = apk.Backend(0)
    yield b
    b.close()


def i32(x):
    return torch.tensor(np.asarray(x, np.int64).astype(np.uint32).view(np.int32), device="cuda")


def new_cache(be, n_pages, page, n_seq, max_pages, planes=2, width=8):
    import allpaka_amd as apk

    region = torch.arange(planes * n_pages * page * width, device="cuda").remainder(4093).to(torch.float16).view(planes, n_pages * page, width).contiguous()
    return apk.PagedCache(be, region, page, n_seq, max_pages)


def same(cache, model):
    """The device's state is the model's, and its free bits, counters and scratch are what they have to be."""
    pool = cache.pool.cpu().numpy().view(np.uint32)
    n = model.n_pages
    assert pool[4:4 + n].tolist() == model.refs
    assert cache.kv_len.cpu().tolist() == model.kv_len
    table = cache.page_table.cpu().numpy()
    for s, t in enumerate(model.table):
        assert table[s, :len(t)].tolist() == t, s
    free = model.free()
    assert pool[0] == len(free)
    words = pool[4 + n:4 + n + ceil_div(n, 32)]
    assert [p for p in range(len(words) * 32) if words[p // 32] >> (p % 32) & 1] == free
    assert not pool[4 + n + len(words):4 + 3 * n + len(words)].any()  # counts and names are zero between calls


def check_step(step, want, rows):
    q_off, positions, slots, pairs = want
    assert step.q_off.cpu().tolist() == q_off
    pad = rows - len(slots)
    assert step.positions.cpu().tolist() == positions + [0] * pad
    assert step.slots.cpu().numpy().view(np.uint32).tolist() == slots + [2 ** 32 - 1] * pad
    k = int(step.n_pairs.item())
    assert [tuple(p) for p in step.pairs.cpu().tolist()[:k]] == pairs


@pytest.mark.parametrize("page", [1, 4, 16, 33])
@pytest.mark.parametrize("n_pages,n_seq", [(1, 1), (40, 5), (700, 33), (5000, 1500)])
def test_random_histories(be, page, n_pages, n_seq):
    """Random steps of every kind, refused ones among them, state compared after each; planes follow the pairs."""
    import allpaka_amd.lib as l

    r = np.random.default_rng([n_pages, n_seq, page])
    max_pages = max(2, min(n_pages, 60))
    cache, model = new_cache(be, n_pages, page, n_seq, max_pages), PageModel(n_pages, page, n_seq, max_pages)
    rows_np = cache.region.cpu().numpy().reshape(2, n_pages, -1)
    same(cache, model)
    share = max(1, n_pages * page // (3 * n_seq))
    refused = 0
    for it in range(40):
        kind = ["extend", "extend", "extend", "fork", "truncate", "compact"][int(r.integers(0, 6))]
        if kind == "extend":
            n_new = r.integers(0, [2, share + 2, 3 * page + 2][int(r.integers(0, 3))], n_seq).tolist()
            rows = sum(n_new) + int(r.integers(-1, 4))
            rows = max(rows, 0)
            want = model.extend(n_new, rows)
            step = cache.extend(i32(n_new), rows)
            be.sync()
            if want is None:
                refused += 1
                assert be.take_faults() & (l.FAULT_NO_PAGES | l.FAULT_ROW_RANGE | l.FAULT_CACHE_RANGE)
                want = ([0] * (n_seq + 1), [], [], [])
            check_step(step, want, rows)
            for a, b in want[3]:
                rows_np[:, a] = rows_np[:, b]
        elif kind == "fork":
            k = int(r.integers(1, min(n_seq, 20) + 1))
            src, dst = r.integers(0, n_seq + (it % 3 == 0), k).tolist(), r.integers(0, n_seq, k).tolist()
            empty = [s for s in range(n_seq) if not model.kv_len[s]]
            if empty and it % 2:
                dst = [int(x) for x in r.permutation(empty)[:k]]
                src = src[:len(dst)]
            bad = model.fork(src, dst)
            cache.fork(i32(src), i32(dst))
            assert be.take_faults() == (l.FAULT_ROW_RANGE if bad else 0)
        elif kind == "truncate":
            cut = [int(r.integers(0, n + 3)) if r.random() < 0.5 else 2 ** 32 - 1 for n in model.kv_len]
            if r.random() < 0.5:
                cut = [0 if r.random() < 0.3 else c for c in cut]
            model.truncate(cut)
            cache.truncate(i32(cut))
        else:
            pairs = model.compact()
            cache.compact()
            be.sync()
            k = int(cache._n_moves.item())
            assert [tuple(p) for p in cache._moves.cpu().tolist()[:k]] == pairs
            for a, b in pairs:
                rows_np[:, a] = rows_np[:, b]
        be.sync()
        same(cache, model)
        assert be.take_faults() == 0
    assert np.array_equal(cache.region.cpu().numpy().reshape(2, n_pages, -1).view(np.uint16), rows_np.view(np.uint16))


def test_a_shared_tail_is_copied_for_all_holders_but_the_last_that_writes(be):
    cache, model = new_cache(be, 12, 4, 4, 6), PageModel(12, 4, 4, 6)
    for m, c in ((model.extend, cache.extend),):
        m([6, 0, 0, 0], 6)
        c(i32([6, 0, 0, 0]), 6)
    model.fork([0, 0, 0], [1, 2, 3])
    cache.fork(i32([0, 0, 0]), i32([1, 2, 3]))
    be.sync()
    same(cache, model)
    assert model.refs[:2] == [4, 4]
    want = model.extend([1, 0, 1, 1], 3)  # sequence 1 does not write: three copies, the old tail stays with it
    assert len(want[3]) == 3
    check_step(cache.extend(i32([1, 0, 1, 1]), 3), want, 3)
    be.sync()
    same(cache, model)
    assert model.refs[1] == 1
    want = model.extend([1, 1, 1, 1], 4)
    assert want[3] == []
    check_step(cache.extend(i32([1, 1, 1, 1]), 4), want, 4)
    model.truncate([0, 0, 0, 0])
    cache.truncate(i32([0, 0, 0, 0]))
    be.sync()
    same(cache, model)
    assert cache.free_pages == 12
    model.extend([6, 0, 0, 0], 6)
    cache.extend(i32([6, 0, 0, 0]), 6)
    model.fork([0], [2])
    cache.fork(i32([0]), i32([2]))
    want = model.extend([2, 0, 3, 0], 5)  # both holders write: one copy, the last one keeps the page
    assert len(want[3]) == 1
    check_step(cache.extend(i32([2, 0, 3, 0]), 5), want, 5)
    be.sync()
    same(cache, model)


def test_refused_steps_change_nothing(be):
    import allpaka_amd.lib as l

    cache, model = new_cache(be, 6, 4, 3, 4), PageModel(6, 4, 3, 4)
    model.extend([5, 3, 0], 8)
    cache.extend(i32([5, 3, 0]), 8)
    model.fork([0], [2])
    cache.fork(i32([0]), i32([2]))
    for n_new, rows, fault in (([8, 8, 8], 30, l.FAULT_NO_PAGES), ([1, 1, 1], 2, l.FAULT_ROW_RANGE), ([12, 0, 0], 12, l.FAULT_CACHE_RANGE | l.FAULT_NO_PAGES),
                               ([0, 2 ** 32 - 1, 0], 8, l.FAULT_CACHE_RANGE)):
        step = cache.extend(i32(n_new), rows)
        got = be.take_faults()
        assert got & fault and not got & ~(fault | l.FAULT_CACHE_RANGE | l.FAULT_ROW_RANGE), (n_new, got)
        check_step(step, ([0] * 4, [], [], []), rows)
        same(cache, model)


def test_foreign_tables_are_reported(be):
    import allpaka_amd.lib as l

    cache, model = new_cache(be, 6, 4, 2, 4), PageModel(6, 4, 2, 4)
    table, n = i32([[1, 99, 0, 0], [2, 3, 0, 0]]), i32([8, 7])
    cache.adopt(table, n)
    assert be.take_faults() == l.FAULT_CACHE_RANGE
    assert cache.refs.cpu().tolist() == [0, 1, 1, 1, 0, 0] and cache.free_pages == 3
    cache.adopt(i32([[1, 4, 0, 0], [2, 3, 0, 0]]), i32([8, 70]))
    assert be.take_faults() == l.FAULT_CACHE_RANGE
    cache.adopt(i32([[1, 4, 0, 0], [2, 3, 0, 0]]), i32([8, 7]))
    model.table, model.kv_len, model.refs = [[1, 4], [2, 3]], [8, 7], [0, 1, 1, 1, 1, 0]
    same(cache, model)
    cache.page_table[0, 1] = 5  # a page nobody holds: its count stays at 0
    cache.truncate(i32([0, 2 ** 32 - 1]))
    assert be.take_faults() == l.FAULT_CACHE_RANGE
    assert cache.refs.cpu().tolist() == [0, 0, 1, 1, 1, 0]


@pytest.mark.parametrize("page_bytes,planes,n_pages", [(16, 3, 50), (48, 1, 9), (2048, 4, 64), (16384, 2, 40), (16400, 3, 21), (100000, 2, 16)])
def test_page_copies(be, page_bytes, planes, n_pages):
    r = np.random.default_rng(page_bytes)
    gap = 64  # bytes of every plane behind its pages: left alone
    plane = n_pages * page_bytes + gap
    host = r.integers(0, 256, (planes, plane), dtype=np.uint8)
    region = torch.from_numpy(host.copy()).cuda()
    order = r.permutation(n_pages)
    k = n_pages // 2
    pairs = np.stack([order[:k], order[k:2 * k]], 1)
    for count, most in ((k, k), (k, k - 1), (3, k), (0, k), (k, 10 * k)):
        before = region.cpu().numpy()
        n = i32([count])
        from allpaka_amd.lib import check

        torch.cuda.synchronize()
        check(be.L.apk_pages_copy(be.h, region.data_ptr(), planes, plane, n_pages, page_bytes, i32(pairs).data_ptr(), n.data_ptr(), most))
        be.sync()
        want = before.copy()
        for a, b in pairs[:min(count, most)]:
            want[:, a * page_bytes:(a + 1) * page_bytes] = before[:, b * page_bytes:(b + 1) * page_bytes]
        assert np.array_equal(region.cpu().numpy(), want), (count, most)
    bad = pairs.copy()
    bad[0, 0], bad[1, 1] = n_pages, -1
    t = i32(bad)
    torch.cuda.synchronize()
    before = region.cpu().numpy()
    check(be.L.apk_pages_copy(be.h, region.data_ptr(), planes, plane, n_pages, page_bytes, t.data_ptr(), i32([2]).data_ptr(), 2))
    assert be.take_faults() == 8
    assert np.array_equal(region.cpu().numpy(), before)


def test_refusals(be):
    import allpaka_amd.lib as l

    L, h = be.L, be.h
    cache = new_cache(be, 8, 4, 2, 4)
    be.sync()
    before = cache.pool.clone()
    one, two = i32([1, 1]), i32([0])
    buf = i32([0] * 16)
    p = buf.data_ptr()
    st = (cache.pool.data_ptr(), 8, 4, cache.page_table.data_ptr(), 4, cache.kv_len.data_ptr(), 2)
    calls = {
        "init": lambda s, ctx=h: L.apk_pages_init(ctx, *s),
        "extend": lambda s, ctx=h, n=one.data_ptr(), q=p, pos=p, sl=p, pr=p, np_=p, rows=2: L.apk_pages_extend(ctx, *s, n, rows, q, pos, sl, pr, np_),
        "fork": lambda s, ctx=h, a=two.data_ptr(), b=one.data_ptr(), n=1: L.apk_pages_fork(ctx, *s, a, b, n),
        "truncate": lambda s, ctx=h, n=one.data_ptr(): L.apk_pages_truncate(ctx, *s, n),
        "compact": lambda s, ctx=h, pr=p, n=p: L.apk_pages_compact(ctx, *s, pr, n),
    }

    def st_with(**kw):
        names = ("pool", "n_pages", "page", "table", "mp", "n", "ns")
        return tuple(kw.get(k, v) for k, v in zip(names, st))

    for name, f in calls.items():
        assert f(st, None) == l.DECLINE_NULL, name
        for kw, rc in ((dict(pool=None), l.DECLINE_NULL), (dict(table=None), l.DECLINE_NULL), (dict(n=None), l.DECLINE_NULL), (dict(n_pages=0), l.DECLINE_SHAPE),
                       (dict(page=0), l.DECLINE_SHAPE), (dict(n_pages=2 ** 28 + 1), l.DECLINE_SHAPE), (dict(n_pages=2 ** 20, page=2 ** 12), l.DECLINE_SHAPE),
                       (dict(mp=0), l.DECLINE_SHAPE), (dict(mp=2 ** 29), l.DECLINE_SHAPE), (dict(ns=2 ** 24 + 1), l.DECLINE_SHAPE)):
            assert f(st_with(**kw)) == rc, (name, kw)
    for kw in (dict(n=None), dict(q=None), dict(pos=None), dict(sl=None), dict(pr=None), dict(np_=None)):
        assert calls["extend"](st, **kw) == l.DECLINE_NULL, kw
    assert calls["extend"](st, rows=2 ** 31) == l.DECLINE_SHAPE
    assert calls["fork"](st, a=None) == l.DECLINE_NULL and calls["fork"](st, b=None) == l.DECLINE_NULL
    assert calls["fork"](st, n=1025) == l.DECLINE_SHAPE and calls["fork"](st, n=0) == 0
    assert calls["truncate"](st, n=None) == l.DECLINE_NULL
    assert calls["compact"](st, pr=None) == l.DECLINE_NULL and calls["compact"](st, n=None) == l.DECLINE_NULL
    reg = cache.region.data_ptr()
    good = [reg, 2, 8 * 64, 8, 64, p, p, 4]
    for i, x, rc in ((0, None, l.DECLINE_NULL), (0, reg + 8, l.DECLINE_SHAPE), (2, 500, l.DECLINE_SHAPE), (2, 7 * 64, l.DECLINE_SHAPE), (4, 60, l.DECLINE_SHAPE),
                     (4, 0, l.DECLINE_SHAPE), (5, None, l.DECLINE_NULL), (6, None, l.DECLINE_NULL), (7, 0, 0), (1, 0, 0), (3, 0, 0), (7, 2 ** 31, l.DECLINE_SHAPE)):
        a = list(good)
        a[i] = x
        assert L.apk_pages_copy(h, *a) == rc, (i, x)
    assert L.apk_pages_copy(None, *good) == l.DECLINE_NULL
    be.sync()
    assert torch.equal(cache.pool, before) and be.take_faults() == 0
    assert L.apk_pages_words(1) == 9 and L.apk_pages_words(64) == 4 + 256 + 2


def _attend_want(region, layer, table, kv_len, q, q_off, page, nq, nkv, hd, scale):
    c = dict(q=q, K=region[2 * layer], V=region[2 * layer + 1], table=table, kv_len=np.array(kv_len, np.int32), q_off=np.array(q_off, np.int32), page=page,
             n_q=nq, n_kv=nkv, hd=hd)
    return attention64(c, scale)


def test_a_serving_run(be, ora):
    """Prompts, a recorded decode step replayed for every token, a fork, drafts taken back, a sequence freed, the pool closed
    up: positions and cache rows handed out on the device drive the rotary rows, the store and the attention of two layers;
    the cache is checked against rows kept per sequence on the host, every attention against its formula."""
    import allpaka_amd as apk

    nq, nkv, hd, page, n_seq, layers, eps = 4, 2, 64, 8, 4, 2, 1e-6
    scale, rows_max = hd ** -0.5, 16
    r = np.random.default_rng(9)
    region = torch.full((2 * layers, 60 * page, nkv * hd), float("nan"), dtype=torch.float16, device="cuda")
    cache = apk.PagedCache(be, region, page, n_seq, 12)
    inv = be.rope_inv_freq(hd, 1e4)
    kept = [[[] for _ in range(layers)] for _ in range(n_seq)]  # (k row, v row) of every token, as stored

    def dev(a):
        return torch.from_numpy(np.ascontiguousarray(a)).cuda()

    bufs = [dict(q=torch.zeros((rows_max, nq * hd), dtype=torch.float16, device="cuda"), k=torch.zeros((rows_max, nkv * hd), dtype=torch.float16, device="cuda"),
                 v=torch.zeros((rows_max, nkv * hd), dtype=torch.float16, device="cuda"), out=torch.zeros((rows_max, nq * hd), dtype=torch.float16, device="cuda"))
            for _ in range(layers)]
    step = apk.backend.PageStep(n_seq, rows_max, be.device)
    table = torch.zeros((rows_max, hd // 2, 2), device="cuda")
    n_new = i32([0] * n_seq)

    def enqueue():
        cache.extend(n_new, rows_max, step)
        be.rope_table_into(step.positions, inv, table)
        for i, b in enumerate(bufs):
            be.L.apk_qknorm_rope_kv_store(be.h, b["q"].data_ptr(), b["k"].data_ptr(), b["v"].data_ptr(), None, None, table.data_ptr(), step.slots.data_ptr(),
                                          region[2 * i].data_ptr(), region[2 * i + 1].data_ptr(), region.shape[1], rows_max, nq, nkv, hd, hd, eps, 1)
            be.attend_paged_chunk_into(b["q"], region[2 * i], region[2 * i + 1], page, cache.page_table, step.q_off, cache.kv_len, nq, nkv, hd, scale, b["out"])

    def one(news, how):
        ins = []
        for b in bufs:
            for n in ("q", "k", "v"):
                b[n].copy_(dev(r.standard_normal(b[n].shape).astype(np.float16)))
            b["out"].fill_(5.0)
            ins.append([b[n].cpu().numpy() for n in ("q", "k", "v")])
        n_new.copy_(i32(news))
        torch.cuda.synchronize()
        how()
        be.sync()
        be.take_faults()  # rows of nobody report the store they were spared
        q_off, pos = step.q_off.cpu().tolist(), step.positions.cpu().tolist()
        host = region.cpu().numpy()
        tab, lens = cache.page_table.cpu().numpy(), cache.kv_len.cpu().tolist()
        total = q_off[-1]
        assert total == sum(news)
        ropes = ora.rope_table(pos[:total], ora.rope_inv_freq(hd, 1e4)) if total else None
        for i, b in enumerate(bufs):
            wq, wk = ins[i][0][:total].astype(np.float32), ins[i][1][:total].astype(np.float32)
            if total:
                ora.qknorm_rope_rows(wq, wk, nq, nkv, hd, None, None, ropes, eps)
                # the device's rotary rows are the oracle's to an ulp of f32: the rows to a rounding of fp16
                assert np.allclose(b["q"].cpu().numpy()[:total].astype(np.float32), wq, rtol=2 ** -10, atol=1e-4)
            got_k = b["k"].cpu().numpy()
            for s in range(n_seq):
                for row in range(q_off[s], q_off[s + 1]):
                    kept[s][i].append((got_k[row].copy(), ins[i][2][row].copy()))
                assert len(kept[s][i]) == lens[s]
                for j, (kr, vr) in enumerate(kept[s][i]):
                    at = tab[s, j // page] * page + j % page
                    assert np.array_equal(host[2 * i, at], kr) and np.array_equal(host[2 * i + 1, at], vr), (s, j)
            out = b["out"].cpu().numpy()
            assert np.all(out[total:] == 5.0)
            want, tol = _attend_want(host, i, tab, lens, b["q"].cpu().numpy()[:total], q_off, page, nq, nkv, hd, scale)
            assert np.all(np.abs(out[:total].astype(np.float64) - want) <= tol)

    one([7, 9, 0, 0], enqueue)
    with be.record() as rec:
        enqueue()
    for _ in range(4):
        one([1, 1, 0, 0], rec.graph.launch)
    cache.fork(i32([1, 0]), i32([2, 3]))
    kept[2], kept[3] = [list(x) for x in kept[1]], [list(x) for x in kept[0]]
    one([1, 1, 1, 1], rec.graph.launch)
    one([4, 0, 5, 1], rec.graph.launch)
    cache.truncate(i32([13, 2 ** 32 - 1, 15, 2 ** 32 - 1]))
    for s, n in ((0, 13), (2, 15)):
        kept[s] = [x[:n] for x in kept[s]]
    one([1, 2, 3, 1], rec.graph.launch)
    cache.truncate(i32([2 ** 32 - 1, 0, 2 ** 32 - 1, 2 ** 32 - 1]))
    kept[1] = [[], []]
    cache.compact()
    be.sync()
    live = int((cache.refs > 0).sum())
    assert torch.all(cache.refs[:live] > 0) and cache.free_pages == 60 - live
    one([1, 6, 1, 1], rec.graph.launch)
    one([2, 1, 0, 3], enqueue)
    rec.graph.destroy()


def test_more_new_pages_in_one_step_than_fit_on_the_chip(be):
    """Thousands of pages taken by one call, by one sequence and by many."""
    for n_seq, new in ((1, [9000]), (3, [1, 4096, 4500]), (2000, [5] * 2000)):
        page = 1 if n_seq < 2000 else 2
        cache, model = new_cache(be, 12000, page, n_seq, 10000 if n_seq < 2000 else 8, width=8), PageModel(12000, page, n_seq, 10000 if n_seq < 2000 else 8)
        rows = sum(new) + 3
        step = cache.extend(i32(new), rows)
        assert be.take_faults() == 0
        check_step(step, model.extend(new, rows), rows)
        same(cache, model)
        step = cache.extend(i32([1] * n_seq), n_seq)
        check_step(step, model.extend([1] * n_seq, n_seq), n_seq)
        same(cache, model)


def test_saved_and_restored(be):
    cache, model = new_cache(be, 40, 4, 3, 8), PageModel(40, 4, 3, 8)
    cache.extend(i32([5, 9, 0]), 14)
    model.extend([5, 9, 0], 14)
    saved = cache.save()
    cache.truncate(i32([0, 2, -1]))
    cache.extend(i32([1, 1, 7]), 9)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        cache.restore(saved)
    be.sync()
    same(cache, model)
    with pytest.raises(AssertionError):
        cache.restore(saved[:-4])
    assert be.take_faults() == 0
