"""Attention over the paged cache (apk_attend_paged, apk_attend_paged_chunk) against its formula in 64 bits, with bounds
counted from roundings (tests/paged_util.py), and its refusals."""
import ctypes as C
import math

import numpy as np
import pytest

from tests.paged_util import attention64, make_case

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def be():
    import allpaka_amd as apk

    b = apk.Backend(0)
    yield b
    b.close()


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def run(be, c, scale, window=0, chunk=True, out=None):
    q, args = dev(c["q"]), (dev(c["K"]), dev(c["V"]), c["page"], dev(c["table"]))
    heads = (c["n_q"], c["n_kv"], c["hd"], scale)
    if chunk:
        got = be.attend_paged_chunk(q, *args, dev(c["q_off"]), dev(c["kv_len"]), *heads, window=window)
    else:
        got = be.attend_paged(q, *args, dev(c["kv_len"]), *heads, window=window)
    assert be.take_faults() == 0
    return got.cpu().numpy()


def close(got, want, tol, what=""):
    err = np.abs(got.astype(np.float64) - want)
    assert np.all(np.isfinite(got)), f"{what}: {np.count_nonzero(~np.isfinite(got))} values are not finite"
    bad = err > tol
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.max(err / tol):.2f} of the bound at {np.unravel_index(np.argmax(err / tol), err.shape)}"


# one token each: lengths of one to several parts, pages that end inside a block of keys, odd groups, more heads than a tile
TOKEN = [
    # lens, n_q, n_kv, hd, page, window
    ([1], 1, 1, 64, 1, 0),
    ([1, 2, 3], 2, 1, 128, 16, 0),
    ([31, 32, 33, 64, 65], 8, 2, 128, 7, 0),
    ([127, 128, 129, 255, 256, 257, 300], 14, 2, 64, 23, 0),
    ([1000, 5, 513], 16, 2, 128, 16, 0),
    ([700, 90], 5, 1, 256, 33, 0),
    ([2100], 64, 2, 64, 64, 0),
    ([1500, 1, 40], 40, 1, 128, 100, 0),
    ([900, 17, 333], 8, 8, 128, 1024, 0),
    ([300, 20], 16, 1, 256, 16, 0),
    ([640, 3, 200, 64], 6, 2, 128, 16, 64),
    ([640, 3, 200, 65], 6, 2, 64, 5, 1),
    ([1300, 1301], 4, 4, 256, 48, 257),
]


@pytest.mark.parametrize("f16", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("i", range(len(TOKEN)))
def test_single_tokens(be, i, f16):
    lens, n_q, n_kv, hd, page, window = TOKEN[i]
    c = make_case(i, lens, [1] * len(lens), n_q, n_kv, hd, page, f16)
    want, tol = attention64(c, hd ** -0.5, window)
    close(run(be, c, hd ** -0.5, window, chunk=False), want, tol, "token entry")
    close(run(be, c, hd ** -0.5, window, chunk=True), want, tol, "chunk entry")


CHUNK = [
    # (cached, new) each, n_q, n_kv, hd, page, window
    ([(0, 1)], 1, 1, 64, 16, 0),
    ([(0, 5), (3, 2), (100, 1)], 4, 2, 128, 16, 0),
    ([(0, 33), (31, 64), (64, 65)], 2, 2, 64, 7, 0),
    ([(0, 70)], 7, 1, 128, 32, 0),
    ([(500, 40), (0, 0), (17, 3)], 8, 1, 128, 33, 0),
    ([(0, 129)], 3, 1, 256, 16, 0),
    ([(1200, 20)], 16, 1, 64, 64, 0),
    ([(40, 50), (3, 130)], 5, 1, 128, 24, 37),
    ([(40, 50), (3, 130)], 4, 2, 64, 1, 1),
    ([(600, 9)], 130, 1, 64, 16, 0),
    ([(2500, 6)], 8, 2, 128, 100, 1000),
    ([(700, 12)], 2, 1, 256, 40, 100),
]


@pytest.mark.parametrize("f16", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("i", range(len(CHUNK)))
def test_chunks(be, i, f16):
    seqs, n_q, n_kv, hd, page, window = CHUNK[i]
    c = make_case(100 + i, [a + b for a, b in seqs], [b for _, b in seqs], n_q, n_kv, hd, page, f16)
    want, tol = attention64(c, hd ** -0.5, window)
    close(run(be, c, hd ** -0.5, window), want, tol)


@pytest.mark.parametrize("hd", [1, 7, 40, 80, 96, 112, 192, 320, 1024])
@pytest.mark.parametrize("f16", [True, False], ids=["f16", "f32"])
def test_other_head_sizes(be, hd, f16):
    c = make_case(200 + hd, [70, 1, 300], [3, 1, 2], 6, 2, hd, 9, f16)
    want, tol = attention64(c, hd ** -0.5, 0)
    close(run(be, c, hd ** -0.5), want, tol)
    c = make_case(201 + hd, [70, 1, 300], [1, 1, 1], 6, 2, hd, 9, f16)
    want, tol = attention64(c, hd ** -0.5, 50)
    close(run(be, c, hd ** -0.5, 50, chunk=False), want, tol)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
@pytest.mark.parametrize("f16", [True, False], ids=["f16", "f32"])
def test_scales(be, scale, f16):
    for chunk in (False, True):
        c = make_case(300, [50, 9], [4, 2] if chunk else [1, 1], 4, 2, 64, 16, f16)
        want, tol = attention64(c, scale)
        close(run(be, c, scale, chunk=chunk), want, tol)


def test_scores_far_apart_and_queries_of_all_sizes(be):
    """A score 60 above the others, first and last; f32 query rows of 1e-30 .. 1e20."""
    for f16 in (True, False):
        for chunk in (False, True):
            c = make_case(310, [400, 130, 129], [2, 3, 1] if chunk else [1, 1, 1], 2, 1, 128, 16, f16)
            for s, j in ((0, 0), (1, 60), (2, 128)):
                row = c["table"][s][j // 16] * 16 + j % 16
                c["K"][row] = 6.0 * np.sign(c["q"][c["q_off"][s], :128]).astype(np.float16)
            want, tol = attention64(c, 0.08)
            close(run(be, c, 0.08, chunk=chunk), want, tol)
    c = make_case(311, [40, 41, 42, 43], [1, 1, 1, 1], 2, 1, 64, 16, False)
    c["q"] *= np.array([[1e-30], [1e-5], [1e8], [1e20]], np.float32)
    for i, scale in enumerate((1.0, 1.0, 1e-9, 1e-21)):
        d = dict(c, q=c["q"][i:i + 1], table=c["table"][i:i + 1], kv_len=c["kv_len"][i:i + 1], q_off=np.array([0, 1], np.int32))
        want, tol = attention64(d, scale)
        for chunk in (False, True):
            close(run(be, d, scale, chunk=chunk), want, tol, f"row {i}")


@pytest.mark.parametrize("hd", [64, 128, 256, 48])
@pytest.mark.parametrize("f16", [True, False], ids=["f16", "f32"])
def test_what_is_masked_does_not_reach_a_row(be, hd, f16):
    """Infinities and NaN in later tokens' K and V, behind the window, and in rows of nobody: earlier rows as without them;
    rows that see such a V get it in its channel alone."""
    c = make_case(400, [40, 70], [30, 66], 4, 2, hd, 16, f16)
    want, tol = attention64(c, hd ** -0.5, 24)
    bad = [(0, 25, 3, np.nan), (0, 39, 1, np.inf), (1, 50, 5, -np.inf), (1, 2, 0, np.nan)]  # sequence, key, channel, value
    for s, j, ch, x in bad:
        row = c["table"][s][j // 16] * 16 + j % 16
        c["V"][row, ch] = x
    kbad = [(0, 37), (1, 60)]
    for s, j in kbad:
        c["K"][c["table"][s][j // 16] * 16 + j % 16] = np.nan
    got = run(be, c, hd ** -0.5, 24)
    for s in range(2):
        for r in range(c["q_off"][s], c["q_off"][s + 1]):
            p = c["kv_len"][s] - (c["q_off"][s + 1] - r)
            sees = lambda j: p - 24 < j <= p  # noqa: E731
            clean = np.ones(c["n_q"] * hd, bool)
            for t, j in kbad:
                if t == s and sees(j):
                    clean[:] = False
            for t, j, ch, x in bad:
                if t == s and sees(j):
                    for h in range(2):  # the heads of kv head 0
                        clean[h * hd + ch] = False
                        assert not np.isfinite(got[r, h * hd + ch]), (s, r, j)
            close(got[r][clean], want[r][clean], tol[r][clean], f"row {r} of sequence {s}")
    # single tokens: nothing behind the last key or before the window counts
    c = make_case(401, [100, 33], [1, 1], 4, 2, hd, 16, f16)
    want, tol = attention64(c, hd ** -0.5, 20)
    for s, n in ((0, 100), (1, 33)):
        for j in (0, n - 21):
            row = c["table"][s][j // 16] * 16 + j % 16
            c["V"][row], c["K"][row] = np.inf, np.nan
    close(run(be, c, hd ** -0.5, 20, chunk=False), want, tol)


def test_released_pages_behind_the_window_are_not_looked_up(be):
    for chunk in (False, True):
        c = make_case(410, [600], [8] if chunk else [1], 4, 2, 128, 16, True)
        want, tol = attention64(c, 0.1, 64)
        c["table"][0, : (600 - 8 - 64) // 16] = -1
        close(run(be, c, 0.1, 64, chunk=chunk), want, tol)


@pytest.mark.parametrize("hd", [64, 128, 256, 24])
@pytest.mark.parametrize("f16", [True, False], ids=["f16", "f32"])
def test_rows_without_keys_and_rows_of_nobody(be, hd, f16):
    """Sequences of length 0, more new rows than tokens, sequences without rows, rows behind the last sequence."""
    c = make_case(420, [0, 3, 20, 0], [2, 5, 0, 0], 4, 2, hd, 8, f16)
    want, tol = attention64(c, 0.2)
    q = np.concatenate([c["q"], np.full((4, 4 * hd), 9.0, c["q"].dtype)])
    out = torch.full(q.shape, 7.0, dtype=torch.float16 if f16 else torch.float32, device="cuda")
    be.attend_paged_chunk_into(dev(q), dev(c["K"]), dev(c["V"]), 8, dev(c["table"]), dev(c["q_off"]), dev(c["kv_len"]), 4, 2, hd, 0.2, out)
    be.sync()
    got = out.cpu().numpy()
    assert np.all(got[7:] == 7.0)
    assert np.all(got[:4] == 0.0)  # length 0, and the two rows at positions -2 and -1
    close(got[:7], want, tol)
    c = make_case(421, [0, 1], [1, 1], 4, 2, hd, 8, f16)
    want, tol = attention64(c, 0.2)
    got = run(be, c, 0.2, chunk=False)
    assert np.all(got[0] == 0.0)
    close(got, want, tol)


@pytest.mark.parametrize("f16", [True, False], ids=["f16", "f32"])
def test_long_caches_are_split_and_joined(be, f16):
    """Lengths far above and far below each other, so that some sequences are split over many workgroups and others not."""
    for chunk in (False, True):
        lens, new = [20011, 1, 300, 9000], ([5, 1, 17, 2] if chunk else [1, 1, 1, 1])
        c = make_case(430, lens, new, 6, 2, 128, 64, f16)
        want, tol = attention64(c, 128 ** -0.5)
        close(run(be, c, 128 ** -0.5, chunk=chunk), want, tol)


@pytest.mark.parametrize("n_seq", [65, 200])
def test_many_sequences(be, n_seq):
    r = np.random.default_rng(5)
    lens = [int(x) for x in r.integers(0, 90, n_seq)]
    lens[n_seq - 3] = 3000
    c = make_case(440, lens, [1] * n_seq, 4, 2, 64, 16, True)
    want, tol = attention64(c, 0.125)
    close(run(be, c, 0.125, chunk=False), want, tol)
    new = [int(r.integers(0, min(n, 3) + 1)) for n in lens]
    c = make_case(441, lens, new, 4, 2, 64, 16, True)
    want, tol = attention64(c, 0.125)
    close(run(be, c, 0.125), want, tol)


def test_small_weights_of_a_long_cache_are_not_lost(be):
    """One key of weight 1, and 60000 of weight 2^-20 each that together weigh 0.057: dropped or rounded to fp16's smallest
    steps they would show."""
    n, hd = 60001, 64
    c = make_case(450, [n], [1], 1, 1, hd, 64, True)
    rows = c["table"][0][np.arange(n) // 64] * 64 + np.arange(n) % 64
    c["q"][:] = 0
    c["q"][0, 0] = 1.0
    c["K"][rows] = 0
    c["K"][rows[777], 0] = 20 * math.log(2)
    c["V"][rows] = 1.0
    c["V"][rows[777]] = 0.0
    want, tol = attention64(c, 1.0)
    for chunk in (False, True):
        close(run(be, c, 1.0, chunk=chunk), want, tol)


def test_cache_rows_past_four_gibibytes(be):
    """Planes of 4.6 GB: pages at their very end, next to page 0."""
    hd, n_kv, page = 128, 8, 64
    n_pages = 36000
    K = torch.empty((n_pages * page, n_kv * hd), dtype=torch.float16, device="cuda")
    V = torch.empty_like(K)
    assert K.numel() * 2 > 2 ** 32
    small = make_case(460, [200, 150], [3, 1], 16, n_kv, hd, page, True)
    where = {p: n_pages - 1 - i * 40 for i, p in enumerate(range(small["n_pages"] - 1))}
    where[small["n_pages"] - 1] = 0
    for p, big in where.items():
        K[big * page:(big + 1) * page] = dev(small["K"][p * page:(p + 1) * page])
        V[big * page:(big + 1) * page] = dev(small["V"][p * page:(p + 1) * page])
    table = np.vectorize(lambda e: where.get(int(e), -1))(small["table"]).astype(np.int32)
    want, tol = attention64(small, 0.09)
    got = be.attend_paged_chunk(dev(small["q"]), K, V, page, dev(table), dev(small["q_off"]), dev(small["kv_len"]), 16, n_kv, hd, 0.09)
    close(got.cpu().numpy(), want, tol)
    one = dict(small, q=small["q"][:2], q_off=np.array([0, 1, 2], np.int32))
    want, tol = attention64(one, 0.09)
    got = be.attend_paged(dev(one["q"]), K, V, page, dev(table), dev(one["kv_len"]), 16, n_kv, hd, 0.09)
    close(got.cpu().numpy(), want, tol)
    assert be.take_faults() == 0


def test_the_output_may_be_the_query(be):
    for chunk in (False, True):
        c = make_case(470, [3000, 40], [9, 3] if chunk else [1, 1], 8, 2, 128, 16, True)
        want = run(be, c, 0.1, chunk=chunk)
        q = dev(c["q"])
        args = (dev(c["K"]), dev(c["V"]), 16, dev(c["table"]))
        if chunk:
            be.attend_paged_chunk_into(q, *args, dev(c["q_off"]), dev(c["kv_len"]), 8, 2, 128, 0.1, q)
        else:
            be.attend_paged_into(q, *args, dev(c["kv_len"]), 8, 2, 128, 0.1, q)
        be.sync()
        assert np.array_equal(q.cpu().numpy().view(np.uint16), want.view(np.uint16))


def test_results_repeat_bit_for_bit(be):
    c = make_case(480, [5000, 700, 3], [4, 90, 3], 8, 2, 128, 16, True)
    first = run(be, c, 0.1)
    for _ in range(3):
        assert np.array_equal(run(be, c, 0.1).view(np.uint16), first.view(np.uint16))


def test_bad_tables_raise_a_fault_and_touch_nothing_else(be):
    import allpaka_amd.lib as apklib

    for chunk in (False, True):
        for hd in (128, 40):
            c = make_case(490, [100, 60], [2, 2] if chunk else [1, 1], 4, 2, hd, 16, True, garbage=0.0)
            want, tol = attention64(c, 0.1)
            for what in ("entry", "length"):
                d = dict(c, table=c["table"].copy(), kv_len=c["kv_len"].copy())
                if what == "entry":
                    d["table"][0, 2] = c["n_pages"]
                else:
                    d["kv_len"][0] = d["table"].shape[1] * 16 + 1
                    d["table"][0] = np.arange(d["table"].shape[1]) % c["n_pages"]
                q, args = dev(d["q"]), (dev(d["K"]), dev(d["V"]), 16, dev(d["table"]))
                out = torch.empty_like(q)
                if chunk:
                    be.attend_paged_chunk_into(q, *args, dev(d["q_off"]), dev(d["kv_len"]), 4, 2, hd, 0.1, out)
                else:
                    be.attend_paged_into(q, *args, dev(d["kv_len"]), 4, 2, hd, 0.1, out)
                assert be.take_faults() == apklib.FAULT_CACHE_RANGE, (chunk, hd, what)
                a = d["q_off"][1]
                close(out.cpu().numpy()[a:], want[a:], tol[a:])
    c = make_case(491, [100, 60], [2, 2], 4, 2, 64, 16, True, garbage=0.0)
    for q_off in ([0, 2, 900], [3, 2, 4]):
        out = torch.full((4, 256), 5.0, dtype=torch.float16, device="cuda")
        be.attend_paged_chunk_into(dev(c["q"]), dev(c["K"]), dev(c["V"]), 16, dev(c["table"]), dev(np.array(q_off, np.int32)), dev(c["kv_len"]), 4, 2, 64,
                                   0.1, out)
        assert be.take_faults() & apklib.FAULT_ROW_RANGE


def test_recorded_and_replayed_with_growing_lengths(be):
    """One recording serves every token: the lengths live on the device.  Two graphs share the context's scratch, with eager
    calls between the replays."""
    c = make_case(500, [2600, 900], [1, 1], 8, 2, 128, 16, True)
    q, K, V, table = dev(c["q"]), dev(c["K"]), dev(c["V"]), dev(c["table"])
    q_off, n = dev(c["q_off"]), dev(c["kv_len"])
    run(be, c, 0.1, chunk=False)
    a, b = torch.empty_like(q), torch.empty_like(q)
    with be.record() as r1:
        be.attend_paged_into(q, K, V, 16, table, n, 8, 2, 128, 0.1, a)
    with be.record() as r2:
        be.attend_paged_chunk_into(q, K, V, 16, table, q_off, n, 8, 2, 128, 0.1, b)
    try:
        for lens in ([2600, 900], [2000, 1], [5, 899], [2599, 640], [2600, 900]):
            n.copy_(torch.tensor(lens, dtype=torch.int32))
            torch.cuda.synchronize()
            d = dict(c, kv_len=np.array(lens, np.int32))
            want, tol = attention64(d, 0.1)
            a.fill_(3.0), b.fill_(3.0)
            torch.cuda.synchronize()
            r1.graph.launch()
            r2.graph.launch()
            r1.graph.launch()
            be.sync()
            eager = run(be, d, 0.1, chunk=False)
            assert np.array_equal(a.cpu().numpy().view(np.uint16), eager.view(np.uint16))
            close(a.cpu().numpy(), want, tol)
            close(b.cpu().numpy(), want, tol)
            assert np.array_equal(b.cpu().numpy().view(np.uint16), run(be, d, 0.1).view(np.uint16))
    finally:
        r1.graph.destroy()
        r2.graph.destroy()


def test_the_first_call_of_a_context_inside_a_recording_is_declined():
    import allpaka_amd as apk

    b = apk.Backend(0)
    c = make_case(510, [2000], [1], 2, 1, 64, 16, True)
    args = (dev(c["q"]), dev(c["K"]), dev(c["V"]), 16, dev(c["table"]), dev(c["kv_len"]), 2, 1, 64, 0.1)
    out = torch.empty_like(args[0])
    b.capture_begin()
    with pytest.raises(apk.Declined) as e:
        b.attend_paged_into(*args, out)
    assert e.value.reason == 7
    b.capture_abort()
    b.attend_paged_into(*args, out)
    b.sync()
    with b.record() as rec:
        b.attend_paged_into(*args, out)
    rec.graph.launch()
    b.sync()
    rec.graph.destroy()
    b.close()


def test_work_queued_on_another_stream_is_waited_for(be):
    c = make_case(520, [300, 7], [1, 1], 4, 2, 128, 16, True)
    want, tol = attention64(c, 0.1)
    side = torch.cuda.Stream()
    q0, K, V, table, n = dev(c["q"]), dev(c["K"]), dev(c["V"]), dev(c["table"]), dev(c["kv_len"])
    big = torch.randn((4096, 4096), device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            big = big @ big * 1e-4
        q = q0.clone()
        out = torch.empty_like(q)
        be.attend_paged_into(q, K, V, 16, table, n, 4, 2, 128, 0.1, out)
    be.sync()
    close(out.cpu().numpy(), want, tol)


def test_refusals(be):
    import allpaka_amd.lib as l

    c = make_case(530, [40], [1], 4, 2, 64, 16, True)
    q, K, V, table, n, q_off = (dev(c[k]) for k in ("q", "K", "V", "table", "kv_len", "q_off"))
    out = torch.full_like(q, 5.0)
    good = dict(q=q.data_ptr(), k=K.data_ptr(), v=V.data_ptr(), cap=K.shape[0], page=16, table=table.data_ptr(), mp=table.shape[1], n=n.data_ptr(), ns=1, nq=4,
                nkv=2, hd=64, scale=0.1, window=0, out=out.data_ptr(), dt=1)

    def call(chunk, **kw):
        a = dict(good, q_off=q_off.data_ptr(), rows=1)
        a.update(kw)
        if chunk:
            return be.L.apk_attend_paged_chunk(be.h, a["q"], a["k"], a["v"], a["cap"], a["page"], a["table"], a["mp"], a["q_off"], a["n"], a["ns"], a["rows"],
                                               a["nq"], a["nkv"], a["hd"], a["scale"], a["window"], a["out"], a["dt"])
        return be.L.apk_attend_paged(be.h, a["q"], a["k"], a["v"], a["cap"], a["page"], a["table"], a["mp"], a["n"], a["ns"], a["nq"], a["nkv"], a["hd"],
                                     a["scale"], a["window"], a["out"], a["dt"])

    for chunk in (False, True):
        for kw, rc in ((dict(dt=2), l.DECLINE_UNSUPPORTED), (dict(hd=0), l.DECLINE_UNSUPPORTED), (dict(hd=1025), l.DECLINE_UNSUPPORTED),
                       (dict(nq=3), l.DECLINE_SHAPE), (dict(nkv=0), l.DECLINE_SHAPE), (dict(nq=0), l.DECLINE_SHAPE), (dict(page=0), l.DECLINE_SHAPE),
                       (dict(cap=15), l.DECLINE_SHAPE), (dict(cap=2 ** 32), l.DECLINE_SHAPE), (dict(mp=0), l.DECLINE_SHAPE), (dict(mp=2 ** 27), l.DECLINE_SHAPE),
                       (dict(scale=math.inf), l.DECLINE_SHAPE), (dict(scale=math.nan), l.DECLINE_SHAPE), (dict(ns=2 ** 31), l.DECLINE_SHAPE),
                       (dict(q=None), l.DECLINE_NULL), (dict(k=None), l.DECLINE_NULL), (dict(v=None), l.DECLINE_NULL), (dict(table=None), l.DECLINE_NULL),
                       (dict(n=None), l.DECLINE_NULL), (dict(out=None), l.DECLINE_NULL), (dict(q=good["q"] + 2), l.DECLINE_SHAPE),
                       (dict(k=good["k"] + 8), l.DECLINE_SHAPE), (dict(out=good["out"] + 4), l.DECLINE_SHAPE)):
            assert call(chunk, **kw) == rc, (chunk, kw)
        assert call(chunk, ns=0) == 0
    assert call(True, q_off=None) == l.DECLINE_NULL
    assert call(True, rows=0, q=None, out=None) == 0
    be.sync()
    assert torch.all(out == 5.0)
    assert be.L.apk_attend_paged(None, *([None] * 3), 16, 16, None, 1, None, 1, 1, 1, 64, 1.0, 0, None, 1) == l.DECLINE_NULL
    for bad in (dict(scale="x"),):
        with pytest.raises(C.ArgumentError):
            call(False, **bad)
    assert be.take_faults() == 0


# chunks over long caches, whose tiles are cut into few and into many parts; groups of more heads than a tile of few rows
LONG = [
    # (cached, new) each, n_q, n_kv, hd, page, window
    ([(9000, 40)], 6, 2, 128, 64, 0),
    ([(20000, 5), (30, 30)], 8, 1, 64, 16, 0),
    ([(7000, 30), (100, 2)], 4, 1, 256, 33, 0),
    ([(6000, 200)], 3, 1, 128, 16, 4000),
    ([(5000, 33), (0, 150), (700, 1)], 9, 3, 64, 24, 0),
    ([(3000, 70)], 6, 2, 256, 16, 700),
    ([(4000, 1), (2500, 1)], 40, 2, 128, 16, 0),
    ([(900, 1), (3, 1)], 100, 1, 256, 16, 0),
]


@pytest.mark.parametrize("f16", [True, False], ids=["f16", "f32"])
@pytest.mark.parametrize("i", range(len(LONG)))
def test_chunks_over_long_caches(be, i, f16):
    seqs, n_q, n_kv, hd, page, window = LONG[i]
    c = make_case(600 + i, [a + b for a, b in seqs], [b for _, b in seqs], n_q, n_kv, hd, page, f16)
    want, tol = attention64(c, hd ** -0.5, window)
    close(run(be, c, hd ** -0.5, window), want, tol, "chunk entry")
    if all(b == 1 for _, b in seqs):
        close(run(be, c, hd ** -0.5, window, chunk=False), want, tol, "token entry")


def test_row_offsets_that_name_rows_twice(be):
    """A descending pair between two ascending ones: more tiles than the rows make.  The call reports it and ends, and rows
    behind are left as they are."""
    import allpaka_amd.lib as apklib

    for hd in (64, 128, 256, 32):
        for lens in ([40, 50, 60], [3000, 50, 2000]):
            c = make_case(620, lens, [4, 0, 0], 16, 1, hd, 16, True, garbage=0.0)
            out = torch.full((4, 16 * hd), 5.0, dtype=torch.float16, device="cuda")
            be.attend_paged_chunk_into(dev(c["q"]), dev(c["K"]), dev(c["V"]), 16, dev(c["table"]), dev(np.array([0, 4, 0, 4], np.int32)),
                                       dev(c["kv_len"]), 16, 1, hd, 0.1, out)
            assert be.take_faults() & apklib.FAULT_ROW_RANGE


def test_heads_that_are_no_power_of_two(be):
    for n_kv, group in ((3, 5), (6, 1), (7, 2)):
        for chunk in (False, True):
            c = make_case(630 + n_kv, [1500, 33, 700], [9, 1, 4] if chunk else [1, 1, 1], n_kv * group, n_kv, 128, 16, True)
            want, tol = attention64(c, 0.09)
            close(run(be, c, 0.09, chunk=chunk), want, tol, f"{n_kv} kv heads")
