"""The paged cache from a stream of torch's that is neither the default one nor the context's: its work before and after a call
is ordered against the call, and arguments may be dropped at once."""
import numpy as np
import pytest

from tests.paged_util import PageModel, attention64, make_case

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def be():
    import allpaka_amd as apk

    b = apk.Backend(0)
    yield b
    b.close()


@pytest.fixture(scope="module")
def busy(be):
    """busy(): some milliseconds of work on the context's stream"""
    a, b = torch.zeros(1 << 28, dtype=torch.int32, device="cuda"), torch.empty(1 << 28, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()

    def run():
        for _ in range(20):
            assert be.L.apk_copy(be.h, a.data_ptr(), b.data_ptr(), a.numel() * 4) == 0

    return run


def i32(x):
    return torch.tensor(np.asarray(x, np.int64).astype(np.uint32).view(np.int32), device="cuda")


def test_what_the_side_stream_does_next_reads_the_result(be, busy):
    for chunk in (False, True):
        c = make_case(900, [3000, 70], [9, 3] if chunk else [1, 1], 8, 2, 128, 16, True)
        want, tol = attention64(c, 0.1)
        t = {k: torch.from_numpy(np.ascontiguousarray(c[k])).cuda() for k in ("q", "K", "V", "table", "q_off", "kv_len")}
        args, heads = (t["K"], t["V"], 16, t["table"]), (8, 2, 128, 0.1)
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            out = torch.full_like(t["q"], 7.0)
            busy()
            q = t["q"].clone()
            if chunk:
                be.attend_paged_chunk_into(q, *args, t["q_off"], t["kv_len"], *heads, out)
            else:
                be.attend_paged_into(q, *args, t["kv_len"], *heads, out)
            size = q.numel()
            del q
            for _ in range(4):
                torch.full((size,), float("nan"), dtype=torch.float16, device="cuda")  # where q was
            got = out.clone()
        side.synchronize()
        assert np.all(np.abs(got.cpu().numpy().astype(np.float64) - want) <= tol)


def test_index_lists_may_be_dropped_at_once(be, busy):
    import allpaka_amd as apk

    n_seq = 6
    region = torch.zeros((2, 40 * 4, 8), dtype=torch.float16, device="cuda")
    cache, model = apk.PagedCache(be, region, 4, n_seq, 8), PageModel(40, 4, n_seq, 8)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()

    def over(n):  # lists of the same size with other contents, where the last ones were
        for _ in range(8):
            torch.full((n,), 5, dtype=torch.int32, device="cuda")

    with torch.cuda.stream(side):
        busy()
        cache.extend(i32([5, 9, 2, 0, 0, 0]), 20)
        over(n_seq), over(20)
        model.extend([5, 9, 2, 0, 0, 0], 20)
        busy()
        cache.fork(i32([0, 1]), i32([3, 4]))
        over(2), over(2)
        model.fork([0, 1], [3, 4])
        busy()
        cache.truncate(i32([3, 9, 0, 4, 1, 0]))
        over(n_seq)
        model.truncate([3, 9, 0, 4, 1, 0])
        busy()
        step = cache.extend(i32([1, 1, 1, 1, 1, 1]), 6)
        want = model.extend([1] * 6, 6)
        lens, slots, refs = cache.kv_len.clone(), step.slots.clone(), cache.refs.clone()
        busy()
        saved = cache.save()
        cache.truncate(i32([0] * n_seq))
        busy()
        cache.restore(saved)
        del saved
        over(cache._all.numel())
        again = cache.kv_len.clone()
    side.synchronize()
    assert lens.cpu().tolist() == again.cpu().tolist() == model.kv_len
    assert refs.cpu().tolist() == model.refs
    assert slots.cpu().tolist() == want[2]
    assert be.take_faults() == 0


def test_torch_on_the_context_s_own_stream(be, busy):
    c = make_case(901, [500, 7], [1, 1], 4, 2, 128, 16, True)
    want, tol = attention64(c, 0.1)
    with torch.cuda.stream(be.stream):
        t = {k: torch.from_numpy(np.ascontiguousarray(c[k])).cuda() for k in ("q", "K", "V", "table", "kv_len")}
        out = torch.empty_like(t["q"])
        busy()
        be.attend_paged_into(t["q"] * 1.0, t["K"], t["V"], 16, t["table"], t["kv_len"], 4, 2, 128, 0.1, out)
        got = out.float() * 2
    be.sync()
    assert np.all(np.abs(got.cpu().numpy() / 2 - want) <= tol)


def test_a_recorded_step_replayed_from_a_side_stream(be, busy):
    """Its arguments are written, and its results read, by the side stream's own work."""
    import allpaka_amd as apk

    n_seq, rows = 3, 8
    region = torch.zeros((2, 40 * 4, 8), dtype=torch.float16, device="cuda")
    cache, model = apk.PagedCache(be, region, 4, n_seq, 8), PageModel(40, 4, n_seq, 8)
    n_new, step = i32([0] * n_seq), apk.backend.PageStep(n_seq, rows, be.device)
    cache.extend(n_new, rows, step)
    with be.record() as rec:
        cache.extend(n_new, rows, step)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    seen = []
    try:
        with torch.cuda.stream(side):
            for news in ([3, 1, 0], [1, 1, 1], [0, 2, 5], [1, 0, 1]):
                n_new.copy_(i32(news))
                busy()
                rec.graph.launch()
                seen.append((step.slots.clone(), cache.kv_len.clone(), model.extend(news, rows)[2], list(model.kv_len)))
        side.synchronize()
        for slots, lens, want, want_lens in seen:
            assert slots.cpu().numpy().view(np.uint32).tolist() == want + [2 ** 32 - 1] * (rows - len(want))
            assert lens.cpu().tolist() == want_lens
        assert be.take_faults() == 0
    finally:
        rec.graph.destroy()
