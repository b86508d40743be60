"""The bookkeeping of the pages at its edges: tables that do not belong to their pool, and tables so wide that the entries of a
thousand sequences pass 32 bits."""
import numpy as np
import pytest

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


@pytest.mark.parametrize("n_seq", [2, 3, 64, 1300])
def test_a_page_named_more_often_than_it_is_held_keeps_its_count(be, n_seq):
    """Every sequence names page 5, which nobody holds, and page 2, which one of them does, in tables changed behind the pool's
    back: the call reports it, page 2 is freed once, and no count goes below zero."""
    import allpaka_amd as apk
    import allpaka_amd.lib as l

    region = torch.zeros((2, 40 * 4, 8), dtype=torch.float16, device="cuda")
    cache = apk.PagedCache(be, region, 4, n_seq, 3)
    cache.adopt(i32([[2, 0, 0]] + [[0, 0, 0]] * (n_seq - 1)), i32([4] + [0] * (n_seq - 1)))
    assert cache.free_pages == 39
    cache.page_table[:, 0], cache.page_table[:, 1] = 5, 2
    cache.kv_len.fill_(8)
    for _ in range(2):  # the second time nobody holds either
        cache.truncate(i32([0] * n_seq))
        assert be.take_faults() == l.FAULT_CACHE_RANGE
        assert cache.refs.cpu().tolist() == [0] * 40 and cache.free_pages == 40
        cache.kv_len.fill_(8)
    cache.kv_len.fill_(0)
    step = cache.extend(i32([4] + [0] * (n_seq - 1)), 4)  # and the pool hands out as before
    assert step.slots.cpu().tolist() == [0, 1, 2, 3] and cache.free_pages == 39
    assert be.take_faults() == 0


def test_tables_whose_entries_pass_32_bits(be):
    """1200 sequences of up to 2^23 pages each (40 GB of table): a round of a thousand of them could not add their entries up
    in 32 bits, so rounds are of 255 here.  Run with short sequences, at the ends of those rounds among others, against the
    model of the bookkeeping."""
    import allpaka_amd as apk
    from tests.paged_util import PageModel

    n_seq, wide, page, n_pages = 1200, 1 << 23, 2, 4000
    region = torch.zeros((2, n_pages * page, 8), dtype=torch.float16, device="cuda")
    cache, model = apk.PagedCache(be, region, page, n_seq, wide), PageModel(n_pages, page, n_seq, wide)
    r = np.random.default_rng(3)

    def same():
        assert be.take_faults() == 0
        assert cache.kv_len.cpu().tolist() == model.kv_len and cache.refs.cpu().tolist() == model.refs
        head = cache.page_table[:, :8].cpu().numpy()
        for s, t in enumerate(model.table):
            assert head[s, :len(t)].tolist() == t, s

    for it in range(3):
        new = r.integers(0, 4, n_seq).tolist()
        cache.extend(i32(new), sum(new)), model.extend(new, sum(new))
        same()
        cut = [0 if r.random() < 0.4 or s in (254, 255, 509, 510, 1019, 1020) else 2 ** 32 - 1 if r.random() < 0.5 else int(r.integers(0, 6)) for s in range(n_seq)]
        cache.truncate(i32(cut)), model.truncate(cut)
        same()
        cache.compact(), model.compact()
        same()
    del cache
    torch.cuda.empty_cache()
