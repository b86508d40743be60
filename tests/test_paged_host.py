"""The host side of the paged cache without a GPU: PagedCache over a stand-in for the library that notes the calls it gets
and declines a copy as the header says."""
import pytest

torch = pytest.importorskip("torch")

import allpaka_amd.backend as backend  # noqa: E402
from allpaka_amd.lib import DECLINE_SHAPE, Declined  # noqa: E402


class Library:
    def __init__(self):
        self.calls = []

    def apk_pages_words(self, n):
        return 4 + 4 * n + (n + 31) // 32

    def apk_pages_copy(self, ctx, region, planes, plane_bytes, n_pages, page_bytes, pairs, n_pairs, most):
        self.calls.append("copy")
        if planes == 0 or n_pages == 0 or most == 0:
            return 0
        ok = region % 16 == 0 and page_bytes % 16 == 0 and plane_bytes % 16 == 0 and page_bytes and page_bytes <= plane_bytes // n_pages
        return 0 if ok else DECLINE_SHAPE

    def __getattr__(self, name):
        def call(*args):
            self.calls.append(name)
            return 0

        return call


class Host(backend.Backend):
    """A Backend without a device."""

    def __init__(self):
        self.L, self.h, self.device, self._recording, self._stream = Library(), 1, torch.device("cpu"), False, None

    def close(self):
        pass

    def _order(self):
        pass


@pytest.fixture
def be(monkeypatch):
    monkeypatch.setattr(backend, "_ptr", lambda t: None if t is None else t.data_ptr())
    return Host()


CHANGES = {"apk_pages_init", "apk_pages_extend", "apk_pages_fork", "apk_pages_truncate", "apk_pages_compact"}


def region(planes, rows, width, skip=0):
    return torch.zeros(planes * rows * width + 8, dtype=torch.float16)[skip:skip + planes * rows * width].view(planes, rows, width)


@pytest.mark.parametrize("planes,rows,width,page,skip", [
    (2, 6, 4, 1, 0),  # pages of 8 bytes
    (2, 12, 7, 1, 0),  # of 14
    (2, 40, 20, 1, 0),  # of 40
    (4, 9, 12, 2, 0),  # of 48, in planes of 216
    (2, 16, 8, 4, 4),  # whole tiles that begin inside one
])
def test_a_cache_whose_pages_cannot_be_copied_is_refused_before_it_has_a_state(be, planes, rows, width, page, skip):
    """Else extend and compact would change the state and then raise, the copies undone."""
    with pytest.raises(Declined) as e:
        backend.PagedCache(be, region(planes, rows, width, skip), page, 3, 4)
    assert e.value.reason == DECLINE_SHAPE
    assert not CHANGES & set(be.L.calls)


def test_pages_of_whole_tiles_are_taken(be):
    for planes, rows, width, page in ((2, 6, 8, 1), (2, 12, 4, 2), (1, 40, 20, 2), (4, 9, 16, 2), (2, 16, 128, 16)):
        c = backend.PagedCache(be, region(planes, rows, width), page, 3, 4)
        c.extend(torch.zeros(3, dtype=torch.int32), 5)
        c.compact()


class Stream:
    def __init__(self, handle, log):
        self.cuda_stream, self.log = handle, log

    def synchronize(self):
        self.log.append("host waits")

    def wait_stream(self, other):
        self.log.append(("waits for", other.cuda_stream))


CONTEXT, SIDE = 4000, 7000


@pytest.fixture
def streams(be, monkeypatch):
    """be with a stream of its own; streams(handle) makes torch's current one."""
    log = be.L.calls
    monkeypatch.setattr(type(be.L), "apk_stream", lambda self, ctx: CONTEXT, raising=False)
    monkeypatch.setattr(Host, "_order", backend.Backend._order)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda handle, device=None: Stream(handle, log))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream(0, log))

    def current(handle):
        monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream(handle, log))
        log.clear()
        return log

    return current


def entries(be):
    """name -> (a call, what it enqueues last)"""
    cache = backend.PagedCache(be, region(2, 64, 16), 16, 3, 4)
    ids, state = torch.zeros(3, dtype=torch.int32), torch.zeros_like(cache._all)
    q = torch.zeros((3, 32), dtype=torch.float16)
    off = torch.zeros(4, dtype=torch.int32)
    step = backend.PageStep(3, 5, be.device)
    paged = (cache.region[0], cache.region[1], 16, cache.page_table)
    return {
        "extend": (lambda: cache.extend(ids, 5, step), "copy"),
        "fork": (lambda: cache.fork(ids, ids), "apk_pages_fork"),
        "truncate": (lambda: cache.truncate(ids), "apk_pages_truncate"),
        "compact": (lambda: cache.compact(), "copy"),
        "restore": (lambda: cache.restore(state), "apk_copy"),
        "adopt": (lambda: cache.adopt(cache.page_table.clone(), cache.kv_len.clone()), "apk_pages_init"),
        "new": (lambda: backend.PagedCache(be, cache.region, 16, 3, 4), "apk_pages_init"),
        "tokens": (lambda: be.attend_paged_into(q, *paged, cache.kv_len, 2, 1, 16, 1.0, q), "apk_attend_paged"),
        "chunk": (lambda: be.attend_paged_chunk_into(q, *paged, off, cache.kv_len, 2, 1, 16, 1.0, q), "apk_attend_paged_chunk"),
        "replay": (lambda: backend.Graph(be, 5).launch(), "apk_graph_launch"),
    }


NAMES = ["extend", "fork", "truncate", "compact", "restore", "adopt", "new", "tokens", "chunk", "replay"]


@pytest.mark.parametrize("name", NAMES)
def test_a_side_stream_comes_before_and_after_what_is_enqueued(be, streams, name):
    """What the side stream does next may read the results, or write over an argument that was freed there."""
    call, last = entries(be)[name]
    log = streams(SIDE)
    call()
    first = min(i for i, x in enumerate(log) if x == "copy" or str(x).startswith(("apk_pages", "apk_attend", "apk_copy", "apk_graph")))
    assert "host waits" in log[:first]
    assert log[-1] == ("waits for", CONTEXT) and log[-2] == last, log


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("handle", [0, CONTEXT])
def test_the_default_stream_and_the_context_s_own_need_no_wait(be, streams, name, handle):
    call, last = entries(be)[name]
    log = streams(handle)
    call()
    assert log[-1] == last and not any(isinstance(x, tuple) for x in log), log


@pytest.mark.parametrize("name", [n for n in NAMES if n not in ("adopt", "replay")])
def test_nothing_waits_for_a_recording(be, streams, name):
    call, last = entries(be)[name]
    log = streams(SIDE)
    be._recording = True
    call()
    assert log[-1] == last and not any(isinstance(x, tuple) for x in log), log


@pytest.mark.parametrize("name", ["extend", "compact"])
def test_a_side_stream_waits_also_where_the_copy_fails(be, streams, name):
    call, _ = entries(be)[name]
    be.L.apk_pages_copy = lambda *a: DECLINE_SHAPE
    log = streams(SIDE)
    with pytest.raises(Declined):
        call()
    assert log[-1] == ("waits for", CONTEXT), log
