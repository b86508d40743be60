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
        self.L, self.h, self.device, self._recording = Library(), 1, torch.device("cpu"), False

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
