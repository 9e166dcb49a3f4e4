"""The pool of pages when a copy fails; the structures of the paged calls in their two forms. No GPU is needed."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from nntrainer_b200 import backend as be  # noqa: E402
from nntrainer_b200 import capi  # noqa: E402


def test_a_fork_whose_copy_fails_changes_nothing():
    """As where the cache lies on another device than the current one, or while a graph is captured."""
    class Failing(be.PagedCache):
        def _copy(self, src, dst):
            raise RuntimeError("no copy now")

    c = Failing(2, 8, 16, 1, 8, device="cpu")
    a = c.new()
    c.reserve([a], [40])
    before = (c.free_pages, sorted(c._free), list(c._refs), {s: (r, list(p)) for s, (r, p) in c._seqs.items()}, c._next)
    for n in (1, 3):
        with pytest.raises(RuntimeError):
            c.fork(a, n)
        assert (c.free_pages, sorted(c._free), list(c._refs), {s: (r, list(p)) for s, (r, p) in c._seqs.items()}, c._next) == before
    c.free(a)
    assert c.free_pages == 8 and not any(c._refs)


def test_a_fork_on_a_cache_that_no_launch_can_reach_changes_nothing():
    c = be.PagedCache(1, 4, 16, 1, 8, device="cpu")  # its copies are refused
    a = c.new()
    c.reserve([a], [17])
    with pytest.raises(ValueError):
        c.fork(a)
    assert c.free_pages == 2 and list(c._seqs) == [a] and sum(c._refs) == 2
    b = c.new()
    c.reserve([b], [16])
    c.free(a)
    pages, refs = c.pages(b), list(c._refs)
    with pytest.raises(ValueError):
        c.compact()
    assert c.pages(b) == pages and c._refs == refs and c.free_pages == 3


def test_the_two_forms_of_the_structures_agree():
    """The calls pack nntr_paged_cache and nntr_paged_batch in one go; capi declares their fields."""
    c = be._PAGED_CACHE.pack(8, 2, 64, 30, 16, 1000, 1 << 40, 0x7f0011223344, 0x7f5566778899)
    want = capi.PagedCache(8, 2, 64, 30, 16, 1000, 1 << 40, 0x7f0011223344, 0x7f5566778899)
    assert len(c) == C.sizeof(capi.PagedCache) and c == bytes(want)
    b = be._PAGED_BATCH.pack(3, 70, 60, 4000, 250, 0x7f0011223344, 0x7f5566778899, 0x7faabbccddee)
    want = capi.PagedBatch(3, 70, 60, 4000, 250, 0x7f0011223344, 0x7f5566778899, 0x7faabbccddee)
    assert len(b) == C.sizeof(capi.PagedBatch)
    for name, kind in capi.PagedBatch._fields_:  # padding between them holds nothing
        at = getattr(capi.PagedBatch, name)
        assert b[at.offset:at.offset + at.size] == bytes(want)[at.offset:at.offset + at.size], name
