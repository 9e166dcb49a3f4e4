"""The paged calls without a GPU: what they refuse before any CUDA work, and the bookkeeping of pages."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from nntrainer_b200 import backend as be  # noqa: E402
from nntrainer_b200 import build as nb_build  # noqa: E402
from nntrainer_b200 import capi  # noqa: E402

BUF = (C.c_uint8 * 65536)()
AT = (C.addressof(BUF) + 255) // 256 * 256  # an aligned address that nothing reads: every call below is refused first


@pytest.fixture(scope="module")
def L():
    nb_build.build()
    return capi.lib()


def cache(**kw):
    c = dict(n_heads_q=8, n_heads_kv=2, head_dim=64, dtype=capi.F16, page_size=16, n_pages=4, page_stride=0, kcache=AT, vcache=AT)
    c.update(kw)
    return capi.PagedCache(*c.values())


def batch(**kw):
    b = dict(batch=2, tokens=2, max_new=1, max_rows=10, ld_table=1, row_start=AT, context=AT, page_table=AT)
    b.update(kw)
    return capi.PagedBatch(*b.values())


BAD_CACHES = [(dict(kcache=None), "INVALID"), (dict(vcache=None), "INVALID"), (dict(dtype=capi.F32), "UNSUPPORTED"), (dict(n_heads_q=7), "INVALID"),
              (dict(n_heads_kv=0), "INVALID"), (dict(n_heads_q=0), "INVALID"), (dict(head_dim=60), "INVALID"), (dict(head_dim=0), "INVALID"),
              (dict(head_dim=136), "UNSUPPORTED"), (dict(page_size=8), "UNSUPPORTED"), (dict(page_size=48), "UNSUPPORTED"),
              (dict(page_size=512), "UNSUPPORTED"), (dict(n_pages=0), "INVALID"), (dict(page_stride=1024), "INVALID"),
              (dict(page_stride=2052), "INVALID"), (dict(kcache=AT + 8), "INVALID"), (dict(vcache=AT + 2), "INVALID")]
BAD_BATCHES = [(dict(batch=70000), "INVALID"), (dict(max_new=3), "INVALID"), (dict(row_start=None), "INVALID"), (dict(context=None), "INVALID"),
               (dict(page_table=None), "INVALID"), (dict(ld_table=1 << 30), "INVALID"), (dict(tokens=1 << 30, max_new=1), "INVALID")]


def attend(L, c, b, q=AT, ld_q=512, window=0xFFFFFFFF, out=AT, out_dtype=capi.F16, ld_out=512):
    return L.nntr_cuda_paged_attention_dev(C.byref(c), C.byref(b), q, ld_q, window, 0, None, out, out_dtype, ld_out, 0, None)


def append(L, c, b, q=AT, k=AT, ld_q=768, ld_kv=768, qg=None, kg=None, cos=AT, out=AT, ld_out=512):
    return L.nntr_cuda_paged_append_dev(C.byref(c), C.byref(b), q, k, AT, ld_q, ld_kv, qg, kg, 1e-6, cos, AT, 16, out, ld_out, 0, None)


@pytest.mark.parametrize("call", [attend, append])
@pytest.mark.parametrize("bad,code", BAD_CACHES)
def test_bad_caches_are_refused(L, call, bad, code):
    assert call(L, cache(**bad), batch()) == getattr(capi, "ERR_" + code)


@pytest.mark.parametrize("call", [attend, append])
@pytest.mark.parametrize("bad,code", BAD_BATCHES)
def test_bad_batches_are_refused(L, call, bad, code):
    assert call(L, cache(), batch(**bad)) == getattr(capi, "ERR_" + code)


@pytest.mark.parametrize("bad", [dict(q=None), dict(out=None), dict(q=AT + 8), dict(out=AT + 2), dict(ld_q=508), dict(ld_q=504), dict(ld_out=516),
                                 dict(window=0)])
def test_bad_attention_operands_are_refused(L, bad):
    assert attend(L, cache(), batch(), **bad) == capi.ERR_INVALID
    assert L.nntr_cuda_last_error()


def test_attention_result_type(L):
    assert attend(L, cache(), batch(), out_dtype=capi.BF16) == capi.ERR_UNSUPPORTED


@pytest.mark.parametrize("bad", [dict(q=None), dict(k=None), dict(cos=None), dict(out=None), dict(out=AT + 4), dict(ld_q=500), dict(ld_kv=100),
                                 dict(ld_out=514), dict(qg=AT), dict(kg=AT)])
def test_bad_append_operands_are_refused(L, bad):
    assert append(L, cache(), batch(), **bad) == capi.ERR_INVALID


def test_empty_batches_do_nothing(L):
    for b in (batch(batch=0), batch(tokens=0, max_new=0)):
        assert attend(L, cache(), b) == capi.OK
        assert append(L, cache(), b) == capi.OK


@pytest.mark.parametrize("args,code", [((None, 1, 0, 4096, 4, AT, AT, 1), "INVALID"), ((AT, 1, 0, 4096, 4, None, AT, 1), "INVALID"),
                                       ((AT, 1, 0, 4096, 4, AT, None, 1), "INVALID"), ((AT, 1, 0, 4088, 4, AT, AT, 1), "INVALID"),
                                       ((AT + 8, 1, 0, 4096, 4, AT, AT, 1), "INVALID"), ((AT, 2, 4096, 4096, 4, AT, AT, 1), "INVALID"),
                                       ((AT, 1, 0, 4096, 0, AT, AT, 1), "INVALID"), ((AT, 1, 0, 0, 4, AT, AT, 1), "INVALID"),
                                       ((AT, 1, 0, 4096, 4, AT, AT, 70000), "UNSUPPORTED"), ((AT, 1, 0, 4096, 4, AT, AT, 0), None),
                                       ((AT, 0, 0, 4096, 4, AT, AT, 1), None)])
def test_copy_pages_refusals(L, args, code):
    assert L.nntr_cuda_copy_pages_dev(*args, 0, None) == (getattr(capi, "ERR_" + code) if code else capi.OK)


@pytest.mark.parametrize("kw,code", [(dict(x=None), "INVALID"), (dict(u=None), "INVALID"), (dict(idx=None), "INVALID"), (dict(n=0), "INVALID"),
                                     (dict(rows=-1), "INVALID"), (dict(ld=50), "INVALID"), (dict(n=(1 << 20) + 1, ld=1 << 21), "UNSUPPORTED"),
                                     (dict(rows=65536), "UNSUPPORTED"), (dict(t=-0.5), "INVALID"), (dict(t=float("nan")), "INVALID"),
                                     (dict(p=-0.1), "INVALID"), (dict(m=-0.1), "INVALID"), (dict(m=1.5), "INVALID"), (dict(rows=0), None)])
def test_sample_refusals(L, kw, code):
    a = dict(x=AT, rows=2, n=100, ld=100, u=AT, t=1.0, k=0, p=1.0, m=0.0, idx=AT)
    a.update(kw)
    rc = L.nntr_cuda_sample_dev(a["x"], a["rows"], a["n"], a["ld"], a["u"], a["t"], a["k"], a["p"], a["m"], None, a["idx"], None, None, 0, None)
    assert rc == (getattr(capi, "ERR_" + code) if code else capi.OK)


def test_host_tensors_are_refused():
    x = torch.zeros(2, 10)
    with pytest.raises(ValueError):
        be.sample(x, torch.zeros(2))
    kv = torch.zeros(1, 2, 4, 16, 2, 8, dtype=torch.float16)
    with pytest.raises(ValueError):
        be.copy_pages(kv, torch.zeros(1, dtype=torch.int32), torch.ones(1, dtype=torch.int32))


class Moved(be.PagedCache):
    """The bookkeeping with copies made on the host."""

    def _copy(self, src, dst):
        assert len(set(dst)) == len(dst) and not set(dst) & set(src)
        if src:
            self.kv[:, :, dst] = self.kv[:, :, src]


def small(pages=8):
    return Moved(2, pages, 16, 1, 8, device="cpu")


def fill(c, seq):
    """Gives every page that the sequence alone holds a content of its own."""
    for k, p in enumerate(c.pages(seq)):
        if c._refs[p] == 1:
            c.kv[:, :, p] = 100 * seq + k + 1


def content(c, seq):
    return [float(c.kv[0, 0, p, 0, 0, 0]) for p in c.pages(seq)]


def test_pages_are_reserved_as_rows_need_them():
    c = small()
    a, b = c.new(), c.new()
    c.reserve([a, b], [1, 16])
    assert (len(c.pages(a)), len(c.pages(b)), c.free_pages) == (1, 1, 6)
    c.reserve([a, b], [15, 1])
    assert (len(c.pages(a)), len(c.pages(b)), c.free_pages) == (1, 2, 5)
    assert (c.rows(a), c.rows(b)) == (16, 17)
    with pytest.raises(MemoryError):
        c.reserve([a, b], [50, 50])
    assert (c.rows(a), c.rows(b), c.free_pages) == (16, 17, 5)
    assert not set(c.pages(a)) & set(c.pages(b))
    for bad in (([a, a], [1, 1]), ([a], [1, 2]), ([a], [-1])):
        with pytest.raises(ValueError):
            c.reserve(*bad)
    c.free(b)
    assert c.free_pages == 7
    with pytest.raises(KeyError):
        c.rows(b)


def test_batch_arrays():
    c = small()
    a, b = c.new(), c.new()
    c.reserve([a, b], [20, 3])
    d = c.batch([b, a], [3, 2])
    assert d["row_start"].tolist() == [0, 3, 5] and d["context"].tolist() == [3, 20]
    assert (d["max_new"], d["max_rows"]) == (3, 20)
    assert d["page_table"].tolist() == [c.pages(b) + [-1], c.pages(a)]
    assert all(t.dtype == torch.int32 and t.is_contiguous() for t in (d["row_start"], d["context"], d["page_table"]))
    for bad in (([], []), ([a], [21]), ([a], [1, 1])):
        with pytest.raises(ValueError):
            c.batch(*bad)


def test_fork_shares_full_pages_and_copies_the_last():
    c = small(10)
    a = c.new()
    c.reserve([a], [40])  # two full pages and a half one
    fill(c, a)
    f, g = c.fork(a, 2)
    assert c.pages(f)[:2] == c.pages(a)[:2] == c.pages(g)[:2]
    assert len({c.pages(s)[2] for s in (a, f, g)}) == 3
    assert content(c, f) == content(c, a) == content(c, g)
    assert c.free_pages == 5
    c.reserve([f], [20])  # into its own page and a new one
    c.free(a)
    assert c.free_pages == 5 and content(c, g) == [1, 2, 3]
    c.free(f)
    c.free(g)
    assert c.free_pages == 10 and not any(c._refs)
    e = c.new()
    assert c.pages(c.fork(e)[0]) == []
    c.reserve([e], [16 * 9])
    c.reserve([e], [1])
    with pytest.raises(MemoryError):  # no page left for the copy of the last one
        c.fork(e)
    assert len(c._seqs) == 2 and all(r <= 1 for r in c._refs)


def test_compact_moves_used_pages_to_the_front():
    c = small(12)
    a, b, d = c.new(), c.new(), c.new()
    for s in (a, b, d, a, b, d):
        c.reserve([s], [20])
    f, = c.fork(d)
    for s in (a, b, d):
        fill(c, s)
    kept = {s: content(c, s) for s in (b, d, f)}
    c.free(a)
    moved = c.compact()
    used = {p for s in (b, d, f) for p in c.pages(s)}
    assert moved > 0 and used == set(range(len(used))) and c.free_pages == 12 - len(used)
    assert {s: content(c, s) for s in (b, d, f)} == kept
    assert c.compact() == 0
    c.reserve([b], [16])
    assert c.pages(b)[-1] == len(used)


def test_more_copies_than_a_launch_takes(monkeypatch):
    calls = []
    monkeypatch.setattr(be, "copy_pages", lambda kv, src, dst: calls.append((src.tolist(), dst.tolist())))
    c = be.PagedCache(1, 4, 16, 1, 8, device="cpu")
    n = 2 * 65535 + 3
    c._copy(list(range(n)), list(range(n, 2 * n)))
    assert [len(s) for s, _ in calls] == [65535, 65535, 3]
    assert sum((s for s, _ in calls), []) == list(range(n)) and sum((d for _, d in calls), []) == list(range(n, 2 * n))
    calls.clear()
    c._copy([], [])
    assert not calls
