"""Calls of the paged operators and of sampling that the documentation allows beside the usual ones: early launches, batches with padding,
logits of other shapes, as many rows as there may be."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_paged_gpu import BF16, F16, Case, be, rng, tables  # noqa: E402, F401
from test_sample import reference  # noqa: E402


@pytest.mark.parametrize("new", [[1] * 9, [70, 1, 200]])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_early_launches_change_nothing(be, dtype, new):
    """Append, attention, a page's copy, attention again and a draw, one behind the other with launches let in early, eager and captured."""
    ctx = [n + 300 for n in new]
    c = Case(new, ctx, (8, 2, 128), dtype, 32, seed=90, junk=0.0)
    cos, sin = tables(be, max(ctx), 128)
    g = rng(91)
    qkv = torch.randn(c.tokens, 12 * 128, generator=g, device="cuda")
    proj, u = torch.randn(1024, 4000, generator=g, device="cuda"), torch.rand(c.tokens, generator=g, device="cuda")
    spare = c.k.shape[0] - 1 if c.k.shape[0] - 1 not in c.table.unique().tolist() else c.k.shape[0] - 2
    while spare in c.table.unique().tolist():
        spare -= 1
    src, dst = c.table[0, :1].clone(), torch.tensor([spare], dtype=torch.int32, device="cuda")
    moved = c.table.clone()
    moved[0, 0] = spare
    kv = torch.stack([c.k, c.v])[None].contiguous()
    start = kv.clone()
    q16 = torch.empty(c.tokens, 8, 128, dtype=dtype, device="cuda")
    o1, o2 = (torch.empty(c.tokens, 8, 128, device="cuda") for _ in range(2))
    drawn = (torch.empty(c.tokens, dtype=torch.int32, device="cuda"), torch.empty(c.tokens, device="cuda"), torch.empty(c.tokens, device="cuda"))

    def chain(pdl):
        b = (c.row_start, c.context, max(new))
        be.paged_append(qkv[:, :1024], qkv[:, 1024:1280], qkv[:, 1280:], kv[0, 0], kv[0, 1], c.table, *b, cos, sin, q_out=q16, pdl=pdl)
        be.paged_attention(q16, kv[0, 0], kv[0, 1], c.table, *b, max(ctx), out=o1, pdl=pdl)
        be.copy_pages(kv, src, dst, pdl=pdl)
        be.paged_attention(q16, kv[0, 0], kv[0, 1], moved, *b, max(ctx), out=o2, pdl=pdl)
        be.sample(o2.view(c.tokens, 1024), u, 0.8, 50, 0.9, out=drawn, pdl=pdl)

    def result():
        torch.cuda.synchronize()
        return [t.clone() for t in (q16, o1, o2, kv, *drawn)]

    chain(False)
    want = result()
    assert torch.equal(want[1], want[2])
    for _ in range(5):
        kv.copy_(start)
        o1.fill_(7)
        o2.fill_(7)
        chain(True)
        assert all(torch.equal(a, b) for a, b in zip(result(), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        chain(True)
    for _ in range(5):
        kv.copy_(start)
        o1.fill_(7)
        o2.fill_(7)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(result(), want))
    be.device_status()


@pytest.mark.parametrize("new", [[1, 1, 1], [90, 7, 33]])
def test_sequences_of_padding_do_nothing(be, new):
    """A batch filled up to the size that a graph was captured for: sequences without rows, without a context, without pages."""
    be.check(be.lib().nntr_cuda_clear_device_status())
    c = Case(new, [200, 90, 333], (8, 2, 64), F16, 16, seed=92, extra_rows=4)
    cos, sin = tables(be, 333, 64)
    x = torch.randn(c.tokens, 12 * 64, device="cuda")
    for pad in (1, 5, 40, 140):
        more = lambda t, v: torch.cat([t, torch.full((pad, *t.shape[1:]), v, dtype=torch.int32, device="cuda")])  # noqa: E731
        table, start, context = more(c.table, -1), more(c.row_start, c.starts[-1]), more(c.context, 0)
        out = torch.full_like(c.q, 5.0)
        be.paged_attention(c.q, c.k, c.v, table, start, context, max(new), 333, out=out)
        c.check(out)
        assert bool((out[c.starts[-1]:] == 5).all())
        k, v, k2, v2 = c.k.clone(), c.v.clone(), c.k.clone(), c.v.clone()
        a = be.paged_append(x[:, :512], x[:, 512:640], x[:, 640:], k, v, table, start, context, max(new), cos, sin, q_out=torch.full_like(c.q, 5.0))
        b = be.paged_append(x[:, :512], x[:, 512:640], x[:, 640:], k2, v2, c.table, c.row_start, c.context, max(new), cos, sin, q_out=torch.full_like(c.q, 5.0))
        assert torch.equal(a, b) and all(torch.equal(p.view(torch.int16), q.view(torch.int16)) for p, q in ((k, k2), (v, v2)))
    be.device_status()


def test_logits_of_other_shapes(be):
    g = rng(93)
    x, u = torch.randn(2, 3, 700, generator=g, device="cuda"), torch.rand(2, 3, generator=g, device="cuda")
    want = be.sample(x.view(6, 700), u.view(6), 0.7, 30)
    assert all(torch.equal(a, b) for a, b in zip(be.sample(x, u, 0.7, 30), want))
    one = be.sample(x[1, 2], u[1, 2:], 0.7, 30)
    assert all(torch.equal(a, b[5:]) for a, b in zip(one, want))


def test_as_many_rows_as_there_may_be(be):
    g = rng(94)
    x, u = torch.randn(65535, 9, generator=g, device="cuda"), torch.rand(65535, generator=g, device="cuda")
    idx = be.sample(x, u, 0.9, 4, 0.95)[0]
    for r in list(range(0, 65535, 1311)) + [65534]:
        i, _, slack = reference(x[r], u[r], t=0.9, k=4, p=0.95)
        assert slack < 1e-6 or int(idx[r]) == i
    with pytest.raises(NotImplementedError):
        be.sample(torch.zeros(65536, 2, device="cuda"), torch.zeros(65536, device="cuda"))


@pytest.mark.parametrize("heads,new,ctx", [((4096, 1, 8), [1], [20]), ((4096, 512, 64), [3], [40]), ((4096, 1, 128), [2, 1], [30, 9])])
def test_as_many_heads_as_there_may_be(be, heads, new, ctx):
    c = Case(new, ctx, heads, F16, 16, seed=95)
    c.check(c.attend(be))


@pytest.mark.parametrize("new", [1, 9])
def test_as_many_sequences_as_there_may_be(be, new):
    """Three sequences, 21845 times: all give what three alone give."""
    c = Case([new] * 3, [new + 4, new, new + 8], (8, 1, 64), BF16, 16, seed=96)
    start = torch.arange(65536, dtype=torch.int32, device="cuda") * new
    out = be.paged_attention(c.q.repeat(21845, 1, 1), c.k, c.v, c.table.repeat(21845, 1), start, c.context.repeat(21845), new, new + 8)
    out = out.view(21845, 3 * new, 8, 64)
    c.check(out[0])
    assert bool((out == out[0]).all())
    be.device_status()
