"""A key/value cache in pages on the GPU: new rows, attention, copies of pages, against the formulas in 64 bits.

Tolerances. A result in a type with epsilon eps is rounded by at most eps / 2 of it (eps = torch.finfo(type).eps). Attention also rounds the
probabilities to the caches' type: with A = sum_j p_j |v_j| / sum_j p_j that moves a result by at most eps / 2 * A, and fp32 arithmetic by at
most 2 * d * A where d bounds the relative error of a probability: the score is a sum of head_dim exact products in fp32, in whatever order,
off by at most head_dim * 2^-23 * (|q| . |k|) / sqrt(head_dim); scaled by log2(e) and less the maximum it is off by 3 * 2^-24 of itself,
where |score| <= (|q| . |k|) / sqrt(head_dim) for the score and the maximum; the exponential by 2^-22 from the special function unit, by
2.82e-6 (fp16) or 1.013e-4 (bf16, whose rounding is 3.9e-3) as a polynomial of fourth or third degree (greatest relative errors of the fits), and
2^-22 for the polynomial's fp32 steps; the sum of L of them and of the products by L * 2^-23. Probabilities below the normal numbers of fp16 are off by 2^-25; the
greatest of a row is 2^6 or more, and so is their sum."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def be():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from nntrainer_b200 import backend, build
    build.build()
    backend.init(0)
    return backend


def rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


class Case:
    """Random inputs of a batch; every cache row that no sequence has is NaN."""

    def __init__(self, new, ctx, heads, dtype=F16, page=16, seed=0, q_scale=2.0, extra_rows=0, junk=math.nan, layout="dense"):
        g = rng(seed)
        self.new, self.ctx, (self.hq, self.hkv, self.hd), self.dtype, self.page = new, ctx, heads, dtype, page
        need = [-(-c // page) for c in ctx]
        pool = sum(need) + 2
        ids = torch.randperm(pool, generator=g, device="cuda").tolist()
        self.table = torch.full((len(ctx), max(need + [1])), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
            at += n
        if layout == "pairs":  # a page's keys and values next to each other
            kv = torch.full((pool, 2, page, self.hkv, self.hd), junk, dtype=dtype, device="cuda")
            self.k, self.v = kv[:, 0], kv[:, 1]
        else:
            self.k = torch.full((pool, page, self.hkv, self.hd), junk, dtype=dtype, device="cuda")
            self.v = self.k.clone()
        self.K, self.V = [], []
        for b, c in enumerate(ctx):
            k, v = (torch.randn(c, self.hkv, self.hd, generator=g, device="cuda").to(dtype) for _ in range(2))
            self.K.append(k)
            self.V.append(v)
            for r in range(0, c, page):
                p = int(self.table[b, r // page])
                self.k[p, :min(page, c - r)] = k[r:r + page]
                self.v[p, :min(page, c - r)] = v[r:r + page]
        self.table = self.table.cuda()
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        self.starts, self.tokens = starts, starts[-1] + extra_rows
        self.row_start = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.context = torch.tensor(ctx, dtype=torch.int32, device="cuda")
        self.q = (q_scale * torch.randn(self.tokens, self.hq, self.hd, generator=g, device="cuda")).to(dtype)
        self.sinks = torch.randn(self.hq, generator=g, device="cuda")

    def attend(self, be, q=None, **kw):
        kw.setdefault("max_rows", max(self.ctx))
        return be.paged_attention(self.q if q is None else q, self.k, self.v, self.table, self.row_start, self.context, max(self.new), **kw)

    def check(self, out, window=None, first_tokens=0, sink=None):
        eps = torch.finfo(self.dtype).eps
        out_eps = torch.finfo(out.dtype).eps
        exponential = 2 ** -22 + (2.82e-6 if self.dtype == F16 else 1.013e-4)
        G = self.hq // self.hkv
        for b, (n, c) in enumerate(zip(self.new, self.ctx)):
            if n == 0:
                continue
            p = torch.arange(c - n, c, device="cuda")[:, None]
            j = torch.arange(c, device="cuda")[None]
            seen = j <= p
            if window is not None:
                seen &= (j > p - window) | (j < first_tokens)
            q = self.q[self.starts[b]:self.starts[b] + n].double()
            for h in range(self.hq):
                k, v = self.K[b][:, h // G].double(), self.V[b][:, h // G].double()
                s = (q[:, h] @ k.T) / math.sqrt(self.hd)
                size = (q[:, h].abs() @ k.abs().T).amax(1) / math.sqrt(self.hd)
                s = s.masked_fill(~seen, -math.inf)
                m = s.amax(1, keepdim=True)
                w = (s - torch.where(m == -math.inf, torch.zeros_like(m), m)).exp()
                den = w.sum(1, keepdim=True)
                if sink is not None:
                    den = den + (sink[h].double() - m).exp()
                w = w / den
                want = torch.nan_to_num(w) @ v if c else torch.zeros(n, self.hd, device="cuda").double()
                A = torch.nan_to_num(w) @ v.abs()
                d = (self.hd * 2 ** -23 + 3 * 2 ** -24 * 2 * 1.4427) * size + exponential + 2 * c * 2 ** -23
                bound = out_eps / 2 * want.abs() + (1 + eps) * (eps / 2 + 2 * d[:, None]) * A + c * 2.0 ** -31 * v.abs().max() + 2.0 ** -24 * (out.dtype == F16)
                got = out[self.starts[b]:self.starts[b] + n, h].double()
                off = (got - want).abs()
                assert bool((off <= bound).all()), (b, h, float((off / bound).max()), n, c)


HEADS = [(8, 2, 128), (4, 4, 64), (8, 1, 128), (6, 2, 96), (16, 2, 64), (5, 1, 8), (7, 1, 40), (32, 1, 128)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_one_token_each(be, heads, dtype, page):
    ctx = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 257, 700]
    c = Case([1] * len(ctx), ctx, heads, dtype, page, seed=page)
    c.check(c.attend(be))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page", [16, 64, 256])
def test_chunks_of_all_lengths(be, heads, dtype, page):
    new = [1, 3, 0, 16, 17, 40, 128, 129, 300, 31, 2]
    ctx = [1, 3, 9, 16, 50, 333, 128, 257, 300, 700, 513]
    c = Case(new, ctx, heads, dtype, page, seed=1)
    c.check(c.attend(be))


@pytest.mark.parametrize("heads", [(8, 2, 128), (16, 2, 64)])
@pytest.mark.parametrize("new,ctx", [([1] * 6, [1, 5, 99, 100, 101, 400]), ([1, 7, 60, 200, 130], [5, 107, 100, 500, 1000])])
@pytest.mark.parametrize("window,first", [(100, 0), (100, 4), (1, 0), (1, 1), (17, 70), (128, 128), (1000, 3), (64, 16)])
@pytest.mark.parametrize("with_sink", [False, True])
def test_windows_first_tokens_and_sinks(be, heads, new, ctx, window, first, with_sink):
    c = Case(new, ctx, heads, F16, 16, seed=2)
    kw = dict(window=window, first_tokens=first, sink=c.sinks if with_sink else None)
    c.check(c.attend(be, **kw), **kw)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new,ctx,window", [(2, 2001, 513), (2, 2001, 512), (3, 2001, 514), (100, 2000, 494), (100, 2000, 493), (100, 2000, 495),
                                            (40, 700, 60), (300, 1000, 129)])
def test_the_first_rows_read_are_out_of_sight_for_some(be, dtype, new, ctx, window):
    """The window of a tile's first query begins at the end of a block that its later ones do not see at all."""
    for heads in ((16, 2, 96), (4, 4, 64)):
        c = Case([new, 1], [ctx, 5], heads, dtype, 32, seed=33)
        c.check(c.attend(be, window=window), window=window)


@pytest.mark.parametrize("new", [1, 65])
def test_what_no_query_sees_may_be_anything(be, new):
    """NaN and infinities in rows that have left the window, in the rest of the last page and in pages of others."""
    c = Case([new] * 3, [400, 333, 290], (8, 2, 128), BF16, 32, seed=3, junk=math.inf)
    for b, n in enumerate(c.ctx):
        oldest = n - new - 100 + 1  # the first row that the first query sees, behind the first tokens
        for r in range(4, oldest):
            page = int(c.table[b, r // 32])
            c.k[page, r % 32] = math.nan
            c.v[page, r % 32] = math.nan
            c.K[b][r] = 0
            c.V[b][r] = 0
    kw = dict(window=100, first_tokens=4)
    out = c.attend(be, **kw)
    assert bool(torch.isfinite(out).all())
    c.check(out, **kw)


@pytest.mark.parametrize("new,ctx", [([1, 1, 1], [30, 100, 7]), ([70, 1, 129], [70, 100, 200])])
def test_results_in_fp32_strided_operands_rows_behind(be, new, ctx):
    c = Case(new, ctx, (8, 2, 96), BF16, 16, seed=4, extra_rows=5, layout="pairs")
    assert not c.k.is_contiguous()
    wide = torch.randn(c.tokens, 8 * 96 + 40, device="cuda").to(BF16)
    q = wide[:, 32:32 + 8 * 96].view(c.tokens, 8, 96)
    q.copy_(c.q)
    out = torch.full((c.tokens, 8 * 96 + 16), 7.0, device="cuda")
    view = out[:, 8:8 + 8 * 96].view(c.tokens, 8, 96)
    assert c.attend(be, q=q, out=view) is view
    c.check(view)
    assert bool((out[:, :8] == 7).all()) and bool((out[:, -8:] == 7).all()) and bool((out[c.starts[-1]:] == 7).all())


@pytest.mark.parametrize("heads", [(8, 2, 128), (8, 1, 64), (3, 1, 96)])
@pytest.mark.parametrize("batch,most", [(150, 1), (129, 3), (70, 5), (33, 90), (40, 16), (3, 16), (2, 8)])
def test_many_sequences_and_few_rows(be, heads, batch, most):
    new = [1 + (7 * b) % most for b in range(batch)]
    ctx = [n + (37 * b) % 211 for b, n in enumerate(new)]
    c = Case(new, ctx, heads, BF16 if batch % 2 else F16, 16, seed=batch)
    c.check(c.attend(be))
    c.check(c.attend(be, window=50, first_tokens=3), window=50, first_tokens=3)


@pytest.mark.parametrize("new", [1, 150])
def test_sharply_peaked_and_large_scores(be, new):
    c = Case([new, new], [700, 150], (8, 2, 64), F16, 64, seed=5, q_scale=60.0)
    c.check(c.attend(be))
    c.K[0][:], c.k[:] = 0, torch.where(torch.isnan(c.k), c.k, torch.zeros_like(c.k))  # all scores equal
    c.K[1][:] = 0
    c.check(c.attend(be))


def test_long_contexts_few_sequences(be):
    for heads, ctx, new in (((8, 1, 128), [30011], [1]), ((4, 4, 64), [20000, 3], [1, 1]), ((8, 2, 128), [9001], [33]), ((32, 8, 128), [5000, 9], [2, 2])):
        c = Case(new, ctx, heads, F16, 64, seed=6)
        for max_rows in (0, 64, max(ctx)):
            c.check(c.attend(be, max_rows=max_rows))


@pytest.mark.parametrize("new", [1, 90])
def test_a_pool_beyond_two_gigaelements(be, new):
    pages, ps, hkv, hd = 8300, 256, 8, 128
    assert pages * ps * hkv * hd > 2 ** 31
    c = Case([new], [500], (8, 8, 128), F16, ps, seed=7)
    k = torch.empty(pages, ps, hkv, hd, dtype=F16, device="cuda")
    v = torch.empty_like(k)
    places = [pages - 1, pages - 2]
    for i, p in enumerate(places):
        k[p], v[p] = c.k[int(c.table[0, i])], c.v[int(c.table[0, i])]
    c.k, c.v = k, v
    c.table = torch.tensor([places], dtype=torch.int32, device="cuda")
    c.check(c.attend(be))


@pytest.mark.parametrize("new", [[1, 2], [70, 3]])
def test_counts_beyond_32_bits(be, new):
    c = Case(new, [100, 300], (8, 2, 64), seed=31)
    want = c.attend(be)
    assert torch.equal(c.attend(be, window=2 ** 32 + 5), want)
    assert torch.equal(c.attend(be, window=5, first_tokens=2 ** 32 + 5), want)


@pytest.mark.parametrize("heads", [(192, 1, 64), (300, 2, 40), (260, 2, 128)])
@pytest.mark.parametrize("new,ctx", [([1, 1], [100, 3]), ([3, 1, 5], [400, 1, 5])])
def test_groups_wider_than_a_tile(be, heads, new, ctx):
    c = Case(new, ctx, heads, F16, 16, seed=32)
    c.check(c.attend(be))


@pytest.mark.parametrize("new", [[1, 1, 1], [60, 2, 9]])
@pytest.mark.parametrize("max_rows", [0, 1, 100, 1 << 29, (1 << 32) - 1])
def test_any_expected_length_is_right(be, new, max_rows):
    c = Case(new, [700, 90, 1100], (8, 2, 128), BF16, 32, seed=33)
    c.check(c.attend(be, max_rows=max_rows))


@pytest.mark.parametrize("new", [1, 40])
def test_rows_in_front_of_the_first_sequence(be, new):
    c = Case([new, new], [200, 90], (8, 2, 128), F16, 16, seed=34)
    q = torch.cat([c.q.new_full((6, 8, 128), math.nan), c.q])
    start = c.row_start + 6
    out = torch.full_like(q, 5.0)
    be.paged_attention(q, c.k, c.v, c.table, start, c.context, new, 200, out=out)
    assert bool((out[:6] == 5).all())
    c.check(out[6:])
    cos, sin = tables(be, 200, 128)
    x = torch.randn(q.shape[0], 12 * 128, device="cuda")
    k, v = c.k.clone(), c.v.clone()
    got = be.paged_append(x[:, :1024], x[:, 1024:1280], x[:, 1280:], k, v, c.table, start, c.context, new, cos, sin, q_out=torch.full_like(q, 5.0))
    k2, v2 = c.k.clone(), c.v.clone()
    want = be.paged_append(x[6:, :1024], x[6:, 1024:1280], x[6:, 1280:], k2, v2, c.table, c.row_start, c.context, new, cos, sin)
    assert bool((got[:6] == 5).all()) and torch.equal(got[6:], want)
    assert torch.equal(torch.nan_to_num(k), torch.nan_to_num(k2)) and torch.equal(torch.nan_to_num(v), torch.nan_to_num(v2))
    be.device_status()


@pytest.mark.parametrize("new", [1, 100])
def test_captured_and_replayed_with_other_contents(be, new):
    c = Case([new, new], [300, 200], (8, 2, 128), F16, 16, seed=8)
    other = Case([new, new - 1 if new > 1 else 1], [270, 333], (8, 2, 128), F16, 16, seed=9)
    wide = max(c.table.shape[1], other.table.shape[1])
    pad = lambda t: torch.cat([t, torch.full((2, wide - t.shape[1]), -1, dtype=torch.int32, device="cuda")], 1).contiguous()  # noqa: E731
    pages = max(c.k.shape[0], other.k.shape[0])
    k, v = (torch.zeros(pages, 16, 2, 128, dtype=F16, device="cuda") for _ in range(2))
    held = [torch.zeros_like(pad(c.table)), c.row_start.clone(), c.context.clone(), torch.zeros(2 * new, 8, 128, dtype=F16, device="cuda")]

    def load(x):
        k[:x.k.shape[0]], v[:x.v.shape[0]] = x.k, x.v
        for d, s in zip(held, (pad(x.table), x.row_start, x.context)):
            d.copy_(s)
        held[3][:x.tokens] = x.q

    out = torch.empty(2 * new, 8, 128, dtype=F16, device="cuda")
    call = lambda: be.paged_attention(held[3], k, v, held[0], held[1], held[2], new, 64, out=out)  # noqa: E731
    load(c)
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        call()
    for x in (other, c):
        load(x)
        out.fill_(9)
        g.replay()
        torch.cuda.synchronize()
        x.check(out)
        assert bool((out[x.starts[-1]:] == 9).all())


def test_two_streams_at_once(be):
    cases = [Case([1] * 5 if i % 2 else [70, 9], [1000, 300, 2, 50, 800] if i % 2 else [700, 9], (8, 2, 128), F16, 16, seed=20 + i) for i in range(4)]
    torch.cuda.synchronize()
    outs, streams = [], [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        outs = []
        for c, st in zip(cases, streams):
            with torch.cuda.stream(st):
                outs.append(c.attend(be))
        torch.cuda.synchronize()
    for c, o in zip(cases, outs):
        c.check(o)


def test_same_bits_every_time(be):
    for new in (1, 77):
        c = Case([new] * 3, [900, 431, 300], (8, 2, 128), BF16, 32, seed=30)
        first = c.attend(be)
        for _ in range(20):
            assert torch.equal(c.attend(be), first)


def test_contradicting_arrays_are_told_and_touch_nothing_out_of_range(be):
    be.check(be.lib().nntr_cuda_clear_device_status())
    for new in (1, 50):
        def told(change, **kw):
            c = Case([new, new], [100, 120], (8, 2, 64), F16, 16, seed=40, extra_rows=3, junk=0.0)
            out = torch.full((c.tokens, 8, 64), 5.0, dtype=F16, device="cuda")
            change(c)
            kw = dict(max_rows=120, out=out) | kw
            n = kw.pop("max_new", new)
            be.paged_attention(c.q, c.k, c.v, c.table, c.row_start, c.context, n, **kw)
            with pytest.raises(ValueError):
                be.device_status()
            be.check(be.lib().nntr_cuda_clear_device_status())
            be.device_status()
            return c, out

        c, out = told(lambda c: c.table[0].fill_(1 << 30))
        assert bool((out[:new] == 0).all())  # its rows read as zeros
        told(lambda c: c.table[1, 2:4].fill_(-5))
        told(lambda c: c.context.copy_(torch.tensor([1 << 30, 120])))
        told(lambda c: c.row_start.copy_(torch.tensor([0, 5 * new, 1 << 28])))
        told(lambda c: c.row_start.copy_(torch.tensor([-7, new, 2 * new])))
        c, out = told(lambda c: c.row_start.copy_(torch.tensor([new, 0, new])))
        if new > 1:
            c, out = told(lambda c: None, max_new=new - 1)
            assert bool((out[new - 1] == 5).all())
            c, out = told(lambda c: c.context.copy_(torch.tensor([new - 2, 120])))
            assert bool((out[:2] == 0).all())


# ---------------------------------------------------------------- new rows
def tables(be, n, hd):
    cos, sin = be.rope_table(hd, n, 1e6)
    return torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()


def append_reference(c, q, k, v, cos, sin, norm):
    """fp64 rows in the order of q, k, v, and each sequence's positions."""
    pos = torch.cat([torch.arange(x - n, x) for n, x in zip(c.new, c.ctx)]).cuda()

    def turned(x, heads, gamma):
        x = x.double().reshape(-1, heads, c.hd)
        if norm is not None:
            x = x / (x.square().mean(-1, keepdim=True) + norm[2]).sqrt() * gamma.double()
        h = c.hd // 2
        co, si = cos[pos].double()[:, None, :h], sin[pos].double()[:, None, :h]
        a, b = x[..., :h], x[..., h:]
        size = torch.cat([a.abs() * co.abs() + b.abs() * si.abs(), a.abs() * si.abs() + b.abs() * co.abs()], -1)
        return torch.cat([a * co - b * si, a * si + b * co], -1), size

    return turned(q, c.hq, norm and norm[0]), turned(k, c.hkv, norm and norm[1]), v.double().reshape(-1, c.hkv, c.hd), pos


def near(got, want, size, hd):
    """One rounding to the result's type; before it fp32 arithmetic: the mean of squares hd * 2^-24, root, quotient and three products 2^-24
    each of the terms, one sum."""
    t = torch.finfo(got.dtype)
    bound = t.eps / 2 * want.abs() + (1 + t.eps) * (hd + 8) * 2.0 ** -24 * size + t.tiny * t.eps
    assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads", HEADS + [(64, 8, 64), (40, 8, 128)])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("new,ctx", [([1] * 5, [1, 16, 17, 100, 64]), ([3, 0, 16, 40, 130], [3, 5, 48, 333, 131])])
def test_append(be, heads, dtype, norm, new, ctx):
    c = Case(new, ctx, heads, dtype, 16, seed=50, extra_rows=2)
    g = rng(51)
    width = (c.hq + 2 * c.hkv) * c.hd
    qkv = 3 * torch.randn(c.tokens, width + 4, generator=g, device="cuda")
    off = 0 if c.hd % 16 else 1  # rows that are not 16-byte aligned too
    qkv = qkv[:, off:off + width]
    q, k, v = qkv[:, :c.hq * c.hd], qkv[:, c.hq * c.hd:(c.hq + c.hkv) * c.hd], qkv[:, (c.hq + c.hkv) * c.hd:]
    nm = (1 + 0.2 * torch.randn(c.hd, generator=g, device="cuda"), 1 + 0.2 * torch.randn(c.hd, generator=g, device="cuda"), 1e-6) if norm else None
    cos, sin = tables(be, max(ctx), c.hd)
    before_k, before_v = c.k.clone(), c.v.clone()
    out = torch.full((c.tokens, c.hq, c.hd), 5.0, dtype=dtype, device="cuda")
    be.paged_append(q, k, v, c.k, c.v, c.table, c.row_start, c.context, max(new), cos, sin, qk_norm=nm, q_out=out)
    n = sum(new)
    (wq, sq), (wk, sk), wv, pos = append_reference(c, q[:n], k[:n], v[:n], cos, sin, nm)
    near(out[:n], wq, sq, c.hd)
    assert bool((out[n:] == 5).all())
    seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).cuda()
    page = c.table[seq, pos // 16].long()
    near(c.k[page, pos % 16], wk, sk, c.hd)
    assert torch.equal(c.v[page, pos % 16], wv.float().to(dtype))
    c.k[page, pos % 16], c.v[page, pos % 16] = before_k[page, pos % 16], before_v[page, pos % 16]
    assert torch.equal(c.k.view(torch.int16), before_k.view(torch.int16)) and torch.equal(c.v.view(torch.int16), before_v.view(torch.int16))


def test_append_tells_what_does_not_fit(be):
    be.check(be.lib().nntr_cuda_clear_device_status())
    for what in range(4):
        c = Case([2, 2], [40, 50], (8, 2, 64), F16, 16, seed=60, junk=1.0)
        cos, sin = tables(be, 50 if what else 45, 64)
        if what == 1:
            c.table[1, 3] = c.k.shape[0]
        if what == 2:
            c.context[0] = 1
        if what == 3:
            c.context[1] = 1 << 20
        qkv = torch.randn(4, 12 * 64, device="cuda")
        before = c.k.clone()
        out = be.paged_append(qkv[:, :512], qkv[:, 512:640], qkv[:, 640:], c.k, c.v, c.table, c.row_start, c.context, 2, cos, sin)
        with pytest.raises(ValueError):
            be.device_status()
        be.check(be.lib().nntr_cuda_clear_device_status())
        changed = int((c.k != before).flatten(1).any(1).sum())
        if what == 0:  # no row of the tables for the second sequence
            assert bool((out[2:] == 0).all()) and changed == 1
        if what == 1:
            assert changed == 1 and bool((out[2:] != 0).any())


# ------------------------------------------------------------ whole pages
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("layers,pages,page,hkv,hd,n", [(1, 4, 16, 1, 8, 1), (3, 40, 16, 2, 64, 11), (2, 9, 256, 8, 128, 4), (5, 33, 32, 3, 40, 16)])
def test_copy_pages(be, dtype, layers, pages, page, hkv, hd, n):
    kv = torch.randn(layers, 2, pages, page, hkv, hd, device="cuda").to(dtype)
    ids = torch.randperm(pages, device="cuda")
    dst, src = ids[:n].int(), ids[n:][torch.randint(pages - n, (n,), device="cuda")].int()
    want = kv.clone()
    want[:, :, dst.long()] = want[:, :, src.long()]
    be.copy_pages(kv, src, dst)
    assert torch.equal(kv, want)
    be.copy_pages(kv, src[:0], dst[:0])
    assert torch.equal(kv, want)


def test_copy_pages_leaves_out_what_is_not_there(be):
    be.check(be.lib().nntr_cuda_clear_device_status())
    kv = torch.randn(2, 2, 6, 16, 2, 64, device="cuda").to(F16)
    want = kv.clone()
    want[:, :, 3] = want[:, :, 1]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    be.copy_pages(kv, i32([1, 6, 0, -1]), i32([3, 2, 1 << 30, 4]))
    with pytest.raises(ValueError):
        be.device_status()
    be.check(be.lib().nntr_cuda_clear_device_status())
    assert torch.equal(kv, want)


def test_pages_beyond_two_gigabytes(be):
    kv = torch.zeros(1, 2, 9000, 256, 4, 128, dtype=F16, device="cuda")  # 2.4 GB a cache
    kv[0, 1, 8999] = 3
    be.copy_pages(kv, torch.tensor([8999], dtype=torch.int32, device="cuda"), torch.tensor([8998], dtype=torch.int32, device="cuda"))
    assert bool((kv[0, 1, 8998] == 3).all()) and bool((kv[0, 0, 8998] == 0).all()) and bool((kv[0, 1, 8997] == 0).all())


# ------------------------------------------------- a run of them together
def test_a_layer_prefilled_in_chunks_forked_and_decoded(be):
    """One attention layer over a cache in pages, as a server runs it: chunks of two prompts, a fork, single tokens of all three; against
    the formula over the rows as they were stored."""
    hq, hkv, hd, ps = 8, 2, 64, 16
    cache = be.PagedCache(2, 40, ps, hkv, hd)
    cos, sin = tables(be, 400, hd)
    g = rng(70)
    nm = tuple(1 + 0.1 * torch.randn(hd, generator=g, device="cuda") for _ in range(2)) + (1e-6,)
    stored = {}

    def step(seqs, new, layer=1):
        cache.reserve(seqs, new)
        b = cache.batch(seqs, new)
        qkv = torch.randn(sum(new), (hq + 2 * hkv) * hd, generator=g, device="cuda")
        q, k, v = qkv[:, :hq * hd], qkv[:, hq * hd:(hq + hkv) * hd], qkv[:, (hq + hkv) * hd:]
        kc, vc = cache.keys(layer), cache.values(layer)
        max_rows = b.pop("max_rows")
        qr = be.paged_append(q, k, v, kc, vc, **b, cos=cos, sin=sin, qk_norm=nm)
        out = torch.empty(sum(new), hq, hd, device="cuda")
        be.paged_attention(qr, kc, vc, **b, max_rows=max_rows, out=out)
        at = 0
        for s, n in zip(seqs, new):
            rows = torch.arange(cache.rows(s), device="cuda")
            pages = torch.tensor(cache.pages(s), device="cuda")[rows // ps]
            K, V = kc[pages, rows % ps], vc[pages, rows % ps]
            old = stored.get(s)
            if old is not None:  # what was there stays
                assert torch.equal(K[:old[0].shape[0]], old[0]) and torch.equal(V[:old[1].shape[0]], old[1])
            stored[s] = (K, V)
            c = Case.__new__(Case)
            c.new, c.ctx, c.hq, c.hkv, c.hd, c.dtype, c.starts, c.q, c.K, c.V = [n], [cache.rows(s)], hq, hkv, hd, F16, [0], qr[at:at + n], [K], [V]
            c.check(out[at:at + n])
            at += n

    a, b = cache.new(), cache.new()
    step([a, b], [33, 70])
    step([b, a], [64, 1])
    f, = cache.fork(b)
    stored[f] = stored[b]
    step([a, b, f], [1, 1, 1])
    step([f, a], [20, 2])
    cache.free(b)
    del stored[b]
    assert cache.compact() > 0
    step([a, f], [1, 1])
    assert bool((cache.kv[0] == 0).all())  # the other layer
    be.device_status()
