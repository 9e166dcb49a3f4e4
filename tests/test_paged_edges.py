"""Attention over a cache in pages and appends to it where a promise ends: scores that rise late, masked values of any size, keys that are not
numbers, pages that nobody needs, contexts that no sequence can have. Bounds: those of test_paged_gpu."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_paged_gpu import BF16, F16, Case, be, tables  # noqa: E402, F401

I32 = torch.int32


def put(c, b, row, k=None, v=None):
    """Another key or value (of every kv head) in row `row` of sequence b."""
    page = int(c.table[b, row // c.page])
    for new, flat, cache in ((k, c.K, c.k), (v, c.V, c.v)):
        if new is not None:
            flat[b][row] = new
            cache[page, row % c.page] = flat[b][row]


LOW = -2 ** 31


@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("context", [LOW, LOW + 1, LOW + 49, -1, -2 ** 30])
def test_negative_contexts_see_nothing_and_are_told(be, new, context):
    be.check(be.lib().nntr_cuda_clear_device_status())
    c = Case([new, new], [100, 120], (8, 2, 64), F16, 16, seed=84, junk=0.0)
    good = c.attend(be)
    c.context[0] = context
    out = torch.full((c.tokens, 8, 64), 5.0, dtype=F16, device="cuda")
    c.attend(be, out=out)
    with pytest.raises(ValueError):
        be.device_status()
    be.check(be.lib().nntr_cuda_clear_device_status())
    assert bool((out[:new] == 0).all()) and torch.equal(out[new:], good[new:])
    cos, sin = tables(be, 120, 64)
    qkv = torch.randn(c.tokens, 12 * 64, device="cuda")
    k, v = c.k.clone(), c.v.clone()
    q = be.paged_append(qkv[:, :512], qkv[:, 512:640], qkv[:, 640:], k, v, c.table, c.row_start, c.context, new, cos, sin)
    with pytest.raises(ValueError):
        be.device_status()
    be.check(be.lib().nntr_cuda_clear_device_status())
    assert bool((q[:new] == 0).all())
    own = c.table[0, :-(-100 // 16)].long()
    assert torch.equal(k[own], c.k[own]) and torch.equal(v[own], c.v[own])  # nothing of the first sequence is stored


def late_peak(height, heads, dtype, new, batch=16, late=128):
    """Flat scores but for one query row of each sequence, which has one key `height` (natural units) above all others: row `late` + b of
    sequence b."""
    c = Case([new] * batch, [400 + new] * batch, heads, dtype, 64, seed=80)
    c.q[:] = 0
    along = math.sqrt(height * math.sqrt(c.hd))
    for b in range(batch):
        c.K[b][:, :, 0] = 0
        for r in range(0, c.ctx[b], c.page):
            rows = c.K[b][r:r + c.page]
            c.k[int(c.table[b, r // c.page]), :rows.shape[0]] = rows
        key = c.K[b][late + b].clone()
        key[:, 0] = along
        put(c, b, late + b, k=key)
        c.q[c.starts[b] + 5 * b % new, b % c.hq, 0] = along
    return c


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads", [(2, 1, 64), (4, 2, 128), (2, 1, 96)])
@pytest.mark.parametrize("new", [1, 64, 128])
@pytest.mark.parametrize("height", [20, 60, 80, 84, 85, 86, 90, 95, 100, 130, 177, 200, 260, 300, 420, 600])
def test_one_score_that_rises_late_and_alone(be, height, new, heads, dtype):
    """At every place modulo 16 of a step whose rows all see everything, far above what the row's maximum was taken from."""
    c = late_peak(height, heads, dtype, new)
    c.check(c.attend(be))
    c.check(c.attend(be, max_rows=64))  # not cut into parts


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads", [(2, 1, 64), (4, 1, 128)])
@pytest.mark.parametrize("new", [2, 9, 40, 128])
def test_values_out_of_sight_have_no_effect_whatever_their_size(be, new, heads, dtype):
    """The last row is seen by the last query alone, row 100 by the first one alone (the window's begin): the others' results keep their bits."""
    c = Case([new], [300], heads, dtype, 32, seed=81)
    window = 300 - new + 1 - 100
    want = c.attend(be, window=window)
    for sign in (1, -1):
        for row in (299, 100):
            put(c, 0, row, v=sign * torch.finfo(dtype).max)
        assert torch.equal(c.attend(be, window=window)[1:-1], want[1:-1])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads", [(2, 1, 64), (4, 1, 128)])
@pytest.mark.parametrize("new", [1, 64, 128])
@pytest.mark.parametrize("at", [0, 130, 270])
def test_a_key_that_is_no_number_shows(be, at, new, heads, dtype):
    """Wherever it lies in a step: the results of the queries that see it are not finite (those of 128 new tokens in front of it do not)."""
    c = Case([new] * 16, [400] * 16, heads, dtype, 16, seed=82)
    for b in range(16):
        put(c, b, at + b, k=math.nan)
    sees = torch.arange(400 - new, 400, device="cuda") >= at + torch.arange(16, device="cuda")[:, None]
    for out in (c.attend(be), c.attend(be, max_rows=64)):
        assert torch.equal(torch.isfinite(out).view(16, new, -1), ~sees[..., None].expand(16, new, c.hq * c.hd))
    c = Case([new] * 16, [400] * 16, heads, dtype, 16, seed=82)
    want = c.attend(be)
    for b in range(16):
        put(c, b, 399, k=math.nan)  # the last query's own row
    got = c.attend(be).view(16, new, -1)
    assert torch.equal(got[:, :-1], want.view(16, new, -1)[:, :-1]) and not bool(torch.isfinite(got[:, -1]).any())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads", [(2, 1, 64), (4, 2, 128)])
@pytest.mark.parametrize("new", [1, 64])
@pytest.mark.parametrize("height", [5, 30, 60, 66])
def test_large_values_behind_a_score_that_rises_late(be, height, new, heads, dtype):
    """Weights refer to a maximum that was taken before the score rose: their products with the values stay inside fp32."""
    c = late_peak(height, heads, dtype, new)
    for b in range(16):
        put(c, b, 128 + b, v=1e12 if dtype == BF16 else 6e4)
    c.check(c.attend(be))
    c.check(c.attend(be, max_rows=64))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads", [(2, 1, 64), (8, 1, 128)])
@pytest.mark.parametrize("ctx", [1, 2, 17, 40])
@pytest.mark.parametrize("kind", ["nan", "inf"])
def test_nothing_but_keys_that_are_no_numbers_shows(be, kind, ctx, heads, dtype):
    """A row that has no finite score at all, or whose score is +inf; the sequence beside it is not affected."""
    c = Case([1, 1], [ctx, 60], heads, dtype, 16, seed=85)
    c.q[:, :, 0] = 1
    want = c.attend(be)[1]
    for r in range(ctx):
        k = c.K[0][r].clone()
        k[:, 0] = math.nan if kind == "nan" else math.inf
        put(c, 0, r, k=k)
    for kw in (dict(), dict(sink=c.sinks), dict(max_rows=1)):
        out = c.attend(be, **kw)
        assert bool(torch.isnan(out[0]).all()) and (kw.get("sink") is not None or torch.equal(out[1], want))


@pytest.mark.parametrize("page", [16, 32, 64, 256])
@pytest.mark.parametrize("new", [1, 20, 65, 200])
@pytest.mark.parametrize("window,first", [(100, 4), (100, 0), (33, 40), (300, 1)])
def test_pages_that_nobody_sees_may_be_given_back(be, window, first, new, page):
    """Page table entries of -1 between the first tokens and the window are no contradiction."""
    be.check(be.lib().nntr_cuda_clear_device_status())
    c = Case([new, new, 1], [1500, 1111, 900], (8, 2, 64), F16, page, seed=83)
    kw = dict(window=window, first_tokens=first)
    gone = 0
    for b, (n, ctx) in enumerate(zip(c.new, c.ctx)):
        oldest = max(0, ctx - n - window + 1)
        for slot in range(-(-ctx // page)):
            if (slot + 1) * page <= oldest and slot * page >= min(first, oldest):
                c.table[b, slot] = -1
                gone += 1
    assert gone > 0
    c.check(c.attend(be, **kw), **kw)
    be.device_status()


@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("pad", [0, 40, 300])
@pytest.mark.parametrize("what", ["backwards", "behind", "negative", "too many", "fewer rows", "no rows, negative", "none"])
def test_append_tells_what_attention_tells(be, what, pad, new):
    """Contradictions of sequences that no token belongs to, too, wherever they stand among sequences of padding."""
    be.check(be.lib().nntr_cuda_clear_device_status())
    c = Case([new, new], [100, 120], (8, 2, 64), F16, 16, seed=86, extra_rows=3, junk=0.0)
    cos, sin = tables(be, 120, 64)
    start, context = c.row_start.tolist() + [2 * new] * pad, [100, 120] + [0] * pad
    table = torch.cat([c.table, torch.full((pad, c.table.shape[1]), -1, dtype=I32, device="cuda")])
    if what == "backwards":
        start[:3] = [new, 0, 2 * new]
    elif what == "behind":
        start[-1] = c.tokens + 1
    elif what == "negative":
        start[0] = -7
    elif what == "too many":
        start[1] += 1
    elif what == "fewer rows":
        context[0] = new - 1
    elif what == "no rows, negative":
        start, context, table = start + [start[-1]], context + [-1], torch.cat([table, table[:1]])
    start, context = (torch.tensor(v, dtype=I32, device="cuda") for v in (start, context))
    qkv = torch.randn(c.tokens, 12 * 64, device="cuda")

    def told():
        if what == "none":
            return be.device_status()
        with pytest.raises(ValueError):
            be.device_status()
        be.check(be.lib().nntr_cuda_clear_device_status())

    be.paged_attention(c.q, c.k, c.v, table, start, context, new)
    told()
    be.paged_append(qkv[:, :512], qkv[:, 512:640], qkv[:, 640:], c.k, c.v, table, start, context, new, cos, sin)
    told()
