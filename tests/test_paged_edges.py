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
