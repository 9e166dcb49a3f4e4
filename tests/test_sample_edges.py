"""Sampling at the ends of its range: the smallest temperatures, the most logits."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_sample import be, check  # noqa: E402, F401


@pytest.mark.parametrize("kw", [dict(), dict(k=40), dict(p=0.9), dict(m=0.1), dict(k=40, p=0.9, m=0.1), dict(k=3000, p=0.99)])
@pytest.mark.parametrize("n", [100, 5000, 9000, 151936])
def test_the_smallest_temperatures_with_a_greatest_logit_of_zero(be, n, kw):
    """Logits less their maximum, as log-probabilities may be given: the other weights are zero, whatever their bits."""
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(4, n, generator=g, device="cuda")
    x -= x.amax(1, keepdim=True)
    x[3, n // 3] = x[3, n - 1] = 0.0  # three of the greatest there
    u = torch.tensor([0.1, 0.5, 0.9, 0.99], device="cuda")
    for t in (1e-300, 1e-100, 1e-45, 1e-40, 3e-39, 1e-38, 1e-30):
        idx = check(be, x, u, t=t, **kw)
        assert torch.equal(idx[:3].long(), x[:3].argmax(1))
    rows = torch.tensor([[1e-40, kw.get("k", 0), kw.get("p", 1.0), kw.get("m", 0.0)]] * 4, device="cuda")
    assert torch.equal(be.sample(x, u, params=rows)[0], check(be, x, u, t=float(rows[0, 0]), **kw))


N = 1 << 20


@pytest.mark.parametrize("rows", [1, 3, 160])
def test_as_many_equal_weights_as_there_can_be(be, rows):
    """2^20 logits of the greatest weight: their sum is the first one that 64 bits do not hold. With equal weights the token is the number of
    whole shares below u, without rounding: u is a multiple of 2^-21."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    i = torch.randint(N, (rows,), generator=g, device="cuda")
    i[0] = N - 1
    u = ((i.double() + 0.5) / N).float()
    assert torch.equal(u.double() * N, i.double() + 0.5)
    flat = torch.full((rows, N), 1.25, device="cuda")
    near = torch.rand(rows, N, generator=g, device="cuda")  # other values, but at this temperature the same weights
    for x, t in ((flat, 1.0), (near, 1e30)):
        idx, idx_f, prob = be.sample(x, u, t)
        assert torch.equal(idx.long(), i) and torch.equal(idx_f.long(), i) and bool((prob == 1 / N).all())
    for p in (0.5, 0.25):  # the lowest indices are kept
        idx, _, prob = be.sample(flat, u, 1.0, 0, p)
        assert torch.equal(idx.long(), (i.double() * p + 0.5 * p).long()) and bool((prob == 1 / (p * N)).all())
    idx, _, prob = be.sample(flat, u, 1.0, 0, 1 - 2.0 ** -53)
    assert torch.equal(idx.long(), i) and bool((prob == 1 / N).all())
    idx, _, prob = be.sample(near, u, 1e30, 0, 0.5)
    kept = near.argsort(dim=1, descending=True, stable=True)[:, :N // 2].sort(1).values
    assert torch.equal(idx.long(), kept.gather(1, (i // 2)[:, None])[:, 0]) and bool((prob == 2 / N).all())
    assert bool((be.sample(flat, torch.ones_like(u))[0] == N - 1).all())
    assert bool((be.sample(flat, torch.zeros_like(u))[0] == 0).all())
