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
