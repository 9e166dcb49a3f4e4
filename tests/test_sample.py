"""Sampling with temperature, top-k, top-p and min-p: the indices equal those of the definition in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from nntrainer_b200 import backend, build
    build.build()
    backend.init(0)
    return backend


def reference(x, u, t=1.0, k=0, p=1.0, m=0.0):
    """(index, probability, distance of the draw and of the cut from the nearest border) of one row, in 64 bits."""
    x = x.double().cpu()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    n = x.numel()
    top = x.max()
    if top == -math.inf:
        return 0, 0.0, 1.0
    if not t > 0:
        t, k = 1.0, 1
    if not p > 0:
        k = 1
    z = torch.where(x == top, torch.zeros_like(x), (x - top) / t)
    w = z.exp()
    order = torch.sort(x, descending=True, stable=True).indices
    order = order[x[order] > -math.inf]
    if 0 < k < n:
        order = order[:k]
    ws = w[order]
    cum = ws.cumsum(0)
    slack = 1.0
    if p < 1:
        goal = p * cum[-1]
        keep = cum - ws < goal
        slack = float(((cum - goal).abs() / cum[-1]).min())
        order = order[keep | (torch.arange(order.numel()) == 0)]
    order = order[(w[order] >= m) | (x[order] == top)]
    kept = torch.sort(order).values
    cum = w[kept].cumsum(0)
    goal = float(u) * cum[-1]
    at = min(int((cum <= goal).sum()), kept.numel() - 1)
    slack = min(slack, float(((cum - goal).abs() / cum[-1]).min()))
    return int(kept[at]), float(w[kept[at]] / cum[-1]), slack


def check(be, x, u, **kw):
    names = dict(t="temperature", k="top_k", p="top_p", m="min_p")
    idx, idx_f, prob = be.sample(x, u, **{names[a]: b for a, b in kw.items()})
    for r in range(x.shape[0]):
        i, pr, slack = reference(x[r], u[r], **kw)
        # A weight is a multiple of 2^-44, the greatest one 1, others are off by less than 2^-44 for that: over n of them no sum is off by more
        # than n * 2^-44. In fp32 the exponent is off by 2^-26 for its rounding and as much for the sum of its two parts, the polynomial by
        # 2^-28.9, its last step and the conversion to 24 bits by 2^-24 each: less than 2^-22 of them in all, of a sum that is no smaller.
        # A border is one sum over another.
        off = 2 * (2.0 ** -22 + x.shape[1] * 2.0 ** -44)
        if slack > off:
            assert int(idx[r]) == i == int(idx_f[r]), (r, kw, slack)
            assert abs(float(prob[r]) - pr) <= pr * (2.0 ** -23 + off) + 1e-38
    return idx


FILTERS = [dict(), dict(t=0.7), dict(k=1), dict(k=5), dict(k=50, t=1.3), dict(k=2000), dict(p=0.9), dict(p=0.5, t=0.6), dict(p=1e-6), dict(p=0.9999),
           dict(m=0.05), dict(m=1.0), dict(k=40, p=0.95), dict(k=40, p=0.8, m=0.1, t=0.8), dict(t=0.0), dict(p=0.0), dict(t=5.0, p=0.97), dict(t=0.05),
           dict(k=20000), dict(k=20000, p=0.9), dict(k=500, p=0.5, t=0.8), dict(k=200, p=0.7, m=1e-3), dict(k=900, p=0.99), dict(p=0.99, m=1e-4), dict(m=1e-6), dict(t=1e-20), dict(t=1e20)]


@pytest.mark.parametrize("kw", FILTERS)
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 2), (2, 31), (4, 257), (3, 1000), (3, 6144), (4, 9000), (2, 32000), (5, 50257), (2, 151936)])
def test_against_the_definition(be, rows, n, kw):
    g = torch.Generator(device="cuda").manual_seed(rows * n)
    x = 2 * torch.randn(rows, n, generator=g, device="cuda")
    x.scatter_add_(1, torch.randint(n, (rows, 12), generator=g, device="cuda"), 6 * torch.rand(rows, 12, generator=g, device="cuda"))
    check(be, x, torch.rand(rows, generator=g, device="cuda"), **kw)


@pytest.mark.parametrize("kw", FILTERS)
def test_many_rows_and_flat_rows(be, kw):
    g = torch.Generator(device="cuda").manual_seed(3)
    check(be, torch.randn(200, 3001, generator=g, device="cuda"), torch.rand(200, generator=g, device="cuda"), **kw)
    check(be, 1e-3 * torch.randn(3, 130001, generator=g, device="cuda"), torch.rand(3, generator=g, device="cuda"), **kw)


@pytest.mark.parametrize("kw", FILTERS)
def test_ties_go_to_the_lowest_index(be, kw):
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randint(-3, 4, (40, 5000), generator=g, device="cuda").float()  # hundreds of equal logits at every border
    x[0] = 1.0
    x[1, ::2] = -0.0
    check(be, x, torch.rand(40, generator=g, device="cuda"), **kw)


@pytest.mark.parametrize("kw", FILTERS)
def test_what_is_masked_is_never_drawn(be, kw):
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(12, 4000, generator=g, device="cuda")
    x[:, torch.randperm(4000, device="cuda")[:3900]] = -math.inf
    x[1, :] = -math.inf
    x[2, :] = math.nan
    x[3, 1:] = -math.inf
    x[4, :-1] = math.nan
    x[5, 100:200] = math.inf
    x[6, 7] = math.inf
    x[7] = torch.finfo(torch.float32).min
    x[8, :2000] = torch.finfo(torch.float32).min
    x[9] *= 1e30
    idx = check(be, x, torch.rand(12, generator=g, device="cuda"), **kw)
    assert int(idx[1]) == 0 and int(idx[2]) == 0 and int(idx[3]) == 0 and int(idx[6]) == 7


def test_the_ends_of_the_random_numbers(be):
    x = torch.tensor([[0.0, 1.0, -math.inf, 2.0, 0.5]], device="cuda").repeat(4, 1)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 1e-30], device="cuda")
    assert be.sample(x, u)[0].tolist() == [0, 4, 4, 0]
    assert be.sample(x, u, top_k=2)[0].tolist() == [1, 3, 3, 1]


def test_parameters_of_each_row(be):
    g = torch.Generator(device="cuda").manual_seed(6)
    sets = [dict(t=0.7), dict(t=0.0), dict(k=3.0), dict(p=0.8), dict(m=0.2), dict(t=1.2, k=30.0, p=0.9, m=0.01), dict(p=0.0), dict()]
    x = 3 * torch.randn(len(sets), 9001, generator=g, device="cuda")
    u = torch.rand(len(sets), generator=g, device="cuda")
    rows = torch.tensor([[s.get("t", 1.0), s.get("k", 0.0), s.get("p", 1.0), s.get("m", 0.0)] for s in sets], device="cuda")
    idx, _, prob = be.sample(x, u, params=rows)
    for r, s in enumerate(sets):
        s = {a: float(torch.tensor(b, dtype=torch.float32)) for a, b in s.items()}  # as the rows hold them
        want = be.sample(x[r:r + 1], u[r:r + 1], s.get("t", 1.0), int(s.get("k", 0)), s.get("p", 1.0), s.get("m", 0.0))
        assert int(idx[r]) == int(want[0]) and float(prob[r]) == float(want[2])


def test_strided_rows_and_given_results(be):
    g = torch.Generator(device="cuda").manual_seed(7)
    wide = torch.randn(6, 5011, generator=g, device="cuda")
    x = wide[:, 3:3 + 5000]
    u = torch.rand(6, generator=g, device="cuda")
    out = (torch.zeros(6, dtype=torch.int32, device="cuda"), torch.zeros(6, device="cuda"), torch.zeros(6, device="cuda"))
    got = be.sample(x, u, 0.8, 100, 0.9, out=out)
    assert got[0] is out[0]
    want = be.sample(x.contiguous(), u, 0.8, 100, 0.9)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_counts_beyond_32_bits_and_the_least_temperature(be):
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(5, 9000, generator=g, device="cuda")
    u = torch.rand(5, generator=g, device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(be.sample(x, u, top_k=2 ** 32 + 1), be.sample(x, u)))
    assert torch.equal(be.sample(x, u, temperature=5e-324, top_p=0.9)[0].long(), x.argmax(1))


def test_greedy_is_the_argmax(be):
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randint(0, 50, (30, 7000), generator=g, device="cuda").float()
    u = torch.rand(30, generator=g, device="cuda")
    assert torch.equal(be.sample(x, u, temperature=0.0)[0], be.argmax(x)[0])


def test_frequencies(be):
    """Of 40000 evenly spread random numbers each token gets its share, one more or less."""
    x = torch.tensor([0.3, -1.0, 2.0, 0.0, -math.inf, 1.0], device="cuda").repeat(40000, 1)
    u = (torch.arange(40000, device="cuda") + 0.5) / 40000
    n = torch.bincount(be.sample(x, u, 0.9)[0].long(), minlength=6).double()
    want = torch.softmax(x[0].double() / 0.9, 0) * 40000
    assert bool(((n - want).abs() <= 1.5).all())


def test_captured_and_replayed(be):
    g = torch.Generator(device="cuda").manual_seed(9)
    x, u = torch.randn(3, 40000, generator=g, device="cuda"), torch.rand(3, generator=g, device="cuda")
    out = (torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda"))
    be.sample(x, u, 0.9, 0, 0.8, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        be.sample(x, u, 0.9, 0, 0.8, out=out)
    for _ in range(3):
        x.normal_(generator=g)
        u.uniform_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        for r in range(3):
            assert int(out[0][r]) == reference(x[r], u[r], t=0.9, p=0.8)[0]
