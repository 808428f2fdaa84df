"""Sampling against the definition in 64 bits (and wider sums): tokens are equal. A random
number within 2^-30 of a border of the running sum, and settings within that of a border of
theirs, would make a case that proves nothing either way; the fixed seeds have none."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def sample(*args, **kw):
    import zipserv_asplos26_b200
    return zipserv_asplos26_b200.sample(*args, **kw)


def one(x, u, t, k, p, m):
    """The definition for one row of float64 logits."""
    if np.isnan(x).any() or x.max() == -math.inf:
        return -1
    if not t > 0:
        return int(x.argmax())
    v = len(x)
    order = np.lexsort((np.arange(v), -x))[:k if k > 0 else v]
    with np.errstate(invalid="ignore"):
        w = np.exp((x[order] - x[order[0]]) / t)
    w[x[order] == x[order[0]]] = 1.0
    w[np.isnan(w)] = 0.0                          # -inf next to +inf
    sums = np.add.accumulate(w.astype(np.longdouble))
    count = len(w) if p >= 1 else int(np.searchsorted(sums, np.longdouble(p) * sums[-1])) + 1
    count = max(1, min(count, int((w >= m).sum())))
    some = order[:count]
    by_index = np.argsort(some)
    sums = np.add.accumulate(w[:count][by_index].astype(np.longdouble))
    return int(some[by_index][min(count - 1, int(np.searchsorted(sums, np.longdouble(u) * sums[-1], side="right")))])


def check(x, u, t=1.0, k=0, p=1.0, m=0.0):
    n = x.shape[0]
    got = sample(x, u, t, k, p, m).tolist()

    def rows(s):
        return s.double().cpu().numpy() if torch.is_tensor(s) else np.full(n, float(s))

    want = [one(r, a, b, int(c), d, e) for r, a, b, c, d, e in
            zip(x.double().cpu().numpy(), rows(u), rows(t), rows(k), rows(p), rows(m))]
    assert got == want
    return got


def logits(n, v, dtype, seed=0, scale=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, v, device="cuda", generator=g) * scale
    x.scatter_add_(1, torch.randint(0, v, (n, 8), device="cuda", generator=g), torch.rand(n, 8, device="cuda", generator=g) * 8)
    return x.to(dtype), torch.rand(n, device="cuda", generator=g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v", [(1, 1), (3, 2), (5, 33), (2, 1024), (2, 1025), (7, 4099), (40, 32000), (3, 131071), (150, 8200)])
@pytest.mark.parametrize("t,k,p,m", [(1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 1000, 0.95, 0.0),
                                     (0.8, 0, 1.0, 0.05), (2.0, 700, 0.8, 0.01), (1.0, 0, 0.999, 0.0)])
def test_against_the_definition(dtype, n, v, t, k, p, m):
    x, u = logits(n, v, dtype, seed=n + v)
    check(x, u, t, k, p, m)


@pytest.mark.parametrize("dtype", TYPES)
def test_settings_of_each_row(dtype):
    n, v = 64, 5003
    x, u = logits(n, v, dtype, seed=4)
    rng = np.random.default_rng(1)

    def pick(values, kind):
        return torch.tensor(rng.choice(values, n), dtype=kind, device="cuda")

    check(x, u, pick([0.0, 0.5, 1.0, 1.7], torch.float32), pick([0, 1, 2, 40, 5002, 5003, 9999], torch.int32),
          pick([0.0, 0.3, 0.9, 1.0], torch.float32), pick([0.0, 0.02, 0.3, 1.0], torch.float32))


@pytest.mark.parametrize("dtype", TYPES)
def test_ties_go_to_the_lowest_index(dtype):
    """Few values, many of each: borders in the middle of equal ones, both zeros equal."""
    v = 3001
    g = torch.Generator(device="cuda").manual_seed(3)
    values = torch.tensor([-2.0, -1.0, -0.0, 0.0, 0.5, 1.0], device="cuda")
    x = values[torch.randint(0, 6, (24, v), device="cuda", generator=g)].to(dtype)
    u = torch.rand(24, device="cuda", generator=g)
    u[0], u[1], u[2] = 0.0, 1 - 2.0 ** -24, 0.5
    for k in (0, 1, 2, 400, 501, 1200, 2999):
        for p in (1.0, 0.5, 0.1, 1e-6):
            check(x, u, 1.0, k, p)
    flat = torch.zeros(4, v, device="cuda", dtype=dtype)
    assert check(flat, torch.tensor([0.0, 0.25, 0.5, 1 - 2.0 ** -24], device="cuda"), 1.0, 0, 1.0)[0] == 0
    assert max(check(flat, u[:4], 1.0, 10)) < 10
    assert check(flat, u[:4], 0.0) == [0] * 4


def test_masked_infinite_and_odd_rows():
    v = 2500
    x, u = logits(9, v, torch.float32, seed=8)
    x[0, 5:] = -math.inf
    x[1, :] = -math.inf
    x[1, 2222] = -3.0
    x[2, :] = -math.inf
    x[3, 77] = math.nan
    x[4, [10, 900, 2400]] = math.inf
    x[4, 11] = -math.inf
    x[5, :] = torch.finfo(torch.float32).min
    x[6, ::2] = torch.finfo(torch.float32).min
    x[7, 3] = math.inf
    x[8, :] = torch.nextafter(torch.tensor(1.0), torch.tensor(2.0)).item()
    x[8, 1000] = 1.0
    for kw in (dict(), dict(k=3), dict(p=0.9), dict(k=2000, p=0.5), dict(m=0.5), dict(t=0.0), dict(t=1e-30), dict(t=1e30)):
        got = check(x, u, **kw)
        assert got[0] < 5 and got[1] == 2222 and got[2] == got[3] == -1 and got[4] in (10, 900, 2400) and got[7] == 3
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    sample(x[4:], u[4:], err=err)
    assert int(err) == 0
    sample(x, u, err=err)
    assert int(err) == 8


def test_many_magnitudes():
    """Logits over all exponents, close ones among them: each digit of the order counts."""
    g = torch.Generator(device="cuda").manual_seed(1)
    bits = torch.randint(0, 2 ** 32, (16, 4000), device="cuda", generator=g).to(torch.int64)
    x = (bits - (bits >= 2 ** 31) * 2 ** 32).to(torch.int32).view(torch.float32)
    x = torch.where(x.isnan(), torch.zeros_like(x), x).clamp(-30, 30)
    base = torch.tensor(7.0, device="cuda").view(torch.int32)
    x[8:] = (base + torch.randint(0, 300, (8, 4000), device="cuda", generator=g, dtype=torch.int32)).view(torch.float32)
    u = torch.rand(16, device="cuda", generator=g)
    for k, p in ((0, 1.0), (100, 1.0), (0, 0.37), (777, 0.6), (3999, 0.99)):
        check(x, u, 1.0, k, p)


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_rows_and_batches(dtype):
    """Rows of any alignment; a row's token is the same alone, in any batch, and any time."""
    big, u = logits(12, 4111, dtype, seed=2)
    whole = sample(big, u, 0.9, 300, 0.9)
    for start, width in ((0, 4111), (1, 4000), (3, 4096), (8, 4103)):
        part = big[:, start:start + width]
        got = sample(part, u, 0.9, 300, 0.9)
        assert torch.equal(got, sample(part.contiguous(), u, 0.9, 300, 0.9))
        assert got.tolist() == [int(sample(part[i:i + 1], u[i:i + 1], 0.9, 300, 0.9)) for i in range(12)]
    many = big.repeat(40, 1)                                   # other clusters
    assert torch.equal(sample(many, u.repeat(40), 0.9, 300, 0.9), whole.repeat(40))
    assert torch.equal(sample(big[::3], u[::3].contiguous(), 0.9, 300, 0.9), whole[::3])
    assert torch.equal(sample(big[:1].expand(5, -1), u[:1].expand(5).contiguous(), 0.9), sample(big[:1], u[:1], 0.9).expand(5))
    assert sample(big[:0], u[:0]).shape == (0,)


def test_the_largest_vocabulary():
    x, u = logits(2, 1 << 20, torch.float32, seed=5)
    for k, p in ((0, 1.0), (0, 0.98), (200000, 0.5)):
        check(x, u, 1.0, k, p)


def test_frequencies():
    """Evenly spaced random numbers find each token as often as its weight says, within one."""
    w = torch.tensor([0.5, 0.0, 0.125, 0.25, 0.0625, 0.0625])
    x = w.log().cuda().expand(4096, 6).contiguous()
    u = (torch.arange(4096, device="cuda") + 0.5) / 4096
    counts = torch.bincount(sample(x, u), minlength=6).cpu()
    assert int((counts - w * 4096).abs().max()) <= 1


def test_graph_streams_and_out():
    x, u = logits(6, 32000, torch.bfloat16, seed=3)
    k = torch.full((6,), 40, dtype=torch.int32, device="cuda")
    out = torch.full((6,), -7, dtype=torch.int64, device="cuda")
    want = sample(x, u, 0.8, k, 0.95)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert sample(x, u, 0.8, k, 0.95, out=out) is out
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sample(x, u, 0.8, k, 0.95, out=out)
    for seed in range(3):
        a, b = logits(6, 32000, torch.bfloat16, seed=10 + seed)
        x.copy_(a)
        u.copy_(b)
        k.fill_(5 + seed)
        graph.replay()
        assert torch.equal(out, sample(a, b, 0.8, 5 + seed, 0.95))


def test_refusals():
    x, u = logits(3, 100, torch.float32)
    k = torch.zeros(3, dtype=torch.int32, device="cuda")
    for bad in (dict(logits=x.double()), dict(logits=x[0]), dict(logits=x.cpu()), dict(logits=x.t()), dict(u=u[:2].contiguous()),
                dict(u=u.double()), dict(temperature=-1.0), dict(temperature=math.nan), dict(top_k=-1), dict(top_k=k.long()),
                dict(top_p=1.5), dict(top_p=-0.1), dict(min_p=2.0), dict(min_p=u[:1].contiguous()), dict(out=k),
                dict(logits=torch.zeros(1, (1 << 20) + 1, device="cuda"), u=u[:1].contiguous()), dict(logits=x[:, :0])):
        with pytest.raises(ValueError):
            sample(**{**dict(logits=x, u=u), **bad})
    with pytest.raises(TypeError):
        sample(x, u, top_k=1.5)
