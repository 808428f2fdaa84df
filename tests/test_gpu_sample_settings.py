"""Sampling's settings at and outside the ends of their ranges: tokens are the definition's
(test_gpu_sample.one), with each setting as the kernel takes it."""
import math

import numpy as np
import pytest
import torch

from test_gpu_sample import TYPES, logits, one, sample

pytestmark = pytest.mark.gpu
LOWEST = torch.finfo(torch.float32).min


@pytest.mark.parametrize("temperature", [5e-324, 1e-310, 1e-300, 1e-45, 1e300])
def test_rows_of_the_lowest_number(temperature):
    """Equal logits weigh the same at any temperature; the lowest number has no next one below."""
    x = torch.full((5, 3000), LOWEST, device="cuda")
    x[1, 1000:] = -math.inf
    x[2, 7:9] = torch.nextafter(torch.tensor(LOWEST), torch.tensor(0.0)).item()
    x[3] = -3.0
    x[4, 1:] = -math.inf
    u = torch.tensor([0.6, 0.6, 0.6, 0.999, 0.5], device="cuda")
    for kw in (dict(), dict(top_k=100), dict(top_p=0.5), dict(top_k=2000, top_p=0.25), dict(min_p=0.5)):
        out = torch.full((5,), -9, dtype=torch.int64, device="cuda")
        sample(x, u, temperature, out=out, **kw)
        xs = x.double().cpu().numpy()
        want = []
        for r, a in zip(xs, u.double().tolist()):
            # far / t passes the doubles' range where t is small: the same weights, from the order alone
            with np.errstate(invalid="ignore", over="ignore"):
                far = np.where(r == r.max(), 0.0, np.where(r == -math.inf, -math.inf, (r - r.max()) / temperature))
            want.append(one(far, a, 1.0, kw.get("top_k", 0), kw.get("top_p", 1.0), kw.get("min_p", 0.0)))
        assert out.tolist() == want


@pytest.mark.parametrize("dtype", TYPES)
def test_a_tensors_settings_outside_their_ranges(dtype):
    """Numbers are refused there, a tensor's count as the nearest end, or as off."""
    n, v = 24, 4001
    x, u = logits(n, v, dtype, seed=6)
    x[::4, 100:200] = -math.inf
    inf, nan = math.inf, math.nan
    taken = [  # name, as given, as taken
        ("temperature", -1.0, 0.0), ("temperature", nan, 0.0), ("temperature", -inf, 0.0), ("temperature", inf, inf),
        ("top_p", -0.5, 0.0), ("top_p", 1.5, 1.0), ("top_p", nan, 1.0), ("top_p", inf, 1.0), ("top_p", -inf, 0.0),
        ("min_p", -0.5, 0.0), ("min_p", 1.5, 1.0), ("min_p", nan, 0.0), ("min_p", inf, 1.0), ("min_p", -inf, 0.0),
        ("top_k", -3, 0), ("top_k", -2 ** 31, 0), ("top_k", 2 ** 31 - 1, 0)]
    rows = x.double().cpu().numpy()
    for name, given, as_taken in taken:
        base = dict(temperature=0.8, top_k=600, top_p=0.9, min_p=0.01)
        if name != "min_p":
            base["min_p"] = 0.0
        t = torch.full((n,), given, dtype=torch.int32 if name == "top_k" else torch.float32, device="cuda")
        got = sample(x, u, **{**base, name: t}).tolist()
        s = {**base, name: as_taken}
        want = [one(r, a, s["temperature"], int(s["top_k"]), s["top_p"], s["min_p"]) for r, a in zip(rows, u.double().tolist())]
        assert got == want, (name, given)


def test_random_numbers_outside_their_range():
    x, _ = logits(1, 700, torch.float32, seed=1)
    x = x.expand(6, -1)
    u = torch.tensor([0.0, -1.0, math.nan, 1.0 - 2.0 ** -24, 1.0, math.inf], device="cuda")
    got = sample(x, u, 1.0, 50).tolist()
    kept = torch.topk(x[0], 50).indices
    assert got[0] == got[1] == got[2] == int(kept.min()) and got[4] == got[5] == int(kept.max())
    assert got[3] in kept.tolist()


def test_a_number_is_a_64_bit_float():
    """0.9 of 2500 equal logits are 2250, which the float32 nearest to 0.9 passes."""
    x, u = torch.zeros(1, 2500, device="cuda"), torch.full((1,), 1 - 2.0 ** -24, device="cuda")
    as_tensor = torch.full((1,), 0.9, device="cuda")
    p = float(as_tensor)
    count = {q: int(np.searchsorted(np.arange(1, 2501), np.longdouble(q) * 2500)) + 1 for q in (0.9, p)}
    assert int(sample(x, u, top_p=0.9)) == count[0.9] - 1
    assert int(sample(x, u, top_p=as_tensor)) == count[p] - 1


def test_numbers_outside_their_ranges_are_refused():
    x, u = logits(2, 50, torch.float32)
    for bad in (dict(temperature=math.inf), dict(temperature=-math.inf), dict(top_p=math.nan), dict(min_p=math.nan),
                dict(min_p=-0.1), dict(top_p=math.inf)):
        with pytest.raises(ValueError):
            sample(x, u, **bad)
