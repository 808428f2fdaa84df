"""Sampling's settings at the ends of their ranges: tokens are the definition's."""
import math

import numpy as np
import pytest
import torch

from test_gpu_sample import one, sample

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
