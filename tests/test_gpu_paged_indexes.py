"""Bad indexes of the paged cache, each in a call of its own: skipped, and flagged with bit 2."""
import pytest
import torch

from test_gpu_paged import BF, DEV, i32, pool, zs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("slot,flagged", [(0, 0), (31, 0), (-1, 0), (-2, 2), (-16, 2), (-2 ** 40, 2), (32, 2), (2 ** 40, 2)])
def test_a_slot_outside_the_pool(slot, flagged):
    q, k, v = (torch.randn(1, h, 64, device=DEV).to(BF) for h in (2, 1, 1))
    kp, vp = pool(2, 16, 1, 64, BF, "heads"), pool(2, 16, 1, 64, BF, "heads")
    cs = torch.cat([torch.ones(1, 32, device=DEV), torch.zeros(1, 32, device=DEV)], 1)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = zs().rope_write(q, k, v, i32([0]), cs, torch.tensor([slot], device=DEV), kp, vp, err=err)
    assert err.item() == flagged and torch.equal(out, q)
    written = 1 if 0 <= slot < 32 else 0
    for p in (kp, vp):
        assert int((~p.isnan()).any(-1).sum()) == written
