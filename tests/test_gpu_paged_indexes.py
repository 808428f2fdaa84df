"""Bad indexes of the paged cache, each in a call of its own: skipped, and flagged with bit 2."""
import numpy as np
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


def plan(table, lens, new, free, count, tokens=40):
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    t, f = i32(table), i32(free)
    p = zs().plan_step(t, i32(lens), i32(new), f, i32([count]), 16, tokens, err=err)
    return p, t, f, err.item()


def test_a_page_missing_from_a_request():
    """The last page of request 1 is not there: its tokens have no slot, the others have."""
    p, _, _, err = plan([[4, -1], [5, -1], [6, -1]], [3, 20, 7], [2, 2, 1], [1, 2], 2)
    assert err == 2
    assert p.slots[:6].tolist() == [4 * 16 + 3, 4 * 16 + 4, -1, -1, 6 * 16 + 7, -1]
    assert p.token_seq[:6].tolist() == [0, 0, 1, 1, 2, -1] and p.positions[:5].tolist() == [3, 4, 20, 21, 7]
    assert p.seq_lens.tolist() == [5, 22, 8]


def test_a_slot_of_a_missing_page_is_never_a_row_of_the_pool():
    """Every row of a page, the last one (-page + page - 1 = -1) among them."""
    for pos in (0, 7, 15):
        p, _, _, err = plan([[-1, -1]], [pos] if pos else [0], [1], [-1, 3], 1)
        assert err == 2 and p.slots[0].item() == -1
        p, _, _, err = plan([[-4, -1]], [pos + 1], [0], [3], 1)
        assert err == 0                                     # nothing of the page is asked for


def test_a_page_missing_from_the_free_list():
    p, t, _, err = plan([[0, -1], [1, -1]], [16, 16], [1, 1], [3, -7], 2)
    assert err == 2 and p.slots[:2].tolist() == [-1, 3 * 16] and t[1].tolist() == [1, 3]


def test_a_missing_page_given_back():
    p, _, f, err = plan([[2, -1], [1, -1]], [30, 3], [-1, 0], [0, 9, 9, 9], 1)
    assert err == 2 and p.free_count.item() == 3
    p, _, f, err = plan([[2, 5], [1, -1]], [30, 3], [-1, 0], [0, 9, 9, 9], 1)
    assert err == 0 and p.free_count.item() == 3 and f[:3].tolist() == [0, 2, 5]


@pytest.mark.parametrize("count,flagged,taken", [(2, 0, 1), (4, 0, 1), (5, 2, 1), (2 ** 31 - 1, 2, 1), (-1, 2, 0), (-2 ** 31, 2, 0)])
def test_a_free_count_outside_the_list(count, flagged, taken):
    """Counts as the nearest that the list can have."""
    p, t, _, err = plan([[-1], [0]], [0, 3], [5, 1], [4, 5, 6, 7], count)
    assert err == flagged | (0 if taken else 4)
    have = max(0, min(count, 4))
    assert p.free_count.item() == have - taken and p.refused.tolist() == [not taken, False]
    if taken:
        assert t[0, 0].item() == 4 + have - 1 and p.slots[0].item() == (4 + have - 1) * 16


def test_good_tables_set_no_bit():
    rng = np.random.default_rng(0)
    order = rng.permutation(200)
    table = np.full((20, 8), -1)
    lens = rng.integers(0, 100, 20)
    at = 0
    for r, n in enumerate(-(-lens // 16)):
        table[r, :n] = order[at:at + n]
        at += n
    free = np.full(200, -1)
    free[:200 - at] = order[at:]
    new = rng.integers(-1, 20, 20)
    p, t, f, err = plan(table, lens, new, free, 200 - at, 400)
    assert err == 0 and not bool(p.refused.any())
    n = p.cu_tokens[-1].item()
    assert bool((p.slots[:n] >= 0).all()) and len(set(p.slots[:n].tolist())) == n
