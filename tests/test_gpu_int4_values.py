"""4-bit attention of values without a range of their own: groups that are one number have a
scale of zero, so nothing but their centres says how large the sums get."""
import pytest
import torch

import int4_plain as plain
from test_gpu_int4 import BF, FP, U, TINY, filled, i32, randn, table_of, zs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("value", [1.0, -1000.0, 2.0 ** 14])
@pytest.mark.parametrize("lens", [[40], [20000, 3]])
def test_constant_values_come_back(value, dtype, lens):
    """The weighted mean of one number is that number: sums of T weights in two bf16 parts
    (2^-16) over sums of the weights, each fp32 sum off by its T / 8 steps of 2^-23."""
    page, dim = 64, 128
    table, blocks = table_of(lens, page)
    kp, vp = filled(blocks, page, 2, dim, 64, seed=3)
    codes, params = plain.quantise(torch.full((blocks, page, 2, dim), value, device="cuda"), 64)
    vp.codes.copy_(codes)
    vp.params.copy_(params)
    assert not vp.params[..., 0, :].any()
    q = randn(len(lens), 8, dim, seed=2).to(dtype)
    o = zs().paged_attention_int4(q, kp, vp, i32(table), i32(lens)).double()
    tol = (U[dtype] + 2.0 ** -16 + 2 * (max(lens) / 8 + 16) * 2.0 ** -23) * abs(value) + TINY[dtype]
    assert float((o - value).abs().max()) <= tol


def test_zeros_and_one_live_group():
    """One group of many has values, in some tokens only."""
    page, dim, lens = 16, 64, [500]
    table, blocks = table_of(lens, page)
    kp, vp = filled(blocks, page, 1, dim, 32, seed=5)
    x = torch.zeros(blocks, page, 1, dim, device="cuda")
    x[::3, 5, 0, 32:] = randn(len(x[::3]), 32, seed=6) * 2.0 ** -20
    codes, params = plain.quantise(x, 32)
    vp.codes.copy_(codes)
    vp.params.copy_(params)
    q = randn(1, 4, dim, seed=2).to(BF)
    o = zs().paged_attention_int4(q, kp, vp, i32(table), i32(lens))
    i = torch.arange(500, device="cuda")
    blk = torch.as_tensor(table[0], device="cuda").long()[i // page]
    k, v = (plain.values(p.codes[blk, i % page], p.params[blk, i % page]) for p in (kp, vp))
    want, _ = plain.attend(q[0], k, v, dim ** -0.5)
    tol = U[BF] * want.abs() + plain.attention_error(q[0], k, v, kp.params, dim ** -0.5, 500) * float(v.abs().max())
    assert bool(((o[0].double() - want).abs() <= tol).all())
    assert not o[0, :, :32].any()


def test_read_refuses_one_output_for_both():
    kp, vp = filled(2, 16, 1, 64, 32)
    slots = torch.arange(4, device="cuda")
    big = torch.empty(8, 1, 64, dtype=BF, device="cuda")
    for out in ((big[:4], big[:4]), (big[:4], big[1:5]), (big[2:6], big[:4])):
        with pytest.raises(ValueError):
            zs().read_int4(kp, vp, slots, out=out)
    k, v = zs().read_int4(kp, vp, slots, out=(big[:4], big[4:]))
    assert torch.equal(torch.cat([k, v]), torch.cat(zs().read_int4(kp, vp, slots)))


@pytest.mark.parametrize("bits", [4, 16])
def test_read_of_slots_outside_a_cache(bits):
    cache = zs().PagedKVCache(4, 1, 4, 2, 64, 16, bits=bits)
    slots = torch.tensor([0, -1, 63], device="cuda")
    cache.read(slots)
    assert cache.check_errors() == 0
    for bad in (-2, 64, 1 << 40):
        cache.err.zero_()
        k, v = cache.read(torch.tensor([3, bad], device="cuda"))
        assert cache.check_errors() == 2 and not k[1].any() and not v[1].any()


@pytest.mark.parametrize("group", [32, 64])
def test_a_head_of_rows_by_token(group):
    """Part of a larger pool, from an odd head on: parameters are aligned to a row of theirs."""
    page, lens, dim = 16, [90], 128
    table, blocks = table_of(lens, page)
    kb, vb = filled(blocks, page, 5, dim, group, "tokens", seed=2)
    kp, vp = (zs().Int4Pages(p.codes[:, :, 3:4], p.params[:, :, 3:4]) for p in (kb, vb))
    own = [zs().Int4Pages(p.codes.contiguous(), p.params.contiguous()) for p in (kp, vp)]
    q = randn(1, 4, dim, seed=2).to(BF)
    o = zs().paged_attention_int4(q, kp, vp, i32(table), i32(lens))
    assert torch.equal(o, zs().paged_attention_int4(q, *own, i32(table), i32(lens)))
    slots = torch.arange(40, device="cuda")
    assert torch.equal(zs().read_int4(kp, vp, slots)[0], zs().read_int4(*own, slots)[0])
    kv = randn(40, 1, dim, seed=4).to(BF)
    cos_sin = torch.cat([torch.ones(1, 64), torch.zeros(1, 64)], 1).cuda()
    before = kb.codes.clone()
    for pools in ((kp, vp), own):
        zs().rope_write_int4(kv, kv, kv, torch.zeros(40, dtype=torch.int32, device="cuda"), cos_sin, slots, *pools)
    assert torch.equal(kp.codes, own[0].codes) and torch.equal(vp.params, own[1].params)
    before[:, :, 3] = kb.codes[:, :, 3]
    assert torch.equal(kb.codes, before)
