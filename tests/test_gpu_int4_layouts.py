"""4-bit attention over pools of other strides and layouts."""
import pytest
import torch

import int4_plain as plain
from test_gpu_int4 import BF, FP, U, TINY, filled, i32, randn, rows_of, table_of, zs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv,dim,page,group,dtype", [
    (12, 3, 128, 64, 64, BF), (7, 1, 128, 16, 32, FP), (18, 2, 64, 32, 32, BF), (48, 2, 128, 16, 64, FP),
    (32, 8, 128, 16, 32, FP), (16, 4, 64, 64, 64, BF)])
@pytest.mark.parametrize("lens", [[4000, 0, 1, 1023, 2500], [9000], [700] * 40])
def test_layouts_give_the_same_sums(hq, hkv, dim, page, group, dtype, lens):
    """Rows by token and by head: equal where the work is dealt alike, which it is unless heads
    go side by side in a CTA (units of a sequence in fours), and there within both forms'
    bounds: attention_error and the output's rounding, once each."""
    table, blocks = table_of(lens, page, seed=3)
    tokens = filled(blocks, page, hkv, dim, group, "tokens", seed=hq)
    heads = []
    for p in tokens:
        x = zs().int4_pages(blocks, page, hkv, dim, group, "heads")
        x.codes.copy_(p.codes)
        x.params.copy_(p.params)
        heads.append(x)
    q = randn(len(lens), hq, dim, seed=1).to(dtype)
    a, b = (zs().paged_attention_int4(q, *pools, i32(table), i32(lens)) for pools in (tokens, heads))
    if hkv * -(-(hq // hkv) // 16) % 4:
        assert torch.equal(a, b)
    for r, n in enumerate(lens[:5]):
        k, v = rows_of(heads[0], table[r], n, page), rows_of(heads[1], table[r], n, page)
        err = plain.attention_error(q[r].float(), k, v, heads[0].params, dim ** -0.5, n) * (float(v.abs().max()) if n else 0.0)
        off = (a[r].double() - b[r].double()).abs()
        most = torch.maximum(a[r].double().abs(), b[r].double().abs())
        assert bool((off <= 2 * (err + U[dtype] * (most + err) + TINY[dtype])).all()), (r, float(off.max()))


def test_a_stride_past_32_bits_is_refused():
    """Attention's addresses are 32-bit multiples; writing and reading take any stride. The pool
    is a view whose second block lies 4 GiB on."""
    big = torch.empty((1 << 32) + 4096, dtype=torch.uint8, device="cuda")
    codes = big.as_strided((2, 16, 1, 64), (1 << 32, 64, 64, 1))
    codes.fill_(0x88)
    params = zs().int4_pages(2, 16, 1, 128).params
    params[..., 1, :] = 3.0
    p = zs().Int4Pages(codes, params)
    q = randn(1, 2, 128).to(BF)
    with pytest.raises(ValueError):
        zs().paged_attention_int4(q, p, p, i32([[1]]), i32([3]))
    k, _ = zs().read_int4(p, p, torch.arange(32, device="cuda"))
    assert bool((k == 3.0).all())
