"""How many bits 4-bit attention holds of a weight: outputs that are what is left of values
that cancel show errors of the weights that the output's own rounding hides elsewhere."""
import pytest
import torch

import int4_plain as plain
from test_gpu_int4 import BF, FP, U, TINY, i32, randn, rows_of, table_of, zs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("n,hq,hkv,dim,group", [(2, 8, 2, 128, 64), (16, 12, 1, 64, 32), (64, 8, 2, 128, 32), (600, 4, 1, 128, 64)])
def test_weights_of_values_that_cancel(dtype, n, hq, hkv, dim, group):
    """Tokens in pairs, the second's values the first's with the other sign, scores a little apart.
    Scores are sums of dim + 8 terms below `most`, each addition losing 2^-23 (attention_error);
    weights in two parts lose 2^-16 with the centres (which are zero here) and 2^-22 with the
    codes, the exponential 2^-22; the sums over n tokens, in steps of 8, 2^-23 each. With one
    part of 11 bits the outputs were off by up to 2^-11 max |v| / 2, four times the bound."""
    page, rows = 16, 24
    table, blocks = table_of([n] * rows, page)
    kp, vp = (zs().int4_pages(blocks, page, hkv, dim, group) for _ in range(2))
    codes, params = plain.quantise(randn(blocks, page, hkv, dim, seed=1) * 0.3, group)
    kp.codes.copy_(codes)
    kp.params.copy_(params)
    g = torch.Generator(device="cuda").manual_seed(2)
    u = torch.randint(1, 16, (blocks, page // 2, hkv, dim), device="cuda", generator=g, dtype=torch.int32)
    u = torch.stack([u, 16 - u], 2).flatten(1, 2)                     # u - 8 and its negative
    vp.codes.copy_((u[..., 0::2] | u[..., 1::2] << 4).to(torch.uint8))
    s = 1 + torch.rand(blocks, page // 2, hkv, dim // group, device="cuda", generator=g)
    vp.params[..., 0, :] = s.to(BF).repeat_interleave(2, 1)
    vp.params[..., 1, :] = 0
    q = (randn(rows, hq, dim, seed=3) * 0.02).to(dtype)
    o = zs().paged_attention_int4(q, kp, vp, i32(table), i32([n] * rows))
    for r in range(rows):
        k, v = (rows_of(p, table[r], n, page) for p in (kp, vp))
        want, _ = plain.attend(q[r], k, v, dim ** -0.5)
        bound = plain.attention_error(q[r].float(), k, v, kp.params, dim ** -0.5, n) - 3 * 2.0 ** -16 + 2.0 ** -20
        off = (o[r].double() - want).abs()
        assert bool((off <= U[dtype] * want.abs() + TINY[dtype] + bound * float(v.abs().max())).all()), \
            (r, float(off.max()), bound * float(v.abs().max()))
