"""Where a rotary write may put its q."""
import pytest
import torch

from test_gpu_paged import BF, DEV, i32, pool, zs

pytestmark = pytest.mark.gpu
HQ, HKV, D = 6, 2, 64


def call(q, k, v, q_out=None):
    n = q.shape[0]
    ang = torch.linspace(0, 3, 9 * D // 2, device=DEV).view(9, D // 2)
    kp, vp = (pool(2, 16, HKV, D, BF, "heads", 0.0) for _ in range(2))
    out = zs().rope_write(q, k, v, i32(range(n)), torch.cat([ang.cos(), ang.sin()], 1), torch.arange(n, device=DEV), kp, vp,
                          q_out=q_out)
    return out, kp, vp


def fused(n):
    x = torch.randn(n, (HQ + 2 * HKV) * D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(n)).to(BF)
    return x, [t.view(n, -1, D) for t in x.split([HQ * D, HKV * D, HKV * D], 1)]


def test_one_token_of_a_fused_projection_in_place():
    x, (q, k, v) = fused(1)
    want, kp, vp = call(*(t.clone() for t in (q, k, v)))
    out, kq, vq = call(q, k, v, q_out=q)
    assert out is q and torch.equal(q, want) and torch.equal(kp, kq) and torch.equal(vp, vq)
    assert torch.equal(x.view(-1, D)[HQ:], fused(1)[0].view(-1, D)[HQ:])        # k and v as they were


def test_in_place_and_beside_the_inputs_in_one_buffer():
    _, (q, k, v) = fused(7)
    want, kp, vp = call(q, k, v)
    arena = torch.empty(7 * (2 * HQ + 2 * HKV) * D, device=DEV, dtype=BF)
    parts = [t.view(7, -1, D) for t in arena.split([7 * h * D for h in (HKV, HQ, HQ, HKV)])]
    for t, s in zip((parts[0], parts[1], parts[3]), (k, q, v)):
        t.copy_(s)
    out, kq, vq = call(parts[1], parts[0], parts[3], q_out=parts[2])             # between the inputs, touching them
    assert torch.equal(out, want) and torch.equal(kp, kq) and torch.equal(vp, vq)
    out, kq, vq = call(parts[1], parts[0], parts[3], q_out=parts[1])
    assert torch.equal(out, want) and torch.equal(kp, kq) and torch.equal(vp, vq)


def test_over_other_tokens_is_refused():
    x, (q, k, v) = fused(7)
    kept = x.clone()
    over = x.view(-1)[:7 * HQ * D].view(7, HQ, D)
    with pytest.raises(ValueError, match="q_out"):
        call(q, k, v, q_out=over)
    qc = q.contiguous()
    for a, b in ((k, v), (v, k)):
        room = torch.zeros(7 * HQ * D + 7 * HKV * D, device=DEV, dtype=BF)
        near = room[-7 * HKV * D - 8:-8].view(7, HKV, D)
        near.copy_(a)
        with pytest.raises(ValueError, match="q_out"):
            call(qc, near, b, q_out=room[:7 * HQ * D].view(7, HQ, D))
        with pytest.raises(ValueError, match="q_out"):
            call(qc, b, near, q_out=room[:7 * HQ * D].view(7, HQ, D))
    assert torch.equal(x, kept)
