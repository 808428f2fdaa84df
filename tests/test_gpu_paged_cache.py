"""PagedKVCache steps in which the rows differ: some have a token, some a whole
prompt, some nothing, one has ended, one is refused. Each token of the plan
attends what its own row holds up to itself; tolerances as in test_gpu_paged.py."""
import math

import numpy as np
import pytest
import torch

from test_gpu_paged import BF, DEV, HF, attend_ref, close, i32, zs

pytestmark = pytest.mark.gpu
HQ, HKV, D, PAGE, MAXPOS = 8, 2, 64, 16, 400


class Rows:
    """A cache, and the keys and values that each of its rows should hold."""

    def __init__(self, blocks, rows, width, dtype, layout):
        self.g = torch.Generator(device=DEV).manual_seed(rows + width)
        ang = torch.rand(MAXPOS, D // 2, device=DEV, generator=self.g) * 6
        self.cs = torch.cat([ang.cos(), ang.sin()], 1)
        self.dtype = dtype
        self.cache = zs().PagedKVCache(blocks, rows, width, HKV, D, PAGE, dtype, layout)
        self.kept = [[] for _ in range(rows)]

    def draw(self, n):
        x = torch.randn(n, HQ + 2 * HKV, D, device=DEV, generator=self.g).to(self.dtype)
        return x[:, :HQ], x[:, HQ:HQ + HKV], x[:, HQ + HKV:]

    def keep(self, new, plan, v):
        for r, n in enumerate(new):
            if n < 0:
                self.kept[r] = []
        for t, (r, slot) in enumerate(zip(plan.token_seq.tolist(), plan.slots.tolist())):
            if r >= 0:
                key = self.cache.k[0][slot // PAGE, slot % PAGE].clone()      # as it was rounded when it was turned
                self.kept[r].append((key, v[t].clone()))

    def check(self, plan, q, out, picked=None):
        """Token by token against the kept keys up to its position; padding is zero."""
        seq, pos = plan.token_seq.tolist(), plan.positions.tolist()
        dense = []
        for r, p in zip(seq, pos):
            x = self.kept[r][:p + 1] if r >= 0 else []
            empty = torch.zeros(0, HKV, D, device=DEV, dtype=self.dtype)
            dense.append((torch.stack([a for a, _ in x]), torch.stack([b for _, b in x])) if x else (empty, empty))
        ref, _, vmax = attend_ref(q, dense, 1 / math.sqrt(D), picked)
        assert close(out, ref, vmax, self.dtype)
        assert bool((out[plan.token_seq < 0] == 0).all())


STEPS = [                           # tokens of rows 0..4, refused rows
    ([30, 0, 17, 1, 0], []),        # prompts beside an idle row
    ([1, 0, 1, 1, 0], []),          # decode, two rows idle
    ([1, 5, -1, 1, 0], []),         # row 2 ends, row 1 starts
    ([1, 1, 0, 0, 1], []),
    ([1, 1, 33, 97, 1], [3]),       # row 3 asks for more than a row of the table holds
    ([-1, 1, 1, 1, 1], []),
]


@pytest.mark.parametrize("dtype,layout", [(BF, "heads"), (HF, "tokens"), (BF, "tokens"), (HF, "heads")])
def test_tokens_attend_their_own_rows(dtype, layout):
    x = Rows(24, 5, 6, dtype, layout)
    cache = x.cache
    for new, refused in STEPS:
        n = sum(t for t in new if t > 0)
        q, k, v = x.draw(n + 3)                              # three tokens of padding
        plan = cache.step(i32(new), n + 3)
        assert plan.refused.nonzero().flatten().tolist() == refused
        rows = cache.token_rows(plan)
        turned = cache.write(q, k, v, x.cs, plan)
        x.keep(new, plan, v)
        assert cache.seqlens.tolist() == [len(r) for r in x.kept]
        x.check(plan, turned, cache.attention(turned, rows=rows))
        out, pages, counts = cache.sparse_attention(turned, 3, rows=rows)
        pg, ct = pages.cpu().numpy(), counts.cpu().numpy()
        want = [min(3, p // PAGE + 1) if r >= 0 else 0
                for r, p in zip(plan.token_seq.tolist(), plan.positions.tolist())]
        assert ct.tolist() == [[c] * HKV for c in want]

        def picked(b, h):
            t = (pg[b, h, :ct[b, h], None] * PAGE + np.arange(PAGE)).ravel()
            return torch.from_numpy(t[t <= int(plan.positions[b])]).to(DEV)

        x.check(plan, turned, out, picked)
    assert cache.check_errors() == 4                         # a request was refused


def test_tokens_attend_their_own_rows_in_a_graph():
    """One graph for all decode steps; which rows have a token is an input of the replay."""
    x = Rows(24, 5, 6, BF, "heads")
    cache = x.cache
    new = i32([0] * 5)
    q, k, v = (t.contiguous() for t in x.draw(5))

    def step():
        plan = cache.step(new, 5)
        rows = cache.token_rows(plan)
        turned = cache.write(q, k, v, x.cs, plan)
        return plan, turned, cache.attention(turned, rows=rows)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()                                               # no tokens: the state stays as it was
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan, turned, out = step()
    asks = [[1, 1, 1, 1, 1], [1, 0, 1, 0, 1], [0, 0, 0, 0, 0], [0, -1, 1, 1, 1], [1, 1, -1, -1, 0], [2, 1, 1, 0, 1],
            [9, 1, 0, 1, 1]]
    refused = [[], [], [], [], [], [], [0, 1, 3, 4]]          # tokens count in order of rows: nothing fits behind nine
    for ask, no in zip(asks, refused):
        new.copy_(i32(ask))
        for t, s in zip((q, k, v), x.draw(5)):
            t.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        assert plan.refused.nonzero().flatten().tolist() == no
        x.keep(ask, plan, v)
        assert cache.seqlens.tolist() == [len(r) for r in x.kept]
        x.check(plan, turned, out)


def test_rows_and_tokens_agree_where_every_row_has_one():
    x = Rows(24, 3, 6, BF, "heads")
    cache = x.cache
    for new in ([20, 33, 1], [1, 1, 1]):
        q, k, v = x.draw(sum(new))
        plan = cache.step(i32(new), sum(new))
        turned = cache.write(q, k, v, x.cs, plan)
    assert torch.equal(cache.attention(turned), cache.attention(turned, rows=cache.token_rows(plan)))


def test_outputs_into_a_given_buffer():
    x = Rows(24, 2, 6, HF, "tokens")
    q, k, v = x.draw(50)
    plan = x.cache.step(i32([40, 10]), 50)
    x.cache.write(q, k, v, x.cs, plan)
    last = torch.randn(2, HQ, D, device=DEV).to(HF)
    want = x.cache.attention(last)
    out, lse = torch.full_like(last, 9.0), torch.zeros(2, HQ, device=DEV)
    got = x.cache.attention(last, out=out, lse=lse)
    assert got.data_ptr() == out.data_ptr() and torch.equal(out, want) and bool(lse.isfinite().all())
