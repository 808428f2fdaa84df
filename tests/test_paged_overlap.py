"""A rotary write whose q_out lies over what other warps still read is refused
(without a GPU: nothing is launched)."""
import ctypes as C
import os
import subprocess

from test_paged_args import ROOT, STRUCTS, _fn, zlib  # noqa: F401

A = 1 << 20
N, HQ, HKV, D, ROW = 5, 4, 2, 64, (4 + 2 * 2) * 64       # a fused projection's row
POOL = (1 << 24, 16 * HKV * D, HKV * D, D, 4, 16, HKV, D, 0)


def status(zlib, q=A, k=A + HQ * D * 2, v=A + (HQ + HKV) * D * 2, q_tok=ROW, kv_tok=ROW, q_out=A, n=N):  # noqa: F811
    far = 1 << 28
    args = STRUCTS["ZsRopeWrite"].pack(0, q, k, v, q_tok, D, kv_tok, D, kv_tok, D, q_out, far, 0, far, far, 0, *POOL, *POOL,
                                       n, HQ, 1, D // 2, 0, 0, 0, 8, D, 0)
    return _fn(zlib, "zs_rope_write")(args)


def test_q_out_over_what_is_read_is_refused(zlib):  # noqa: F811
    assert status(zlib) == 1                                             # q's own start, q a slice of a wider row
    for k_or_v in ("k", "v"):
        kw = dict(q=8 * A, q_tok=HQ * D, q_out=2 * A, k=4 * A, v=6 * A, kv_tok=HKV * D)
        kw[k_or_v] = 2 * A + (N * HQ * D - 8) * 2                        # the last 8 values of q_out
        assert status(zlib, **kw) == 1
        kw[k_or_v] = 2 * A - (N * HKV * D - 8) * 2                       # the first 8
        assert status(zlib, **kw) == 1
    contiguous = dict(q_tok=HQ * D, k=4 * A, v=6 * A, kv_tok=HKV * D)
    for shift in (16, -16, (N * HQ * D - 8) * 2):
        assert status(zlib, q_out=A + shift, **contiguous) == 1          # contiguous, but not q itself


def test_rows_meet_against_every_pair_of_elements(tmp_path):
    src = tmp_path / "meet.cpp"
    src.write_text(r'''
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "rows_meet.h"
int main() {
    srand(3);
    long met = 0, apart = 0;
    for (int c = 0; c < 200000; ++c) {
        const int n = 1 + rand() % 4, heads = 1 + rand() % 4, dim = 1 + rand() % 5, len = 1 + rand() % 9;
        const int tok = rand() % 41 - 20, head = rand() % 41 - 20, at = rand() % 161 - 80;
        bool want = false;
        for (int t = 0; t < n; ++t)
            for (int h = 0; h < heads; ++h)
                for (int i = 0; i < dim; ++i) {
                    const int x = t * tok + h * head + i;
                    want |= x >= at && x < at + len;
                }
        const uintptr_t base = 1 << 20;
        const bool got = zs::rows_meet((void*)base, n, heads, dim, tok, head, (void*)(base + 2 * (intptr_t)at), len);
        if (got != want) {
            printf("n %d heads %d dim %d tok %d head %d at %d len %d: %d\n", n, heads, dim, tok, head, at, len, got);
            return 1;
        }
        (want ? met : apart)++;
    }
    printf("%ld %ld\n", met, apart);
    return met > 20000 && apart > 20000 ? 0 : 2;
}
''')
    exe = tmp_path / "meet"
    subprocess.check_call(["g++", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover",
                           "-I" + os.path.join(ROOT, "zipserv_asplos26_b200", "csrc"), str(src), "-o", str(exe)])
    subprocess.check_call([str(exe)])
