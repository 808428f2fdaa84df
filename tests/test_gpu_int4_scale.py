"""The largest softmax scales of 4-bit attention, and those past them."""
import ctypes as C
import math

import pytest
import torch

from test_gpu_int4 import BF, FP, check_attention, filled, i32, randn, table_of, zs
from test_int4_args import attention, zlib  # noqa: F401


@pytest.mark.parametrize("scale", [2.0 ** 57, -(2.0 ** 57), 2.0 ** 100, math.inf, math.nan])
def test_scales_out_of_range_are_refused_without_a_gpu(zlib, scale):  # noqa: F811
    assert zlib.zs_paged_attention_int4(C.byref(attention(softmax_scale=scale))) == 1
    assert zlib.zs_paged_attention_int4(C.byref(attention(B=0, softmax_scale=2.0 ** 56))) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,power", [(BF, 56), (BF, 40), (FP, 14)])
def test_large_scales(dtype, power):
    page, lens = 16, [50, 700]
    table, blocks = table_of(lens, page)
    for sign in (1, -1):
        kp, vp = filled(blocks, page, 1, 64, 32, seed=3)
        q = (randn(2, 3, 64, seed=2) * 2.0 ** -power).to(dtype)
        check_attention(q, kp, vp, table, lens, page, scale=sign * 2.0 ** (power - 3))


@pytest.mark.gpu
def test_scales_out_of_range_are_refused():
    kp, vp = filled(2, 16, 1, 64, 32)
    q = randn(1, 2, 64).to(BF)
    for scale in (2.0 ** 57, -(2.0 ** 60), math.nan, 1e300):
        with pytest.raises(ValueError):
            zs().paged_attention_int4(q, kp, vp, i32([[0]]), i32([3]), scale)
