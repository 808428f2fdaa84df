"""Sampling without a GPU: the C struct, and refusals before anything is launched."""
import ctypes as C

import pytest
import torch


class Sample(C.Structure):
    _fields_ = [("stream", C.c_void_p), ("logits", C.c_void_p), ("row_stride", C.c_int64)] + \
        [(n, C.c_void_p) for n in ("u", "temperature", "top_k", "top_p", "min_p", "out", "err")] + \
        [(n, C.c_int) for n in ("B", "V", "dtype", "top_k1")] + \
        [(n, C.c_double) for n in ("temperature1", "top_p1", "min_p1")]


@pytest.fixture(scope="module")
def zlib():
    from zipserv_asplos26_b200.build_lib import build
    build()
    from zipserv_asplos26_b200._lib import lib
    return lib()


@pytest.mark.parametrize("bad", [dict(B=-1), dict(V=0), dict(V=(1 << 20) + 1), dict(dtype=3), dict(dtype=-1), dict(row_stride=-1),
                                 dict(logits=0), dict(u=0), dict(out=0), dict(logits=258), dict(B=1 << 30)])
def test_bad_arguments_are_refused(zlib, bad):
    good = dict(logits=256, u=256, out=256, B=1, V=10, row_stride=10, dtype=2, temperature1=1.0, top_p1=1.0)
    assert zlib.zs_sample(C.byref(Sample(**{**good, **bad}))) == 1
    assert zlib.zs_sample(C.byref(Sample(**{**good, "B": 0}))) == 0
    assert zlib.zs_sample(None) == 1


def test_cpu_tensors_are_refused():
    import zipserv_asplos26_b200 as zs
    with pytest.raises(ValueError):
        zs.sample(torch.zeros(1, 4), torch.zeros(1))
