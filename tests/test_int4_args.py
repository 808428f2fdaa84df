"""4-bit paged-cache operators without a GPU: the format's error bound, refusals of the C ABI
and of the cache class."""
import ctypes as C

import pytest
import torch

import int4_plain as plain
from zipserv_asplos26_b200 import paged


@pytest.fixture(scope="module")
def zlib():
    from zipserv_asplos26_b200.build_lib import build
    build()
    from zipserv_asplos26_b200._lib import lib
    return lib()


class Pool(C.Structure):
    _fields_ = [("codes", C.c_void_p), ("params", C.c_void_p)] + \
        [(n, C.c_int64) for n in ("codes_block", "codes_token", "codes_head", "params_block", "params_token", "params_head")] + \
        [(n, C.c_int) for n in ("num_blocks", "page_size", "num_heads", "head_dim", "group", "reserved")]


class Attention(C.Structure):
    _fields_ = [("stream", C.c_void_p), ("q", C.c_void_p), ("block_table", C.c_void_p), ("table_stride", C.c_int64)] + \
        [(n, C.c_void_p) for n in ("seq_lens", "pages", "counts", "ws")] + [("ws_bytes", C.c_size_t)] + \
        [(n, C.c_void_p) for n in ("out", "lse", "err")] + [("k_pool", Pool), ("v_pool", Pool)] + \
        [(n, C.c_int) for n in ("B", "Hq", "width", "top")] + [("softmax_scale", C.c_float)] + \
        [(n, C.c_int) for n in ("max_seqlen", "dtype")]


class Read(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("stream", "slots", "k_out", "v_out", "err")] + \
        [("k_pool", Pool), ("v_pool", Pool), ("N", C.c_int), ("dtype", C.c_int)]


def pool(**over):
    p = Pool(codes=256, params=512, codes_block=16 * 2 * 64, codes_token=64, codes_head=16 * 64, params_block=16 * 2 * 4,
             params_token=4, params_head=16 * 4, num_blocks=4, page_size=16, num_heads=2, head_dim=128, group=64)
    for k, v in over.items():
        setattr(p, k, v)
    return p


def attention(k=None, v=None, **over):
    a = Attention(q=256, block_table=256, table_stride=2, seq_lens=256, out=256, k_pool=k or pool(), v_pool=v or pool(),
                  B=1, Hq=4, width=2, softmax_scale=0.1)
    for n, x in over.items():
        setattr(a, n, x)
    return a


def test_the_formulas_error():
    g = torch.Generator().manual_seed(0)
    for scale, offset in ((1.0, 0.0), (1e-3, 5.0), (100.0, -3000.0), (1e30, 0.0), (1e-36, 0.0)):
        x = torch.randn(200, 128, generator=g) * scale + offset
        for group in (32, 64):
            codes, params = plain.quantise(x, group)
            s, c = params.double().unbind(-2)
            off = (plain.values(codes, params) - x.double()).abs().unflatten(-1, (-1, group))
            assert bool((off <= (s / 2 + (15 * s + c.abs()) / 256).unsqueeze(-1)).all())


BAD_POOLS = [dict(codes=0), dict(params=0), dict(codes=8), dict(params=4), dict(codes_token=72), dict(params_token=6),
             dict(codes_block=-64), dict(num_blocks=0), dict(page_size=24), dict(page_size=8), dict(num_heads=0),
             dict(head_dim=96), dict(head_dim=256), dict(group=16), dict(group=128)]


@pytest.mark.parametrize("bad", BAD_POOLS)
def test_bad_pools_are_refused(zlib, bad):
    for k, v in ((pool(**bad), pool(**bad)), (pool(), pool(**bad))):
        a = attention(k, v, B=0)
        assert zlib.zs_paged_attention_int4(C.byref(a)) == 1
        assert zlib.zs_read_int4(C.byref(Read(k_pool=k, v_pool=v, N=0))) == 1
    assert zlib.zs_paged_attention_int4(C.byref(attention(B=0))) == 0
    assert zlib.zs_read_int4(C.byref(Read(k_pool=pool(), v_pool=pool(), N=0))) == 0


@pytest.mark.parametrize("bad", [dict(q=0), dict(q=8), dict(out=0), dict(out=4), dict(block_table=0), dict(seq_lens=0),
                                 dict(Hq=3), dict(Hq=0), dict(B=-1), dict(width=0), dict(table_stride=1), dict(dtype=2),
                                 dict(softmax_scale=float("inf")), dict(pages=256), dict(pages=256, counts=256, top=0),
                                 dict(width=1 << 28, table_stride=1 << 28)])
def test_bad_attention_arguments_are_refused(zlib, bad):
    a = attention(**bad)
    assert zlib.zs_paged_attention_int4(C.byref(a)) == 1


def test_long_calls_need_their_workspace(zlib):
    f = zlib.zs_paged_attention_int4_workspace
    f.restype = C.c_size_t
    a = attention(width=4096, table_stride=4096)
    need = f(C.byref(a))
    assert need > 0
    for ws, n in ((0, need), (8, need), (256, need - 1)):
        a.ws, a.ws_bytes = ws, n
        assert zlib.zs_paged_attention_int4(C.byref(a)) == 1
    assert f(C.byref(attention())) == 0 and f(None) == 0


def test_null_is_refused(zlib):
    for name in ("zs_rope_write_int4", "zs_read_int4", "zs_paged_attention_int4"):
        assert getattr(zlib, name)(None) == 1


@pytest.mark.parametrize("over", [dict(bits=8), dict(bits=4, bounds=True), dict(bits=4, group=128), dict(bits=4, group=16)])
def test_cache_refusals(over):
    with pytest.raises(ValueError):
        paged.PagedKVCache(4, 1, 4, 2, device="cpu", **over)


def test_cache_pools():
    c = paged.PagedKVCache(4, 1, 4, 2, 128, 16, bits=4, num_layers=2, device="cpu")
    assert c.codes is None and len(c.k) == 2 and c.k[0].codes.shape == (4, 16, 2, 64)
    assert c.k[0].params.shape == (4, 16, 2, 2, 2)
    assert not plain.values(c.k[0].codes, c.k[0].params).any()
    assert paged.PagedKVCache(4, 1, 4, 2, device="cpu").codes is not None
    for bad in (dict(num_blocks=0), dict(head_dim=96), dict(page_size=20), dict(layout="x"), dict(group=7)):
        with pytest.raises(ValueError):
            paged.int4_pages(**{**dict(num_blocks=1, page_size=16, num_heads=1, head_dim=64, device="cpu"), **bad})


def test_cpu_tensors_are_refused():
    kp = paged.int4_pages(1, 16, 1, 64, device="cpu")
    q = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        paged.paged_attention_int4(q, kp, kp, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError):
        paged.read_int4(kp, kp, torch.zeros(1, dtype=torch.long))
    with pytest.raises(ValueError):
        paged.rope_write_int4(q, q, q, torch.zeros(1, dtype=torch.int32), torch.zeros(1, 64), torch.zeros(1, dtype=torch.long),
                              kp, kp)
