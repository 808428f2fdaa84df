"""Paged-cache operators without a GPU: the argument structs of the C ABI as a
ctypes caller packs them, and refusals before anything is launched."""
import ctypes as C
import os
import re
import struct
import subprocess

import pytest
import torch

from zipserv_asplos26_b200 import paged

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def zlib():
    from zipserv_asplos26_b200.build_lib import build
    build()
    from zipserv_asplos26_b200._lib import lib
    return lib()


_POOL = "Qqqqiiiii4x"
STRUCTS = {"ZsPlanStep": struct.Struct("<QQq12Q6i"), "ZsRopeWrite": struct.Struct("<QQQQ6qQQqQQQ" + _POOL * 2 + "3i4i3i"),
           "ZsPagedAttention": struct.Struct("<QQQqQQQQQQQQ" + _POOL * 2 + "4ifi"),
           "ZsPageBounds": struct.Struct("<QQqQQQQQ" + _POOL + "4i"),
           "ZsSelectPages": struct.Struct("<QQQQQqQQQQ12i")}


def _fn(zlib, name, args=(C.c_char_p,), res=C.c_int):
    f = getattr(zlib, name)
    f.argtypes, f.restype = list(args), res
    return f


def test_packed_structs_match_the_header(tmp_path):
    """Sizes, and the offset of every field, against a C compiler's."""
    header = open(os.path.join(ROOT, "include", "zipserv_b200.h")).read()
    src, names = ['#include <stdio.h>', '#include <stddef.h>', '#include "zipserv_b200.h"', "int main(void) {"], []
    for s in STRUCTS:
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (s, s), header, re.S).group(1)
        src.append(f'printf("{s} . %zu\\n", sizeof({s}));')
        for decl in body.split(";"):
            for part in decl.split(","):
                m = re.search(r"(\w+)(\[\d+\])?\s*$", part.strip())
                if m:
                    src.append(f'printf("{s} {m.group(1)} %zu\\n", offsetof({s}, {m.group(1)}));')
                    names.append((s, m.group(1)))
    src.append("return 0; }")
    c = tmp_path / "sizes.c"
    c.write_text("\n".join(src))
    subprocess.check_call(["gcc", "-std=c11", f"-I{ROOT}/include", str(c), "-o", str(tmp_path / "sizes")])
    seen = {}
    for line in subprocess.check_output([str(tmp_path / "sizes")], text=True).splitlines():
        s, f, off = line.split()
        seen.setdefault(s, []).append((f, int(off)))
    for s, fmt in STRUCTS.items():
        got = dict(seen[s])
        assert got.pop(".") == fmt.size, s
        # offsets by packing one field after another
        offs, at = [], 0
        text = fmt.format[1:]
        items = re.findall(r"(\d*)([a-zA-Z])", text)
        flat = []
        for n, ch in items:
            flat += ["4x"] if ch == "x" else [ch] * int(n or 1)
        for ch in flat:
            if ch != "4x":
                offs.append(at)
            at += struct.calcsize("<" + ch)
        for f, off in got.items():
            assert off in offs, (s, f, off)


def test_null_and_bad_arguments_are_refused(zlib):
    for name in ("zs_plan_step", "zs_rope_write", "zs_paged_attention", "zs_page_bounds", "zs_select_pages"):
        f = _fn(zlib, name)
        assert f(None) == 1, name
        size = {"zs_plan_step": 144, "zs_rope_write": 280, "zs_paged_attention": 232, "zs_page_bounds": 136,
                "zs_select_pages": 128}[name]
        assert f(bytes(size)) == 1, name
    ok = (1 << 20, 2048, 128, 2048, 4, 16, 1, 128, 0)
    for i, bad in ((0, 0), (0, (1 << 20) + 8), (1, 2049), (2, -8), (4, 0), (5, 24), (5, 512), (6, 0), (8, 2)):
        pool = list(ok)
        pool[i] = bad
        args = STRUCTS["ZsPageBounds"].pack(0, 1 << 20, 4, 1 << 20, 1 << 20, 1 << 20, 1 << 20, 0, *pool, 0, 4, 8, 0)
        assert _fn(zlib, "zs_page_bounds")(args) == 1, (i, bad)
    assert _fn(zlib, "zs_page_bounds")(STRUCTS["ZsPageBounds"].pack(0, 1 << 20, 4, 1 << 20, 1 << 20, 1 << 20, 1 << 20, 0, *ok,
                                                          0, 4, 8, 0)) == 0          # no sequences: nothing to do


def test_plan_outputs_are_other_buffers(zlib):
    """Every thread block reads lengths, asks and count, so none of them may be written."""
    a = 1 << 20
    names = ("table", "seq_lens", "new_lens", "free_blocks", "free_count", "out_lens", "out_count")
    for same in (("out_lens", "seq_lens"), ("out_lens", "new_lens"), ("out_count", "free_count")):
        at = {n: a + 4096 * i for i, n in enumerate(names)}
        at[same[0]] = at[same[1]]
        args = STRUCTS["ZsPlanStep"].pack(0, at["table"], 4, at["seq_lens"], at["new_lens"], at["free_blocks"],
                                          at["free_count"], at["out_lens"], at["out_count"], *[2 * a] * 5, 0, 1, 4, 8, 16, 8, 0)
        assert _fn(zlib, "zs_plan_step")(args) == 1, same


def test_workspace_bytes(zlib):
    f = _fn(zlib, "zs_paged_attention_workspace_bytes", [C.c_int] * 4, C.c_size_t)
    assert f(0, 32, 8, 128) == 0 and f(1, 30, 8, 128) == 0
    assert f(1, 32, 8, 128) >= 2 * 148 * 16 * (128 + 2) * 4
    assert f(1 << 20, 32, 8, 128) > f(1, 32, 8, 128)


def test_tensors_must_be_on_a_gpu():
    x = torch.zeros(2, 16, 1, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        paged.paged_attention(torch.zeros(1, 1, 64, dtype=torch.bfloat16), x, x, i.view(1, 1), i)
    with pytest.raises(ValueError, match="CUDA"):
        paged.plan_step(i.view(1, 1), i, i, i, i, 16, 1)
    with pytest.raises(ValueError, match="CUDA"):
        paged.page_bounds(x, i.view(1, 1), i, i, torch.zeros(2, 1, 2, 64, dtype=torch.int8), torch.zeros(2, 1), 1)
    with pytest.raises(ValueError, match="layout"):
        paged.PagedKVCache(1, 1, 1, 1, layout="rows")
    with pytest.raises(ValueError, match="page_size"):
        paged.PagedKVCache(1, 1, 1, 1, page_size=48)
