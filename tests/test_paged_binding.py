"""The binding of the paged-cache operators belongs to one torch and one Python:
after an upgrade of either it is built anew, and the old file is not loaded."""
import os
import sysconfig

import pytest
import torch

from zipserv_asplos26_b200 import build_lib, paged
from zipserv_asplos26_b200._lib import ZipServError

SUFFIX = sysconfig.get_config_var("EXT_SUFFIX")


def test_the_file_names_what_it_was_built_for():
    here = build_lib.binding_path(torch.__version__, SUFFIX)
    assert paged.BINDING == build_lib.BINDING == here
    others = {here, build_lib.binding_path(torch.__version__ + "1", SUFFIX), build_lib.binding_path(torch.__version__, ".cpython-399.so")}
    assert len(others) == 3 and all(os.path.dirname(p) == build_lib.LIBDIR for p in others)


def test_another_torch_builds_its_own(monkeypatch):
    build_lib.build()
    ran = []

    def run(cmd, **kw):
        ran.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return type("R", (), {"returncode": 0})

    monkeypatch.setattr(build_lib.subprocess, "run", run)
    build_lib.build()
    assert not ran                                           # up to date
    path = build_lib.binding_path("0.0.0", SUFFIX)
    monkeypatch.setattr(build_lib, "BINDING", path)
    try:
        build_lib.build()
        assert len(ran) == 1 and os.path.exists(path)
    finally:
        if os.path.exists(path):
            os.remove(path)


def test_another_torchs_file_is_not_loaded(monkeypatch):
    build_lib.build()
    monkeypatch.setattr(paged, "_native", None)
    monkeypatch.setattr(paged, "BINDING", build_lib.binding_path("0.0.0", SUFFIX))
    with pytest.raises(ZipServError, match="not built"):
        paged._load()
