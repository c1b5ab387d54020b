"""build.py where the torch binding cannot be built: the C-ABI library is built alone."""
import os
import shutil
import stat

import pytest


@pytest.fixture()
def sandbox(tmp_path, monkeypatch):
    """build.py with an nvcc that only writes its output file, in a folder of its own."""
    import build

    fake = tmp_path / "nvcc"
    fake.write_text('#!/bin/sh\nwhile [ $# -gt 0 ]; do [ "$1" = -o ] && : > "$2"; shift; done\n')
    fake.chmod(fake.stat().st_mode | stat.S_IXUSR)
    monkeypatch.setenv("NVCC", str(fake))
    for name, path in (("BUILD_DIR", "objects"), ("LIB_DIR", "lib"), ("LIB_PATH", "lib/lib.so"), ("EXT_PATH", "lib/ext.so")):
        monkeypatch.setattr(build, name, str(tmp_path / path))
    return build


def test_the_library_is_built_without_a_binding(sandbox, monkeypatch, capsys):
    real = shutil.which
    monkeypatch.setattr(shutil, "which", lambda name, *a, **k: None if name == "g++" else real(name, *a, **k))
    assert sandbox.why_no_binding() == "no g++"
    os.makedirs(sandbox.LIB_DIR)
    open(sandbox.EXT_PATH, "w").close()  # an older binding must not stay beside the new library
    assert sandbox.build(force=True) == sandbox.LIB_PATH
    assert os.path.exists(sandbox.LIB_PATH) and not os.path.exists(sandbox.EXT_PATH)
    assert "no g++" in capsys.readouterr().err
    assert sandbox.up_to_date()


def test_missing_headers_are_named(sandbox, monkeypatch):
    assert sandbox.why_no_binding() == ""
    monkeypatch.setattr(sandbox.sysconfig, "get_paths", lambda: {"include": "/nowhere"})
    assert sandbox.why_no_binding() == "no /nowhere/Python.h"


def test_a_missing_binding_is_out_of_date_where_it_can_be_built(sandbox):
    os.makedirs(sandbox.LIB_DIR)
    open(sandbox.LIB_PATH, "w").close()
    assert not sandbox.up_to_date()
