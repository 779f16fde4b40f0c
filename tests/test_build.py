"""When a source of the library is compiled again (style_transfer_amd/build.py); nothing is compiled here."""
import os
import types

import pytest


@pytest.fixture
def compiler(monkeypatch, tmp_path):
    """build.py with a compiler that notes its commands and writes an empty object."""
    from style_transfer_amd import build
    ran = []

    def run(cmd, **_):
        ran.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(build, "OBJ_DIR", str(tmp_path))
    monkeypatch.setattr(build, "subprocess", types.SimpleNamespace(run=run))
    return build, ran


def test_an_object_is_made_again_when_its_command_changes(compiler, monkeypatch):
    build, ran = compiler
    src = build.sources()[0]
    obj = build._compile(src, False, False)
    assert build._compile(src, False, False) == obj and len(ran) == 1
    monkeypatch.setattr(build, "COMMON_FLAGS", [*build.COMMON_FLAGS, "-DOTHER"])
    build._compile(src, False, False)
    assert len(ran) == 2 and "-DOTHER" in ran[1]
    build._compile(src, False, False)
    assert len(ran) == 2
    build._compile(src, True, False)
    assert len(ran) == 3


def test_an_object_is_made_again_when_its_source_is_newer(compiler):
    build, ran = compiler
    src = build.sources()[0]
    obj = build._compile(src, False, False)
    os.utime(obj, (1, 1))
    build._compile(src, False, False)
    assert len(ran) == 2
