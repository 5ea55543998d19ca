"""_torch_ops.so is built anew for another torch or Python, which it is linked to."""
import importlib.metadata
import shutil
import sysconfig

import pytest

from indecis_b200 import build


@pytest.fixture
def commands(monkeypatch, tmp_path):
    """The commands that a build would run, after one that is up to date."""
    build.build()
    stamp = getattr(build, "TORCH_OPS_STAMP", None)
    if stamp:
        monkeypatch.setattr(build, "TORCH_OPS_STAMP", shutil.copy(stamp, tmp_path / "stamp"))
    ran = []
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **_: ran.append(cmd))
    return ran


def torch_ops(ran):
    return [c for c in ran if build.TORCH_OPS in c]


def test_up_to_date(commands):
    build.build()
    assert commands == []


def test_another_torch(commands, monkeypatch):
    real = importlib.metadata.version
    monkeypatch.setattr(importlib.metadata, "version", lambda name: "99.0" if name == "torch" else real(name))
    build.build()
    assert len(torch_ops(commands)) == 1
    build.build()
    assert len(commands) == 1  # built for that one now


def test_another_python(commands, monkeypatch):
    real = sysconfig.get_config_var
    monkeypatch.setattr(sysconfig, "get_config_var", lambda name: "cpython-399" if name == "SOABI" else real(name))
    build.build()
    assert len(torch_ops(commands)) == 1
