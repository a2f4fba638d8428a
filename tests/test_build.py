"""When the module for torch tensors is built: the compiler is not run."""

import importlib.util
import os
from pathlib import Path

import pytest

BUILD = Path(__file__).resolve().parents[1] / "distributed-kge-poplar_b200" / "build.py"


@pytest.fixture
def build(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("_kge_build_tested", BUILD)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    monkeypatch.setattr(module, "HERE", tmp_path)
    monkeypatch.setattr(module, "TORCH_MODULE", tmp_path / "libkge_torch.so")
    module.ran = []

    def run(cmd, verbose):
        module.ran.append(cmd)
        module.TORCH_MODULE.write_bytes(b"")

    monkeypatch.setattr(module, "_run", run)
    return module


def test_without_torch_the_rest_stands(build, monkeypatch, capsys):
    def missing(name):
        raise build.importlib.metadata.PackageNotFoundError(name)

    monkeypatch.setattr(build.importlib.metadata, "version", missing)
    for force in (False, True):
        build._build_torch_module(force, False)
    assert not build.ran and "no torch" in capsys.readouterr().err


def test_another_torch_is_built_for_anew(build, monkeypatch):
    pytest.importorskip("torch")
    version = ["1.0"]
    monkeypatch.setattr(build, "_torch_version", lambda: version[0])
    for expected, change in [(1, None), (1, None), (2, "2.0"), (2, None)]:
        version[0] = change or version[0]
        build._build_torch_module(False, False)
        assert len(build.ran) == expected
    os.utime(build.TORCH_MODULE, (1, 1))  # older than its source
    build._build_torch_module(False, False)
    assert len(build.ran) == 3
