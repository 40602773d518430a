"""csrc/build.py puts the library and the binding in place together or not at all."""
import importlib.util
import json
import os
import subprocess
from pathlib import Path

import pytest
import torch

from h3_speedkit import _lib

CSRC = Path(__file__).resolve().parents[1] / "comfyui-h3-speedkit_b200" / "csrc"


@pytest.fixture
def kernel_build(tmp_path, monkeypatch):
    """The build script with its commands replaced: each writes its output, or fails."""
    spec = importlib.util.spec_from_file_location("h3sk_build_under_test", CSRC / "build.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.NATIVE, module.BUILD, module.failing, module.turn = tmp_path / "native", tmp_path / "build", None, 0

    def run(cmd):
        out = Path(cmd[cmd.index("-o") + 1])
        if module.failing and module.failing in out.name:
            return subprocess.CompletedProcess(cmd, 1, "", f"no {out.name}")
        out.write_text(f"{out.name} {module.turn}")
        return subprocess.CompletedProcess(cmd, 0, "", "")
    monkeypatch.setattr(module, "run", run)
    return module


def contents(module):
    return [(module.NATIVE / name).read_text() for name in (module.LIB_NAME, module.BINDING_NAME)]


@pytest.mark.parametrize("failing", ["rope.o", "libh3sk_b200.so", "h3sk_torch.so"])
def test_a_failed_build_leaves_the_last_one_and_is_not_up_to_date(kernel_build, failing, monkeypatch):
    kernel_build.build()
    assert kernel_build.up_to_date()
    before = contents(kernel_build)
    for name in (kernel_build.LIB_NAME, kernel_build.BINDING_NAME):    # a source changes
        os.utime(kernel_build.NATIVE / name, (1, 1))
    kernel_build.failing, kernel_build.turn = failing, 1
    for _ in range(2):
        assert not kernel_build.up_to_date()
        with pytest.raises(RuntimeError, match=f"no {failing}"):
            kernel_build.build()
        assert contents(kernel_build) == before
        assert f"no {failing}" in (kernel_build.NATIVE / "build.log").read_text()
    kernel_build.failing = None
    kernel_build.build()
    assert kernel_build.up_to_date() and contents(kernel_build) == [f"{kernel_build.LIB_NAME} 1", f"{kernel_build.BINDING_NAME} 1"]


def test_a_stale_or_foreign_binding_is_built_again(kernel_build, monkeypatch):
    kernel_build.build()
    os.utime(kernel_build.NATIVE / kernel_build.BINDING_NAME, (1, 1))
    assert not kernel_build.up_to_date()
    kernel_build.build()
    assert kernel_build.up_to_date()
    hosts = kernel_build.hosts()
    for name in hosts:
        with monkeypatch.context() as patch:
            patch.setattr(kernel_build, "hosts", lambda: hosts | {name: "another"})
            assert not kernel_build.up_to_date()
    (kernel_build.NATIVE / kernel_build.BINDING_NAME).unlink()
    assert not kernel_build.up_to_date()


def test_manifest_names_the_binding(kernel_build):
    kernel_build.build()
    binding = json.loads((kernel_build.NATIVE / "build.json").read_text())["binding"]
    assert binding["sha256"] == kernel_build.sha256(kernel_build.NATIVE / kernel_build.BINDING_NAME)
    assert binding["library_sha256"] == kernel_build.sha256(kernel_build.NATIVE / kernel_build.LIB_NAME)
    assert binding["torch"] == torch.__version__


def test_a_binding_of_another_torch_is_not_loaded(tmp_path, monkeypatch):
    _lib.load()
    (tmp_path / "h3sk_torch.so").write_text("")
    (tmp_path / "build.json").write_text(json.dumps({"binding": {"torch": "0.0"}}))
    monkeypatch.setattr(_lib, "NATIVE", tmp_path)
    monkeypatch.setattr(_lib, "_binding", None)
    with pytest.raises(RuntimeError, match="built for torch 0.0"):
        _lib.binding()


def test_argument_blocks_are_declared_once():
    """The library and its binding take them from the public header."""
    for source in CSRC.glob("*.cu"):
        text = source.read_text()
        assert "struct H3RopeArgs {" not in text and "struct H3MaskedAttentionArgs {" not in text
