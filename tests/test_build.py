"""CPU: what the build does where torch or g++ is missing. The C libraries need neither."""
import shutil
import sys

import pytest

from tabby_b200 import build


@pytest.fixture
def only_the_extension_is_stale(monkeypatch, tmp_path):
    monkeypatch.setattr(build, "DECODE_TORCH", str(tmp_path / "tabby_decode_torch.so"))
    monkeypatch.setattr(build, "_stale", lambda lib, sources: lib == build.DECODE_TORCH)
    ran = []
    monkeypatch.setattr(build, "_run", lambda cmd, what: ran.append(cmd))
    return ran


def test_without_torch_the_libraries_are_enough(only_the_extension_is_stale, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)
    assert build.build() == build.LIB
    assert not only_the_extension_is_stale
    assert "torch is missing" in capsys.readouterr().err


def test_a_torch_without_cuda_is_none(only_the_extension_is_stale, monkeypatch, capsys):
    torch = pytest.importorskip("torch")
    monkeypatch.setattr(torch.version, "cuda", None)
    assert build.build() == build.LIB
    assert not only_the_extension_is_stale
    assert "torch with CUDA is missing" in capsys.readouterr().err


def test_without_a_host_compiler_too(only_the_extension_is_stale, monkeypatch, capsys):
    pytest.importorskip("torch")
    which = shutil.which
    monkeypatch.setattr(shutil, "which", lambda name: None if name == "g++" else which(name))
    assert build.build() == build.LIB
    assert not only_the_extension_is_stale
    assert "g++ is missing" in capsys.readouterr().err


def test_a_compiler_error_is_one(only_the_extension_is_stale, monkeypatch):
    pytest.importorskip("torch")
    if shutil.which("g++") is None:
        pytest.skip("no g++")

    def fail(cmd, what):
        raise RuntimeError(what)

    monkeypatch.setattr(build, "_run", fail)
    with pytest.raises(RuntimeError, match="decode_torch"):
        build.build()


def test_the_toolkits_headers_go_with_its_compiler(only_the_extension_is_stale, monkeypatch,
                                                   tmp_path):
    pytest.importorskip("torch")
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    nvcc = tmp_path / "kit" / "bin" / "nvcc"
    nvcc.parent.mkdir(parents=True)
    nvcc.touch()
    monkeypatch.setenv("NVCC", str(nvcc))
    monkeypatch.setattr(build.os, "replace", lambda a, b: None)
    build.build()
    (cmd,) = only_the_extension_is_stale
    assert f"-I{tmp_path}/kit/include" in cmd
