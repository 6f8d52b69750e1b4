"""What the build makes of a machine that lacks something: the library comes first, and does without the extension module."""
import fcntl
import os
import subprocess

import pytest

from tpp_pytorch_extension_b200 import _build


@pytest.fixture
def made(monkeypatch, tmp_path):
    """A build that writes files of no content under a folder of its own, and a list of what it made."""
    done = []
    monkeypatch.setattr(_build, "SO", str(tmp_path / "lib.so"))
    monkeypatch.setattr(_build, "TORCH_SO", str(tmp_path / "module.so"))
    monkeypatch.setattr(_build, "OBJ_DIR", str(tmp_path / "build"))

    def check_call(cmd, **kw):
        if cmd[0] == "g++":
            done.append("module")
        elif "-shared" in cmd:
            done.append("library")
        open(cmd[cmd.index("-o") + 1], "w").close()

    monkeypatch.setattr(_build.subprocess, "check_call", check_call)
    return done


def build():
    return _build.build(so=_build.SO)


def test_once_and_the_library_first(made):
    assert build() == _build.SO and made == ["library", "module"]
    build()
    assert made == ["library", "module"] and not _build.module_stale()


@pytest.mark.parametrize("error", [subprocess.CalledProcessError(1, "g++"), FileNotFoundError("g++")])
def test_without_the_module_there_is_still_a_library(made, monkeypatch, error):
    plain = _build.subprocess.check_call

    def check_call(cmd, **kw):
        if cmd[0] == "g++":
            raise error
        plain(cmd, **kw)

    monkeypatch.setattr(_build.subprocess, "check_call", check_call)
    with pytest.warns(UserWarning, match="_tpx_torch"):
        assert build() == _build.SO
    assert made == ["library"] and os.path.exists(_build.SO) and not os.path.exists(_build.TORCH_SO)


def test_another_torch_has_the_module_built_anew(made, monkeypatch):
    build()
    monkeypatch.setattr(_build, "_made_for", lambda: "another torch")
    assert _build.module_stale()
    build()
    assert made == ["library", "module", "module"] and not _build.module_stale()


@pytest.mark.parametrize("nvcc", ["nvcc", "/usr/local/cuda/bin/nvcc", "nowhere/nvcc"])
def test_cuda_headers_are_found_wherever_the_compiler_is(monkeypatch, tmp_path, nvcc):
    if not os.path.exists("/usr/local/cuda/bin/nvcc"):
        pytest.skip("no CUDA toolkit here")
    monkeypatch.setenv("NVCC", nvcc)
    monkeypatch.setenv("PATH", "/usr/local/cuda/bin" + os.pathsep + os.environ["PATH"])
    monkeypatch.chdir(tmp_path)
    inc = _build.cuda_include()
    assert os.path.isabs(inc) and os.path.exists(os.path.join(inc, "cuda_runtime_api.h"))


def test_one_build_at_a_time(made):
    with _build._alone():
        with open(os.path.join(_build.OBJ_DIR, "lock")) as other, pytest.raises(BlockingIOError):
            fcntl.flock(other, fcntl.LOCK_EX | fcntl.LOCK_NB)


def test_what_is_up_to_date_needs_no_folder_to_write_to(made, monkeypatch):
    build()

    def locked():
        raise PermissionError("read-only")

    monkeypatch.setattr(_build, "_alone", locked)
    assert build() == _build.SO and made == ["library", "module"]
