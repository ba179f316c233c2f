"""When the library's objects are compiled again. The compiler is a script that writes down what it is asked for."""
import os
import stat

import pytest

from omni_attention_b200 import build


@pytest.fixture
def compiled(tmp_path, monkeypatch):
    """A function: builds, and returns how many objects were compiled and how often the library was linked."""
    log, nvcc = tmp_path / "log", tmp_path / "nvcc"
    nvcc.write_text(f'#!/bin/sh\necho "$@" >> {log}\nwhile [ $# -gt 1 ]; do if [ "$1" = -o ]; then touch "$2"; fi; shift; done\n')
    nvcc.chmod(nvcc.stat().st_mode | stat.S_IXUSR)
    monkeypatch.setenv("NVCC", str(nvcc))
    monkeypatch.setattr(build, "OBJ_DIR", str(tmp_path / "obj"))
    monkeypatch.setattr(build, "LIB_PATH", str(tmp_path / "lib.so"))

    def run(**kw):
        log.write_text("")
        build.build_library(**kw)
        lines = log.read_text().splitlines()
        return sum(" -c " in f" {line} " for line in lines), sum("-shared" in line for line in lines)
    return run


def test_objects_follow_sources_flags_and_compiler(compiled, monkeypatch, tmp_path):
    n = len(build.CUDA_SOURCES)
    assert compiled() == (n, 1)
    assert compiled() == (0, 0)
    os.utime(os.path.join(build.OBJ_DIR, "omni_bwd.o"), (0, 0))       # older than its source: only that one
    os.utime(build.LIB_PATH, (0, 0))
    assert compiled() == (1, 1)
    monkeypatch.setattr(build, "NVCC_FLAGS", [*build.NVCC_FLAGS, "-DSOMETHING"])
    assert compiled() == (n, 1)
    assert compiled() == (0, 0)
    other = tmp_path / "nvcc2"
    other.write_bytes((tmp_path / "nvcc").read_bytes())
    other.chmod(0o755)
    monkeypatch.setenv("NVCC", str(other))
    assert compiled() == (n, 1)


def test_a_verbose_build_compiles_everything(compiled):
    n = len(build.CUDA_SOURCES)
    assert compiled() == (n, 1)
    assert compiled(verbose=True) == (n, 1)
    assert compiled() == (0, 0)
    assert compiled(force=True) == (n, 1)


def test_a_build_that_failed_is_done_again(compiled, monkeypatch, tmp_path):
    n = len(build.CUDA_SOURCES)
    assert compiled() == (n, 1)
    monkeypatch.setattr(build, "NVCC_FLAGS", [*build.NVCC_FLAGS, "-DSOMETHING"])
    nvcc = tmp_path / "nvcc"
    good = nvcc.read_text()
    nvcc.write_text("#!/bin/sh\nexit 1\n")
    with pytest.raises(Exception):
        compiled()
    nvcc.write_text(good)
    assert compiled() == (n, 1)
