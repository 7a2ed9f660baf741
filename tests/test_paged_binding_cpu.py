"""Where the torch binding of the paged cache can be built, and which file is its; nothing is compiled."""
import os

import pytest

from bmo_jetson_b200 import build

CUDA_FILES = ["include/c10/cuda/CUDAGuard.h", "lib/libc10_cuda.so"]


@pytest.fixture
def torch_dir(tmp_path, monkeypatch):
    """An installed torch with CUDA, as far as the build looks at it."""
    for f, text in [(f, "") for f in CUDA_FILES] + [("version.py", "__version__ = '2.11.0+cu128'\n")]:
        path = tmp_path / f
        path.parent.mkdir(parents=True, exist_ok=True)
        path.write_text(text)
    monkeypatch.setattr(build, "_torch_dir", lambda: str(tmp_path))
    monkeypatch.setattr(build, "_compile", lambda cmd: pytest.fail("compiles"))
    if build.binding_path() is None:
        pytest.skip("no Python or CUDA headers here")
    return tmp_path


@pytest.mark.parametrize("missing", CUDA_FILES + ["version.py"])
def test_torch_without_cuda_is_left_out(torch_dir, missing):
    """The library needs no torch: its build goes on without the binding."""
    (torch_dir / missing).unlink()
    assert build.binding_path() is None and build.build_binding() is None and build.build_binding(force=True) is None


def test_no_torch(monkeypatch):
    monkeypatch.setattr(build, "_torch_dir", lambda: None)
    assert build.build_binding() is None


def test_another_version_is_another_file(torch_dir, monkeypatch, tmp_path):
    first = build.binding_path()
    assert os.path.dirname(first) == os.path.dirname(build.LIB) and first == build.binding_path()
    (torch_dir / "version.py").write_text("__version__ = '2.12.0+cu128'\n")
    second = build.binding_path()
    assert second != first
    monkeypatch.setattr(build.sysconfig, "get_config_var", lambda name: "cpython-313")
    third = build.binding_path()
    assert third not in (first, second)
    source = tmp_path / "changed.cpp"
    with open(build.BINDING_SRC) as f:
        source.write_text(f.read() + "//\n")
    monkeypatch.setattr(build, "BINDING_SRC", str(source))
    assert build.binding_path() not in (first, second, third)


def test_the_binding_in_use_is_this_ones():
    paged = pytest.importorskip("bmo_jetson_b200.paged")
    assert paged._ext.__file__ == build.binding_path()
