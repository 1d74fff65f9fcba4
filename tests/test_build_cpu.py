"""CPU suite: what build.py makes again, and what it does without, with the compilers replaced."""
import importlib.util
import os
import types
import warnings

import pytest

from conftest import ROOT


class _Build:
    def __init__(self, tmp_path):
        spec = importlib.util.spec_from_file_location("l3_build_under_test", os.path.join(ROOT, "llama3.np_b200", "build.py"))
        self.m = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(self.m)
        self.ran, self.gxx = [], 0
        self.m.OBJ, self.m.LIB = str(tmp_path / "build"), str(tmp_path / "lib.so")
        self.m.TORCH_OPS_STAMP = str(tmp_path / "build" / "ops.stamp")
        self.m.TORCH_OPS, self.m.NVCC = str(tmp_path / "ops.so"), str(tmp_path / "nvcc")
        open(self.m.NVCC, "w").close()
        self.torch = tmp_path / "torch"
        (self.torch / "lib").mkdir(parents=True)
        (self.torch / "version.py").write_text("1.0")
        self.m._torch_folder = lambda: str(self.torch)
        self.m.subprocess = types.SimpleNamespace(run=self.run)

    def with_cuda(self):
        (self.torch / "lib" / "libc10_cuda.so").write_text("")
        return self

    def run(self, cmd, **_):
        name = os.path.basename(cmd[0])
        self.ran.append("link" if name == "nvcc" and "-shared" in cmd else name)
        if name == "g++" and self.gxx == "missing":
            raise FileNotFoundError("g++")
        rc = self.gxx if name == "g++" else 0
        if rc == 0:
            open(cmd[cmd.index("-o") + 1], "w").close()
        return types.SimpleNamespace(returncode=rc, stdout="", stderr="no Python.h" if rc else "")

    def __call__(self, **kw):
        self.ran.clear()
        with warnings.catch_warnings(record=True) as seen:
            warnings.simplefilter("always")
            assert self.m.build(**kw) == self.m.LIB
        assert os.path.exists(self.m.LIB)
        self.warned = [str(w.message) for w in seen]
        return self.ran.count("nvcc"), self.ran.count("link"), self.ran.count("g++"), os.path.exists(self.m.TORCH_OPS)


@pytest.fixture
def build(tmp_path):
    return _Build(tmp_path)


def test_torch_without_cuda_and_no_torch(build):
    """The library does without torch: a torch for the CPU alone, or none, is no reason for it to fail."""
    units = len(build.m._sources())
    build.gxx = 1
    assert build() == (units, 1, 0, False) and not build.warned
    build.m._torch_folder = lambda: None
    assert build(force=True) == (units, 1, 0, False) and not build.warned


@pytest.mark.parametrize("how", [1, "missing"])
def test_extension_that_cannot_be_built(build, how):
    """The library is there all the same; the extension's failure is a warning, its old file does not stay, and the next call tries again."""
    build.with_cuda()
    assert build()[2:] == (1, True)
    (build.torch / "version.py").write_text("2.0")
    build.gxx = how
    assert build() == (0, 0, 1, False) and "torch_ops.cpp" in build.warned[0]
    build.gxx = 0
    assert build() == (0, 0, 1, True) and not build.warned
    assert build() == (0, 0, 0, True)


def test_what_is_made_again(build):
    build.with_cuda()
    units = len(build.m._sources())
    assert build() == (units, 1, 1, True)
    assert build() == (0, 0, 0, True)
    (build.torch / "version.py").write_text("1.1")   # another torch: its extension alone
    assert build() == (0, 0, 1, True)
    os.remove(build.m.TORCH_OPS)
    assert build() == (0, 0, 1, True)
    build.m.FLAGS = build.m.FLAGS + ["-DX"]
    assert build() == (units, 1, 0, True)
    assert build(force=True) == (units, 1, 1, True)
