"""The torch module of the row operators: what is built, and what is there without it."""
import subprocess
import sys
import types

import pytest

from hephaestus_b200 import build


def test_the_other_torch_entry_points_do_not_need_it():
    code = """
import sys
class Absent:
    def find_spec(self, name, path=None, target=None):
        if name == "hephaestus_b200._torch_rows":
            raise ImportError("not here")
sys.meta_path.insert(0, Absent())
import torch
from hephaestus_b200 import InvalidConfiguration, torch_ops as T
x = torch.ones(4, 4)
for call in (T.sum, T.cumsum, lambda t: T.argmax_axis(t, 0)):
    try:
        call(x)
    except InvalidConfiguration as e:
        assert "needs CUDA tensors" in str(e), e
try:
    T.rms_norm(x)
except ImportError as e:
    assert "rms_norm needs" in str(e) and "not here" in str(e), e
    print("as it should be")
"""
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert out.returncode == 0 and "as it should be" in out.stdout, out.stderr


@pytest.fixture
def compiler(monkeypatch, tmp_path):
    """A host compiler that fails, and an older module in a folder of its own."""
    module = tmp_path / "_torch_rows.so"
    module.write_text("older")
    monkeypatch.setattr(build, "TORCH_MODULE", str(module))
    monkeypatch.setattr(build, "nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    said = types.SimpleNamespace(module=module, cmd=None)

    def run(cmd, **kw):
        said.cmd = cmd
        return types.SimpleNamespace(returncode=1, stderr="no Python.h")

    monkeypatch.setattr(build.subprocess, "run", run)
    return said


def test_a_module_that_does_not_compile_is_left_out(compiler, capsys):
    build._torch_module_or_note(True)  # the library stays good
    err = capsys.readouterr().err
    assert "_torch_rows.so" in err and "left out" in err and "no Python.h" in err
    assert not compiler.module.exists()
    with pytest.raises(RuntimeError, match="no Python.h"):
        build.build_torch_module(True)


def test_it_is_built_for_the_installed_torch(compiler, monkeypatch):
    import torch
    for abi in (True, False):
        monkeypatch.setattr(torch, "compiled_with_cxx11_abi", lambda: abi)
        with pytest.raises(RuntimeError):
            build.build_torch_module(True)
        assert f"-D_GLIBCXX_USE_CXX11_ABI={int(abi)}" in compiler.cmd


def test_without_a_cuda_torch_it_is_left_out(monkeypatch, capsys):
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda name: None)
    build._torch_module_or_note()
    assert "left out: no CUDA build of torch" in capsys.readouterr().err
