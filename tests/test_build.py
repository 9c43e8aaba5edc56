"""build.py: the Python extension module beside the C libraries."""
import importlib.util
from pathlib import Path
from types import SimpleNamespace

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture
def build(monkeypatch, tmp_path):
    """build.py with its commands recorded instead of run, its outputs under tmp_path, and a torch for CUDA there."""
    spec = importlib.util.spec_from_file_location("exl3_build", ROOT / "xiaomi-hexagon-exl3_b200" / "build.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    (tmp_path / "torch" / "lib").mkdir(parents=True)
    (tmp_path / "torch" / "lib" / "libc10_cuda.so").touch()
    (tmp_path / "torch" / "version.py").write_text("__version__ = '2.11.0+cu128'\n")
    mod.TORCH_LIB, mod.BUILD = tmp_path / "exl3cu_torch.so", tmp_path
    mod.commands = []

    def run(cmd):
        mod.commands.append(cmd)
        mod.TORCH_LIB.touch()

    mod._run = run
    mod.found = SimpleNamespace(origin=str(tmp_path / "torch" / "__init__.py"))
    monkeypatch.setattr(mod.importlib.util, "find_spec", lambda name: mod.found)
    mod.package = tmp_path / "torch"
    return mod


CC = "/usr/local/cuda/bin/nvcc"


@pytest.mark.skipif(not (Path(importlib.import_module("sysconfig").get_paths()["include"]) / "Python.h").exists(),
                    reason="no Python headers")
class TestTorchModule:
    def test_is_built_once(self, build):
        assert build.build_torch_module(CC) and len(build.commands) == 1
        assert build.build_torch_module(CC) and len(build.commands) == 1
        assert build.build_torch_module(CC, force=True) and len(build.commands) == 2

    def test_is_built_again_for_another_torch_or_python(self, build, monkeypatch):
        assert build.build_torch_module(CC) and "2.11.0+cu128" in " ".join(build.commands[0])
        (build.package / "version.py").write_text("__version__ = '2.12.0+cu130'\n")
        assert build.build_torch_module(CC) and "2.12.0+cu130" in " ".join(build.commands[1])
        assert build.build_torch_module(CC) and len(build.commands) == 2
        monkeypatch.setattr(build.sysconfig, "get_config_var", lambda name: "cpython-399-none")
        assert build.build_torch_module(CC) and "cpython-399-none" in " ".join(build.commands[2])

    def test_is_built_again_after_a_build_that_failed(self, build, monkeypatch):
        def fail(cmd):
            build.TORCH_LIB.touch()
            raise RuntimeError

        with monkeypatch.context() as m:
            m.setattr(build, "_run", fail)
            with pytest.raises(RuntimeError):
                build.build_torch_module(CC)
        assert build.build_torch_module(CC) and len(build.commands) == 1

    def test_is_left_out_without_torch(self, build, capsys):
        build.found = None
        assert not build.build_torch_module(CC, force=True)
        assert "torch is not installed" in capsys.readouterr().err and not build.commands

    def test_is_left_out_without_cuda(self, build, capsys):
        (build.package / "lib" / "libc10_cuda.so").unlink()
        assert not build.build_torch_module(CC)
        assert "not one for CUDA" in capsys.readouterr().err and not build.commands


def test_build_without_torch_still_makes_the_c_libraries(build, monkeypatch, tmp_path):
    """All of build(), its commands recorded: without torch it ends with the library as ever."""
    build.found = None
    monkeypatch.setattr(build, "nvcc", lambda: CC)
    monkeypatch.setattr(build, "LIB", tmp_path / "libexl3cu.so")
    monkeypatch.setattr(build, "GGML_LIB", tmp_path / "libexl3cu_ggml.so")
    monkeypatch.setattr(build, "_newer", lambda target, deps: True)

    def run(cmd):
        build.commands.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).touch()
        return ""

    monkeypatch.setattr(build, "_run", run)
    assert build.build() == tmp_path / "libexl3cu.so"
    made = {Path(c[c.index("-o") + 1]).name for c in build.commands}
    assert {"libexl3cu.so", "libexl3cu_ggml.so"} <= made and "exl3cu_torch.so" not in made


def test_module_of_another_torch_is_refused(monkeypatch):
    """What was built says for which torch and Python; loaded into another, an error names both."""
    import torch
    from exl3_b200 import attention

    attention._native()  # as built
    monkeypatch.setattr(torch, "__version__", "1.2.3")
    with pytest.raises(ImportError, match="built for .*" + str(attention._native().built_for.split()[-1]).replace("+", "\\+") + ".*1.2.3"):
        attention._native.__wrapped__()
