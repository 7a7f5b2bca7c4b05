"""The extension for torch tensors is built where there is a torch with CUDA, again for another torch, and after all that needs none."""
import importlib.util
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture
def build(tmp_path):
    """build.py with its outputs in an empty folder and commands that only touch what they would write."""
    spec = importlib.util.spec_from_file_location("build_under_test", ROOT / "quanta.cpp_b200" / "build.py")
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    b.BUILD, b.LIB = tmp_path / "_build", tmp_path / "lib"
    b.made = []

    def run(cmd):
        out = Path(cmd[cmd.index("-o") + 1])
        out.write_text("")
        b.made.append(out.name)

    b._run = run
    return b


def folder_of_torch(tmp_path, name, with_cuda):
    """A package `torch` that is nothing but its files."""
    d = tmp_path / name / "torch"
    (d / "lib").mkdir(parents=True)
    (d / "__init__.py").write_text("class _C:\n    _GLIBCXX_USE_CXX11_ABI = True\n")
    (d / "lib" / "libtorch_cpu.so").write_text("")
    if with_cuda:
        (d / "lib" / "libtorch_cuda.so").write_text("")
    info = tmp_path / name / "torch-9.9.dist-info"
    info.mkdir()
    (info / "METADATA").write_text(f"Metadata-Version: 2.1\nName: torch\nVersion: 9.{name}\n")
    return tmp_path / name


def use(monkeypatch, where):
    for m in [m for m in sys.modules if m == "torch" or m.startswith("torch.")]:
        monkeypatch.delitem(sys.modules, m)
    monkeypatch.syspath_prepend(str(where))


def test_torch_without_cuda(build, monkeypatch, tmp_path):
    use(monkeypatch, folder_of_torch(tmp_path, "cpu", with_cuda=False))
    build.build()
    assert "quanta_b200" in build.made and "quanta_b200_torch.so" not in build.made


def test_the_driver_does_not_wait_for_the_extension(build):
    build.build()
    assert build.made.index("quanta_b200") < build.made.index("quanta_b200_torch.so")


def test_built_again_for_another_torch(build, monkeypatch, tmp_path):
    with monkeypatch.context() as m:
        use(m, folder_of_torch(tmp_path, "1", with_cuda=True))
        build.build()
        assert "quanta_b200_torch.so" in build.made
        build.made.clear()
        build.build()
        assert build.made == []
    with monkeypatch.context() as m:
        use(m, folder_of_torch(tmp_path, "2", with_cuda=True))
        build.build()
        assert build.made == ["quanta_b200_torch.so"]


def test_the_phase_timed_library_has_one_of_its_own(build, tmp_path):
    build.PKG = tmp_path
    build.build(stamps=True)
    assert "quanta_b200_torch.so" in build.made and (tmp_path / "lib_stamps" / "quanta_b200_torch.so").exists()
