"""The build without torch, in directories of the test's own."""
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

from neural_block_textures_b200 import build as b


@pytest.fixture
def apart(tmp_path, monkeypatch):
    """The build's outputs below tmp_path, made of one quick source."""
    if not (shutil.which(b.nvcc()) or Path(b.nvcc()).exists()):
        pytest.skip("no nvcc")
    monkeypatch.setattr(b, "OUT_DIR", tmp_path / "lib")
    monkeypatch.setattr(b, "BUILD_DIR", tmp_path / "obj")
    monkeypatch.setattr(b, "LIB", tmp_path / "lib" / b.LIB.name)
    monkeypatch.setattr(b, "TORCH_LIB", tmp_path / "lib" / b.TORCH_LIB.name)
    monkeypatch.setattr(b, "SOURCES", ["ntcb_format.cpp"])
    return tmp_path


def test_without_torch_the_library_is_built(apart, monkeypatch, capsys):
    monkeypatch.setattr(b.importlib.util, "find_spec", lambda name: None)
    assert b.build() == b.LIB and b.LIB.exists() and not b.TORCH_LIB.exists()
    assert "torch is not installed" in capsys.readouterr().err


def test_without_python_headers_the_library_is_built(apart, monkeypatch, capsys):
    monkeypatch.setattr(b.sysconfig, "get_paths", lambda: {"include": str(apart / "nowhere")})
    assert b.build() == b.LIB and b.LIB.exists() and not b.TORCH_LIB.exists()
    assert "headers" in capsys.readouterr().err


def test_a_torch_that_does_not_compile_leaves_the_library(apart, monkeypatch):
    """The failure is raised, after the library that does not need torch was linked."""
    def failing():
        raise RuntimeError("these headers do not fit")
    monkeypatch.setattr(b, "_compile_torch_host", failing)
    with pytest.raises(RuntimeError, match="do not fit"):
        b.build()
    assert b.LIB.exists()


def test_another_torch_is_compiled_for_again(apart, monkeypatch):
    """The host side uses torch's C++ classes: an object of another torch, or of one that moved, does not stay."""
    from types import SimpleNamespace
    made = []

    def compiler(cmd, **kw):
        out = Path(cmd[cmd.index("-o") + 1])
        made.append(out.name)
        out.write_text("object")
        return SimpleNamespace(returncode=0, stdout="", stderr="")

    def torch(name, version):
        where = apart / name
        where.mkdir(exist_ok=True)
        (where / "version.py").write_text(f"__version__ = '{version}'\n")
        monkeypatch.setattr(b.importlib.util, "find_spec", lambda _: SimpleNamespace(submodule_search_locations=[str(where)]))
        before = len(made)
        b._compile_torch_host()
        return len(made) - before
    monkeypatch.setattr(b.subprocess, "run", compiler)
    b.BUILD_DIR.mkdir()
    assert [torch("a", "1.0"), torch("a", "1.0"), torch("a", "1.1"), torch("a", "1.1"), torch("b", "1.1"), torch("a", "1.1")] == [1, 0, 1, 0, 1, 1]


def test_star_import_does_without_torch():
    """`import *` gives the names that need no torch and loads none; the operators come by name."""
    code = ("import sys\n"
            "sys.modules['torch'] = None\n"   # an import of it raises
            "from neural_block_textures_b200 import *\n"
            "assert callable(Trainer) and callable(config) and 'neural_block_textures_b200.symbols' not in sys.modules\n"
            "import neural_block_textures_b200 as n\n"
            "assert 'AdamW' in dir(n) and 'symbol_logprobs' in dir(n) and 'AdamW' not in globals()\n"
            "try:\n"
            "    n.AdamW\n"
            "except ImportError:\n"
            "    print('fine')\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, cwd=b.ROOT)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr
