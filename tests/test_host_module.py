"""CPU: _host.so runs only beside the library and the sources that it was built from."""
import os
import shutil
import subprocess
import sys

import pytest

from framefusion_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_module_carries_the_hash_of_its_sources():
    assert _lib.host() is not None
    assert _lib.file_stamp(_lib.HOST_PATH) == _lib.file_stamp(_lib.LIB_PATH) == _lib.source_hash()
    assert "ff_host.cpp" in _lib.hashed_sources()


@pytest.fixture
def tree(tmp_path):
    """The package as built, its host module of another build."""
    _lib.host()
    pkg = tmp_path / "framefusion_amd"
    shutil.copytree(os.path.join(ROOT, "framefusion_amd"), pkg, ignore=shutil.ignore_patterns("*.o", "__pycache__"))
    shutil.copytree(os.path.join(ROOT, "include"), tmp_path / "include")
    blob = (pkg / "_host.so").read_bytes()
    stamp = b"FFSRCHASH:" + _lib.source_hash().encode()
    assert stamp in blob
    (pkg / "_host.so").write_bytes(blob.replace(stamp, b"FFSRCHASH:0123456789abcdef"))

    def run(**env):
        code = ("from framefusion_amd import _lib\n_lib.load()\n"
                "try:\n    _lib.host()\nexcept _lib.FrameFusionHipError as e:\n    print('refused:', e)\nelse:\n    print('loaded')")
        return subprocess.run([sys.executable, "-c", code], cwd=tmp_path, env={**os.environ, "PYTHONPATH": str(tmp_path), **env}, capture_output=True, text=True)
    return pkg, run


def test_a_module_of_other_sources_is_not_loaded(tree):
    pkg, run = tree
    out = run(FF_AUTO_BUILD="0")
    assert "refused:" in out.stdout and "0123456789abcdef" in out.stdout and "other sources" in out.stdout, out


def test_a_module_of_another_build_than_the_library_is_not_loaded(tree):
    """Without the sources nothing can be hashed: the module asks the library."""
    pkg, run = tree
    shutil.rmtree(pkg / "csrc")
    out = run()
    assert "refused:" in out.stdout and "0123456789abcdef" in out.stdout and "than the library beside it" in out.stdout, out


def test_the_library_alone_needs_no_torch_to_build():
    """make without a target is what a host of the C ABI runs; the package's own build makes both."""
    def commands(*target):
        return subprocess.run(["make", "-n", "-B", "-C", _lib.CSRC, *target], capture_output=True, text=True, check=True).stdout
    assert "-ltorch" not in commands() and "-o ../libframefusion_hip" in commands()
    assert "-ltorch" in commands("all")


def test_the_library_is_built_without_the_module(monkeypatch, tmp_path):
    """A process that only reduces prefills asks for the library alone, also where it has to build it."""
    asked = []
    monkeypatch.setattr(_lib, "build", lambda verbose=False, force=False, target="all": asked.append(target))
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setattr(_lib, "LIB_PATH", str(tmp_path / "nope.so"))
    with pytest.raises(_lib.FrameFusionHipError):
        _lib.load()
    assert asked and set(asked) == {"lib"}
