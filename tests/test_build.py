"""librbq_torch.so is tied to the torch that it was compiled against; librbq.so and the index are not."""
import os
import shutil
import subprocess
import sys

import pytest

from neurosamble_b200 import _lib, build_ext, torch_ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_library_is_stale_under_another_torch(tmp_path, monkeypatch):
    assert _lib.TORCH_VERSION_PATH == build_ext.TORCH_VERSION and _lib.TORCH_LIB_PATH == build_ext.TORCH_LIB
    lib, version = tmp_path / "librbq_torch.so", tmp_path / "librbq_torch.so.torch"
    monkeypatch.setattr(build_ext, "TORCH_LIB", str(lib))
    monkeypatch.setattr(build_ext, "TORCH_VERSION", str(version))
    assert build_ext._torch_stale()
    lib.write_bytes(b"")
    assert build_ext._torch_stale()  # no record of its torch
    version.write_text("0.0.1\n")
    assert build_ext._torch_stale()
    version.write_text(build_ext.torch_version() + "\n")
    assert not build_ext._torch_stale()
    os.utime(lib, (1, 1))
    assert build_ext._torch_stale()  # older than its sources


def test_another_torch_leaves_the_index_usable(tmp_path):
    """The package imports, says what is missing and how to get it, and keeps the index and its operators."""
    package = tmp_path / "neurosamble_b200"
    shutil.copytree(os.path.join(ROOT, "neurosamble_b200"), package, ignore=shutil.ignore_patterns("_lib", "csrc", "__pycache__"))
    (package / "_lib").mkdir()
    (package / "_lib" / "librbq_torch.so").write_bytes(b"not to be read")
    (package / "_lib" / "librbq_torch.so.torch").write_text("0.0.1\n")
    code = ("import warnings, torch\n"
            "with warnings.catch_warnings(record=True) as seen:\n"
            "    warnings.simplefilter('always')\n"
            "    import neurosamble_b200 as n\n"
            "said = [str(w.message) for w in seen if 'build_ext' in str(w.message)]\n"
            "assert len(said) == 1 and 'against torch 0.0.1' in said[0], said\n"
            "assert n.IndexIVFRaBitQ and hasattr(torch.ops.rbq, 'search') and not hasattr(torch.ops.rbq, 'linear')\n")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=tmp_path)


def test_a_library_that_cannot_be_loaded_is_a_warning(tmp_path, monkeypatch):
    bad = tmp_path / "librbq_torch.so"
    bad.write_bytes(b"not a library")
    monkeypatch.setattr(_lib, "TORCH_LIB_PATH", str(bad))
    with pytest.warns(UserWarning, match="build_ext"):
        assert not torch_ops._load_encoder_operators()
    monkeypatch.setattr(_lib, "TORCH_LIB_PATH", str(tmp_path / "none.so"))
    assert not torch_ops._load_encoder_operators()


def test_what_is_built_when(monkeypatch):
    """Each library when it is out of date, and the operators of torch only with torch."""
    done = []
    monkeypatch.setattr(build_ext, "build_library", lambda verbose=False: done.append("rbq"))
    monkeypatch.setattr(build_ext, "build_torch", lambda: done.append("torch"))
    for stale, torch_stale, version, want in [(False, False, "2", []), (False, True, "2", ["torch"]), (True, False, "2", ["rbq"]),
                                              (True, True, "2", ["rbq", "torch"]), (True, True, "", ["rbq"])]:
        monkeypatch.setattr(build_ext, "_stale", lambda: stale)
        monkeypatch.setattr(build_ext, "_torch_stale", lambda: torch_stale)
        monkeypatch.setattr(build_ext, "torch_version", lambda: version)
        done.clear()
        assert build_ext.build() == build_ext.LIB and done == want
