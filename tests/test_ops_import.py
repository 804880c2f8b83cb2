"""The operator module without the library of the drafted-tree operators, and when that library is built anew."""
import importlib.util
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import torch
import exact_llm_b200.ops as ops
with torch._subclasses.fake_tensor.FakeTensorMode():
    y = torch.ops.exact.gemv(torch.empty(256, dtype=torch.int16), torch.empty(8, 256, dtype=torch.int8),
                             torch.empty(8, 2, dtype=torch.int64))
assert y.shape == (8,) and y.dtype == torch.int64
assert ops.tree_masks([-1, 0], [0, 2]).tolist() == [[1], [3]]
for name in ("tree_attention", "tree_verify", "kv_compact_", "kv_copy_pages_"):
    try:
        getattr(torch.ops.exact, name)(1, 2, three=3)
    except ImportError as e:
        assert name in str(e) and "build.py" in str(e) and "libexactb200_torch.so" in str(e), e
    else:
        raise AssertionError(name)
"""


@pytest.mark.parametrize("there", ["nothing", "not a library", "another library"])
def test_ops_without_the_torch_library(tmp_path, there):
    """exact::gemv needs libexactb200.so alone: the import works, and only the operators that are missing raise."""
    pytest.importorskip("torch")
    pkg = tmp_path / "exact_llm_b200"
    pkg.mkdir()
    for f in os.listdir(os.path.join(ROOT, "exact_llm_b200")):
        if f.endswith(".py") or f == "libexactb200.so":
            os.symlink(os.path.join(ROOT, "exact_llm_b200", f), pkg / f)
    lib = pkg / "libexactb200_torch.so"
    if there == "not a library":
        lib.write_bytes(b"not a library")
    elif there == "another library":                         # it loads, and has no entry to bind
        src = tmp_path / "empty.c"
        src.write_text("int nothing;\n")
        subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(lib), str(src)], check=True)
    (tmp_path / "use.py").write_text(PROGRAM)
    r = subprocess.run([sys.executable, str(tmp_path / "use.py")], cwd=tmp_path, capture_output=True, text=True,
                       env=dict(os.environ, PYTHONPATH=str(tmp_path)), timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


def test_torch_library_is_built_anew_for_another_torch(tmp_path, monkeypatch):
    torch = pytest.importorskip("torch")
    spec = importlib.util.spec_from_file_location("exb_build_copy", os.path.join(ROOT, "exact_llm_b200", "build.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    calls = []

    def compiler(cmd, **kw):
        calls.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("library")

    monkeypatch.setattr(b, "TORCH_LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(b, "OBJ", str(tmp_path / "obj"))
    monkeypatch.setattr(b.subprocess, "run", compiler)
    for version, builds in (("9.1", 1), ("9.1", 1), ("9.2", 2), ("9.2", 2), ("9.1", 3)):
        monkeypatch.setattr(torch, "__version__", version)
        assert b.build_torch() == str(tmp_path / "lib.so") and len(calls) == builds, version
    b.build_torch(force=True)
    assert len(calls) == 4
