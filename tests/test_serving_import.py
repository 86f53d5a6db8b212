"""What a missing or unfitting library of the serving ops means: other modules work, a serving op says why it
does not."""

import os
import shutil
import subprocess
import sys

import pytest

from conftest import ROOT

PROBE = """
import torch, mzoo_b200
from mzoo_b200 import _lib, csa2_attn, gqa_attn, indexer, kv_pages, ops, sparse_mla, swa_attn
from torch._subclasses.fake_tensor import FakeTensorMode
assert mzoo_b200.__file__.startswith({here!r}) and not _lib.torch_ops_loaded
with FakeTensorMode():
    q = torch.empty(3, 2, 64, dtype=torch.bfloat16, device="cuda:0")
    assert gqa_attn.prefill(q, q, q, torch.empty(2, dtype=torch.int32, device="cuda:0"))[0].shape == q.shape
try:
    ops._launch("x", torch.zeros(1), False, lambda err: None)
except ImportError as e:
    print(e)
"""


@pytest.mark.parametrize("files,why", [((), "is missing"), (("libmzb200_torch.so",), "libmzb200.so is missing"),
                                       (("libmzb200.so", "libmzb200_torch.so"), "does not fit this package")])
def test_import_without_the_libraries(tmp_path, files, why):
    here = tmp_path / "mzoo_b200"
    shutil.copytree(os.path.join(ROOT, "mzoo_b200"), here, ignore=shutil.ignore_patterns("*.so", "*.tmp", "csrc", "__pycache__"))
    for name in files:
        (here / name).write_text("not a library")
    r = subprocess.run([sys.executable, "-c", PROBE.format(here=str(tmp_path))], cwd=tmp_path, capture_output=True, text=True,
                       env={**os.environ, "PYTHONPATH": str(tmp_path)})
    assert r.returncode == 0, r.stderr
    assert why in r.stdout


def test_a_library_of_other_sources_is_named(tmp_path):
    """A library without the entry that this package calls (an older build)."""
    src, lib = tmp_path / "old.c", tmp_path / "libmzb200_torch.so"
    src.write_text("int mzb_torch_register(void) { return 0; }")
    subprocess.run(["gcc", "-shared", "-fPIC", str(src), "-o", str(lib)], check=True)
    code = ("from mzoo_b200 import _lib, build\n"
            "build.build()\n"
            f"_lib.TORCH_LIB_PATH, _lib.torch_ops_loaded = {str(lib)!r}, False\n"
            "try:\n    _lib.load_torch_ops()\nexcept ImportError as e:\n    print(e)\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert "does not fit this package" in r.stdout and "--force" in r.stdout
