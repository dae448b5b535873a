"""The paged cache's sources, build and imports, without a GPU."""
import os
import re
import shutil
import subprocess
import sys

import pytest

from smlm_b200 import _lib as L

PKG = os.path.dirname(os.path.dirname(os.path.abspath(L.__file__)))


@pytest.mark.parametrize("name", ["paged.cuh", "paged_attn.cu", "pages.cu"])
def test_no_load_that_assumes_nobody_writes_while_the_kernel_runs(name):
    """These kernels begin while their predecessor, which writes pages and tables, still runs: the non-coherent load
    (ld.global.nc, __ldg, or what a compiler makes of a const __restrict__ pointer) is specified for memory that nobody
    writes during the kernel's whole life."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(PKG, "csrc", name)).read())
    assert not re.search(r"\.nc\b|__ldg\b|const\s+[\w:]+\s*\*\s*__restrict__|texture|tex1D", text)


def test_the_other_modules_work_without_the_paged_binding(tmp_path):
    """smlm_b200.decode (GraphDecoder) needs the C library alone; a call of the paged functions names what is missing."""
    shutil.copytree(os.path.join(PKG, "smlm_b200"), tmp_path / "smlm_b200",
                    ignore=shutil.ignore_patterns("_paged.so", "__pycache__"))
    code = ("import smlm_b200.decode as d, smlm_b200.paged as p, torch\n"
            "d.GraphDecoder, d.PagedDecoder, p.PagedKVCache\n"
            "try:\n    p.paged_attention(*[torch.zeros(1)] * 5)\n"
            "except ImportError as e:\n    assert '_paged.so' in str(e), e\n"
            "else:\n    raise SystemExit('no error')\n")
    env = dict(os.environ, PYTHONPATH=str(tmp_path))
    subprocess.run([sys.executable, "-c", code], check=True, env=env, cwd=tmp_path, timeout=300)


def test_the_default_build_needs_no_torch():
    """`make` alone builds the C library; the Python binding has a target of its own."""
    out = subprocess.run(["make", "-C", os.path.join(PKG, "csrc"), "-n", "-B", "PYTHON=/nonexistent"], check=True,
                         capture_output=True, text=True, timeout=60)
    assert "libsmlm_b200.so" in out.stdout and "binding.cpp" not in out.stdout and "nonexistent" not in out.stderr
    out = subprocess.run(["make", "-C", os.path.join(PKG, "csrc"), "-n", "-B", "binding", f"PYTHON={sys.executable}"],
                         check=True, capture_output=True, text=True, timeout=120)
    assert "binding.cpp" in out.stdout and "_paged.so" in out.stdout
