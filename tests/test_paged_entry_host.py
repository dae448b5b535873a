"""The paged cache's sources, build, imports and size checks, without a GPU."""
import ctypes
import os
import re
import shutil
import subprocess
import sys

import pytest

from smlm_b200 import _lib as L

PKG = os.path.dirname(os.path.dirname(os.path.abspath(L.__file__)))
P = ctypes.c_void_p(0x1000)      # never dereferenced: the checks fail before any launch


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


def attention(batch, hq, hkv, blocks, page=16, window=0, sinks=0):
    """Without scratch: a call that passes the checks and takes the list is refused for that."""
    strides = (ctypes.c_int64 * 6)(1024, 512, 64, 1024, 512, 64)
    return L.lib().smlm_paged_attention(P, P, P, L.BF16, strides, P, blocks, P, batch, hq, hkv, 64, 8, page, blocks,
                                        0.125, window, sinks, P, None, None, 0, None, None)


@pytest.mark.parametrize("args", [
    dict(batch=1024, hq=64, hkv=8, blocks=131072 * 2),                            # 8192 items of 131073 tiles
    dict(batch=65535, hq=32, hkv=4, blocks=65536, window=1024, sinks=4),          # 262140 items of at most 40 tiles
    dict(batch=4000, hq=4096, hkv=4, blocks=1024)])
def test_attention_takes_what_its_list_of_tiles_can_hold(args):
    """The list has one item per key head and up to 16 query heads of it, and a window bounds an item's tiles."""
    assert attention(**args) == L.ERR_WORKSPACE, L.lib().smlm_last_error()


@pytest.mark.parametrize("args", [dict(batch=65535, hq=64, hkv=64, blocks=65536),
                                  dict(batch=65535, hq=4096, hkv=4096, blocks=256),
                                  dict(batch=65535, hq=1024, hkv=1024, blocks=65536, window=4096)])
def test_attention_refuses_more_than_31_bits_of_tiles(args):
    assert attention(**args) == L.ERR_INVALID and b"fewer rows" in L.lib().smlm_last_error()
