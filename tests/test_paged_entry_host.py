"""The paged cache's sources, without a GPU."""
import os
import re

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
