"""What the block-scaled kernels' sources may not contain."""
import re
from pathlib import Path

import pytest

from h3b import _lib


@pytest.mark.parametrize("name", ["blocks.cu", "gemm_blocks.cu"])
def test_kernels_that_start_early_read_by_plain_loads(name):
    """These kernels may run while the kernel ahead of them writes their inputs, so no load may take them for constant."""
    code = re.sub(r"//[^\n]*", "", (Path(_lib.__file__).parents[1] / "csrc" / name).read_text())
    assert "pdl_wait()" in code
    assert not re.findall(r"__ldg|\.nc\b|const\s+\w+\s*\*\s*__restrict__", code)
