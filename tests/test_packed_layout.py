"""What the packed cache's kernels lay out, as far as it shows without a GPU."""

import ctypes
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ferrisinfer_b200", "csrc")


@pytest.mark.parametrize("file", ["packed_cache.cu", "packed_attention.cu"])
def test_shared_memory_that_is_read_by_16_bytes_begins_on_16(file):
    """Dynamic shared memory stands behind the static: where it begins is the declaration's alignment, and no more."""
    source = open(os.path.join(CSRC, file)).read()
    found = re.findall(r"extern __shared__ ([^;]*);", source)
    assert found and all("__align__(16)" in one for one in found), found
