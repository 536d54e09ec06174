"""What can be seen of the 8-bit operators' calls without a GPU."""

import re

from pare_b200.kernels import _lib

CSRC = _lib.LIB_PATH.parent.parent / "csrc"


def _code(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


def test_the_cache_is_not_read_as_read_only_memory():
    """Each kernel of the paged cache is launched while the one before it still writes, so the loads that need memory that nobody writes while the
    kernel lives are out of place there."""
    for name in ("paged_cache.cu", "paged_attn.cu"):
        found = re.findall(r"ld_stream_v4|__ldg\b|ld\.global(?:\.\w+)*\.nc\b|__restrict__", _code(name))
        assert not found, (name, found)
