"""What can be seen of the 8-bit operators' calls without a GPU."""

import ctypes
import re

import pytest

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


@pytest.mark.parametrize("block_size,heads", [(64, 32768), (64, 65535)])
def test_more_heads_than_a_grid_has_room_for(block_size, heads):
    buf = (ctypes.c_char * 4160)()
    p = (ctypes.addressof(buf) + 63) // 64 * 64                # never read: the call is refused first
    layer = _lib.PagedLayerStruct(p, p, p, p, p, p, 4, 2, heads, block_size, 128, 0)
    tables = _lib.PagedTablesStruct(p, p, 4, 4, 2, 2, block_size)
    got = _lib.lib().pare_paged_append(p, p, heads * 128, 128, heads * 128, 128, ctypes.addressof(layer), ctypes.addressof(tables), None)
    assert got == _lib.UNSUPPORTED
