"""Which rows the calls that move cache rows take, before any CUDA call (no slots: nothing is launched)."""
import ctypes as C

import pytest

from semi_pd_b200 import _lib

MB = 1 << 20


@pytest.mark.parametrize("row_bytes,planes,code", [
    (MB, 1, 0), (MB + 16, 1, 0), (2 * MB, 32, 0), (4 * MB + 6, 3, 0), (1 << 30, 1, 0),
    (MB + 1, 1, -2),                    # an odd number of bytes
    ((1 << 30) + 2, 1, -3),             # longer than any row
    (32768, 65534, 0), (32770, 32767, 0), (32770, 32768, -3), (2 * MB, 1024, -3)])
def test_lengths(row_bytes, planes, code):
    buf = (C.c_char * 64)()
    p = (C.addressof(buf) + 15) & ~15
    s = _lib.KVPlaneSet(p, 4 * row_bytes // 2 * 2, 4, row_bytes, planes)
    assert _lib.lib.spd_kv_copy(C.addressof(s), 1, None, None, 0, None) == code
