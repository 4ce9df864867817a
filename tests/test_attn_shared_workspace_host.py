"""attn_decode_shared refuses a workspace that its kernels could not address, before any CUDA call."""
import ctypes as C

import pytest

from semi_pd_b200 import _lib


@pytest.mark.parametrize("offset", [1, 2, 4, 8])
@pytest.mark.parametrize("tokens", [False, True])
def test_alignment(offset, tokens):
    lib = _lib.lib
    buf = (C.c_char * 4096)()
    p = (C.addressof(buf) + 15) & ~15
    need = lib.spd_attn_decode_shared_workspace_bytes(4, 8, 2, 128)
    args = (p, p, p, p, p, p, p, p, p, 4, 1)
    rest = (64, 8, 2, 128, 1024, 1024, 8, 0.1, 0, p + offset, need, 0, None)
    if tokens:
        assert lib.spd_attn_decode_shared_tokens(*args, 0, 0, 0, 0, *rest) == -2
    else:
        assert lib.spd_attn_decode_shared(*args, 512, *rest) == -2
    assert b"aligned" in lib.spd_last_error_string()
