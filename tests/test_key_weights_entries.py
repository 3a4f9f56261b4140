"""The C entries for the weights of keys take the rows that their rules give them, and refuse more before anything runs."""
import ctypes

import pytest
import torch

from photon_infer_b200.csrc.build import compile_module
from photon_infer_b200.kernels import ops

UNSUPPORTED = -2


def _entry(name, tokens, group=4, dtype=1, packed=0, d=64, lse=256, scratch=256):
    """The status of a call that no kernel may see: its pointers are none."""
    call = ops._KEY_WEIGHTS_CALL.pack(256, 256, 256, 256, 256, 256, 0, 0, lse, scratch, 0, group * 2 * d, 64, dtype, packed, 4, 1, 64, 2 * group, 2, d, 16, 4, 0, 1, tokens, 0, 0.125, 0.0)
    f = getattr(ctypes.CDLL(compile_module(name)), "photon_" + name)
    f.argtypes, f.restype = [ctypes.c_char_p, ctypes.c_void_p], ctypes.c_int
    return f(call, None)


@pytest.mark.skipif(torch.cuda.is_available(), reason="pointers to nothing: only where no kernel can run")
@pytest.mark.parametrize("lse", [0, 256])
@pytest.mark.parametrize("packed", [0, 1])
@pytest.mark.parametrize("name,dtype,most", [("key_weights", 0, 8), ("key_weights", 1, 8), ("key_weights_mma", 1, 32)])
def test_more_rows_are_refused(name, dtype, most, packed, lse):
    for tokens, group in ((most // 4 + 1, 4), (most + 1, 1), (1, most + 1), (4096, 4)):
        assert _entry(name, tokens, group, dtype, packed, lse=lse) == UNSUPPORTED
    assert _entry(name, 0, 4, dtype, packed, lse=lse) == 0               # nothing to do


def test_the_rule_keeps_to_them():
    for dtype in (torch.bfloat16, torch.float32):
        for d in (64, 96, 128):
            for rows in range(1, 70):
                for packed in (False, True):
                    for known in (False, True):
                        name = ops._key_weights_route(dtype, d, 16, 1000, packed, known, 3, 2, rows, 500, 100, 148)[0]
                        assert rows <= {"key_weights": 8, "kv4_key_weights": 8, "key_weights_mma": 32}.get(name, 1 << 30)
