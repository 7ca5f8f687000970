"""A library without the hybrid layers' entry points (include/ns_layer.h) - one that an engine built before they were there - loads as it did, and says
which one is missing where one is called."""
import ctypes as C
import types

import pytest

from nextsycl_amd import Error
from nextsycl_amd.attn import ATTN_H, LAYER_H, Kernels, Ops


class Library:
    """An Api whose entry points all return 0, but for those it lacks."""

    def __init__(self, lacks):
        self.lacks = lacks

    def symbol(self, name, restype, argtypes):
        if name in self.lacks:
            raise OSError("lib.so: missing symbol " + name)
        return C.CFUNCTYPE(restype, *argtypes)(lambda *a: 0)

    def error(self):
        return ""


def buffers():
    return types.SimpleNamespace(ptr=4096, len=1 << 20)


def test_a_library_without_the_layers_loads():
    ops = Ops(types.SimpleNamespace(raw=C.c_void_p(4096), handle=4096), Kernels(Library(set(LAYER_H))))
    b = buffers()
    for call, name in ((lambda: ops.norm_gated(0, b, 16, b, 16, None, b, 16, 1, 16, 1, 1e-5), "ns_norm_gated"),
                       (lambda: ops.norm_residual(0, 0, b, 16, b, 16, b, 16, b, 16, 1, 16, 1e-5), "ns_norm_residual"),
                       (lambda: ops.ssm_prompt_scratch(1, 1, 1, 1, 1, 1), "ns_ssm_prompt_scratch"), (lambda: ops.q4_bytes(1, 1, 32), "ns_q4_bytes"),
                       (lambda: ops.q4_pack(0, b, 16, 1, 16, 32, b), "ns_q4_bytes"), (lambda: ops.q4_product(0, b, 16, b, 32, b, 16, 1, 16, 16), "ns_q4_bytes"),
                       (lambda: ops.ssm_step(0, b, 6, b, 1, b, None, b, None, None, b, 4, 0, 1, 1, 2, 2, 1, 1, None, b, b, 2), "ns_ssm_step")):
        with pytest.raises(Error, match="missing symbol " + name):
            call()


def test_one_that_lacks_some_of_them_calls_the_others():
    ops = Ops(types.SimpleNamespace(raw=C.c_void_p(4096), handle=4096), Kernels(Library({"ns_ssm_step"})))
    b = buffers()
    ops.norm_gated(0, b, 16, b, 16, None, b, 16, 1, 16, 1, 1e-5)
    with pytest.raises(Error, match="missing symbol ns_ssm_step"):
        ops.ssm_step(0, b, 6, b, 1, b, None, b, None, None, b, 4, 0, 1, 1, 2, 2, 1, 1, None, b, b, 2)


def test_the_attention_entry_points_stay_required():
    with pytest.raises(OSError, match="missing symbol"):
        Kernels(Library({next(iter(ATTN_H))}))
