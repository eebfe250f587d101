"""A call that the device refuses fails alone."""

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

import mojodgl.ops as ops  # noqa: E402
from mojodgl import _lib  # noqa: E402


def test_a_failed_call_leaves_nothing_for_the_next_one():
    lib = _lib.lib()
    x = torch.randn(8, 64, device="cuda")
    clean = ops.layer_norm(x)
    handle, offset, opened = ctypes.create_string_buffer(64), ctypes.c_int64(), ctypes.c_void_p()
    assert lib.bgl_ipc_export(x.data_ptr(), x.numel() * 4, handle, ctypes.byref(offset)) == 0
    # a buffer cannot be opened by the process that it belongs to: the runtime says so
    assert lib.bgl_ipc_open(handle, offset.value, x.numel() * 4, ctypes.byref(opened)) != 0
    assert b"cudaIpcOpenMemHandle" in lib.bgl_last_error()
    assert torch.equal(ops.layer_norm(x), clean)
