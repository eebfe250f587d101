"""The element type that operands of mixed types are worked on in: read from the
types, without a converted copy."""

import numpy as np
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from mojodgl import _tensor as T
from mojodgl.base import DGLError


class Count(TorchDispatchMode):
    calls = 0

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.calls += 1
        return func(*args, **(kwargs or {}))


F16, BF16, F32, F64 = (torch.ones(4, 6, dtype=t) for t in (torch.float16, torch.bfloat16, torch.float32, torch.float64))


@pytest.mark.parametrize("operands,want", [
    ((F16,), torch.float32), ((BF16, F32), torch.float32), ((F32, BF16, F16), torch.float32), ((BF16, BF16), torch.bfloat16),
    ((F32.t(), F16.t()), torch.float32), ((F64[:, ::2], BF16), torch.float64), ((F16, F64), torch.float64)])
def test_no_operand_is_copied_to_read_its_type(operands, want):
    with Count() as count:
        assert T.float_type(*operands) == want
    assert count.calls == 0


def test_numpy_and_whole_numbers():
    a = np.ones((3, 2))
    assert T.float_type(a.astype(np.float32)) == T.float_type(a.astype(np.float32), BF16) == torch.float32
    assert T.float_type(a) == T.float_type(a.astype(np.float16)) == T.float_type(a.astype(np.int32), F32) == torch.float64
    assert T.float_type(torch.ones(3, dtype=torch.int32)) == torch.float64
    for bad in (a.astype(np.complex64), torch.ones(2, dtype=torch.complex64), np.array([2 ** 53 + 1], dtype=np.uint64)):
        with pytest.raises(DGLError):
            T.float_type(bad)
        with pytest.raises(DGLError):
            T.float_type(F32, bad)
