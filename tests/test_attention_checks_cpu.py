"""Host-side checks of the attention calls that need no GPU."""
import ctypes

import pytest
import torch

from reax_engine_b200 import _lib as L
from reax_engine_b200 import attention as A
from test_attention_cpu import call


def test_an_empty_output_shares_nothing():
    """Empty tensors all have the data pointer 0."""
    q = torch.empty(0, 4, 64, dtype=torch.bfloat16)
    for out in (torch.empty(0, 4, 64, dtype=torch.bfloat16), q):
        assert A._output(out, q, (q, q, q)) is out
    t = torch.empty(3, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        A._output(t[1:], t[:2], (t,))
