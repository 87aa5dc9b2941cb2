"""The 8-bit layer operators' refusals and workspace sizes that need no GPU, beside tests/test_lowbit_cpu.py."""
import pytest
import torch

from nicecore import _lib as L
from nicecore import lowbit


def test_a_bias_that_requires_grad_is_refused():
    """quantized_linear has no gradient for the bias either: dropping it silently would freeze it."""
    rows = lowbit.CodedRows(torch.zeros(4, 128, dtype=torch.uint8), torch.ones(4), 8, torch.Size([4]), torch.float32,
                            L.NC_CODES_ROW)
    bias = torch.zeros(4, requires_grad=True)
    with pytest.raises(L.NiceCoreError, match="bias.detach"):
        lowbit.quantized_linear(rows, rows, bias)
    with torch.no_grad(), pytest.raises(L.NiceCoreError, match="bias must be"):  # (taken; the next check's turn)
        lowbit.quantized_linear(rows, rows, torch.zeros(3, requires_grad=True))
