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


def test_backward_workspace_goes_by_its_outputs():
    """Frozen parts of a layer cost no scratch: dW's parts and decoded values only with dW, W^T only with dx; more
    outputs never need less."""
    import ctypes
    import itertools
    from nicecore import build as B
    B.build()
    lib = L.load()

    def need(dtype, m, k, n, **out):
        a = L.NcLayerArgs(abi_version=L.NC_ABI_VERSION, dtype=dtype, relu=1, rows=m, inputs=k, outputs=n, w=256, w_stride=k,
                          codes=256, steps=256, code_stride=(k + 127) // 128 * 128, dy=256, dy_stride=n, dx_stride=k, **out)
        return lib.nc_layer_workspace_bytes(ctypes.byref(a), 1)

    outs = [dict(zip(c, (256,) * 3)) for r in range(4) for c in itertools.combinations(("dx", "dw", "db"), r)]
    for dtype in (L.NC_F32, L.NC_F16, L.NC_BF16):
        for m, k, n in ((1, 1, 1), (200, 93, 256), (600, 1, 1), (8192, 4096, 4096), (220000, 256, 4), (64, 55, 4616), (70, 2048, 2048)):
            size = {frozenset(o): need(dtype, m, k, n, **o) for o in outs}
            for p, q in itertools.product(size, size):
                assert p - q or 0 < size[p] <= size[q], (dtype, m, k, n, p, q)
    # 8192 x 4096 x 4096: a transposed weight for dx alone; the values of the codes, one part, for dW alone
    assert need(L.NC_BF16, 8192, 4096, 4096, dx=256) == 4096 * 4096 * 2
    assert need(L.NC_BF16, 8192, 4096, 4096, dw=256) == 8192 * 4096 * 2
    assert need(L.NC_BF16, 8192, 4096, 4096, db=256) < 1 << 20


def test_a_quantised_mlp_renders_no_rays():
    from nicecore import imap
    q = object.__new__(imap.QuantizedMLP)
    with pytest.raises(L.NiceCoreError, match="point queries"):
        imap.render_rays(q, torch.zeros(1, 3), torch.ones(1, 3), torch.zeros(3, 2))
