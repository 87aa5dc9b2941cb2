"""The 8-bit layer operators' refusals and host side (no GPU): nicecore.lowbit's argument checks
and the C entries' (include/nicecore.h, ABI v12), and the oracle's own definitions."""
import ctypes

import pytest
import torch

from nicecore import _lib as L
from nicecore import build as B
from nicecore import lowbit
from oracle import lowbit_oracle as LO


@pytest.fixture(scope="module")
def lib():
    B.build()
    return L.load()


def test_struct_layouts_match(lib):
    assert lib.nc_struct_size(14) == ctypes.sizeof(L.NcCodesArgs)
    assert lib.nc_struct_size(15) == ctypes.sizeof(L.NcQlinearArgs)
    assert lib.nc_struct_size(16) == ctypes.sizeof(L.NcLayerArgs)


def test_cpu_tensors_are_refused():
    x, w = torch.randn(4, 8), torch.randn(3, 8)
    for call in (lambda: lowbit.quantize_rows(x), lambda: lowbit.pack_activations(x),
                 lambda: lowbit.checkpointed_linear(x, w)):
        with pytest.raises(L.NiceCoreError, match="HIP device"):
            call()
    with pytest.raises(L.NiceCoreError, match="tensor"):
        lowbit.quantize_rows([1.0])
    with pytest.raises(L.NiceCoreError, match="HIP device"):
        lowbit.quantized_linear(x, w)


def test_coded_rows_are_checked():
    rows = lowbit.CodedRows(torch.zeros(4, 128, dtype=torch.uint8), torch.ones(4), 8, torch.Size([4]), torch.float32,
                            L.NC_CODES_ROW)
    groups = lowbit.CodedRows(torch.zeros(4, 128, dtype=torch.uint8), torch.ones(4, 4, dtype=torch.uint8), 8,
                              torch.Size([4]), torch.float32, L.NC_CODES_GROUP)
    assert rows.shape == (4, 8) and rows.codes.shape == (4, 8) and rows.scales.shape == (4,) and groups.scales.shape == (4, 1)
    narrow = lowbit.CodedRows(torch.zeros(4, 128, dtype=torch.uint8), torch.ones(4), 7, torch.Size([4]), torch.float32,
                              L.NC_CODES_ROW)
    for x, w, kw, msg in ((rows, torch.zeros(4, 8), {}, "weight must be"), (rows, groups, {}, "weight must be"),
                          (groups, rows, {}, "x must be"), (rows, narrow, {}, "channels differ"),
                          (rows, rows, dict(out_dtype=torch.float64), "out_dtype"),
                          (rows, rows, dict(bias=torch.zeros(3)), "bias must be")):
        with pytest.raises(L.NiceCoreError, match=msg):
            lowbit.quantized_linear(x, w, **kw)
    with pytest.raises(L.NiceCoreError, match="decode"):
        rows.dequantize(torch.float64)


def codes_args(**kw):
    a = L.NcCodesArgs(abi_version=L.NC_ABI_VERSION, dtype=L.NC_F32, format=L.NC_CODES_ROW, rows=4, cols=100, stride=100,
                      code_stride=128, x=16, codes=32, scales=16, values=16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_codes_args_validated(lib):
    for kw, msg in ((dict(dtype=3), b"dtype"), (dict(format=3), b"format"), (dict(format=-1), b"format"),
                    (dict(rows=-1), b"rows"), (dict(cols=0), b"inputs"), (dict(cols=L.NC_MAX_INPUTS + 1), b"131072"),
                    (dict(code_stride=96), b"code_stride"), (dict(code_stride=130), b"code_stride"),
                    (dict(codes=40), b"aligned"), (dict(stride=-1), b"stride"), (dict(codes=0), b"NULL"),
                    (dict(scales=0), b"NULL"), (dict(x=0, values=0), b"NULL")):
        a = codes_args(**kw)
        for f in (lib.nc_encode_rows, lib.nc_decode_rows):
            assert f(ctypes.byref(a), None) == -1, kw
            assert msg in lib.nc_last_error(), (kw, lib.nc_last_error())
    a = codes_args(abi_version=L.NC_ABI_VERSION - 1)
    assert lib.nc_encode_rows(ctypes.byref(a), None) == -2
    assert lib.nc_encode_rows(None, None) == -1
    assert lib.nc_encode_rows(ctypes.byref(codes_args(rows=0)), None) == 0


def test_qlinear_args_validated(lib):
    def args(**kw):
        a = L.NcQlinearArgs(abi_version=L.NC_ABI_VERSION, rows=4, inputs=100, outputs=8, x=16, x_stride=100,
                            code_stride=128, w_codes=32, w_scales=16, out=16, out_stride=8)
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    for kw, msg in ((dict(dtype=9), b"dtype"), (dict(out_dtype=9), b"dtype"), (dict(bias=16, bias_dtype=9), b"dtype"),
                    (dict(outputs=0), b"outputs"), (dict(inputs=L.NC_MAX_INPUTS + 1, code_stride=1 << 20), b"131072"),
                    (dict(code_stride=64), b"code_stride"), (dict(w_codes=8), b"aligned"), (dict(x=0, x_codes=8), b"aligned"),
                    (dict(out_stride=-1), b"stride")):
        a = args(**kw)
        assert lib.nc_quantized_linear_workspace_bytes(ctypes.byref(a)) == 0, kw
        assert msg in lib.nc_last_error(), (kw, lib.nc_last_error())
        assert lib.nc_quantized_linear(ctypes.byref(a), 256, 1 << 30, None) == -1
    a = args(rows=100, inputs=300, code_stride=384)  # (few rows are encoded within the product)
    n = lib.nc_quantized_linear_workspace_bytes(ctypes.byref(a))
    assert n >= 100 * 384 + 400
    assert lib.nc_quantized_linear(ctypes.byref(a), 256, n - 1, None) == -1 and b"workspace" in lib.nc_last_error()
    assert lib.nc_quantized_linear(ctypes.byref(a), None, n, None) == -1
    assert lib.nc_quantized_linear(ctypes.byref(args(out=0)), 256, n, None) == -1 and b"NULL" in lib.nc_last_error()
    assert lib.nc_quantized_linear(ctypes.byref(args(rows=0)), None, 0, None) == 0


def test_layer_args_validated(lib):
    def args(**kw):
        a = L.NcLayerArgs(abi_version=L.NC_ABI_VERSION, rows=4, inputs=100, outputs=8, x=16, x_stride=100, w=16, w_stride=100,
                          y=16, y_stride=8, codes=32, steps=16, code_stride=128, dy=16, dy_stride=8, dx=16, dx_stride=100, dw=16, db=16)
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    for kw, msg in ((dict(dtype=5), b"dtype"), (dict(rows=-2), b"rows"), (dict(rows=1 << 31), b"2^31"),
                    (dict(inputs=0), b"inputs"), (dict(outputs=L.NC_MAX_INPUTS + 1), b"131072"),
                    (dict(x_stride=-1), b"stride"), (dict(dy_stride=-1), b"stride"), (dict(x_stride=(1 << 22) + 1), b"2^22"), (dict(dx_stride=-1), b"stride")):
        a = args(**kw)
        for back in (0, 1):
            assert lib.nc_layer_workspace_bytes(ctypes.byref(a), back) == 0, kw
            assert msg in lib.nc_last_error(), (kw, lib.nc_last_error())
        assert lib.nc_layer_forward(ctypes.byref(a), 256, 1 << 40, None) == -1
        assert lib.nc_layer_backward(ctypes.byref(a), 256, 1 << 40, None) == -1
    big = 1 << 40
    for kw, f in ((dict(x=0), 0), (dict(w=0), 0), (dict(y=0), 0), (dict(steps=0), 0), (dict(code_stride=64), 0),
                  (dict(dy=0), 1), (dict(codes=0), 1), (dict(w=0), 1), (dict(codes=8), 1)):
        call = lib.nc_layer_backward if f else lib.nc_layer_forward
        assert call(ctypes.byref(args(**kw)), 256, big, None) == -1, kw
    a = args()
    for back, call in ((0, lib.nc_layer_forward), (1, lib.nc_layer_backward)):
        n = lib.nc_layer_workspace_bytes(ctypes.byref(a), back)
        assert n > 0
        assert call(ctypes.byref(a), 256, n - 1, None) == -1 and b"workspace" in lib.nc_last_error()
    assert lib.nc_layer_forward(ctypes.byref(args(rows=0)), None, 0, None) == 0
    assert lib.nc_layer_backward(ctypes.byref(args(dx=0, dw=0, db=0)), None, 0, None) == 0


def test_oracle_codes():
    """The definitions on values worked out by hand."""
    q, s = LO.row_codes(torch.tensor([[127.0, 1.5, 2.5, -0.5, -127.0]]))
    assert s.item() == 1.0 and q.tolist() == [[127.0, 2.0, 2.0, 0.0, -127.0]]
    q, byte, v = LO.group_codes(torch.tensor([[127.0, 0.5, 1.5, -3.0]]), False)
    assert byte.item() == 127 and q.tolist() == [[127.0, 0.0, 2.0, -3.0]]
    q, byte, v = LO.group_codes(torch.tensor([[127.5, 0.5, 1.5, -3.0]]), False)
    assert byte.item() == 128 and v.tolist() == [[128.0, 0.0, 2.0, -4.0]]
    q, byte, v = LO.group_codes(torch.tensor([[254.0, 0.25, 1.5, -3.0]]), True)
    assert byte.item() == 127 and q.tolist() == [[255.0, 1.0, 3.0, 0.0]] and v.tolist() == [[254.0, 0.0, 2.0, 0.0]]


def test_imap_flags_validated(lib):
    """The iMAP* entries with 8-bit checkpoints: less than half the workspace; other flags are refused."""
    def points(flags, n=1000):
        a = L.NcImapPointsArgs(abi_version=L.NC_ABI_VERSION, flags=flags, n_points=n)
        return lib.nc_imap_points_workspace_bytes(ctypes.byref(a)), a
    full, _ = points(L.NC_SAVE_FOR_BACKWARD, 200000)
    coded, a = points(L.NC_SAVE_FOR_BACKWARD | L.NC_CODED_ACTIVATIONS, 200000)
    assert 0 < coded < full / 2
    assert lib.nc_imap_points_activation_offset(ctypes.byref(a), 0) == -1
    assert points(L.NC_CODED_ACTIVATIONS)[0] == points(0)[0]  # nothing to keep
    assert points(L.NC_DETERMINISTIC)[0] == 0
    assert lib.nc_imap_features(None, -1, None, None, None) == -1
    assert lib.nc_imap_features(None, 5, None, None, None) == -1 and b"NULL" in lib.nc_last_error()
    assert lib.nc_imap_features(None, 0, None, None, None) == 0


def test_activation_names_are_checked():
    from nicecore import decoder as D
    from nicecore import imap
    m = D.build_imap(seed=0)
    with pytest.raises(L.NiceCoreError, match="activations"):
        imap.eval_points(m, torch.zeros(4, 3), activations="fp8")
    with pytest.raises(L.NiceCoreError, match="HIP device"):
        m.quantize()


def test_overlaps_and_sizes_are_refused(lib):
    """Rows of an output that overlap, codes with other strides, more threads than a launch has."""
    def layer(**kw):
        a = L.NcLayerArgs(abi_version=L.NC_ABI_VERSION, rows=4, inputs=100, outputs=8, x=16, x_stride=100, w=16, w_stride=100,
                          y=16, y_stride=8, codes=32, steps=16, code_stride=128, dy=16, dy_stride=8, dx=16, dx_stride=100, dw=16, db=16)
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    for kw, msg in ((dict(y_stride=7), b"overlap"), (dict(dx_stride=99), b"overlap"), (dict(rows=1 << 28), b"2^34")):
        for back, call in ((0, lib.nc_layer_forward), (1, lib.nc_layer_backward)):
            assert lib.nc_layer_workspace_bytes(ctypes.byref(layer(**kw)), back) == 0 and msg in lib.nc_last_error(), kw
            assert call(ctypes.byref(layer(**kw)), 256, 1 << 60, None) == -1, kw
    assert lib.nc_layer_workspace_bytes(ctypes.byref(layer(rows=1, y_stride=0, dx_stride=0)), 1) > 0  # one row overlaps with none
    for call in (lib.nc_layer_forward, lib.nc_layer_backward):
        assert call(ctypes.byref(layer(code_stride=256)), 256, 1 << 60, None) == -1 and b"code_stride" in lib.nc_last_error()
    assert lib.nc_decode_rows(ctypes.byref(codes_args(stride=99)), None) == -1 and b"overlap" in lib.nc_last_error()
    assert lib.nc_encode_rows(ctypes.byref(codes_args(code_stride=256)), None) == -1
    a = L.NcQlinearArgs(abi_version=L.NC_ABI_VERSION, rows=4, inputs=100, outputs=8, x=16, x_stride=100, code_stride=128, w_codes=32,
                        w_scales=16, out=16, out_stride=7)
    assert lib.nc_quantized_linear_workspace_bytes(ctypes.byref(a)) == 0 and b"overlap" in lib.nc_last_error()
