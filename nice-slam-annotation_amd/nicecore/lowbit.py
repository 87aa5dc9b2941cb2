"""8-bit operators for the layers of a scene MLP (include/nicecore.h, ABI v12), HIP only.

The reference evaluates and trains its decoders in float32 (src/conv_onet/models/decoder.py:
190-219: ``net = pts_linear(net); net = F.relu(net)``).  Beside that path:

  quantize_rows(x)              codes of rows: int8 with one float32 scale per row
  quantized_linear(x, W8, b)    the product of such rows (a token's, a channel's scale)
  pack_activations(a)           an 8-bit checkpoint: 32 neighbouring channels share a power of two
  checkpointed_linear(x, W, b)  a layer for training whose backward keeps only that checkpoint

Inputs are float32, float16 or bfloat16, ``[..., channels]``; sums are held in 32 bits (int32
for products of codes, which are exact).  Rows may be strided; channels must be contiguous
(a copy is made otherwise).  No call synchronises; work goes to the current stream of the
tensors' device.
"""
from __future__ import annotations

import contextlib
import ctypes

import torch

from . import _lib as L

_DTYPES = {torch.float32: L.NC_F32, torch.float16: L.NC_F16, torch.bfloat16: L.NC_BF16}
GROUP = 32


def _code_stride(cols: int) -> int:
    return (cols + 127) // 128 * 128


def _dtype(t, what):
    if t.dtype not in _DTYPES:
        raise L.NiceCoreError(f"{what} must be float32, float16 or bfloat16, got {t.dtype}")
    return _DTYPES[t.dtype]


def _device(t, what):
    if not isinstance(t, torch.Tensor):
        raise L.NiceCoreError(f"{what} must be a tensor, got {type(t).__name__}")
    if t.device.type != "cuda":
        raise L.NiceCoreError(f"nicecore's 8-bit operators run on a HIP device; {what} is on {t.device}")
    return t.device


def _same_device(dev, t, what):
    if t.device != dev:
        raise L.NiceCoreError(f"{what} is on {t.device}, the input on {dev}")


def _rows(x, what):
    """[..., cols] as ([rows, cols] with contiguous columns, lead shape)."""
    if x.dim() < 1:
        raise L.NiceCoreError(f"{what} needs at least one dimension")
    cols = x.shape[-1]
    if not 1 <= cols <= L.NC_MAX_INPUTS:
        raise L.NiceCoreError(f"{what} must have 1 to {L.NC_MAX_INPUTS} channels, got {cols}")
    x2 = x.detach()
    lead = x2.shape[:-1]
    x2 = x2.unsqueeze(0) if x2.dim() == 1 else x2.reshape(-1, cols)
    if cols > 1 and x2.stride(1) != 1:
        x2 = x2.contiguous()
    return x2, lead


def _on(dev):
    """The library launches on the current device: make it the tensors'."""
    if torch.cuda.current_device() == dev.index:
        return contextlib.nullcontext()
    return torch.cuda.device(dev)


class CodedRows:
    """8-bit rows: ``codes`` [..., channels] (int8, or uint8 of a ReLU's output) and
    ``scales``: float32 [...] of a row, or uint8 [..., groups], the biased exponent of a
    group's step."""

    def __init__(self, storage, scales, cols, lead, dtype, fmt):
        self._storage, self._scales = storage, scales
        self._cols, self._lead, self.dtype, self._fmt = cols, lead, dtype, fmt

    @property
    def shape(self):
        return torch.Size((*self._lead, self._cols))

    @property
    def device(self):
        return self._storage.device

    @property
    def codes(self):
        return self._storage[:, :self._cols].view(torch.int8 if self._fmt != L.NC_CODES_RELU else torch.uint8) \
            .reshape(self.shape)

    @property
    def scales(self):
        if self._fmt == L.NC_CODES_ROW:
            return self._scales.reshape(self._lead)
        return self._scales[:, :(self._cols + GROUP - 1) // GROUP].reshape(*self._lead, -1)

    def nbytes(self):
        return self._storage.numel() + self._scales.numel() * self._scales.element_size()

    def dequantize(self, dtype=None):
        """The values that the codes stand for, in ``dtype`` (default: the encoded tensor's)."""
        dtype = dtype or self.dtype
        if dtype not in _DTYPES:
            raise L.NiceCoreError(f"codes decode to float32, float16 or bfloat16, not {dtype}")
        lib = L.load()
        rows = self._storage.shape[0]
        out = torch.empty(rows, self._cols, device=self.device, dtype=dtype)
        a = L.NcCodesArgs(abi_version=L.NC_ABI_VERSION, dtype=_DTYPES[dtype], format=self._fmt, rows=rows,
                          cols=self._cols, stride=self._cols, code_stride=self._storage.shape[1],
                          codes=self._storage.data_ptr(), scales=self._scales.data_ptr(), values=out.data_ptr())
        with _on(self.device):
            L.check(lib.nc_decode_rows(ctypes.byref(a), L.raw_stream(self.device)), "nc_decode_rows")
        return out.reshape(self.shape)


def _encode(x, fmt, what):
    dev = _device(x, what)
    dt = _dtype(x, what)
    x2, lead = _rows(x, what)
    rows, cols = x2.shape
    lib = L.load()
    stride = _code_stride(cols)
    codes = torch.empty(rows, stride, device=dev, dtype=torch.uint8)
    if fmt == L.NC_CODES_ROW:
        scales = torch.empty(rows, device=dev, dtype=torch.float32)
    else:
        scales = torch.empty(rows, stride // GROUP, device=dev, dtype=torch.uint8)
    a = L.NcCodesArgs(abi_version=L.NC_ABI_VERSION, dtype=dt, format=fmt, rows=rows, cols=cols, stride=x2.stride(0),
                      code_stride=stride, x=x2.data_ptr(), codes=codes.data_ptr(), scales=scales.data_ptr())
    with _on(dev):
        L.check(lib.nc_encode_rows(ctypes.byref(a), L.raw_stream(dev)), "nc_encode_rows")
    return CodedRows(codes, scales, cols, lead, x.dtype, fmt)


def quantize_rows(x):
    """int8 codes of ``x`` [..., channels] with one float32 scale per row:
    s = max(amax |x| / 127, 2^-126), q = the integer nearest to x / s (ties to even), value q s.
    A row that holds an infinity or NaN decodes to NaN.  A layer's weight [outputs, inputs] is
    encoded the same way (a scale per output channel).  Carries no gradient."""
    return _encode(x, L.NC_CODES_ROW, "x")


def pack_activations(x, relu=False):
    """The 8-bit checkpoint of ``x`` (``relu``: of max(x, 0), in codes whose 0 says x <= 0): 32
    neighbouring channels share a step, the least power of two of which 127 (254) hold the
    group's largest magnitude.  1.03 bytes a channel; half a step of error.  Carries no gradient."""
    return _encode(x, L.NC_CODES_RELU if relu else L.NC_CODES_GROUP, "x")


def quantized_linear(x, weight, bias=None, relu=False, out_dtype=None):
    """y = x8 W8^T + bias [, ReLU]: ``x`` [..., inputs] is encoded by quantize_rows within the call
    (or given as its CodedRows), ``weight`` = quantize_rows(W), W [outputs, inputs].  The sum of the
    code products is exact (int32); y has ``out_dtype`` (default: x's).  For inference: x must
    not require grad."""
    coded = isinstance(x, CodedRows)
    dev = x.device if coded else _device(x, "x")
    if not isinstance(weight, CodedRows) or weight._fmt != L.NC_CODES_ROW or len(weight._lead) != 1:
        raise L.NiceCoreError("weight must be quantize_rows(W) of a [outputs, inputs] matrix")
    if coded and x._fmt != L.NC_CODES_ROW:
        raise L.NiceCoreError("x must be a tensor or quantize_rows(x)")
    if x.shape[-1:] != weight.shape[-1:]:
        raise L.NiceCoreError(f"x has shape {tuple(x.shape)}, the weight {tuple(weight.shape)}: channels differ")
    if not coded and x.requires_grad and torch.is_grad_enabled():
        raise L.NiceCoreError("quantized_linear has no gradient: call it under torch.no_grad() or with x.detach() "
                              "(checkpointed_linear is the layer for training)")
    out_dtype = out_dtype or x.dtype
    if out_dtype not in _DTYPES:
        raise L.NiceCoreError(f"out_dtype must be float32, float16 or bfloat16, got {out_dtype}")
    _same_device(dev, weight, "weight")
    outputs, inputs = weight.shape
    a = L.NcQlinearArgs(abi_version=L.NC_ABI_VERSION, out_dtype=_DTYPES[out_dtype], relu=1 if relu else 0,
                        inputs=inputs, outputs=outputs, code_stride=weight._storage.shape[1],
                        w_codes=weight._storage.data_ptr(), w_scales=weight._scales.data_ptr())
    if coded:
        lead, rows = x._lead, x._storage.shape[0]
        a.x_codes, a.x_scales = x._storage.data_ptr(), x._scales.data_ptr()
    else:
        a.dtype = _dtype(x, "x")
        x2, lead = _rows(x, "x")
        rows = x2.shape[0]
        a.x, a.x_stride = x2.data_ptr(), x2.stride(0)
    a.rows = rows
    if bias is not None:
        _same_device(dev, bias, "bias")
        if bias.shape != (outputs,):
            raise L.NiceCoreError(f"bias must be [{outputs}], got {tuple(bias.shape)}")
        bias = bias.detach().contiguous()
        a.bias_dtype, a.bias = _dtype(bias, "bias"), bias.data_ptr()
    out = torch.empty(rows, outputs, device=dev, dtype=out_dtype)
    if rows:
        a.out, a.out_stride = out.data_ptr(), outputs
        lib = L.load()
        nbytes = lib.nc_quantized_linear_workspace_bytes(ctypes.byref(a))
        if nbytes == 0:
            L.check(-1, "nc_quantized_linear_workspace_bytes")
        ws = torch.empty(nbytes, device=dev, dtype=torch.uint8)
        with _on(dev):
            L.check(lib.nc_quantized_linear(ctypes.byref(a), ws.data_ptr(), nbytes, L.raw_stream(dev)),
                    "nc_quantized_linear")
    return out.reshape(*lead, outputs)


class _CheckpointedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, relu):
        dev = _device(x, "x")
        dt = _dtype(x, "x")
        for t, what in ((weight, "weight"), (bias, "bias")):
            if t is None:
                continue
            _same_device(dev, t, what)
            if t.dtype != x.dtype:
                raise L.NiceCoreError(f"{what} is {t.dtype}, x {x.dtype}")
        if weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
            raise L.NiceCoreError(f"weight must be [outputs, {x.shape[-1]}], got {tuple(weight.shape)}")
        outputs, inputs = weight.shape
        if not 1 <= outputs <= L.NC_MAX_INPUTS:
            raise L.NiceCoreError(f"weight must have 1 to {L.NC_MAX_INPUTS} outputs, got {outputs}")
        if bias is not None and bias.shape != (outputs,):
            raise L.NiceCoreError(f"bias must be [{outputs}], got {tuple(bias.shape)}")
        x2, lead = _rows(x, "x")
        w2 = weight.detach()
        if inputs > 1 and w2.stride(1) != 1:
            w2 = w2.contiguous()
        b2 = bias.detach().contiguous() if bias is not None else None
        rows = x2.shape[0]
        ctx.set_materialize_grads(False)
        need = ctx.needs_input_grad
        y = torch.empty(rows, outputs, device=dev, dtype=x.dtype)
        stride = _code_stride(inputs)
        a = L.NcLayerArgs(abi_version=L.NC_ABI_VERSION, dtype=dt, relu=1 if relu else 0, rows=rows, inputs=inputs,
                          outputs=outputs, x=x2.data_ptr(), x_stride=x2.stride(0), w=w2.data_ptr(),
                          w_stride=w2.stride(0), bias=b2.data_ptr() if b2 is not None else None, y=y.data_ptr(),
                          y_stride=outputs, code_stride=stride)
        codes = steps = None
        if rows and (need[1] or (need[0] and relu)):
            codes = torch.empty(rows, stride, device=dev, dtype=torch.uint8)
            steps = torch.empty(rows, stride // GROUP, device=dev, dtype=torch.uint8)
            a.codes, a.steps = codes.data_ptr(), steps.data_ptr()
        if rows:
            lib = L.load()
            nbytes = lib.nc_layer_workspace_bytes(ctypes.byref(a), 0)
            if nbytes == 0:
                L.check(-1, "nc_layer_workspace_bytes")
            ws = torch.empty(nbytes, device=dev, dtype=torch.uint8)
            with _on(dev):
                L.check(lib.nc_layer_forward(ctypes.byref(a), ws.data_ptr(), nbytes, L.raw_stream(dev)), "nc_layer_forward")
        ctx.save_for_backward(weight if need[0] else None, codes, steps)
        ctx.lead, ctx.sizes, ctx.relu, ctx.dtype = lead, (rows, inputs, outputs), bool(relu), x.dtype
        return y.reshape(*lead, outputs)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        if dy is None:
            return None, None, None, None
        weight, codes, steps = ctx.saved_tensors
        rows, inputs, outputs = ctx.sizes
        need = ctx.needs_input_grad
        dev = dy.device
        dy2, _ = _rows(dy, "the gradient")
        dx = torch.empty(rows, inputs, device=dev, dtype=ctx.dtype) if need[0] else None
        dw = torch.empty(outputs, inputs, device=dev, dtype=ctx.dtype) if need[1] else None
        db = torch.empty(outputs, device=dev, dtype=ctx.dtype) if need[2] else None
        a = L.NcLayerArgs(abi_version=L.NC_ABI_VERSION, dtype=_DTYPES[ctx.dtype], relu=1 if ctx.relu else 0, rows=rows,
                          inputs=inputs, outputs=outputs, code_stride=_code_stride(inputs), dy=dy2.data_ptr(),
                          dy_stride=dy2.stride(0))
        w2 = None
        if need[0]:
            w2 = weight.detach()
            if inputs > 1 and w2.stride(1) != 1:
                w2 = w2.contiguous()
            a.w, a.w_stride = w2.data_ptr(), w2.stride(0)
        if codes is not None:
            a.codes, a.steps = codes.data_ptr(), steps.data_ptr()
        a.dx, a.dw, a.db = (t.data_ptr() if t is not None else None for t in (dx, dw, db))
        lib = L.load()
        nbytes = lib.nc_layer_workspace_bytes(ctypes.byref(a), 1)
        if nbytes == 0:
            L.check(-1, "nc_layer_workspace_bytes")
        ws = torch.empty(nbytes, device=dev, dtype=torch.uint8)
        with _on(dev):
            L.check(lib.nc_layer_backward(ctypes.byref(a), ws.data_ptr(), nbytes, L.raw_stream(dev)), "nc_layer_backward")
        return dx.reshape(*ctx.lead, inputs) if dx is not None else None, dw, db, None


def checkpointed_linear(x, weight, bias=None, relu=False):
    """y = a W^T + bias with a = x, or max(x, 0) when ``relu`` (the activation before the layer):
    one layer of a scene MLP (decoder.py:190-219), differentiable in x, weight and bias.

    Instead of the input its backward keeps the 8-bit checkpoint of ``a`` (pack_activations: 1.03
    bytes a channel):  dx = (dy W) [x > 0 if relu]  and  db  are those of the full layer, dW = dy^T a8
    sees the checkpoint's values.  All tensors have one dtype; sums are held in float32, and a
    float32 product is accurate to float32.  A chain of such layers trains an MLP."""
    return _CheckpointedLinear.apply(x, weight, bias, bool(relu))
