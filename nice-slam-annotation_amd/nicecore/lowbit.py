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
    """[..., cols] as ([rows, cols] with contiguous columns, rows, cols, row stride)."""
    dims = x.dim()
    if dims < 1:
        raise L.NiceCoreError(f"{what} needs at least one dimension")
    cols = x.shape[-1]
    if not 1 <= cols <= L.NC_MAX_INPUTS:
        raise L.NiceCoreError(f"{what} must have 1 to {L.NC_MAX_INPUTS} channels, got {cols}")
    if dims != 2:
        x = x.detach()
        x = x.unsqueeze(0) if dims == 1 else x.reshape(-1, cols)
    stride, one = x.stride()
    if (cols > 1 and one != 1) or stride > L.NC_MAX_STRIDE:
        x = x.detach().contiguous()
        stride = cols
    return x, x.shape[0], cols, stride


_HERE = contextlib.nullcontext()


def _on(dev):
    """The library launches on the current device: make it the tensors'."""
    return _HERE if torch._C._cuda_getDevice() == dev.index else torch.cuda.device(dev)


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
            return self._scales if len(self._lead) == 1 else self._scales.reshape(self._lead)
        return self._scales[:, :(self._cols + GROUP - 1) // GROUP].reshape(*self._lead, -1)

    def nbytes(self):
        return self._storage.numel() + self._scales.numel() * self._scales.element_size()

    def dequantize(self, dtype=None):
        """The values that the codes stand for, in ``dtype`` (default: the encoded tensor's)."""
        dtype = dtype or self.dtype
        if dtype not in _DTYPES:
            raise L.NiceCoreError(f"codes decode to float32, float16 or bfloat16, not {dtype}")
        codes = self._storage
        rows, cols = codes.shape[0], self._cols
        dev = codes.device
        out = torch.empty((rows, cols), device=dev, dtype=dtype)
        if rows:
            a = L.NcCodesArgs(L.NC_ABI_VERSION, _DTYPES[dtype], self._fmt, 0, rows, cols, cols, codes.shape[1], None,
                              codes.data_ptr(), self._scales.data_ptr(), out.data_ptr())
            with _on(dev):
                L.check(L.load().nc_decode_rows(ctypes.byref(a), L.raw_stream(dev)), "nc_decode_rows")
        if len(self._lead) == 1:
            return out
        return out.reshape(self.shape)


def _encode(x, fmt, what):
    dev = _device(x, what)
    dt = _dtype(x, what)
    x2, rows, cols, x_stride = _rows(x, what)
    stride = _code_stride(cols)
    codes = torch.empty((rows, stride), device=dev, dtype=torch.uint8)
    if fmt == L.NC_CODES_ROW:
        scales = torch.empty(rows, device=dev, dtype=torch.float32)
    else:
        scales = torch.empty((rows, stride // GROUP), device=dev, dtype=torch.uint8)
    if rows:
        a = L.NcCodesArgs(L.NC_ABI_VERSION, dt, fmt, 0, rows, cols, x_stride, stride, x2.data_ptr(), codes.data_ptr(),
                          scales.data_ptr(), None)
        with _on(dev):
            L.check(L.load().nc_encode_rows(ctypes.byref(a), L.raw_stream(dev)), "nc_encode_rows")
    return CodedRows(codes, scales, cols, x.shape[:-1], x.dtype, fmt)


def quantize_rows(x):
    """int8 codes of ``x`` [..., channels] with one float32 scale per row:
    s = max(amax |x| fl(1 / 127), 2^-126) in float32 (what ``amax / 127`` of a float32 tensor gives on the device; within
    one unit of the rounded quotient), q = the integer nearest to x / s (ties to even), value q s.
    A row that holds an infinity or NaN decodes to NaN.  A layer's weight [outputs, inputs] is
    encoded the same way (a scale per output channel).  Carries no gradient."""
    return _encode(x, L.NC_CODES_ROW, "x")


def pack_activations(x, relu=False):
    """The 8-bit checkpoint of ``x`` (``relu``: of max(x, 0), in codes whose 0 says x <= 0): 32
    neighbouring channels share a step, the least power of two of which 127 (254) hold the
    group's largest magnitude.  1.03 bytes a channel; half a step of error.  As float16 a value of 65536 (the
    nearest one to a magnitude over 65024) is float16's largest number, 65504.  Carries no gradient."""
    return _encode(x, L.NC_CODES_RELU if relu else L.NC_CODES_GROUP, "x")


def quantized_linear(x, weight, bias=None, relu=False, out_dtype=None):
    """y = x8 W8^T + bias, ``relu``: max(y, 0), the activation after the layer (checkpointed_linear's is the one before
    it): ``x`` [..., inputs] is encoded by quantize_rows within the call
    (or given as its CodedRows), ``weight`` = quantize_rows(W), W [outputs, inputs].  The sum of the
    code products is exact (int32); y has ``out_dtype`` (default: x's).  For inference: x and
    bias must not require grad."""
    coded = isinstance(x, CodedRows)
    dev = x.device if coded else _device(x, "x")
    if not isinstance(weight, CodedRows) or weight._fmt != L.NC_CODES_ROW or len(weight._lead) != 1:
        raise L.NiceCoreError("weight must be quantize_rows(W) of a [outputs, inputs] matrix")
    if coded and x._fmt != L.NC_CODES_ROW:
        raise L.NiceCoreError("x must be a tensor or quantize_rows(x)")
    if x.shape[-1:] != weight.shape[-1:]:
        raise L.NiceCoreError(f"x has shape {tuple(x.shape)}, the weight {tuple(weight.shape)}: channels differ")
    if torch.is_grad_enabled():
        for t, what in ((None if coded else x, "x"), (bias, "bias")):
            if t is not None and t.requires_grad:
                raise L.NiceCoreError(f"quantized_linear has no gradient: call it under torch.no_grad() or with "
                                      f"{what}.detach() (checkpointed_linear is the layer for training)")
    out_dtype = out_dtype or x.dtype
    if out_dtype not in _DTYPES:
        raise L.NiceCoreError(f"out_dtype must be float32, float16 or bfloat16, got {out_dtype}")
    _same_device(dev, weight, "weight")
    w_codes = weight._storage
    outputs, inputs = w_codes.shape[0], weight._cols
    x_dt, x_ptr, x_stride, x_codes, x_scales = 0, None, 0, None, None
    if coded:
        rows = x._storage.shape[0]
        x_codes, x_scales = x._storage.data_ptr(), x._scales.data_ptr()
    else:
        x_dt = _dtype(x, "x")
        x2, rows, _, x_stride = _rows(x, "x")
        x_ptr = x2.data_ptr()
    b_dt, b_ptr = 0, None
    if bias is not None:
        _same_device(dev, bias, "bias")
        if bias.dim() != 1 or bias.shape[0] != outputs:
            raise L.NiceCoreError(f"bias must be [{outputs}], got {tuple(bias.shape)}")
        if bias.stride(0) != 1:
            bias = bias.detach().contiguous()
        b_dt, b_ptr = _dtype(bias, "bias"), bias.data_ptr()
    out = torch.empty((rows, outputs), device=dev, dtype=out_dtype)
    if rows:
        a = L.NcQlinearArgs(L.NC_ABI_VERSION, x_dt, _DTYPES[out_dtype], b_dt, 1 if relu else 0, 0, rows, inputs, outputs,
                            x_ptr, x_stride, x_codes, x_scales, w_codes.shape[1], w_codes.data_ptr(),
                            weight._scales.data_ptr(), b_ptr, out.data_ptr(), outputs)
        lib, ref = L.load(), ctypes.byref(a)
        nbytes = lib.nc_quantized_linear_workspace_bytes(ref)
        if nbytes == 0:
            L.check(-1, "nc_quantized_linear_workspace_bytes")
        ws = torch.empty(nbytes, device=dev, dtype=torch.uint8)
        with _on(dev):
            L.check(lib.nc_quantized_linear(ref, ws.data_ptr(), nbytes, L.raw_stream(dev)), "nc_quantized_linear")
    lead = x.shape[:-1]
    return out if len(lead) == 1 else out.reshape(*lead, outputs)


def _weight_rows(w, inputs):
    if (inputs > 1 and w.stride(1) != 1) or w.stride(0) < 0:
        w = w.detach().contiguous()
    return w, w.stride(0)


def _came_back(t, what, dev, dtype, size):
    """A saved tensor is what a hook made of it: nothing else is read."""
    if t.device != dev or t.dtype != dtype or t.numel() != size:
        raise L.NiceCoreError(f"the saved {what} came back as {t.numel()} x {t.dtype} on {t.device}, "
                              f"kept were {size} x {dtype} on {dev}")


class _CheckpointedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, relu):
        dev = _device(x, "x")
        dt = _dtype(x, "x")
        for t, what in ((weight, "weight"), (bias, "bias")):
            if t is not None:
                _same_device(dev, t, what)
                if t.dtype != x.dtype:
                    raise L.NiceCoreError(f"{what} is {t.dtype}, x {x.dtype}")
        x2, rows, inputs, x_stride = _rows(x, "x")
        if weight.dim() != 2 or weight.shape[1] != inputs:
            raise L.NiceCoreError(f"weight must be [outputs, {inputs}], got {tuple(weight.shape)}")
        outputs = weight.shape[0]
        if not 1 <= outputs <= L.NC_MAX_INPUTS:
            raise L.NiceCoreError(f"weight must have 1 to {L.NC_MAX_INPUTS} outputs, got {outputs}")
        b_ptr = None
        if bias is not None:
            if bias.dim() != 1 or bias.shape[0] != outputs:
                raise L.NiceCoreError(f"bias must be [{outputs}], got {tuple(bias.shape)}")
            if bias.stride(0) != 1:
                bias = bias.detach().contiguous()
            b_ptr = bias.data_ptr()
        w2, w_stride = _weight_rows(weight, inputs)
        ctx.set_materialize_grads(False)
        need = ctx.needs_input_grad
        y = torch.empty((rows, outputs), device=dev, dtype=x.dtype)
        stride = _code_stride(inputs)
        # the checkpoint: codes, then steps
        kept = None
        a = L.NcLayerArgs(L.NC_ABI_VERSION, dt, 1 if relu else 0, 0, rows, inputs, outputs, x2.data_ptr(), x_stride,
                          w2.data_ptr(), w_stride, b_ptr, y.data_ptr(), outputs, None, None, stride)
        if rows:
            if need[1] or (need[0] and relu):
                kept = torch.empty(rows * (stride + stride // GROUP), device=dev, dtype=torch.uint8)
                a.codes = kept.data_ptr()
                a.steps = a.codes + rows * stride
            lib, ref = L.load(), ctypes.byref(a)
            nbytes = lib.nc_layer_workspace_bytes(ref, 0)
            if nbytes == 0:
                L.check(-1, "nc_layer_workspace_bytes")
            ws = torch.empty(nbytes, device=dev, dtype=torch.uint8)
            with _on(dev):
                L.check(lib.nc_layer_forward(ref, ws.data_ptr(), nbytes, L.raw_stream(dev)), "nc_layer_forward")
        # (the weight is checked for changes in place; the backward frees the checkpoint)
        ctx.save_for_backward(weight if need[0] else None, kept)
        ctx.args, ctx.shape, ctx.dtype = a, x.shape, x.dtype
        return y if x.dim() == 2 else y.reshape(*x.shape[:-1], outputs)

    @staticmethod
    def backward(ctx, dy):
        if dy is None:
            return None, None, None, None
        if torch.is_grad_enabled():
            raise L.NiceCoreError("checkpointed_linear has no second derivative (backward with create_graph=True)")
        weight, kept = ctx.saved_tensors
        a, dtype = ctx.args, ctx.dtype
        rows, inputs, outputs, stride = a.rows, a.inputs, a.outputs, a.code_stride
        need = ctx.needs_input_grad
        dev = dy.device
        if weight is not None:
            _came_back(weight, "weight", dev, dtype, outputs * inputs)
        if kept is not None:
            _came_back(kept, "checkpoint", dev, torch.uint8, rows * (stride + stride // GROUP))
        dy2, _, _, dy_stride = _rows(dy, "the gradient")
        dx = torch.empty(ctx.shape, device=dev, dtype=dtype) if need[0] else None
        dw = torch.empty((outputs, inputs), device=dev, dtype=dtype) if need[1] else None
        db = torch.empty(outputs, device=dev, dtype=dtype) if need[2] else None
        w_ptr, w_stride, codes = None, 0, None
        if need[0]:
            w2, w_stride = _weight_rows(weight, inputs)
            w_ptr = w2.data_ptr()
        if kept is not None:
            kept = kept.contiguous()
            codes = kept.data_ptr()
        b = L.NcLayerArgs(L.NC_ABI_VERSION, a.dtype, a.relu, 0, rows, inputs, outputs, None, 0, w_ptr, w_stride, None, None, 0,
                          codes, codes + rows * stride if codes else None, stride, dy2.data_ptr(), dy_stride,
                          dx.data_ptr() if need[0] else None, inputs, dw.data_ptr() if need[1] else None,
                          db.data_ptr() if need[2] else None)
        lib, ref = L.load(), ctypes.byref(b)
        nbytes = lib.nc_layer_workspace_bytes(ref, 1)
        if nbytes == 0:
            L.check(-1, "nc_layer_workspace_bytes")
        ws = torch.empty(nbytes, device=dev, dtype=torch.uint8)
        with _on(dev):
            L.check(lib.nc_layer_backward(ref, ws.data_ptr(), nbytes, L.raw_stream(dev)), "nc_layer_backward")
        return dx, dw, db, None


def checkpointed_linear(x, weight, bias=None, relu=False):
    """y = a W^T + bias with a = x, or max(x, 0) when ``relu`` (the activation before the layer):
    one layer of a scene MLP (decoder.py:190-219), differentiable in x, weight and bias.

    Instead of the input its backward keeps the 8-bit checkpoint of ``a`` (pack_activations: 1.03
    bytes a channel):  dx = (dy W) [x > 0 or NaN if relu]  and  db  are those of the full layer, dW = dy^T a8
    sees the checkpoint's values.  All tensors have one dtype; sums are held in float32.  y and dx of a
    float32 layer keep 22 bits of a value of x or dy down to 2^-25 of the largest in its row (a floor of 2^-47 of
    that) and of W down to 2^-17 of the largest in its row (of W^T for dx; 2^-38), and are as near to the exact result as a
    plain float32 product unless rows span more: an input of 1e8 beside ones of 1, with a weight of 1e-8, leaves
    1.4e-5 (float32 3e-7).  An infinity in float32 x, W or dy gives the infinities and NaNs of the formula, but NaN where its
    factor is below the digits above (a weight under 2^-28, an x or dy under 2^-36 of the row's largest) or infinite too.
    A chain of such layers trains an MLP.  Has no second derivative.
    The checkpoint is a saved tensor: a backward frees it, and saved-tensor hooks may move it."""
    if not torch.is_grad_enabled():  # no backward, no checkpoint (a Function sees the inputs' own requires_grad)
        x, weight, bias = (t.detach() if isinstance(t, torch.Tensor) else t for t in (x, weight, bias))
    return _CheckpointedLinear.apply(x, weight, bias, bool(relu))
