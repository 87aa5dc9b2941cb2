"""The 8-bit layer operators (nicecore.lowbit) at the ends of their types, at the sizes of a mapper
iteration, and what their autograd graph and workspaces hold.

Tolerances are those of tests/test_gpu_lowbit.py: u = 2^-24 is half a float32 step, sums of
products as in sum_tol, the output's rounding as in out_tol.
"""
import ctypes
import math

import pytest
import torch
import torch.utils.checkpoint

from oracle import lowbit_oracle as LO
from test_gpu_lowbit import BF16, F16, F32, TYPES, U, acts, check, gen, layer_run, lb, out_tol, sum_tol

pytestmark = pytest.mark.gpu


def check_dw(dw, x, dy, relu):
    """dW against the float64 sum over the checkpoint's values."""
    v = LO.group_codes(x, relu)[2]
    want = dy.double().t() @ v
    t = sum_tol(dy.double().abs().t() @ v.abs(), x.shape[0], 3 if x.dtype == F32 else 1)
    assert torch.isfinite(want).all() and torch.isfinite(dw).all()
    check(dw, want, t + out_tol(want.abs() + t, x.dtype))


# small tiles decode while they stage, the large ones of 2048 x 2048 take the values written out
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("m,k,n", [(5, 96, 40), (200, 300, 130), (70, 2048, 2048)])
def test_half_checkpoints_of_the_largest_numbers(m, k, n, relu):
    """float16's largest numbers: the nearest code of a magnitude over 65024 (65280 with relu) stands for 65536,
    which as float16 is its largest number, 65504."""
    x = acts(m, k, F16, 3)
    top = torch.tensor([65024., 65056., 65280., 65312., 65472., 65504.], dtype=F16)
    for i, t in enumerate(top):  # alone in its group, and beside values of every size
        x[i % m, (33 * i) % k] = t
        x[(i + 2) % m, (33 * i + 7) % k] = -t
    x[:, 60] = 6e-8  # the least subnormal
    x[1, 64:96] = (1e-6 * x[1, 64:96].float()).to(F16)  # a group of them
    p = lb().pack_activations(x.cuda(), relu=relu)
    v = LO.group_codes(x, relu)[2]
    assert v.abs().max() == 65504 and torch.equal(p.dequantize().cpu().double(), v)
    a = torch.relu(x.double()) if relu else x.double()
    step = torch.ldexp(torch.ones_like(p.scales.cpu(), dtype=torch.float64), p.scales.cpu().int() - 127)
    assert ((v - a).abs() <= step.repeat_interleave(32, 1)[:, :k] / 2).all()
    wide = v.clone()
    wide[v.abs() == 65504] = 65536 * v[v.abs() == 65504].sign()  # the code's own value
    assert torch.equal(p.dequantize(F32).cpu().double(), wide)
    g = gen(4)
    w = (1e-4 * torch.randn(n, k, generator=g)).to(F16)
    dy = (1e-3 * torch.randn(m, n, generator=g)).to(F16)
    y, _, dw = layer_run(x, w, None, dy, relu)
    assert torch.isfinite(y).all()
    check_dw(dw, x, dy, relu)


def test_half_values_of_float32_codes():
    """Codes of float32 rows as float16: 65536 ends at 65504 too, larger values are infinite, subnormals rounded."""
    x = torch.tensor([65536., -65536., 65535.5, 131072., 3., -3., 0., 1.])[:, None].expand(8, 32).contiguous()
    x = torch.cat([x, x * 2.0 ** -40])
    d = lb().pack_activations(x.cuda()).dequantize(F16).cpu()
    want = LO.group_codes(x, False)[2]
    want = torch.where(want.abs() == 65536, 65504 * want.sign(), want).to(F16)
    assert torch.equal(d, want)
    assert d[3].isinf().all() and d[0, 0] == 65504 and d[1, 0] == -65504


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,k,n", [(5, 96, 40), (200, 300, 130), (70, 2048, 2048)])
def test_checkpoints_of_the_largest_numbers(m, k, n, dtype, relu):
    """Magnitudes up to the largest float: their groups' step is 2^121, which 128 times would not be finite."""
    x = acts(m, k, dtype, 5)
    end = torch.finfo(dtype).max
    for i, t in enumerate((1.6e38, 1.69e38, 1.8e38, 3e38, 3.37e38, end)):
        x[i % m, (33 * i) % k] = min(t, end)
        x[(i + 2) % m, (33 * i + 7) % k] = -min(t, end)
    p = lb().pack_activations(x.cuda(), relu=relu)
    v = LO.group_codes(x, relu)[2]
    assert torch.equal(p.dequantize(F32).cpu().double(), v)
    g = gen(6)
    w = (1e-30 * torch.randn(n, k, generator=g)).to(dtype)
    dy = (1e-30 * torch.randn(m, n, generator=g)).to(dtype)
    y, _, dw = layer_run(x, w, None, dy, relu)
    assert torch.isfinite(y).all()
    check_dw(dw, x, dy, relu)


# one and few rows, short sums, tiles, sums cut in parts; the third size of rows is coded before the call
@pytest.mark.parametrize("m,k,n", [(1, 256, 64), (16, 300, 33), (200, 93, 256), (50, 700, 40), (700, 256, 384), (2100, 512, 640), (90, 8200, 33),
                                   (300, 4096, 256)])
@pytest.mark.parametrize("coded", [False, True])
def test_quantized_linear_of_far_scales(m, k, n, coded):
    """Scales whose product is no normal number, where y is one."""
    x, w = acts(m, k, F32, m), acts(n, k, F32, n)
    for sx, sw in ((1e-20, 1e-21), (1e-36, 1e-3), (1e-3, 1e-36), (1e34, 1e-36), (1e34, 1e6), (1e6, 1e34), (1e-30, 1e-30)):
        xs, ws = x * sx, w * sw
        xs[0, :] = 0
        xs[0, :2] = 100 * sx  # a sum of exactly 0 with the first channel, whatever the scales
        ws[0, :] = 0
        ws[0, 0], ws[0, 1] = 100 * sw, -100 * sw
        q, w8 = lb().quantize_rows(xs.cuda()), lb().quantize_rows(ws.cuda())
        y = lb().quantized_linear(q if coded else xs.cuda(), w8).double().cpu()
        xq, xsc = LO.row_codes(xs)
        wq, wsc = LO.row_codes(ws)
        want = LO.quantized_linear(xq, xsc, wq, wsc)
        assert y[0, 0] == 0
        big = torch.finfo(F32).max
        fits = want.abs() * (1 + 4 * U) < big
        check(y[fits], want[fits], 4 * U * want[fits].abs() + 2.0 ** -148)
        over = want.abs() * (1 - 4 * U) > big
        assert torch.equal(y[over], math.inf * want[over].sign())


def step_leaves(dtype=F32, m=300, k=256, n=96):
    x, w, dy = acts(m, k, dtype, 1).cuda(), acts(n, k, dtype, 2).cuda(), acts(m, n, dtype, 3).cuda()
    b = torch.ones(n, device="cuda", dtype=dtype)
    return [t.requires_grad_(True) for t in (x, w, b)], dy


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_the_checkpoint_is_a_saved_tensor(dtype, relu):
    """Hooks on saved tensors see the codes, may move them, and the gradients are the same."""
    leaves, dy = step_leaves(dtype)
    want = torch.autograd.grad(lb().checkpointed_linear(*leaves, relu=relu), leaves, dy)
    seen = []

    def pack(t):
        seen.append((t.dtype, t.numel()))
        return t.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.cuda()):
        y = lb().checkpointed_linear(*leaves, relu=relu)
    assert (torch.uint8, 300 * (256 + 8)) in seen
    for a, b in zip(torch.autograd.grad(y, leaves, dy), want):
        assert torch.equal(a, b)
    with torch.autograd.graph.save_on_cpu():
        y = lb().checkpointed_linear(*leaves, relu=relu)
    for a, b in zip(torch.autograd.grad(y, leaves, dy), want):
        assert torch.equal(a, b)

    def layer(*t):
        return lb().checkpointed_linear(*t, relu=relu)

    y = torch.utils.checkpoint.checkpoint(layer, *leaves, use_reentrant=False)
    for a, b in zip(torch.autograd.grad(y, leaves, dy), want):
        assert torch.equal(a, b)


def test_the_checkpoint_is_freed_by_the_backward():
    """An output that is kept after the backward holds no codes; a graph that is kept does, and serves again."""
    leaves, dy = step_leaves(m=40000)
    codes = 40000 * (256 + 8)
    y = lb().checkpointed_linear(*leaves)
    first = [t.cpu() for t in torch.autograd.grad(y, leaves, dy, retain_graph=True)]
    held = torch.cuda.memory_allocated()
    second = [t.cpu() for t in torch.autograd.grad(y, leaves, dy)]
    assert held - torch.cuda.memory_allocated() >= codes
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, leaves, dy)


@pytest.mark.parametrize("unpack", [lambda t: t, lambda t: t.cuda().short(), lambda t: t.cuda()[:1]])
def test_a_checkpoint_that_comes_back_otherwise_is_refused(unpack):
    """Saved tensors that hooks give back on another device, as another type or cut short are not read."""
    from nicecore import _lib as L
    leaves, dy = step_leaves()
    leaves[0].requires_grad_(False)  # (the weight is not saved then)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), unpack):
        y = lb().checkpointed_linear(*leaves)
    with pytest.raises(L.NiceCoreError, match="checkpoint came back"):
        torch.autograd.grad(y, leaves[1:], dy)
