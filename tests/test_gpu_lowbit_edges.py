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
from test_gpu_lowbit import BF16, F16, F32, TYPES, U, acts, check, gen, layer_case, layer_run, lb, out_tol, sum_tol

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


def in_guard(nbytes):
    """A workspace of NaNs with as much behind it."""
    return torch.full((nbytes + (1 << 20),), 255, device="cuda", dtype=torch.uint8)


def intact(guard, nbytes):
    torch.cuda.synchronize()
    return bool((guard[nbytes:] == 255).all())


# odd and whole sizes; cut sums of every product; few rows; the decoded values of the large tiles
SIZES = [(77, 100, 50), (700, 200, 130), (2048, 64, 1), (200, 4096, 256), (500, 1024, 1024), (3000, 33, 70), (70, 2048, 2048)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_layers_stay_in_the_workspace_that_they_ask_for(m, k, n, dtype):
    """Forward and backward, each choice of outputs, from exactly as many bytes as the query says."""
    from nicecore import _lib as L
    lib, s = L.load(), L.raw_stream(torch.device("cuda", 0))
    x, w, b, dy = acts(m, k, dtype, 1).cuda(), acts(n, k, dtype, 2).cuda(), acts(1, n, dtype, 3)[0].cuda(), acts(m, n, dtype, 4).cuda()
    want = layer_run(x, w, b, dy, True)
    leaves = b.clone().requires_grad_()
    alone = torch.autograd.grad(lb().checkpointed_linear(x, w, leaves, relu=True), leaves, dy)[0]
    kp = (k + 127) // 128 * 128
    codes, steps = torch.empty(m, kp, device="cuda", dtype=torch.uint8), torch.empty(m, kp // 32, device="cuda", dtype=torch.uint8)
    y = torch.empty_like(dy)
    kind = {F32: L.NC_F32, F16: L.NC_F16, BF16: L.NC_BF16}[dtype]

    def run(call, back, **out):
        a = L.NcLayerArgs(abi_version=L.NC_ABI_VERSION, dtype=kind, relu=1, rows=m, inputs=k, outputs=n, x=x.data_ptr(), x_stride=k,
                          w=w.data_ptr(), w_stride=k, bias=b.data_ptr(), y=y.data_ptr(), y_stride=n, codes=codes.data_ptr(),
                          steps=steps.data_ptr(), code_stride=kp, dy=dy.data_ptr(), dy_stride=n, dx_stride=k,
                          **{o: t.data_ptr() for o, t in out.items()})
        size = lib.nc_layer_workspace_bytes(ctypes.byref(a), back)
        guard = in_guard(size)
        assert call(ctypes.byref(a), guard.data_ptr(), size, s) == 0
        assert intact(guard, size)
        if size > 256:
            assert call(ctypes.byref(a), guard.data_ptr(), size - 1, s) < 0

    run(lib.nc_layer_forward, 0)
    assert torch.equal(y, want[0])
    for names in (("dx", "dw", "db"), ("dw", "db"), ("dx",), ("dw",), ("db",), ("dx", "db")):
        out = {"dx": torch.full_like(x, math.nan), "dw": torch.full_like(w, math.nan), "db": torch.full_like(b, math.nan)}
        run(lib.nc_layer_backward, 1, **{o: out[o] for o in names})
        for o, t in zip(("dx", "dw", "db"), want[1:]):
            # (db without dW adds its rows in other parts)
            assert torch.equal(out[o], alone if o == "db" and "dw" not in names else t) if o in names else out[o].isnan().all(), (names, o)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,k,n", [(1, 256, 64), (64, 4096, 40), (200, 93, 256), (90, 8200, 33), (300, 4096, 256), (2100, 512, 640)])
@pytest.mark.parametrize("coded", [False, True])
def test_products_stay_in_the_workspace_that_they_ask_for(m, k, n, dtype, coded):
    from nicecore import _lib as L
    lib, s = L.load(), L.raw_stream(torch.device("cuda", 0))
    x = acts(m, k, dtype, 1).cuda()
    q, w8 = lb().quantize_rows(x), lb().quantize_rows(acts(n, k, F32, 2).cuda())
    want = lb().quantized_linear(q if coded else x, w8)
    out = torch.full((m, n), math.nan, device="cuda", dtype=dtype)
    kind = L.NC_F32 if dtype == F32 else L.NC_BF16
    a = L.NcQlinearArgs(abi_version=L.NC_ABI_VERSION, dtype=kind, out_dtype=kind, rows=m, inputs=k, outputs=n,
                        x=None if coded else x.data_ptr(), x_stride=k, x_codes=q._storage.data_ptr(), x_scales=q._scales.data_ptr(),
                        code_stride=w8._storage.shape[1], w_codes=w8._storage.data_ptr(), w_scales=w8._scales.data_ptr(),
                        out=out.data_ptr(), out_stride=n)
    size = lib.nc_quantized_linear_workspace_bytes(ctypes.byref(a))
    guard = in_guard(size)
    assert lib.nc_quantized_linear(ctypes.byref(a), guard.data_ptr(), size, s) == 0
    assert intact(guard, size)
    assert torch.equal(out, want)


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("far,kind", [(1e4, "unused"), (1e6, "unused"), (1e7, "unused"), (1e4, "scaled"), (1e6, "scaled"), (1e8, "scaled")])
@pytest.mark.parametrize("m,k,n", [(70, 256, 130), (300, 93, 256), (2000, 1024, 300), (4100, 256, 1500)])
def test_float32_products_of_rows_with_a_far_value(m, k, n, far, kind, back):
    """One input (one output's gradient) is far larger than the others, and its weights are 0 or as much smaller.
    x = (x0 + x1) / scale with the largest so far at 2^11 or above: x0 is off by 2^-11 of x or 2^-25, x1 is that
    remainder times 2^11, off by as much again: 2^-22 of x, or 2^-36 = 2^-47 of the largest.  W's planes, the largest at
    2^14 or above, are off by 2^-22 of w or 2^-25 = 2^-39 of the largest, and as much for W's first plane times 2^-11,
    which multiplies x1 2^11, no larger than x.  The rest as in test_gpu_lowbit.py."""
    g = gen(k + n)
    kk, nn = (n, k) if back else (k, n)  # the sum's length, the results
    a, w = torch.randn(m, kk, generator=g), torch.randn(nn, kk, generator=g) / math.sqrt(kk)
    a[:, 17] *= far
    w[:, 17] *= 0.0 if kind == "unused" else 1 / far
    if back:
        got = layer_run(torch.randn(m, k, generator=g), w.t().contiguous(), None, a, False)[1]
    else:
        got = layer_run(a, w, None, torch.zeros(m, n), False)[0]
    a, w = a.double(), w.double()
    want = a @ w.t()
    floors = 2.0 ** -47 * a.abs().amax(1, keepdim=True) * w.abs().sum(1) + 2.0 ** -38 * a.abs().sum(1, keepdim=True) * w.abs().amax(1)
    t = sum_tol(a.abs() @ w.abs().t(), kk, 6) + floors
    check(got, want, t + out_tol(want.abs() + t, F32))
    if far <= 1e6 or kind == "unused":  # the floors are below the other roundings: as near as ordinary rows
        rel = ((got.detach().double().cpu() - want).norm() / want.norm()).item()
        assert rel <= 4 * U * math.sqrt(6 * kk / 32 + 16), rel


def test_a_quantised_mlp_is_called_as_the_module():
    """decoders(p, c_grid=None), as the reference's renderer and mesher call the scene MLP."""
    from nicecore import decoder as D
    m = D.build_imap(seed=1).cuda()
    q = m.quantize()
    p = torch.rand(50, 3, generator=gen(1), dtype=torch.float64).cuda()
    assert torch.equal(q(p, c_grid=None), q(p)) and q(p, c_grid=None).shape == m(p, c_grid=None).shape


@pytest.mark.parametrize("k,n,relu", [(93, 256, False), (256, 256, True), (256, 4, True)])
def test_layers_of_a_mapper_iteration(k, n, relu):
    """The scene MLP's layers on 5,000 rays of 44 samples, against the float64 layer on the device."""
    m = 220000
    g = torch.Generator(device="cuda").manual_seed(k + n)
    x = torch.randn(m, k, generator=g, device="cuda")
    w = torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)
    b, dy = torch.randn(n, generator=g, device="cuda"), torch.randn(m, n, generator=g, device="cuda")
    got = layer_run(x, w, b, dy, relu)
    v = lb().pack_activations(x, relu=relu).dequantize().double()
    rows = torch.randint(m, (4096,), generator=gen(1))  # of the codes against their definition
    assert torch.equal(v[rows.cuda()].cpu(), LO.group_codes(x[rows.cuda()].cpu(), relu)[2])
    a = (torch.relu(x) if relu else x).double()
    w, dy = w.double(), dy.double()

    def near(out, want, terms, count, planes):
        tol = sum_tol(terms, count, planes)
        assert ((out.detach().double() - want).abs() <= tol + U * (want.abs() + tol)).all()
        rel = ((out.detach().double() - want).norm() / want.norm()).item()
        assert rel <= 4 * U * math.sqrt(planes * count / 32 + 16), rel

    wt, ones = w.t().contiguous(), torch.ones(1, m, device="cuda", dtype=torch.float64)
    near(got[0], a @ wt + b.double(), a.abs() @ wt.abs() + b.double().abs(), k, 6)
    mask = (x > 0).double() if relu else torch.ones_like(a)
    near(got[1], (dy @ w) * mask, dy.abs() @ w.abs(), n, 6)
    dyt = dy.t().contiguous()
    near(got[2], dyt @ v, dyt.abs() @ v.abs(), m, 3)
    sums, terms = (ones @ dy)[0], (ones @ dy.abs())[0]
    tol = (m / 8 + 300) * U * terms
    assert ((got[3].detach().double() - sums).abs() <= tol + U * sums.abs()).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_row_scales_are_those_of_the_devices_own_division(dtype):
    """A float32 tensor's amax / 127 on the device is the product with the rounded 1 / 127: the scales' definition."""
    x = acts(4000, 200, dtype, 8).cuda()
    assert torch.equal(lb().quantize_rows(x).scales, x.float().abs().amax(1) / 127)
    ends = torch.tensor([torch.finfo(dtype).max, torch.finfo(dtype).tiny, 1.0], device="cuda", dtype=dtype)[:, None]
    q = lb().quantize_rows(ends)
    assert torch.equal(q.scales, (ends.float().abs().amax(1) / 127).clamp_min(2.0 ** -126))
    assert torch.isfinite(q.dequantize()).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_offsets_past_32_bits(dtype):
    """1,100,000 rows of 2,048 channels: the last rows' codes, products and gradients, and the sums over all."""
    m, k, n, last = 1100000, 2048, 64, 1000
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(m, k, generator=g, device="cuda", dtype=dtype).requires_grad_()
    w = (torch.randn(n, k, generator=g, device="cuda") / 45).to(dtype).requires_grad_()
    b = torch.zeros(n, device="cuda", dtype=dtype, requires_grad=True)
    dy = torch.randn(m, n, generator=g, device="cuda", dtype=dtype)
    end = x.detach()[-last:]
    with torch.no_grad():
        q, part = lb().quantize_rows(x), lb().quantize_rows(end)
        assert torch.equal(q.codes[-last:], part.codes) and torch.equal(q.scales[-last:], part.scales)
        assert torch.equal(q.dequantize()[-last:], part.dequantize())
        w8 = lb().quantize_rows(w)
        assert torch.equal(lb().quantized_linear(x, w8)[-last:], lb().quantized_linear(end, w8))  # (exact sums)
        del q
        p, part = lb().pack_activations(x, relu=True), lb().pack_activations(end, relu=True)
        assert torch.equal(p.codes[-last:], part.codes) and torch.equal(p.scales[-last:], part.scales)
    y = lb().checkpointed_linear(x, w, b, relu=True)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    wd, ed = w.detach().double(), dy[-last:].double()
    f = 6 if dtype == F32 else 1

    def near(out, want, terms, count, planes):
        tol = sum_tol(terms, count, planes)
        step = torch.finfo(dtype).eps / 2
        assert ((out.detach().double() - want).abs() <= tol + step * (want.abs() + tol)).all()

    a = torch.relu(end).double()
    wt = wd.t().contiguous()
    near(y[-last:], a @ wt, a.abs() @ wt.abs(), k, f)
    near(dx[-last:], (ed @ wd) * (end > 0), ed.abs() @ wd.abs(), n, f)
    want, terms, sums, mags = torch.zeros_like(wd), torch.zeros_like(wd), torch.zeros(n, device="cuda", dtype=torch.float64), 0
    for at in range(0, m, 100000):
        v = lb().pack_activations(x.detach()[at:at + 100000], relu=True).dequantize().double()
        d = dy[at:at + 100000].double().t().contiguous()
        want, terms, sums, mags = want + d @ v, terms + d.abs() @ v, sums + d.sum(1), mags + d.abs().sum(1)
    near(dw, want, terms, m, 3 if dtype == F32 else 1)
    tol = (m / 8 + 300) * U * mags
    assert ((db.detach().double() - sums).abs() <= tol + torch.finfo(dtype).eps / 2 * (sums.abs() + tol)).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(3, 131072, 5), (3, 5, 131072), (140, 131072, 3)])
def test_layers_of_the_most_channels(m, k, n, dtype):
    layer_case(m, k, n, dtype, True, m + k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("stride", [1 << 22, (1 << 22) + 8])
def test_rows_far_apart(dtype, stride):
    """The longest row stride that is read in place, and one that is copied: rows of x and dy 2^22 elements apart."""
    m, k, n = 260, 192, 64
    x, w, dy = acts(m, k, dtype, 1).cuda(), acts(n, k, dtype, 2).cuda(), acts(m, n, dtype, 3).cuda()
    want = layer_run(x, w, None, dy, True)
    room = torch.empty(m * stride, device="cuda", dtype=dtype)
    far = room.as_strided((m, k), (stride, 1))
    fard = room.as_strided((m, n), (stride, 1), 1 << 20)
    far.copy_(x)
    fard.copy_(dy)
    leaves = [far.requires_grad_(), w.clone().requires_grad_()]
    y = lb().checkpointed_linear(*leaves, relu=True)
    for a, b in zip((y, *torch.autograd.grad(y, leaves, fard)), want):
        assert torch.equal(a, b)
    with torch.no_grad():
        w8 = lb().quantize_rows(w)
        assert torch.equal(lb().quantized_linear(far, w8), lb().quantized_linear(x, w8))
        assert torch.equal(lb().pack_activations(far).codes, lb().pack_activations(x).codes)


@pytest.mark.parametrize("dtype", TYPES)
def test_empty_leading_dimensions_and_weights_of_other_types(dtype):
    w = acts(12, 40, dtype, 1).cuda()
    for shape in ((0, 5, 40), (2, 0, 40), (0, 40)):
        x = torch.empty(shape, device="cuda", dtype=dtype, requires_grad=True)
        wl = w.clone().requires_grad_()
        y = lb().checkpointed_linear(x, wl, relu=True)
        assert y.shape == (*shape[:-1], 12)
        dx, dw = torch.autograd.grad(y, (x, wl), torch.empty_like(y))
        assert dx.shape == x.shape and not dw.any()
        with torch.no_grad():
            assert lb().quantized_linear(x, lb().quantize_rows(w)).shape == y.shape
            assert lb().quantize_rows(x).dequantize().shape == x.shape and lb().pack_activations(x).codes.shape == x.shape
    x = acts(30, 40, F32, 2)
    xq, xs = LO.row_codes(x)
    wq, ws = LO.row_codes(w.cpu())
    want = LO.quantized_linear(xq, xs, wq, ws)
    check(lb().quantized_linear(x.cuda(), lb().quantize_rows(w)), want, 4 * U * want.abs())


def test_graphs_that_share_a_pool_and_eager_calls_between():
    """Two captured training steps of one memory pool, replayed in turn with eager steps between them."""
    cases = []
    pool = torch.cuda.graph_pool_handle()
    for i, (m, k, n, dtype) in enumerate(((300, 256, 64, F32), (777, 100, 50, BF16))):
        x, w, dy = acts(m, k, dtype, i).cuda(), acts(n, k, dtype, i + 5).cuda(), acts(m, n, dtype, i + 9).cuda()

        def body(x, w=w, dy=dy):
            leaves = [t.detach().requires_grad_() for t in (x, w)]
            y = lb().checkpointed_linear(*leaves, relu=True)
            return (y.detach(), *torch.autograd.grad(y, leaves, dy))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            body(x)
        torch.cuda.current_stream().wait_stream(side)
        graph, held = torch.cuda.CUDAGraph(), x.clone()
        with torch.cuda.graph(graph, pool=pool):
            out = body(held)
        cases.append((graph, held, x, body, out))
    for r in range(3):
        for graph, held, x, body, out in cases:
            held.copy_(x.roll(r, 0))
            graph.replay()
            got = [t.clone() for t in out]  # (the other graph writes the shared pool)
            for a, b in zip(got, body(x.roll(r, 0))):
                assert torch.equal(a, b)


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("m,k,n", [(5, 40, 30), (300, 93, 256), (2000, 256, 256), (140, 2100, 300), (4100, 1024, 1500)])
def test_float32_infinities(m, k, n, relu):
    """Infinities in x, W or dy of a float32 layer: infinite or NaN where the formula is, finite elsewhere."""
    g = gen(m)
    x, w = acts(m, k, F32, 1), torch.randn(n, k, generator=g)
    dy = torch.randn(m, n, generator=g)
    plain = (x.clone(), w.clone(), dy.clone())

    def same(got, want, terms, count, planes):
        got, fine = got.detach().double().cpu(), torch.isfinite(want)
        assert torch.equal(torch.isfinite(got), fine) and torch.equal(got.isnan(), want.isnan())
        over = ~fine & ~want.isnan()
        assert torch.equal(got[over], want[over])
        t = sum_tol(terms, count, planes)
        check(got[fine], want[fine], (t + out_tol(want.abs() + t, F32))[fine])

    for place in range(3):
        x, w, dy = (t.clone() for t in plain)
        t = (x, w, dy)[place]
        t[1, 3], t[-1, -1], t[2, 5], t[2, 9] = math.inf, -math.inf, math.inf, -math.inf
        if place == 0:
            w[4, 3] = 0.0  # inf x 0
        elif place == 1:
            x[3, 3] = 0.0
            dy[3, 1] = 0.0
        else:
            w[1, 7] = 0.0 if m > 5 else w[1, 7]
        y, dx, dw = layer_run(x, w, None, dy, relu)
        a = torch.relu(x.double()) if relu else x.double()
        wd, d = w.double(), dy.double()
        nz = lambda u: torch.nan_to_num(u.abs(), posinf=0.0)  # noqa: E731
        same(y, a @ wd.t(), nz(a) @ nz(wd).t(), k, 6)
        full = d @ wd
        same(dx, torch.where(x > 0, full, torch.zeros_like(full)) if relu else full, nz(d) @ nz(wd), n, 6)
        if place != 0:  # (x's infinities make NaN of their groups in the checkpoint)
            v = LO.group_codes(x, relu)[2]
            same(dw, d.t() @ v, nz(d).t() @ nz(v), m, 3)
