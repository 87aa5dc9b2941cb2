"""The 8-bit layer operators (nicecore.lowbit) against their definitions in float64
(oracle/lowbit_oracle.py).

Tolerances.  u = 2^-24 is half a float32 step, e = finfo(out).eps / 2 the output's rounding.
Codes, scales and step bytes are equal.  A decoded value is one float32 product rounded to its
type.  quantized_linear: the integer sum is exact, then four float32 roundings (sum to float,
scale product, their product, bias) and the output's.  The layer's products: a matrix
instruction adds 32 products to a float32 sum; its error is taken as 2 roundings of the
running sum (1.9 measured) for each of the n / 32 instructions, and one for each of its 32
products; a float32 product is 6 (weight gradient 3) such sums of planes and leaves out 2^-25.
The float32 products of y and dx (half planes: three products for each 32 columns, n / 32 x 3 x 2 roundings of
the running sum; a representation of 2^-22 on either side and a product of 2^-22 left out; products of 11-bit
numbers are exact) are inside that bound: (6 n / 32 + 12 + 4) u against (12 n / 32 + 40) u.
"""
import ctypes
import math

import pytest
import torch

from oracle import lowbit_oracle as LO

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]


def lb():
    from nicecore import lowbit
    return lowbit


def gen(seed):
    return torch.Generator().manual_seed(seed)


def acts(m, k, dtype, seed):
    g = gen(seed)
    x = torch.randn(m, k, generator=g) * torch.exp(torch.randn(k, generator=g))
    x = torch.where(torch.rand(m, k, generator=g) < 0.01, 20 * x, x)
    return x.to(dtype)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def out_tol(y, dtype):
    """The rounding of y to dtype: half a step, of the least normal number below it."""
    return half_step(dtype) * y.abs().clamp_min(torch.finfo(dtype).tiny)


def check(got, want, tol):
    got = got.detach().double().cpu()
    err = (got - want).abs()
    worst = (err / tol.clamp_min(1e-300)).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"worst error {worst:.3f} of its bound"


ROWS = [(1, 1), (3, 31), (5, 93), (4, 128), (130, 256), (7, 513), (4, 1000), (3, 1025), (2, 4096), (2, 8192),
        (2, 8200), (1, 20001)]


# ---- codes --------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", ROWS)
def test_row_codes(m, k, dtype):
    x = acts(m, k, dtype, 10 * m + k)
    q = lb().quantize_rows(x.cuda())
    want, s = LO.row_codes(x)
    assert torch.equal(q.codes.cpu().double(), want)
    assert torch.equal(q.scales.cpu(), s)
    assert not q._storage[:, k:].any()
    assert q.shape == x.shape and q.codes.dtype == torch.int8
    assert torch.equal(q.dequantize().cpu(), (want.float() * s[:, None]).to(dtype))


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", ROWS)
def test_group_codes(m, k, dtype, relu):
    x = acts(m, k, dtype, 7 * m + k)
    p = lb().pack_activations(x.cuda(), relu=relu)
    q, byte, v = LO.group_codes(x, relu)
    assert torch.equal(p.codes.cpu().double(), q)
    assert torch.equal(p.scales.cpu().long(), byte)
    assert not p._storage[:, k:].any()
    assert torch.equal(p.dequantize().cpu().double(), v.to(dtype).double())
    # half a step of error, and the value is exact in the 16-bit types
    a = torch.relu(x.double()) if relu else x.double()
    step = torch.ldexp(torch.ones_like(byte, dtype=torch.float64), (byte - 127).int()).repeat_interleave(32, 1)[:, :k]
    assert ((v - a).abs() <= step / 2).all()
    assert torch.equal(v.to(dtype).double(), v)


def test_codes_next_to_ties_and_at_the_ends():
    """Quotients on and one ulp beside a half, zero rows, the least and the largest numbers."""
    s = (torch.tensor(3.0) * torch.tensor(1 / 127, dtype=F32)).item()
    k = torch.arange(-126, 126)
    mid = ((k.double() + 0.5) * torch.tensor(s, dtype=F32).double()).float()
    up, dn = torch.nextafter(mid, torch.full_like(mid, 9.)), torch.nextafter(mid, torch.full_like(mid, -9.))
    rows = [torch.cat([torch.tensor([3.0]), r]) for r in (mid, up, dn)]
    n = rows[0].numel()
    rows += [torch.arange(n).float() + 0.5 - n // 2 for _ in range(1)]  # exact ties with s = amax / 127 off a power of two
    rows += [torch.cat([torch.tensor([127.0]), (k.float() + 0.5)])]     # s = 1: exact ties
    rows += [torch.zeros(n), torch.full((n,), 1e-45), torch.full((n,), 3.4e38), torch.full((n,), -1.2e-38)]
    x = torch.stack(rows)
    x[5, 0], x[5, 1] = -0.0, 0.0
    q = lb().quantize_rows(x.cuda())
    want, sc = LO.row_codes(x)
    assert torch.equal(q.codes.cpu().double(), want) and torch.equal(q.scales.cpu(), sc)
    for relu in (False, True):
        p = lb().pack_activations(x.cuda(), relu=relu)
        wq, byte, v = LO.group_codes(x, relu)
        assert torch.equal(p.codes.cpu().double(), wq) and torch.equal(p.scales.cpu().long(), byte)
        assert torch.equal(p.dequantize().cpu().double(), v.float().double())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_codes_of_rows_that_are_not_finite(bad, dtype):
    x = acts(4, 100, dtype, 1)
    x[2, 40] = bad
    q = lb().quantize_rows(x.cuda())
    d = q.dequantize().cpu()
    assert torch.isnan(d[2]).all() and torch.isfinite(d[[0, 1, 3]]).all()
    for relu in (False, True):
        p = lb().pack_activations(x.cuda(), relu=relu)
        wq, byte, v = LO.group_codes(x, relu)
        assert torch.equal(p.codes.cpu().double(), wq) and torch.equal(p.scales.cpu().long(), byte)
        d = p.dequantize().cpu()
        hit = torch.zeros(4, 100, dtype=torch.bool)
        hit[2, 32:64] = not (relu and bad == -float("inf"))
        assert torch.equal(torch.isnan(d), hit)


@pytest.mark.parametrize("dtype", TYPES)
def test_codes_of_strided_rows(dtype):
    base = acts(12, 600, dtype, 3).cuda()
    for x in (base[:, 1:301], base[::3, 8:264], base.t()[5:50], base.view(3, 4, 600)[:, 1:3, :77], base[0], base[:1].expand(5, -1)):
        q, p = lb().quantize_rows(x), lb().pack_activations(x)
        flat = x.reshape(-1, x.shape[-1]).cpu()
        want, s = LO.row_codes(flat)
        assert q.codes.shape == x.shape and q.scales.shape == x.shape[:-1]
        assert torch.equal(q.codes.reshape(flat.shape).cpu().double(), want)
        assert torch.equal(q.scales.reshape(-1).cpu(), s)
        assert torch.equal(p.codes.reshape(flat.shape).cpu().double(), LO.group_codes(flat, False)[0])
        assert p.dequantize().shape == x.shape


# ---- the 8-bit product ----------------------------------------------------------------------------

def product_case(m, k, n, dtype, out_dtype, bias, relu, seed):
    x, w = acts(m, k, dtype, seed), acts(n, k, F32, seed + 1)
    b = (5 * torch.randn(n, generator=gen(seed + 2))).to(bias) if bias else None
    w8 = lb().quantize_rows(w.cuda())
    y = lb().quantized_linear(x.cuda(), w8, b.cuda() if bias else None, relu=relu, out_dtype=out_dtype)
    xq, xs = LO.row_codes(x)
    wq, ws = LO.row_codes(w)
    raw = LO.quantized_linear(xq, xs, wq, ws)
    want = LO.quantized_linear(xq, xs, wq, ws, b, relu)
    tol = 4 * U * (raw.abs() + (b.double().abs() if bias else 0)) * (1 + 1e-6) + 2.0 ** -148
    check(y, want, tol + out_tol(want.abs() + tol, out_dtype))
    assert y.dtype == out_dtype and y.shape == (m, n)
    return y


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 64, 65, 130, 300])
@pytest.mark.parametrize("k,n", [(1, 1), (31, 4), (93, 256), (128, 129), (256, 256), (517, 33), (1024, 1001)])
def test_quantized_linear(m, k, n):
    product_case(m, k, n, F32, F32, F32, (m + k) % 2 == 0, 3 * m + k)


@pytest.mark.parametrize("dtype,out_dtype,bias", [(F16, F16, F16), (BF16, BF16, BF16), (BF16, F32, F32), (F32, BF16, None),
                                                  (F16, F32, None)])
@pytest.mark.parametrize("m,k,n", [(1, 2048, 520), (5, 300, 77), (40, 640, 256), (257, 192, 384), (600, 128, 515)])
def test_quantized_linear_types(m, k, n, dtype, out_dtype, bias):
    product_case(m, k, n, dtype, out_dtype, bias, False, m + n)


@pytest.mark.parametrize("m,k,n", [(1, 8192, 2048), (3, 16384, 256), (1024, 768, 1536), (2100, 512, 640), (64, 4096, 4096),
                                   (16, 2048, 300), (17, 256, 4100), (700, 250, 517), (300, 2049, 1027), (90, 8200, 33),
                                   (6000, 96, 2050)])
def test_quantized_linear_larger(m, k, n):
    product_case(m, k, n, BF16, BF16, F32, True, m)


def test_quantized_linear_saturated_sums():
    """Every code at 127 over the longest rows: the sum reaches 127^2 131072 < 2^31."""
    from nicecore import _lib as L
    k = L.NC_MAX_INPUTS
    x = torch.ones(3, k)
    x[1] = -1
    w = torch.ones(5, k)
    y = lb().quantized_linear(x.cuda(), lb().quantize_rows(w.cuda()))
    want = torch.tensor([k, -k, k]).double()[:, None].expand(3, 5)
    check(y, want, 6 * U * want.abs())


def test_quantized_linear_of_codes_and_leading_dimensions():
    x = acts(24, 96, BF16, 5)
    w8 = lb().quantize_rows(acts(40, 96, F32, 6).cuda())
    y = lb().quantized_linear(x.cuda(), w8)
    q = lb().quantize_rows(x.view(2, 3, 4, 96).cuda())
    assert torch.equal(lb().quantized_linear(q, w8).view(24, 40), y)
    assert torch.equal(lb().quantized_linear(x[7].cuda(), w8), y[7])
    assert lb().quantized_linear(x[:0].cuda(), w8).shape == (0, 40)
    wide = acts(24, 200, BF16, 5).cuda()
    wide[:, 50:146] = x.cuda()
    assert torch.equal(lb().quantized_linear(wide[:, 50:146], w8), y)


def test_quantized_linear_keeps_faults_visible():
    x = acts(70, 64, F32, 8)
    x[3, 5] = float("nan")
    x[66, 1] = float("inf")
    w8 = lb().quantize_rows(acts(20, 64, F32, 9).cuda())
    for relu in (False, True):
        y = lb().quantized_linear(x.cuda(), w8, relu=relu).cpu()
        bad = torch.zeros(70, dtype=torch.bool)
        bad[[3, 66]] = True
        assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all()


# ---- the layer with an 8-bit checkpoint -----------------------------------------------------------

def sum_tol(terms, n, planes):
    """A sum of n products whose magnitudes add up to ``terms``."""
    return (2 * (planes * math.ceil(n / 32) + 4) + 32) * U * terms + 2.0 ** -25 * terms


def layer_run(x, w, b, dy, relu):
    leaves = [t.detach().cuda().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    y = lb().checkpointed_linear(*leaves, relu=relu)
    wanted = [t for t in leaves if t is not None]
    return (y, *torch.autograd.grad(y, wanted, dy.cuda()))


def layer_case(m, k, n, dtype, relu, seed, bias=True):
    g = gen(seed)
    x = acts(m, k, dtype, seed + 1)
    w = (torch.randn(n, k, generator=g) / math.sqrt(k)).to(dtype)
    b = torch.randn(n, generator=g).to(dtype) if bias else None
    dy = torch.randn(m, n, generator=g).to(dtype)
    got = layer_run(x, w, b, dy, relu)
    y, dx, dw, db = LO.layer(x, w, b, dy, relu)
    f = 6 if dtype == F32 else 1
    a = torch.relu(x.double()) if relu else x.double()
    v = LO.group_codes(x, relu)[2]

    def one(out, want, terms, count, planes):
        assert out.dtype == dtype and out.shape == want.shape
        t = sum_tol(terms, count, planes)
        check(out, want, t + out_tol(want.abs() + t, dtype))
        # roundings of a random sign: well inside that bound
        if dtype == F32 and want.norm() > 0:
            rel = ((out.detach().double().cpu() - want).norm() / want.norm()).item()
            assert rel <= 4 * U * math.sqrt(planes * count / 32 + 16), rel

    one(got[0], y, a.abs() @ w.double().abs().t() + (b.double().abs() if bias else 0), k, f)
    one(got[1], dx, dy.double().abs() @ w.double().abs(), n, f)
    one(got[2], dw, dy.double().abs().t() @ v.abs(), m, 3 if dtype == F32 else 1)
    if bias:
        t = (m / 8 + 300) * U * dy.double().abs().sum(0)
        check(got[3], db, t + out_tol(db.abs() + t, dtype))
    if relu:
        assert not got[1].cpu()[x <= 0].any()
    return got


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 256, 256), (2, 33, 5), (31, 93, 256), (32, 64, 64), (65, 128, 129),
                                   (200, 256, 4), (129, 517, 260), (257, 192, 320), (513, 96, 640)])
def test_layer(m, k, n, dtype, relu):
    layer_case(m, k, n, dtype, relu, m + k + n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(5000, 93, 256), (3001, 256, 256), (1024, 1024, 768), (640, 512, 2048), (70, 1100, 55),
                                   (64, 55, 4616), (150, 2047, 1033), (1, 4096, 96), (33000, 40, 300), (9000, 300, 130)])
def test_layer_larger(m, k, n, dtype):
    layer_case(m, k, n, dtype, True, m, bias=m % 2 == 0)


def test_layer_strides_and_leading_dimensions():
    g = gen(11)
    for dtype in TYPES:
        big = torch.randn(40, 300, generator=g).to(dtype).cuda()
        wide = torch.randn(50, 300, generator=g).to(dtype).cuda()
        dyb = torch.randn(40, 150, generator=g).to(dtype).cuda()
        for cut, wcut, dcut in ((slice(0, 128), slice(64, 192), slice(0, 50)), (slice(3, 95), slice(1, 93), slice(7, 57))):
            x, w, dy = big[:, cut], wide[:, wcut], dyb[:, dcut]
            ref = layer_run(x.contiguous(), w.contiguous(), None, dy.contiguous(), True)
            for got in (layer_run(x, w, None, dy, True), layer_run(x.t().contiguous().t(), w.t().contiguous().t(), None,
                                                                   dy.t().contiguous().t(), True)):
                for a, b in zip(got, ref):
                    assert torch.equal(a, b)
            x4 = x.reshape(2, 5, 4, -1)
            got = layer_run(x4, w, None, dy.reshape(2, 5, 4, -1), True)
            assert got[0].shape == (2, 5, 4, 50) and got[1].shape == x4.shape
            assert torch.equal(got[0].reshape(40, 50), ref[0]) and torch.equal(got[1].reshape(x.shape), ref[1])
            assert torch.equal(got[2], ref[2])


@pytest.mark.parametrize("dtype", TYPES)
def test_layer_partial_gradients_and_empty_batches(dtype):
    x, w = acts(9, 40, dtype, 1).cuda(), acts(6, 40, dtype, 2).cuda()
    b = torch.ones(6, device="cuda", dtype=dtype)
    dy = torch.randn(9, 6, generator=gen(3)).to(dtype).cuda()
    full = layer_run(x, w, b, dy, True)
    for pick in range(1, 8):
        leaves = [t.clone().requires_grad_(bool(pick >> i & 1)) for i, t in enumerate((x, w, b))]
        y = lb().checkpointed_linear(*leaves, relu=True)
        y.backward(dy)
        for i, t in enumerate(leaves):
            assert torch.equal(t.grad, full[1 + i]) if pick >> i & 1 else t.grad is None
    with torch.no_grad():
        assert torch.equal(lb().checkpointed_linear(x, w, b, relu=True), full[0])
    leaves = [t.requires_grad_(True) for t in (x[:0].clone(), w.clone(), b.clone())]
    y = lb().checkpointed_linear(*leaves)
    assert y.shape == (0, 6)
    y.sum().backward()
    assert leaves[0].grad.shape == (0, 40) and not leaves[1].grad.any() and not leaves[2].grad.any()
    y = lb().checkpointed_linear(x.clone().requires_grad_(True), w, b)
    y.sum().backward()  # an expanded gradient


def test_layer_gradients_against_differences():
    """The layer is linear in each argument apart from the checkpoint: a central difference of the
    float64 definition along a direction equals the gradient's product with it, up to the sums'
    roundings, and for W up to the checkpoint's half steps besides."""
    m, k, n = 40, 70, 30
    g = gen(21)
    x = torch.randn(m, k, generator=g)
    x = torch.where(x.abs() < 0.05, torch.full_like(x, 0.3), x)  # no ReLU changes sides below
    w, b = torch.randn(n, k, generator=g), torch.randn(n, generator=g)
    dy = torch.randn(m, n, generator=g)
    _, dx, dw, db = layer_run(x, w, b, dy, True)
    h = 2.0 ** -6

    def value(x, w, b):
        return (LO.layer(x, w, b, dy, True)[0] * dy.double()).sum()

    for i, (leaf, grad) in enumerate(((x, dx), (w, dw), (b, db))):
        v = torch.sign(torch.randn(leaf.shape, generator=g)).double()
        hi, lo = [x.double(), w.double(), b.double()], [x.double(), w.double(), b.double()]
        hi[i], lo[i] = hi[i] + h * v, lo[i] - h * v
        fd = (value(*hi) - value(*lo)) / (2 * h)
        got = (grad.double().cpu() * v).sum()
        mags = {0: dy.abs().double() @ w.abs().double(), 1: dy.abs().double().t() @ x.abs().double(), 2: dy.abs().double().sum(0)}[i]
        tol = (sum_tol(mags, max(m, n, k), 6)).sum()
        if i == 1:
            step = torch.ldexp(torch.ones(m, 3, dtype=torch.float64), (LO.group_codes(x, True)[1] - 127).int())
            tol = tol + (dy.abs().double().t() @ (step / 2).repeat_interleave(32, 1)[:, :k]).sum()
        assert (got - fd).abs() <= tol


@pytest.mark.parametrize("dtype", TYPES)
def test_layer_keeps_faults_visible(dtype):
    x, w = acts(70, 96, dtype, 4), acts(33, 96, dtype, 5)
    dy = torch.randn(70, 33, generator=gen(6)).to(dtype)
    x[68, 40] = float("nan")
    y, dx, dw = layer_run(x, w, None, dy, True)
    rows = torch.arange(70) != 68
    assert torch.isnan(y.cpu()[68]).all() and torch.isfinite(y.cpu()[rows]).all()
    assert torch.isfinite(dx).all()
    cols = torch.zeros(96, dtype=torch.bool)
    cols[32:64] = True  # the group that holds it
    assert torch.isnan(dw.cpu()[:, cols]).all() and torch.isfinite(dw.cpu()[:, ~cols]).all()
    x[68, 40] = 1
    dy[69, 7] = float("inf")
    y, dx, dw = layer_run(x, w, None, dy, False)
    assert not torch.isfinite(dx.cpu()[69]).any() and torch.isfinite(dx.cpu()[:69]).all()
    n = torch.arange(33) == 7
    assert not torch.isfinite(dw.cpu()[n]).any() and torch.isfinite(dw.cpu()[~n]).all()


def test_layer_float32_range():
    """Float products keep float32's range: large, small and mixed magnitudes."""
    for scale in (1e18, 1e-15, 1.0):
        g = gen(31)
        x = torch.randn(50, 160, generator=g) * scale
        w = torch.randn(70, 160, generator=g) * torch.exp(4 * torch.randn(70, 1, generator=g))
        dy = torch.randn(50, 70, generator=g)
        y, dx, dw = layer_run(x, w, None, dy, False)
        wy, wdx, wdw, _ = LO.layer(x, w, None, dy, False)
        check(y, wy, sum_tol(x.double().abs() @ w.double().abs().t(), 160, 6))
        check(dx, wdx, sum_tol(dy.double().abs() @ w.double().abs(), 70, 6))
        check(dw, wdw, sum_tol(dy.double().abs().t() @ LO.group_codes(x, False)[2].abs(), 50, 3))


def test_runs_are_identical_and_scratch_is_not_read():
    """Two runs agree to the bit, also where the allocator hands out memory full of NaNs."""
    for dtype, (m, k, n) in ((F32, (700, 200, 130)), (BF16, (513, 320, 260))):
        x, w = acts(m, k, dtype, 1), acts(n, k, dtype, 2)
        b, dy = acts(1, n, dtype, 3)[0], acts(m, n, dtype, 4)
        one = layer_run(x, w, b, dy, True)
        w8 = lb().quantize_rows(w.cuda())
        y1 = lb().quantized_linear(x.cuda(), w8)
        poison = [torch.full((1 << s,), 255, device="cuda", dtype=torch.uint8) for s in (16, 20, 22, 24) for _ in range(6)]
        del poison
        two = layer_run(x, w, b, dy, True)
        for p, q in zip(one, two):
            assert torch.equal(p, q)
        assert torch.equal(lb().quantized_linear(x.cuda(), w8), y1)


def test_another_stream():
    x, w = acts(300, 256, F32, 1).cuda(), acts(256, 256, F32, 2).cuda()
    dy = acts(300, 256, F32, 3).cuda()
    ref = layer_run(x, w, None, dy, True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = layer_run(x, w, None, dy, True)
        q = lb().quantized_linear(x, lb().quantize_rows(w))
    torch.cuda.current_stream().wait_stream(s)
    for p, r in zip(got, ref):
        assert torch.equal(p, r)
    assert torch.equal(q, lb().quantized_linear(x, lb().quantize_rows(w)))


def test_a_captured_chain_replays():
    """Encode, product and a training step of two layers in one graph: every replay equals the
    eager step on the same inputs, with eager work between the replays."""
    g = gen(41)
    x = torch.randn(333, 93, generator=g).cuda()
    ws = [torch.randn(256, 93, generator=g).cuda() / 9, torch.randn(4, 256, generator=g).cuda() / 16]
    bs = [torch.randn(256, generator=g).cuda(), torch.randn(4, generator=g).cuda()]
    dy = torch.randn(333, 4, generator=g).cuda()
    w8 = lb().quantize_rows(ws[0])

    def body(x, dy):
        leaves = [t.detach().requires_grad_(True) for t in (x, *ws, *bs)]
        h = lb().checkpointed_linear(leaves[0], leaves[1], leaves[3])
        y = lb().checkpointed_linear(h, leaves[2], leaves[4], relu=True)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy), lb().quantized_linear(x, w8, bs[0], relu=True))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    sx, sdy = x.clone(), dy.clone()
    with torch.cuda.stream(side):
        body(sx, sdy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = body(sx, sdy)
    for r in range(4):
        sx.copy_(x * (1 + r))
        sdy.copy_(dy.roll(r, 0))
        eager = body(sx.clone(), sdy.clone())
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert torch.equal(a, b)


def test_chain_follows_the_full_mlp():
    """Four layers as the scene MLP stacks them: outputs and input gradient as the float64 MLP,
    weight gradients within the checkpoints' half steps."""
    g = gen(51)
    m, widths = 900, [93, 256, 256, 256, 4]
    ws = [torch.randn(o, i, generator=g) * math.sqrt(2 / i) for i, o in zip(widths, widths[1:])]
    bs = [0.1 * torch.randn(o, generator=g) for o in widths[1:]]
    x = torch.sin(3 * torch.randn(m, 93, generator=g))
    dy = torch.randn(m, 4, generator=g)
    dev = [t.cuda().requires_grad_(True) for t in (x, *ws, *bs)]
    h = dev[0]
    for l in range(4):
        h = lb().checkpointed_linear(h, dev[1 + l], dev[5 + l], relu=l > 0)
    got = torch.autograd.grad(h, dev, dy.cuda())
    ref = [t.double().requires_grad_(True) for t in (x, *ws, *bs)]
    r = ref[0]
    for l in range(4):
        r = torch.nn.functional.linear(torch.relu(r) if l else r, ref[1 + l], ref[5 + l])
    want = torch.autograd.grad(r, ref, dy.double())
    rel = lambda a, b: ((a.detach().double().cpu() - b).norm() / b.norm()).item()  # noqa: E731
    assert rel(h, r.detach()) < 1e-5
    # dx, and the biases: float32 sums (a ReLU within rounding of 0 may fall on the other side)
    for k in (0, 5, 6, 7, 8):
        assert rel(got[k], want[k]) < 1e-3, k
    # half a step of at most amax / 127 (64 codes a power of two at the least): uniform, so
    # step / sqrt(12) rms against activations of rms >= amax / 8
    for k in (1, 2, 3, 4):
        assert rel(got[k], want[k]) < 8 * (1 / 63.5) / math.sqrt(12), k


def test_workspace_sizes_are_enough():
    """The C entries take exactly the workspace that they ask for, full of NaNs."""
    from nicecore import _lib as L
    lib = L.load()
    x, w = acts(77, 100, F32, 1).cuda(), acts(50, 100, F32, 2).cuda()
    y = torch.empty(77, 50, device="cuda")
    a = L.NcLayerArgs(abi_version=L.NC_ABI_VERSION, dtype=L.NC_F32, rows=77, inputs=100, outputs=50, x=x.data_ptr(),
                      x_stride=100, w=w.data_ptr(), w_stride=100, y=y.data_ptr(), y_stride=50, code_stride=128)
    n = lib.nc_layer_workspace_bytes(ctypes.byref(a), 0)
    guard = torch.full((n + 4096,), 255, device="cuda", dtype=torch.uint8)
    s = L.raw_stream(x.device)
    assert lib.nc_layer_forward(ctypes.byref(a), guard.data_ptr(), n, s) == 0
    assert lib.nc_layer_forward(ctypes.byref(a), guard.data_ptr(), n - 1, s) < 0
    torch.cuda.synchronize()
    assert bool((guard[n:] == 255).all())
    with torch.no_grad():
        assert torch.equal(y, lb().checkpointed_linear(x, w))


# large outputs (256 x 256 tiles, the codes' values written out), one part and several, both formats; float sums
# cut over large tiles; many cuts of a long batch
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("m,k,n,dtype", [(777, 2048, 1030, F16), (1000, 1100, 2100, BF16), (64, 4096, 1024, BF16), (300, 2100, 1100, F32),
                                         (1030, 260, 4100, F32), (40000, 60, 130, BF16), (70001, 20, 30, F32)])
def test_layer_cuts(m, k, n, dtype, relu):
    layer_case(m, k, n, dtype, relu, m + n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(1, 40, 50), (70, 40, 50), (1000, 300, 40), (130, 2048, 1100)])
def test_layer_bias_gradient_alone(m, k, n, dtype):
    """db without dW, and dW without db, are what both together give."""
    x, w = acts(m, k, dtype, 1).cuda(), acts(n, k, dtype, 2).cuda()
    b, dy = acts(1, n, dtype, 3)[0].cuda(), acts(m, n, dtype, 4).cuda()
    wl, bl = w.clone().requires_grad_(), b.clone().requires_grad_()
    dw, db = torch.autograd.grad(lb().checkpointed_linear(x, wl, bl), (wl, bl), dy)
    alone, = torch.autograd.grad(lb().checkpointed_linear(x, w, bl), bl, dy)
    # (other parts of the sum: its roundings, not its terms)
    t = 2 * (m / 8 + 300) * U * dy.double().abs().sum(0).cpu()
    check(alone, db.double().cpu(), t + 2 * out_tol(db.double().cpu().abs() + t, dtype))
    assert torch.equal(torch.autograd.grad(lb().checkpointed_linear(x, wl, b), wl, dy)[0], dw)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m,k,n", [(1, 40, 50), (70, 256, 50), (193, 300, 300), (130, 2048, 1100)])
def test_layer_infinite_gradient_in_the_last_row(m, k, n, dtype):
    """Rows behind the last one take no part: dW and db are infinite or NaN where the formula's are."""
    x, dy = acts(m, k, dtype, 5), acts(m, n, dtype, 6)
    x[-1, ::3] = 0.0  # codes of 0: inf x 0 is NaN
    dy[-1, 7] = float("inf")
    _, dw, db = layer_run(x, acts(n, k, dtype, 7), torch.zeros(n, dtype=dtype), dy, False)[1:]
    v = LO.group_codes(x, False)[2]
    want = torch.where(v[-1] == 0, math.nan, torch.where(v[-1] > 0, math.inf, -math.inf))
    assert torch.equal(torch.nan_to_num(dw[7].double().cpu(), nan=5.0), torch.nan_to_num(want.double(), nan=5.0))
    assert db[7].item() == math.inf
    # the others are infinite only where the formula's value is beyond the type's range (float16: these inputs reach
    # sums of |dy v| of 10^5, its largest number is 65504)
    rest = [j for j in range(n) if j != 7]
    exact = dy[:, rest].double().t() @ v
    inside = exact.abs() + sum_tol(dy[:, rest].double().abs().t() @ v.abs(), m, 1) < torch.finfo(dtype).max
    assert inside.double().mean() > 0.9 and torch.isfinite(dw[rest].cpu()[inside]).all() and torch.isfinite(db[rest]).all()


@pytest.mark.parametrize("m,k,n", [(2000, 200, 64), (3000, 100, 128), (300, 4096, 1024), (1000, 2100, 1000), (4096, 300, 1500)])
def test_quantized_linear_tiles(m, k, n):
    """Few channels, the middle tiles, cut sums."""
    x, w = acts(m, k, BF16, m).cuda(), acts(n, k, F32, n).cuda()
    q, w8 = lb().quantize_rows(x), lb().quantize_rows(w)
    got = lb().quantized_linear(x, w8, out_dtype=F32).double().cpu()
    acc = q.codes.double().cpu() @ w8.codes.double().cpu().t()
    want = acc * q.scales.double().cpu()[:, None] * w8.scales.double().cpu()
    check(got, want, 4 * U * want.abs())
    assert torch.equal(lb().quantized_linear(q, w8), lb().quantized_linear(x, w8))


@pytest.mark.parametrize("shape", ["grows", "shrinks", "zeros first", "one spike", "rows apart"])
@pytest.mark.parametrize("m,k,n", [(70, 700, 130), (300, 1024, 257), (2000, 96, 300), (40, 4096, 256)])
def test_layer_float32_scales_within_rows(m, k, n, shape):
    """The power of two that a row's values are split by follows the row: a value is off by at most 2^-22 of itself or
    2^-36 of the largest in its row (of W 2^-40), beside the bound of the sums."""
    g = gen(k + n)
    x, w = torch.randn(m, k, generator=g), torch.randn(n, k, generator=g)
    dy = torch.randn(m, n, generator=g)
    if shape == "grows":
        x = x * torch.exp2(torch.linspace(-30, 30, k))
        dy = dy * torch.exp2(torch.linspace(-30, 30, n))
    elif shape == "shrinks":
        x = x * torch.exp2(torch.linspace(30, -30, k))
        dy = dy * torch.exp2(torch.linspace(30, -30, n))
    elif shape == "zeros first":
        x[:, :k // 2] = 0.0
        dy[:, :n // 2] = 0.0
    elif shape == "one spike":
        x[torch.arange(m), torch.randint(k, (m,), generator=g)] = 3e4
        dy[torch.arange(m), torch.randint(n, (m,), generator=g)] = -2e5
        w[torch.arange(n), torch.randint(k, (n,), generator=g)] = 1e3
    else:
        x, dy = x * torch.exp2(torch.linspace(-60, 40, m))[:, None], dy * torch.exp2(torch.linspace(40, -60, m))[:, None]
        w = w * torch.exp2(torch.linspace(-12, 12, n))[:, None]
    y, dx, _ = layer_run(x, w, None, dy, False)

    def bound(a, b):  # of a b^T
        a, b = a.double().abs(), b.double().abs()
        small = 2.0 ** -36 * a.amax(1, keepdim=True) * b.sum(1) + 2.0 ** -40 * a.sum(1, keepdim=True) * b.amax(1)
        return sum_tol(a @ b.t(), a.shape[1], 6) + small

    check(y, x.double() @ w.double().t(), bound(x, w))
    check(dx, dy.double() @ w.double(), bound(dy, w.t()))
