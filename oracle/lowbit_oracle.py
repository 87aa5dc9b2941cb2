"""ORACLE — TEST INFRASTRUCTURE ONLY.  Never imported by the product path.

The 8-bit layer operators (nicecore.lowbit) from their definitions, in float64 on the CPU.
The reference has no such operators: parity unpinned; the layer itself is the reference's
(``net = pts_linear(net); net = F.relu(net)``, src/conv_onet/models/decoder.py:190-219).
"""
from __future__ import annotations

import torch

GROUP = 32


def row_codes(x):
    """(codes float64 [M, K], scales float32 [M]): s = max(fl32(amax fl32(1 / 127)), 2^-126), q the integer
    nearest to x / s.  The float64 quotient of two float32 numbers is within 2^-53 of the exact
    one, which is a half-integer or at least 2^-49 (relative) from it: no code can differ."""
    x = x.double()
    top = x.abs().amax(1)
    inv = torch.tensor(1 / 127, dtype=torch.float32).double()  # (the product is exact in float64)
    s = (top * inv).to(torch.float32).clamp_min(torch.finfo(torch.float32).tiny)
    q = torch.round(x / s.double()[:, None]).clamp(-127, 127)
    bad = ~torch.isfinite(top)
    q[bad] = 0
    s[bad] = float("nan")
    return q, s


def group_codes(x, relu):
    """(codes float64 [M, K] as stored, bytes int64 [M, ceil(K / 32)], values float64 [M, K]).  float16's largest
    number ends the values of a float16 x: the one code value beyond it, 65536, is 65504 there."""
    m, k = x.shape
    half = x.dtype == torch.float16
    x = x.double()
    a = torch.where(x > 0, x, torch.zeros_like(x)) if relu else x
    a = torch.where(torch.isnan(x), x, a)
    most = 254 if relu else 127
    g = torch.nn.functional.pad(a, (0, -k % GROUP)).view(m, -1, GROUP)
    top = g.abs().amax(2)
    bad = ~torch.isfinite(top)
    safe = torch.where(bad, torch.ones_like(top), top)
    frac, e = torch.frexp(safe)  # safe = frac 2^e
    bits = 8 if relu else 7
    e = e.long() - bits + (frac > most / 2.0 ** bits)
    # a float32 exponent has a least value, and none above 254: the largest magnitudes saturate
    byte = (e + 127).clamp(1, 254 - (7 if relu else 6))
    byte = torch.where(top == 0, torch.ones_like(byte), byte)
    step = torch.ldexp(torch.ones_like(top), (byte - 127).to(torch.int32))
    clean = torch.where(bad[..., None], torch.zeros_like(g), g)
    q = torch.round(clean / step[..., None]).clamp(-most, most)
    v = torch.where(bad[..., None], torch.full_like(q, float("nan")), q * step[..., None])
    if half:
        v = v.clamp(-65504, 65504)
    q, v = (t.reshape(m, -1)[:, :k] for t in (q, v))
    if relu:
        q = torch.where((x > 0) | torch.isnan(x), q + 1, torch.zeros_like(q))
    return q, torch.where(bad, torch.full_like(byte, 255), byte), v


def quantized_linear(xq, xs, wq, ws, bias=None, relu=False):
    y = (xq @ wq.t()) * xs.double()[:, None] * ws.double()
    if bias is not None:
        y = y + bias.double()
    return torch.relu(y) if relu else y


def layer(x, w, b, dy, relu):
    """y, dx, dw, db of the checkpointed layer."""
    x, w, dy = x.double(), w.double(), dy.double()
    a = torch.relu(x) if relu else x
    y = a @ w.t()
    if b is not None:
        y = y + b.double()
    dx = dy @ w
    if relu:
        dx = torch.where(x > 0, dx, torch.zeros_like(dx))
    return y, dx, dy.t() @ group_codes(x, relu)[2], dy.sum(0)
