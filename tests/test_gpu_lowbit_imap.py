"""The 8-bit operators where the framework uses them: iMAP* training with 8-bit checkpoints
(Renderer with rendering.activations = 'int8', imap.eval_points) and the quantised scene MLP's
queries, on the golden scene and synthetic points.

Tolerances.  Outputs, point, ray and bias gradients are float32 computations: within OUT_TOL /
GRAD_TOL of the default path's (the tolerances of tests/test_gpu_imap.py), which itself is held to
the reference.  A ReLU whose input is within rounding of 0 may open on one path alone; with 1024 units
a point that happens at one point in some thousands, whose gradient then differs by that unit's
share: `open_units` finds the units in float64 and adds up what they can change.  A weight gradient sees each activation off by at most
half a step (activations of a ReLU: 1 / 254 of the group's largest at most, rms step / sqrt(12)).
"""
import json
import math
import os
import types

import numpy as np
import pytest
import torch

from oracle import lowbit_oracle as LO

pytestmark = pytest.mark.gpu
GOLD = os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden")
META = json.load(open(os.path.join(GOLD, "imap_meta.json")))
CASES = [c["name"] for c in META["cases"]]
OUT_TOL, GRAD_TOL = 2e-5, 2e-4


def load(name):
    with np.load(os.path.join(GOLD, f"imap_{name}.npz")) as z:
        return {k: torch.from_numpy(z[k]) for k in z.files}


def model():
    from nicecore import decoder as D
    d = load("scene")
    m = D.build_imap(seed=None)
    m.load_state_dict({k[len("param/"):]: v for k, v in d.items() if k.startswith("param/")})
    return m.cuda(), d["bound"]


def renderer(bound, n_importance, activations):
    from nicecore.renderer import Renderer
    cfg = {"rendering": {"lindisp": False, "perturb": 0.0, "N_samples": META["n_samples"], "N_surface": 0,
                         "N_importance": n_importance, "activations": activations}, "scale": 1, "occupancy": False}
    slam = types.SimpleNamespace(nice=False, bound=bound, H=64, W=80, fx=60., fy=60., cx=40., cy=32.)
    return Renderer(cfg, None, slam)


def rel_max(a, b):
    a, b = a.detach().double(), b.detach().double()
    return float((a - b).abs().max() / b.abs().max().clamp_min(1e-30))


def rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    return float((a - b).norm() / b.norm().clamp_min(1e-30))


WEIGHTS = [f"pts_linears.{l}.weight" for l in range(4)] + ["output_linear.weight"]
# half-step noise, rms, against activations whose rms is at least 1/16 of their group's largest
WEIGHT_REL = 16 * (1 / 127) / math.sqrt(12)


def open_units(m, p, up):
    """For points p and upstream gradients up: which points have a hidden unit whose input is within
    rounding of 0 (float64; 2^-18 of the sum of its terms' magnitudes: both paths add some 300 float32
    terms of which each rounds by at most 2^-23 of that sum, through four layers), and by how much
    those units can change each gradient: the sum, point by point, of |gradient with them open -
    gradient with them closed|."""
    prm = {k: v.detach().double().cpu() for k, v in m.named_parameters()}
    p, up = p.detach().double().cpu(), up.detach().double().cpu()

    near, masks = [], []
    h = torch.sin(p @ prm["embedder._B"])
    for l in range(4):
        w, b = prm[f"pts_linears.{l}.weight"], prm[f"pts_linears.{l}.bias"]
        z = torch.nn.functional.linear(h, w, b)
        near.append(z.abs() < 2.0 ** -18 * (h.abs() @ w.abs().t() + b.abs()))
        masks.append(z > 0)
        h = torch.relu(z)
    hit = torch.stack([n.any(1) for n in near]).any(0)
    change = {k: torch.zeros_like(v) for k, v in prm.items()}
    for i in hit.nonzero().flatten().tolist():
        grads = []
        for opened in (True, False):
            q = {k: v.clone().requires_grad_(True) for k, v in prm.items()}
            h = torch.sin(p[i:i + 1] @ q["embedder._B"])
            for l in range(4):
                z = torch.nn.functional.linear(h, q[f"pts_linears.{l}.weight"], q[f"pts_linears.{l}.bias"])
                keep = (masks[l][i] | near[l][i]) if opened else (masks[l][i] & ~near[l][i])
                h = z * keep
            raw = torch.nn.functional.linear(h, q["output_linear.weight"], q["output_linear.bias"])
            grads.append(torch.autograd.grad((raw * up[i]).sum(), list(q.values())))
        for k, a, b in zip(change, *grads):
            change[k] += (a - b).abs()
    return hit, change


def compare(full, coded, change=None):
    for name, g in full.items():
        if name in WEIGHTS:
            assert rel(coded[name], g) < WEIGHT_REL, (name, rel(coded[name], g))
            continue
        tol = GRAD_TOL * g.abs().max().double() + (change[name].to(g.device) if change else 0.0)
        worst = ((coded[name].double() - g.double()).abs() / tol.clamp_min(1e-30)).max().item()
        assert worst < 1, (name, worst)


@pytest.mark.parametrize("case", CASES)
def test_render_with_checkpoints(case):
    rec = load(case)
    n_imp = next(c for c in META["cases"] if c["name"] == case)["n_importance"]
    got = {}
    for act in ("float32", "int8"):
        m, bound = model()
        r = renderer(bound, n_imp, act)
        ro, rd = rec["rays_o"].cuda().requires_grad_(True), rec["rays_d"].cuda().requires_grad_(True)
        dep = rec["gt_depth"].cuda() if "nodepth" not in case else None
        d, v, c = r.render_batch_ray(None, m, rd, ro, "cuda", "color", dep)
        (d.sum() + c.sum()).backward()
        grads = {"rays_o": ro.grad, "rays_d": rd.grad, **{n: p.grad for n, p in m.named_parameters()}}
        got[act] = (d, v, c, grads)
    for k in range(3):
        assert rel_max(got["int8"][k], got["float32"][k]) < (OUT_TOL if k != 1 else 10 * OUT_TOL)
    compare(got["float32"][3], got["int8"][3])


@pytest.mark.parametrize("n", [1, 31, 700, 20011])
def test_points_with_checkpoints(n):
    from nicecore import imap
    m, _ = model()
    g = torch.Generator().manual_seed(n)
    p = torch.rand(n, 3, generator=g, dtype=torch.float64) * 2 - 1
    up = torch.randn(n, 4, generator=g).cuda()
    got = {}
    for act in (None, "int8"):
        x = p.cuda().requires_grad_(True)
        for q in m.parameters():
            q.grad = None
        raw = imap.eval_points(m, x, activations=act)
        raw.backward(up)
        got[act] = (raw, {k: q.grad.clone() for k, q in m.named_parameters()}, x.grad.clone())
    assert rel_max(got["int8"][0], got[None][0]) < OUT_TOL
    hit, change = open_units(m, p.float(), up)
    compare(got[None][1], got["int8"][1], change)
    sure = ~hit.cuda()
    assert sure.float().mean() > 0.8
    compare({"p": got[None][2][sure]}, {"p": got["int8"][2][sure]})
    with torch.no_grad():  # nothing to keep: the default path
        assert torch.equal(imap.eval_points(m, p.cuda(), activations="int8"), imap.eval_points(m, p.cuda()))


def test_points_with_checkpoints_frozen_and_empty():
    from nicecore import imap
    m, _ = model()
    for q in m.parameters():
        q.requires_grad_(False)
    p = torch.rand(300, 3, dtype=torch.float64, generator=torch.Generator().manual_seed(1)).cuda().requires_grad_(True)
    a, = torch.autograd.grad(imap.eval_points(m, p).square().sum(), p)
    b, = torch.autograd.grad(imap.eval_points(m, p, activations="int8").square().sum(), p)
    assert rel_max(b, a) < GRAD_TOL
    for q in m.parameters():
        q.requires_grad_(True)
    e = torch.zeros(0, 3, dtype=torch.float64, device="cuda")
    raw = imap.eval_points(m, e, activations="int8")
    raw.sum().backward()
    assert raw.shape == (0, 4) and all(not q.grad.any() for q in m.parameters())


def test_a_captured_step_with_checkpoints_replays():
    """A mapper step (render, loss, backward) with 8-bit checkpoints as a graph: each replay equals the
    eager step on the same rays (dB is a float-atomic sum: compared to rounding), eager work in between."""
    from nicecore.graph import GraphedStep
    m, bound = model()
    r = renderer(bound, 0, "int8")
    rec = load(CASES[0])
    ro, rd = rec["rays_o"].cuda().repeat(40, 1), rec["rays_d"].cuda().repeat(40, 1)
    dep = rec["gt_depth"].cuda().repeat(40)

    def body():
        for q in m.parameters():
            q.grad = None
        d, v, c = r.render_batch_ray(None, m, rd, ro, "cuda", "color", dep)
        loss = (dep - d).abs().sum() + c.square().sum()
        loss.backward()
        return loss.detach()

    step = GraphedStep(body)
    captured = {n: q.grad for n, q in m.named_parameters()}  # what every replay writes
    for k in range(4):
        ro.add_(0.01 * k)
        step()
        torch.cuda.synchronize()
        graph = {n: g.clone() for n, g in captured.items()}
        body()
        torch.cuda.synchronize()
        for n, q in m.named_parameters():
            if n == "embedder._B":
                assert rel(graph[n], q.grad) < 1e-5
            else:
                assert torch.equal(graph[n], q.grad), (k, n)


def test_quantized_mlp():
    from nicecore import imap, lowbit
    m, bound = model()
    q8 = m.quantize()
    p = (torch.rand(5000, 3, dtype=torch.float64, generator=torch.Generator().manual_seed(2)) * 2 - 1).cuda()
    f = q8.features(p)
    x = p.float() @ m.embedder._B  # the argument in float32, as the reference
    want = torch.sin(p.float().double() @ m.embedder._B.double())
    # sin of an argument that three float32 products and sums rounded: 3 steps of the largest partial
    tol = 4 * 2.0 ** -24 * (p.float().abs().double() @ m.embedder._B.abs().double()) + 2.0 ** -23
    assert ((f[:, :93].double() - want).abs() <= tol).all() and not f[:, 93:].any()
    # the chain of public operators
    h = f
    for l, (w, b) in enumerate(zip(q8.weights, q8.biases)):
        h = lowbit.quantized_linear(h, w, b, relu=l < 4, out_dtype=torch.float32 if l == 4 else torch.bfloat16)
    raw = q8(p)
    assert torch.equal(raw, h) and raw.shape == (5000, 4) and raw.dtype == torch.float32
    with torch.no_grad():
        full = imap.eval_points(m, p)
    # each of 5 layers: activations off by amax / (127 sqrt(12)) rms of rows whose amax is below 8 rms, weights by
    # as much of rows whose amax is below 4 rms, bfloat16 2^-9: independent, so the squares add up; twice that
    one = (8 / 127 / math.sqrt(12)) ** 2 + (4 / 127 / math.sqrt(12)) ** 2 + 2.0 ** -18
    assert rel(raw, full) < 2 * math.sqrt(5 * one), rel(raw, full)
    # in the renderer's place, with its bound mask
    r = renderer(bound, 0, None)
    with torch.no_grad():
        a, b = r.eval_points(p, q8), r.eval_points(p, m)
    out = (b[:, 3] == 100.0)
    assert bool((a[:, 3] == 100.0)[out].all()) and torch.equal(a[~out], raw[~out])
    assert q8(p[:0]).shape == (0, 4)
    from nicecore import _lib as L
    with pytest.raises(L.NiceCoreError, match="no gradient"):
        q8(p.clone().requires_grad_(True))
    with pytest.raises(L.NiceCoreError, match="points are on"):
        q8(p.cpu())


def test_nice_renderer_refuses_coded_activations():
    m, bound = model()
    r = renderer(bound, 0, "int8")
    r.nice = r.occupancy = True
    with pytest.raises(NotImplementedError, match="int8"):
        r.render_batch_ray(None, m, None, None, "cuda", "color")


def test_backward_twice_with_checkpoints():
    """A graph that is kept gives the same gradients again: the backward leaves what it reads."""
    from nicecore import decoder as D
    from nicecore import imap
    m = D.build_imap(seed=3).cuda()
    p = torch.rand(3000, 3, generator=torch.Generator().manual_seed(4), dtype=torch.float64).cuda().requires_grad_()
    raw = imap.eval_points(m, p, activations="int8")
    g = torch.randn(raw.shape, generator=torch.Generator().manual_seed(5)).to(raw.dtype).cuda()
    leaves = [p, *m.parameters()]
    first = torch.autograd.grad(raw, leaves, g, retain_graph=True)
    second = torch.autograd.grad(raw, leaves, g)
    for (name, _), a, b in zip([("p", None), *m.named_parameters()], first, second):
        if name.endswith("_B"):  # its sum's order is the atomics'
            assert rel(a, b) < GRAD_TOL
        else:
            assert torch.equal(a, b), name
