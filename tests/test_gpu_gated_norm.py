"""ops.gated_residual_norm (norm after a block, gate, scaled residual, next norm in one pass) against the same
formulas in float64.

Tolerances, derived: between loads and stores every value is float32, with at most 256 roundings of 2^-24 on the
way of any element of a row (sums over a row are formed from lane sums of at most 32 terms, six cross-lane
additions and at most 16 waves; a gradient passes four such sums), each relative to the largest term of its row; the
store rounds by half a step (2^-8 relative to the value for bfloat16).  Column sums over R rows add at most
R + 64 roundings relative to the sum of the terms' magnitudes."""

import pytest
import torch

from helpers import gen

BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def reference(t, norm, alpha, eps, dh=None, dn=None):
    """(h, n, grads, scales): float64; scales hold per-element bounds of the terms' magnitudes."""
    v = {k: None if x is None else x.detach().cpu().double().requires_grad_(True) for k, x in t.items()}
    d = v["x"].shape[-1]

    def nrm(y, w, b):
        mu = y.mean(-1, keepdim=True) if norm == "layer" else torch.zeros_like(y[..., :1])
        rs = 1 / torch.sqrt((y - mu).square().mean(-1, keepdim=True) + eps)
        hat = (y - mu) * rs
        out = hat * w
        return (out if b is None else out + b), hat, rs

    if v["w1"] is not None:
        u, xh, r1 = nrm(v["x"], v["w1"], v["b1"])
    else:
        u, xh, r1 = v["x"], v["x"], torch.ones_like(v["x"][..., :1])
    g = v["gate"] if v["gate"] is not None else torch.ones((), dtype=torch.float64)
    h = alpha * v["r"] + g * u
    n = hh = r2 = None
    if v["w2"] is not None:
        n, hh, r2 = nrm(h, v["w2"], v["b2"])
    grads, scale = {}, {}
    amax = lambda y: y.detach().abs().amax(-1, keepdim=True)
    scale["h"] = (abs(alpha) * amax(v["r"]) + amax(g * u) + amax(g * xh)).expand(h.shape)
    if n is not None:
        scale["n"] = ((scale["h"][..., :1] * r2.detach() + 1) * (1 + amax(hh)) * v["w2"].detach().abs().max()
                      + (0 if v["b2"] is None else v["b2"].detach().abs().max())).expand(h.shape)
    if dh is not None or dn is not None:
        outs = [(o, y.cpu().double()) for o, y in ((h, dh), (n, dn)) if y is not None]
        leaves = {k: x for k, x in v.items() if x is not None}
        got = torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [y for _, y in outs], allow_unused=True)
        grads = {k: (torch.zeros_like(x) if gr is None else gr) for (k, x), gr in zip(leaves.items(), got)}
        dH = 0 if dh is None else amax(dh.cpu().double())
        if dn is not None:
            g2 = amax(dn.cpu().double()) * v["w2"].detach().abs().max()
            cancel = 1 + scale["h"][..., :1] * r2.detach()
            dH = dH + r2.detach() * g2 * (1 + amax(hh)) ** 2 * cancel
        gmax = amax(g.expand(h.shape))
        w1m = 1 if v["w1"] is None else v["w1"].detach().abs().max()
        x_cancel = 1 + amax(v["x"]) * r1.detach()
        scale["r"] = (abs(alpha) * dH).expand(h.shape)
        scale["x"] = (r1.detach() * gmax * dH * w1m * (1 + amax(xh)) ** 2 * x_cancel).expand(h.shape)
        scale["gate"] = (dH * (amax(u) + amax(xh) * w1m)).expand(h.shape)
        scale["w1"] = (gmax * dH * (1 + amax(xh)) * x_cancel).expand(h.shape)
        scale["b1"] = (gmax * dH).expand(h.shape)
        if dn is not None:
            scale["w2"] = (amax(dn.cpu().double()) * (1 + amax(hh)) * cancel).expand(h.shape)
            scale["b2"] = amax(dn.cpu().double()).expand(h.shape)
    return (None if h is None else h.detach()), (None if n is None else n.detach()), grads, scale


def check(name, got, want, scale, dtype):
    """|got - want| <= half a step of the output's type + 256 float32 roundings of the terms."""
    got = got.detach().cpu().double()
    half = torch.finfo(dtype).eps / 2
    # (summed over broadcast axes: the terms' magnitudes add up, and each addition rounds)
    while scale.dim() > got.dim():
        scale = scale.sum(0)
    extra = 1
    for i, s in enumerate(got.shape):
        if s != scale.shape[i]:
            extra += scale.shape[i]
            scale = scale.sum(i, keepdim=True)
    tol = half * want.abs() * (1 + 2 ** -8) + (256 + extra) * U * scale + 1e-38
    bad = (got - want).abs() > tol
    worst = ((got - want).abs() / tol).max().item() if got.numel() else 0.0
    print(f"{name}: worst {worst:.3f} of the tolerance", flush=True)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} elements, worst {worst:.2f} of the tolerance"


def make(shape, xdt, rdt, norm, gate, seed, post=True, pre=True, dev="cpu"):
    g0 = gen(seed)
    d = shape[-1]
    t = {"x": (torch.randn(*shape, generator=g0) * 0.5 + 0.2).to(xdt),
         "r": (torch.randn(*shape, generator=g0) * 2 - 0.3).to(rdt),
         "w1": torch.randn(d, generator=g0) * 0.3 + 1 if post else None,
         "b1": torch.randn(d, generator=g0) * 0.2 if post and norm == "layer" else None,
         "w2": torch.randn(d, generator=g0) * 0.3 + 1 if pre else None,
         "b2": torch.randn(d, generator=g0) * 0.2 if pre and norm == "layer" else None}
    gs = {"none": None, "scalar": (1,), "channel": (d,), "token": shape[:-1] + (1,), "full": shape}[gate]
    t["gate"] = None if gs is None else (torch.randn(*gs, generator=g0) * 0.5 + 0.4).to(
        F32 if gate in ("scalar", "channel") else xdt)
    dh = torch.randn(*shape, generator=g0).to(rdt)
    dn = torch.randn(*shape, generator=g0).to(xdt) if pre else None
    return t, dh, dn


def run(t, dev, norm, alpha, eps, dh, dn, out_dtype=None):
    from memory_amd import ops
    leaf = {k: None if x is None else x.detach().to(dev).requires_grad_(True) for k, x in t.items()}
    h, n = ops.gated_residual_norm(leaf["x"], leaf["r"], post_weight=leaf["w1"], post_bias=leaf["b1"], gate=leaf["gate"],
                                   residual_scale=alpha, pre_weight=leaf["w2"], pre_bias=leaf["b2"], eps=eps, norm=norm,
                                   out_dtype=out_dtype)
    outs = [(o, y.to(dev)) for o, y in ((h, dh), (n, dn)) if o is not None and y is not None]
    names = [k for k, x in leaf.items() if x is not None]
    grads = torch.autograd.grad([o for o, _ in outs], [leaf[k] for k in names], [y for _, y in outs], allow_unused=True)
    return h, n, dict(zip(names, grads))


def compare(t, dev, norm, alpha, eps, dh, dn, out_dtype=None):
    h, n, grads = run(t, dev, norm, alpha, eps, dh, dn, out_dtype)
    wh, wn, wg, sc = reference(t, norm, alpha, eps, dh, dn)
    assert h.dtype == t["r"].dtype and h.shape == wh.shape
    check("h", h, wh, sc["h"], h.dtype)
    if wn is not None:
        assert n.dtype == (out_dtype or t["x"].dtype)
        check("n", n, wn, sc["n"], n.dtype)
    for k, g in grads.items():
        if g is None:
            assert not wg[k].any()
            continue
        assert g.dtype == t[k].dtype and g.shape == t[k].shape
        check("d" + k, g, wg[k], sc[k], g.dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["none", "scalar", "channel", "token", "full"])
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("xdt,rdt", [(BF, BF), (BF, F32), (F32, F32), (F32, BF)])
def test_types_and_gates(gpu_device, xdt, rdt, norm, gate):
    t, dh, dn = make((2, 37, 96), xdt, rdt, norm, gate, 11)
    compare(t, gpu_device, norm, 0.7, 1e-5, dh, dn)


@pytest.mark.gpu
@pytest.mark.parametrize("R,d", [(1, 1), (3, 7), (5, 64), (1, 768), (300, 768), (9, 1000), (4, 1025), (7, 2048), (2, 2049),
                                 (6, 4096), (2, 4104), (1030, 40), (2, 8200), (1, 16384), (2, 16383), (2100, 8)])
@pytest.mark.parametrize("norm,gate,xdt", [("rms", "channel", BF), ("layer", "token", F32)])
def test_sizes(gpu_device, R, d, norm, gate, xdt):
    t, dh, dn = make((R, d), xdt, xdt, norm, gate, R * 7 + d)
    if d == 1 and norm == "layer":
        t["x"] = t["x"] * 0 + 1       # one element is its own mean
    compare(t, gpu_device, norm, 1.0, 1e-6, dh, dn)


@pytest.mark.gpu
@pytest.mark.parametrize("post,pre,use_h,use_n", [(True, False, True, False), (False, True, True, True), (True, True, False, True),
                                                  (True, True, True, False), (False, False, True, False)])
def test_parts(gpu_device, post, pre, use_h, use_n):
    """Either norm left out, and a gradient that arrives through one result only."""
    t, dh, dn = make((65, 264), BF, F32, "layer", "channel", 5, post, pre)
    compare(t, gpu_device, "layer", -0.5, 1e-5, dh if use_h else None, dn if use_n and pre else None)


@pytest.mark.gpu
def test_other_types_and_layouts(gpu_device):
    """float16 rows, an output type of its own, and operands that are views: transposed, offset to an odd address,
    expanded."""
    t, dh, dn = make((33, 72), torch.float16, torch.float16, "rms", "full", 3)
    compare(t, gpu_device, "rms", 1.0, 1e-5, dh, dn)
    t, dh, dn = make((33, 72), BF, F32, "rms", "token", 4)
    compare(t, gpu_device, "rms", 1.0, 1e-5, dh, dn.float(), out_dtype=F32)
    from memory_amd import ops
    t, dh, dn = make((33, 72), BF, BF, "rms", "full", 4)
    want = ops.gated_residual_norm(*(t[k].to(gpu_device) for k in ("x", "r")), gate=t["gate"].to(gpu_device),
                                   post_weight=t["w1"].to(gpu_device), pre_weight=t["w2"].to(gpu_device))
    x_t = t["x"].to(gpu_device).t().contiguous().t()
    r_off = torch.zeros(33 * 72 + 1, device=gpu_device, dtype=BF)[1:].view(33, 72)
    r_off.copy_(t["r"])
    wide = torch.zeros(33, 80, device=gpu_device, dtype=BF)
    wide[:, 5:77] = t["gate"].to(gpu_device)
    got = ops.gated_residual_norm(x_t, r_off, gate=wide[:, 5:77], post_weight=t["w1"].to(gpu_device).to(BF).float() * 0
                                  + t["w1"].to(gpu_device), pre_weight=t["w2"].to(gpu_device))
    for a, b in zip(got, want):   # (the scalar-load variant adds a row's terms in another order)
        assert torch.allclose(a.float(), b.float(), rtol=2 ** -7, atol=1e-6)


@pytest.mark.gpu
def test_rows_stand_alone(gpu_device):
    """A row of NaN, infinities or zeros leaves every other row as it is; a zero block with a zero residual is 0."""
    from memory_amd import ops
    t, _, _ = make((12, 768), BF, F32, "rms", "channel", 8)
    a = {k: None if v is None else v.to(gpu_device) for k, v in t.items()}
    go = lambda: ops.gated_residual_norm(a["x"], a["r"], post_weight=a["w1"], gate=a["gate"], pre_weight=a["w2"])
    h0, n0 = go()
    a["x"][3, 5] = float("nan")
    a["r"][6, 0] = float("inf")
    a["x"][9] = 0
    a["r"][9] = 0
    h1, n1 = go()
    rest = [i for i in range(12) if i not in (3, 6, 9)]
    assert torch.equal(h0[rest], h1[rest]) and torch.equal(n0[rest], n1[rest])
    assert torch.isnan(h1[3]).all() and torch.isnan(n1[3]).all() and torch.isinf(h1[6, 0])
    assert not h1[9].any() and not n1[9].any()


@pytest.mark.gpu
def test_empty_and_repeatable(gpu_device):
    t, dh, dn = make((0, 96), BF, BF, "layer", "scalar", 1)
    h, n, g = run(t, gpu_device, "layer", 1.0, 1e-5, dh, dn)
    assert h.shape == n.shape == (0, 96) and all(not x.any() for x in g.values())
    t, dh, dn = make((4097, 328), BF, BF, "layer", "scalar", 2)
    first = run(t, gpu_device, "layer", 1.0, 1e-5, dh, dn)
    for _ in range(2):
        again = run(t, gpu_device, "layer", 1.0, 1e-5, dh, dn)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
        assert all(torch.equal(first[2][k], again[2][k]) for k in first[2])


@pytest.mark.gpu
def test_graph_replays_forward_and_backward(gpu_device):
    """Captured with its backward, replayed on new inputs with eager work between the replays."""
    t, dh, dn = make((130, 256), BF, F32, "layer", "token", 6)
    from memory_amd import ops
    leaf = {k: v.to(gpu_device).requires_grad_(True) for k, v in t.items() if v is not None}
    dh, dn = dh.to(gpu_device), dn.to(gpu_device)

    def step():
        h, n = ops.gated_residual_norm(leaf["x"], leaf["r"], post_weight=leaf["w1"], post_bias=leaf["b1"],
                                       gate=leaf["gate"], residual_scale=0.9, pre_weight=leaf["w2"], pre_bias=leaf["b2"],
                                       norm="layer")
        return (h.detach(), n.detach(), *torch.autograd.grad([h, n], list(leaf.values()), [dh, dn]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for rep in range(3):
        with torch.no_grad():
            leaf["x"].copy_(torch.randn(130, 256, generator=gen(rep)).to(BF))
        graph.replay()
        got = [o.clone() for o in out]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step())), f"replay {rep}"


@pytest.mark.gpu
def test_second_derivatives_are_refused(gpu_device):
    """A recorded backward gives first derivatives and refuses to be differentiated itself."""
    from memory_amd import ops
    x = torch.randn(5, 64, device=gpu_device, requires_grad=True)
    w = torch.ones(64, device=gpu_device)
    h, n = ops.gated_residual_norm(x, x.detach() * 2, post_weight=w, pre_weight=w)
    (g,) = torch.autograd.grad(n.square().sum(), x, create_graph=True)
    h2, n2 = ops.gated_residual_norm(x, x.detach() * 2, post_weight=w, pre_weight=w)
    assert torch.equal(g, torch.autograd.grad(n2.square().sum(), x)[0])
    with pytest.raises(RuntimeError):
        g.sum().backward()
    z = torch.randn(5, 33, device=gpu_device, requires_grad=True)
    (g,) = torch.autograd.grad(ops.router_select(z, 4, 1)[1].square().sum(), z, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_refusals():
    from memory_amd import ops
    x, w = torch.zeros(3, 8), torch.ones(8)
    for bad in (dict(norm="batch"), dict(post_bias=w), dict(post_weight=w, post_bias=w), dict(post_weight=torch.ones(7)),
                dict(gate=torch.ones(3)), dict(gate=torch.ones(2, 1)), dict(out_dtype=torch.int32)):
        with pytest.raises(ValueError):
            ops.gated_residual_norm(x, x, **bad)
    with pytest.raises(ValueError, match="one shape"):
        ops.gated_residual_norm(x, torch.zeros(3, 9))
    with pytest.raises(ValueError, match="one shape"):
        ops.gated_residual_norm(torch.zeros(3, 0), torch.zeros(3, 0))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.gated_residual_norm(x, x, post_weight=w)
    from memory_amd import _lib as L
    import ctypes
    a = ops._GatedNormArgs(rows=1, d=8)
    with pytest.raises(ValueError, match="null pointer"):
        L.call("moc_gated_norm_fwd", ctypes.addressof(a), None)
    a.x = a.residual = a.h = 16
    a.d = 16385
    with pytest.raises(ValueError, match="16384"):
        L.call("moc_gated_norm_fwd", ctypes.addressof(a), None)
    a.d, a.norm, a.norm2, a.gate_mode = 8, 1, 1, 9
    with pytest.raises(ValueError, match="gate mode"):
        L.call("moc_gated_norm_fwd", ctypes.addressof(a), None)


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["scalar", "channel", "token"])
def test_parameter_gradients_hold_no_workspace(gpu_device, gate):
    """What stays allocated behind the parameters' gradients is their own size, not the backward's workspace."""
    d = 768
    t, dh, dn = make((2048, d), BF, F32, "layer", gate, 21)
    _, _, g = run(t, gpu_device, "layer", 1.0, 1e-5, dh, dn)
    for name in ("w1", "b1", "w2", "b2") + (("gate",) if gate != "token" else ()):
        assert g[name].untyped_storage().nbytes() <= 4 * (5 * d + 64), name


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["x", "r", "gate", "w1", "w2"])
def test_forward_mode_is_refused(gpu_device, which):
    """A tangent raises, as in the single norm: it is never dropped."""
    import torch.autograd.forward_ad as fwd
    from memory_amd import ops
    t, _, _ = make((5, 64), F32, F32, "rms", "channel", 1)
    t = {k: v.to(gpu_device) for k, v in t.items() if v is not None}
    go = lambda v: ops.gated_residual_norm(v["x"], v["r"], gate=v["gate"], post_weight=v["w1"], pre_weight=v["w2"])
    want = go(t)
    with fwd.dual_level():
        with pytest.raises(NotImplementedError):
            ops.row_norm(fwd.make_dual(t["x"], torch.ones_like(t["x"])), t["w1"], None, 1e-6, "rms")
        with pytest.raises(NotImplementedError):
            go({**t, which: fwd.make_dual(t[which], torch.ones_like(t[which]))})
        got = go(t)                                  # (no tangent: as outside)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
